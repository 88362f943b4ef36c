"""The gated delta rule and group_norm as a program uses them: captured and replayed, on several streams and from several threads, with
retained graphs, values that must not spread, and betas that leave nothing of a row."""
import threading

import pytest
import torch

from tests import gdr_testlib as lib

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32

KINDS = [dict(B=2, T=150, H=1, HV=2, K=128, V=128, dtype=BF), dict(B=1, T=2000, H=1, HV=1, K=128, V=128, dtype=BF),
         dict(B=2, T=150, H=1, HV=2, K=64, V=128, dtype=F32)]


def tensors(x):
    return [x[n].detach().clone().requires_grad_() for n in lib.NAMES if n in x]


def call(leaf, **kw):
    from openkimi_b200 import chunk_gated_delta_rule

    q, k, v, g, beta, A, bias, h0 = leaf
    return chunk_gated_delta_rule(q, k, v, g, beta, A_log=A, dt_bias=bias, initial_state=h0, output_final_state=True, use_qk_l2norm_in_kernel=True,
                                  use_gate_in_kernel=True, use_beta_sigmoid_in_kernel=True, **kw)


def step(leaf, x, **kw):
    o, ht = call(leaf, **kw)
    return [o.detach(), ht.detach(), *torch.autograd.grad([o, ht], leaf, [x["do"], x["dht"]])]


def equal(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("kind", KINDS)
def test_two_captured_training_steps(kind):
    """Two graphs over the same leaves, replayed in turn with new inputs: each has memory of its own."""
    xs = [lib.make(**kind, seed=s) for s in (1, 2)]
    want = [step(tensors(x), x) for x in xs]
    leaf = tensors(xs[0])
    x = dict(do=xs[0]["do"].clone(), dht=xs[0]["dht"].clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(leaf, x)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(leaf, x)
        graphs.append((graph, out))
    for turn in (0, 1, 1, 0):
        with torch.no_grad():
            for t, n in zip(leaf, lib.NAMES):
                t.copy_(xs[turn][n])
        x["do"].copy_(xs[turn]["do"])
        x["dht"].copy_(xs[turn]["dht"])
        for graph, out in graphs:
            graph.replay()
            assert equal(out, want[turn])


def test_a_graph_keeps_the_tables_of_its_documents():
    from openkimi_b200 import gated_delta, ops

    docs = [0, 100, 331, 700]
    x = lib.make(1, 700, 1, 2, 128, 128, BF, docs=docs)
    cu = torch.tensor(docs)
    with torch.no_grad():
        leaf = tensors(x)
        run = lambda: call(leaf, cu_seqlens=cu.cuda() if not torch.cuda.is_current_stream_capturing() else None, cu_seqlens_cpu=cu)  # noqa: E731
        want = run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        gated_delta._offsets.cache_clear()
        ops._chunk_tables_cached.cache_clear()
        junk = [torch.full((1 << i,), 0x7f7f7f7f, dtype=torch.int32, device="cuda") for i in range(2, 14) for _ in range(8)]
        graph.replay()
        assert equal(out, want)
    del junk


def test_streams_and_threads_at_once():
    xs = [lib.make(**KINDS[i % 3], seed=i) for i in range(6)]
    want = [step(tensors(x), x) for x in xs]
    torch.cuda.synchronize()
    got = [None] * 6

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(3):
                got[i] = step(tensors(xs[i]), xs[i])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(equal(a, b) for a, b in zip(got, want))


def test_retained_graph_and_second_derivative():
    from openkimi_b200 import group_norm

    x = lib.make(**KINDS[0])
    leaf = tensors(x)
    o, ht = call(leaf)
    first = torch.autograd.grad([o, ht], leaf, [x["do"], x["dht"]], retain_graph=True)
    assert equal(first, torch.autograd.grad([o, ht], leaf, [x["do"], x["dht"]], retain_graph=True))
    d = torch.autograd.grad([o, ht], leaf, [x["do"], x["dht"]], create_graph=True)
    assert equal(first, d)
    with pytest.raises(RuntimeError, match="not differentiable"):
        (o.float().sum() + d[0].float().sum()).backward()
    a = torch.randn(20, 32, device="cuda", requires_grad=True)
    (d,) = torch.autograd.grad(group_norm(a, 4, activation="silu").sum(), a, create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        (a.sum() + d.square().sum()).backward()


def test_an_input_changed_before_the_backward_is_noticed():
    x = lib.make(**KINDS[0])
    leaf = tensors(x)
    o, ht = call(leaf)
    with torch.no_grad():
        leaf[2].mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        o.sum().backward()


@pytest.mark.parametrize("dtype", [F32, BF])
def test_only_some_outputs_and_inputs(dtype):
    """The final state alone, the outputs alone, and gradients of one input: the same numbers as all at once with zeros."""
    x = lib.make(1, 200, 1, 2, 128, 128, dtype)
    leaf = tensors(x)
    o, ht = call(leaf)
    zero = torch.zeros_like
    for ends, given, full in (([ht], [x["dht"]], [zero(o), x["dht"]]), ([o], [x["do"]], [x["do"], zero(ht)])):
        some = torch.autograd.grad(ends, leaf, given, retain_graph=True, allow_unused=True)
        whole = torch.autograd.grad([o, ht], leaf, full, retain_graph=True)
        assert equal(some, whole)
    for i in range(len(leaf)):
        alone = [t.detach() for t in leaf]
        alone[i].requires_grad_()
        o, ht = call(alone)
        (d,) = torch.autograd.grad([o, ht], [alone[i]], [x["do"], x["dht"]])
        leaf2 = tensors(x)
        o2, ht2 = call(leaf2)
        assert torch.equal(d, torch.autograd.grad([o2, ht2], leaf2, [x["do"], x["dht"]])[i])


def test_not_a_number_stays_in_its_document_and_head():
    docs = [0, 90, 220, 400]
    x = lib.make(1, 420, 2, 4, 128, 128, BF, docs=docs)
    want = lib.device_run(x)
    for name in ("q", "k", "v", "do"):
        y = dict(x)
        y[name] = x[name].clone()
        head = 2 if name in ("v", "do") else 1
        y[name][0, 100, head] = float("nan")
        y[name][0, 405:] = float("inf")  # rows of no document
        got = lib.device_run(y)
        heads = [2] if head == 2 else [2, 3]
        other = [h for h in range(4) if h not in heads]
        for n in ("o", "dv", "dg", "dbeta"):
            a, b = got[n], want[n]
            assert torch.equal(a[:, :90], b[:, :90]) and torch.equal(a[:, 220:], b[:, 220:]) and torch.equal(a[:, :, other], b[:, :, other]), (name, n)
        for n in ("ht", "dh0"):
            assert torch.equal(got[n][0], want[n][0]) and torch.equal(got[n][2], want[n][2]) and torch.equal(got[n][1][other], want[n][1][other])
        for n in ("dq", "dk"):
            a, b = got[n], want[n]
            assert torch.equal(a[:, :90], b[:, :90]) and torch.equal(a[:, 220:], b[:, 220:]) and torch.equal(a[:, :, 0], b[:, :, 0])


@pytest.mark.parametrize("V,dtype", [(128, BF), (64, BF), (128, F32)])
@pytest.mark.parametrize("beta", [0.0, 1e-30, 1e-12, -1.0, 2.0])
def test_betas_at_the_ends(V, dtype, beta):
    """Betas given as they are; some rows take none of the error, all of it twice, or so little that 1 / beta has no place in FP32.
    (With |1 - beta| <= 1 the states stay bounded; -1 is held to a few rows.)"""
    x = lib.make(1, 150, 1, 2, 128, V, dtype, gate=False)
    rows = slice(None) if beta >= 0 else slice(40, 45)
    x["beta"][:, rows, 0] = beta
    ref = lib.reference(x)
    lib.check(lib.device_run(x), ref)


def test_many_value_heads_of_one_key_head():
    x = lib.make(1, 130, 1, 10, 128, 128, BF)
    ref = lib.add_terms(lib.reference(x), x)
    lib.check(lib.device_run(x), ref)


def test_unaligned_and_strided_inputs():
    x = lib.make(**KINDS[0])
    want = lib.device_run(x)
    y = dict(x)
    for n in ("q", "k", "v", "do", "g", "beta", "h0", "A_log", "dt_bias"):
        flat = torch.empty(x[n].numel() + 1, dtype=x[n].dtype, device="cuda")[1:].view(x[n].shape)
        y[n] = flat.copy_(x[n])
    leaf = [y[n].detach().requires_grad_() for n in lib.NAMES]
    got = step(leaf, y)
    assert equal(got, [want[n] for n in ("o", "ht", *("d" + n for n in lib.NAMES))])
    wide = torch.randn(2, 150, 1, 3 * 128, device="cuda").to(BF)
    wide[..., 128:256] = x["k"]
    leaf = [t.detach().requires_grad_() for t in (x[n] for n in lib.NAMES)]
    leaf[1] = wide[..., 128:256].detach().requires_grad_()
    leaf[2] = x["v"].transpose(1, 2).contiguous().transpose(1, 2).detach().requires_grad_()
    assert equal(step(leaf, x), got)


def test_captured_norm_and_layer_backward():
    from openkimi_b200 import group_norm

    for shape in ((300, 96), (2, 257, 96)):
        x, dy = torch.randn(*shape, device="cuda"), torch.randn(*shape, device="cuda")
        w, b = torch.rand(96, device="cuda"), torch.randn(96, device="cuda")
        leaf = [t.requires_grad_() for t in (x, w, b)]

        def run():
            y = group_norm(x, 3, w, b, activation="silu")
            return [y.detach(), *torch.autograd.grad(y, leaf, dy)]

        want = run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        for t in out:
            t.zero_()
        graph.replay()
        assert equal(out, want)

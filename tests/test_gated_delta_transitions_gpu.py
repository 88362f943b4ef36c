"""Segmented walks of a training call: which transitions (what a segment makes of the state it is entered with) are computed, and two
segments against one."""
import ctypes as C

import pytest
import torch

from tests.gdr_testlib import UNIT, make

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
SHORT = [0, 300, 600, 900, 1200, 1500, 3500]  # one document of them is cut, in two


class Call:
    """A call through the C entry points, in workspaces of its own; ``hint``: chunks of the longest document (0: no segments)."""

    def __init__(self, x, docs, hint):
        from openkimi_b200 import _lib, gated_delta, ops

        self.lib, self.x, self.keep = _lib.load(), x, []
        p = self.p = _lib.KdaGdrParams()
        (_, p.T, p.H, p.dk), (p.HV, p.dv) = x["q"].shape, x["v"].shape[2:]
        seq, off, nt, tab, longest = ops._chunk_tables(None, torch.tensor(docs), x["q"].device, p.T)
        p.B, p.N, p.NT, p.max_chunks = 1, len(docs) - 1, nt, longest if hint else 0
        p.dtype, p.g_dtype, p.flags, p.scale = _lib.DTYPE_BF16, _lib.DTYPE_F32, _lib.FLAG_QK_L2NORM, p.dk ** -0.5
        for n, t in dict(q=x["q"], k=x["k"], v=x["v"], g=x["g"], beta=x["beta"], h0=x["h0"], chunk_seq=seq, seq_chunk_off=off, chunk_tab=tab,
                         cu_seqlens=gated_delta._offsets(tuple(docs), x["q"].device.index)).items():
            setattr(p, n, t.data_ptr())
            self.keep.append(t)
        new = lambda t: torch.empty_like(t)  # noqa: E731
        self.out = dict(o=new(x["v"]), ht=new(x["h0"]))
        self.grads = dict(grad_q=new(x["q"]), grad_k=new(x["k"]), grad_v=new(x["v"]), grad_g=new(x["g"]), grad_beta=new(x["beta"]), grad_h0=new(x["h0"]))
        sizes = []
        for flags in (p.flags | _lib.FLAG_NO_SAVE, p.flags):
            p.flags = flags
            a, b = C.c_size_t(), C.c_size_t()
            assert self.lib.kda_gdr_workspace_bytes(C.byref(p), C.byref(a), C.byref(b)) == 0
            sizes.append(a.value)
        self.no_save = sizes[0]
        self.ws = torch.full((sizes[1],), 0xA5, dtype=torch.uint8, device="cuda")
        self.scratch = torch.empty(b.value, dtype=torch.uint8, device="cuda")
        p.workspace, p.workspace_bytes, p.bwd_scratch, p.bwd_scratch_bytes = self.ws.data_ptr(), sizes[1], self.scratch.data_ptr(), b.value
        for n, t in (*self.out.items(), *self.grads.items(), ("grad_o", x["do"]), ("grad_ht", x["dht"])):
            setattr(p, n, t.data_ptr())

    def run(self, backward=True):
        stream = torch.cuda.current_stream().cuda_stream
        assert self.lib.kda_gdr_fwd(C.byref(self.p), stream) == 0
        if backward:
            assert self.lib.kda_gdr_bwd(C.byref(self.p), stream) == 0
        torch.cuda.synchronize()
        return {**self.out, **self.grads}


def _pair(HV, docs):
    x = make(1, docs[-1], 1, HV, 128, 128, BF, docs=docs, gate=False, seed=HV)
    cut, whole = Call(x, docs, True), Call(x, docs, False)
    matrix = 128 * 128 * 4 * (len(docs) - 1) * HV  # of one segment of every walk
    return cut, whole, (cut.no_save - whole.no_save) // (2 * matrix)


@pytest.mark.parametrize("HV,docs,segments", [(16, SHORT, 2), (100, SHORT, 2), (2, [0, 1300, 1900], None)])
def test_transitions_that_are_read(HV, docs, segments):
    """Of the segments' transitions (the last of what a forward without a backward keeps) those of the first and of a document's last
    segment are left as they were."""
    cut, whole, segs = _pair(HV, docs)
    assert segs == segments if segments else segs > 2
    cut.run()
    x = cut.ws[cut.no_save - 128 * 128 * 4 * (len(docs) - 1) * HV * segs:cut.no_save].view(len(docs) - 1, HV, segs, -1)
    chunks = [(b - a + 63) // 64 for a, b in zip(docs, docs[1:])]
    size = -(-max(chunks) // segs)
    for n, c in enumerate(chunks):
        last = min(segs, -(-c // size)) - 1
        for s in range(segs):
            untouched = bool((x[n, :, s] == 0xA5).all())
            assert untouched == (not 1 <= s < last), (n, s)


@pytest.mark.parametrize("HV,docs", [(16, SHORT), (100, SHORT)])
def test_two_segments_against_one(HV, docs):
    """The same call with sequences whole and cut in two: FP32 results to the bound of their products, BF16 ones to a rounding more."""
    cut, whole, segs = _pair(HV, docs)
    assert segs == 2
    a, b = cut.run(), whole.run()
    for n in a:
        p, q = a[n].double(), b[n].double()
        step = 2.0 ** -7 if a[n].dtype == BF else 0.0  # either side is rounded to BF16
        assert ((p - q).abs() <= step * q.abs() + 8 * UNIT * q.abs().max()).all(), n

"""The index tables of packed documents on a stream that did not make them."""
import gc

import pytest
import torch

from tests.gdr_testlib import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["gdr", "kda"])
def test_dropped_tables_wait_for_the_stream_that_reads_them(kind):
    """Tables made by a call on one stream, used on another that is far behind, and then dropped: their memory is not given out again
    before that stream has passed the call.  (Only where memory lies is looked at; nothing is written to it.)"""
    from openkimi_b200 import chunk_gated_delta_rule, chunk_kda, gated_delta, ops

    docs = (0, 101, 333, 699)  # (a layout that no other test captures)
    cu = torch.tensor(docs)
    x = make(1, 699, 1, 1, 128, 128, torch.bfloat16, docs=docs, gate=False, h0=False)
    on_device = cu.cuda()

    def call():
        with torch.no_grad():
            if kind == "gdr":
                return chunk_gated_delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], use_qk_l2norm_in_kernel=True, cu_seqlens_cpu=cu)[0]
            g = x["g"][..., None].expand(1, 699, 1, 128)
            return chunk_kda(x["q"], x["k"], x["v"], g, x["beta"], use_qk_l2norm_in_kernel=True, cu_seqlens=on_device, cu_seqlens_cpu=cu)[0]

    ops._chunk_tables_cached.cache_clear()
    gated_delta._offsets.cache_clear()
    want = call()
    index = x["q"].device.index
    held = [t for t in ops._chunk_tables_cached(docs, index) if isinstance(t, torch.Tensor)]
    if kind == "gdr":
        held.append(gated_delta._offsets(docs, index))
    places = {t.data_ptr() for t in held}
    torch.cuda.synchronize()
    late = torch.cuda.Stream()
    with torch.cuda.stream(late):
        torch.cuda._sleep(1_000_000_000)  # half a second
        got = call()
    passed = late.record_event()
    ops._chunk_tables_cached.cache_clear()
    gated_delta._offsets.cache_clear()
    del held
    gc.collect()
    new = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in (1, 512, 1024) for _ in range(400)]
    assert not passed.query()
    assert not places & {t.data_ptr() for t in new}
    torch.cuda.synchronize()
    assert torch.equal(got, want)

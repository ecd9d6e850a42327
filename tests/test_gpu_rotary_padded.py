"""Rotary positions with the cache write of a batch that is padded behind its last slot: the same as the two
steps, rotary positions of every row and a cache write of as many tokens as there are slots."""
import pytest

from test_gpu_rotary import inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["nhd", "packed"])
@pytest.mark.parametrize("rows,slots", [(8, 5), (33, 32), (3, 1), (4, 0), (300, 299), (7, 7)])
@pytest.mark.parametrize("in_place", [False, True])
def test_rows_behind_the_last_slot(rows, slots, layout, in_place):
    import torch
    from kvx_b200 import ops
    q, k, v, positions = inputs("bf16", rows, 4, 2, 64, pad=8, seed=rows, fused=True)
    shape = (40, 16, 2, 64) if layout == "nhd" else (40, 2, 8, 16, 8)
    caches = [torch.full(shape, 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    at = torch.randperm(640, device="cuda")[:slots].to(torch.int32)
    freq, factor = ops.rotary_inv_freq(64, device="cuda")
    want, turned = ops.rotary_embedding(q, k, positions, freq, factor=factor)
    ops.reshape_and_cache_flash_kvx(turned, v, caches[2], caches[3], at)
    got = ops.rotary_and_cache(q, k, v, positions, freq, caches[0], caches[1], at, factor=factor, query_out=q if in_place else None)
    torch.cuda.synchronize()
    for a, b in ((got, want), (caches[0], caches[2]), (caches[1], caches[3])):
        same = torch.equal(a, b)
        assert same


def test_more_slots_than_rows_are_refused():
    import torch
    from kvx_b200 import ops
    q, k, v, positions = inputs("bf16", 4, 4, 2, 64, fused=True)
    freq, _ = ops.rotary_inv_freq(64, device="cuda")
    for shape in ((40, 16, 2, 64), (40, 2, 8, 16, 8)):
        c = torch.zeros(shape, dtype=torch.bfloat16, device="cuda")
        with pytest.raises((RuntimeError, ValueError)):
            ops.rotary_and_cache(q, k, v, positions, freq, c, c.clone(), torch.arange(5, device="cuda"))
        assert not bool(c.any())

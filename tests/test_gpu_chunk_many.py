"""Chunk attention of more sequences than the attention kernels plan for themselves (32): the plan is then made by a
kernel of its own, for every way of reading the pages."""
import pytest

from test_gpu_chunk_attention import check, make

pytestmark = pytest.mark.gpu

WAYS = [dict(dtype="f32", dim=64), dict(dtype="f32", dim=128, layout="hnd"), dict(dtype="f32", dim=66), dict(dtype="f32", dim=320),
        dict(cache="f8", dim=128), dict(dtype="f16", cache="f8", dim=64, block_size=32), dict(dtype="f32", cache="f8", dim=64),
        dict(dim=64, layout="packed"), dict(dim=128, block_size=6), dict(dim=256), dict(dim=80, cache="f8", block_size=4)]


def _lengths(count, seed):
    import torch
    g = torch.Generator().manual_seed(seed)
    some = [0, 1, 2, 15, 16, 17, 127, 128, 129, 255, 256, 257, 300, 511, 640, 2500]
    n = torch.randint(0, 9, (count,), generator=g).tolist()
    t = [some[i] for i in torch.randint(0, len(some), (count,), generator=g).tolist()]
    return tuple(zip(n, t))


@pytest.mark.parametrize("way", range(len(WAYS)))
@pytest.mark.parametrize("count", [32, 33, 150])
def test_many_sequences(way, count):
    check(make(lens=_lengths(count, count + way), kv_heads=2, group=3, seed=way, **WAYS[way]))
    check(make(lens=_lengths(count, count + way)[::-1], kv_heads=1, group=4, seed=way, **WAYS[way]), causal=False)


@pytest.mark.parametrize("way", range(len(WAYS)))
def test_one_long_sequence_among_many(way):
    """Tiles that are cut between shares, behind a plan of its own kernel."""
    lens = _lengths(40, way)
    check(make(lens=lens[:20] + ((130, 7000),) + lens[20:], kv_heads=1, group=2, seed=way, **WAYS[way]))

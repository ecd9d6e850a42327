"""NaN and infinities in V under chunk attention: a token that a row may not see has no influence on it,
one that it sees has, other sequences of the batch keep their bits, and none of it holds up the call
(the kernel's waits on its own work are bounded: a row that took too long would leave others unwritten)."""
import math

import pytest

from test_gpu_chunk_attention import check, make, run

pytestmark = pytest.mark.gpu


def _put(c, s, token, head, dims, value):
    """V of one token's head from now on."""
    page, at = int(c["table"][s][token // c["block_size"]]), token % c["block_size"]
    fp8 = c["ks"] is not None
    v = c["vc"].view(__import__("torch").uint8) if fp8 else c["vc"]
    value = 0x7F if fp8 else value
    if c["layout"] == "nhd":
        v[page, at, head, dims] = value
    elif c["layout"] == "hnd":
        v[page, head, at, dims] = value
    else:
        for d in range(*dims.indices(c["dim"])):
            v[page, head, d // 8, at, d % 8] = value


def _timed(c):
    import torch
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    a.record()
    out = run(c, c["dim"] ** -0.5)
    b.record()
    torch.cuda.synchronize()
    return out, a.elapsed_time(b)


@pytest.mark.parametrize("dtype,cache,dim,layout,group", [("bf16", "same", 128, "nhd", 4), ("f16", "f8", 128, "nhd", 4),
                                                          ("bf16", "same", 256, "hnd", 4), ("f16", "same", 64, "packed", 3),
                                                          ("bf16", "same", 64, "nhd", 1), ("f32", "same", 128, "nhd", 2)])
def test_one_token_of_a_long_sequence(dtype, cache, dim, layout, group):
    """A NaN that every row of a long sequence sees, and one that only its last rows see."""
    import torch
    c = make(dtype=dtype, cache=cache, dim=dim, layout=layout, group=group, kv_heads=2, seed=31,
             lens=((300, 40000), (3, 129), (150, 150), (1, 3000)))
    clean = check(c)
    _put(c, 0, 5, 0, slice(0, 3), math.nan)
    _put(c, 0, 39900, 1, slice(dim - 2, dim), math.inf)
    out = check(c)
    kept = torch.equal(out[300:], clean[300:])
    assert kept, "other sequences changed"
    assert bool(out[:300, :group, :3].isnan().all())
    same = torch.equal(out[:300, :group, 3:], clean[:300, :group, 3:])
    assert same, "other dims changed"
    early, late = out[:200, group:], out[200:300, group:]
    assert bool(early.isfinite().all())
    assert not bool(late[..., dim - 2:].isfinite().any()) and bool(late[..., :dim - 2].isfinite().all())


@pytest.mark.parametrize("dim,group", [(64, 1), (64, 4), (128, 1), (128, 3), (128, 16), (256, 1), (256, 4), (80, 5)])
def test_the_last_new_token(dim, group):
    """V of the last token all NaN: every row but the last one's keeps its value, in tiles of one stream
    and of two, whole and cut, where the masked tokens lie in one tile of tokens, two or three."""
    for i, (n, total) in enumerate([(2, 2), (129, 129), (300, 300), (257, 3000), (64, 20000), (130, 1153)]):
        c = make(dim=dim, group=group, kv_heads=2, lens=((n, total), (5, 700)), seed=40 + i)
        _put(c, 0, total - 1, 0, slice(0, dim), math.nan)
        _put(c, 0, total - 1, 1, slice(0, 1), -math.inf)
        out = check(c)
        assert bool(out[:n - 1].isfinite().all())
        assert bool(out[n - 1, :group].isnan().all())


@pytest.mark.parametrize("dtype,cache,dim,layout", [("bf16", "same", 128, "nhd"), ("bf16", "same", 256, "nhd"), ("f16", "f8", 128, "nhd"),
                                                    ("bf16", "same", 128, "packed")])
def test_a_sequence_without_a_finite_value(dtype, cache, dim, layout):
    """All of V of a long prompt is NaN: the worst case for the rows' repair, in every one of its tiles.
    The others' bits stay, and the call stays far below the two seconds after which waits give up."""
    import torch
    import kvx_b200
    c = make(dtype=dtype, cache=cache, dim=dim, layout=layout, kv_heads=2, group=4, seed=50,
             lens=((8000, 8000), (3, 129), (150, 150), (1, 3000)))
    _timed(c)
    clean, usual = _timed(c)
    used = c["table"][0][:500].long()
    if cache == "f8":
        c["vc"].view(torch.uint8)[used] = 0x7F
    else:
        c["vc"][used] = math.nan
    out, ms = _timed(c)
    print(f"{dtype} {cache} {dim} {layout}: {ms:.2f} ms, finite {usual:.2f}")
    assert kvx_b200.lib().kvx_attention_device_error(0) == 0
    assert bool(out[:8000].isnan().all())
    kept = torch.equal(out[8000:], clean[8000:])
    assert kept
    assert ms < 500

"""Chunk attention where one token outweighs a long context of tokens of little weight each: what those
weigh together has to come out, although each of their weights is next to nothing in 16 bits.

One dominant token has V = 0 and score 0, all others V = 1 and the weight w = 2^-bits, so a row that sees
p others and the dominant one has out = p w / (1 + p w).  Tolerance (u = half a unit in the last place):
  * rounding of the weights: u relative; in f16 a weight is carried as 2^7 times itself, so what lies
    below 2^-21 of the largest is off by at most half of f16's smallest step, 2^-25 / 2^7 = 2^-32
    absolute; p of them (the denominator counts them exactly): p 2^-32;
  * rounding of the result: u relative;
  * p products added 16 at a time in f32, at most 2^-22 each time: (p / 16) 2^-22 relative;
  * the f32 sum of the weights, at most one addition per pair of a tile's tokens and one per tile: (64 + p / 128) 2^-24,
    the exponential and its argument (below 64): 2^-22 + 2^-18; all below 2^-13 here.
"""
import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [25.1, 24.7, 20.36, 12.0])
@pytest.mark.parametrize("where", ["first", "middle", "late"])
@pytest.mark.parametrize("dtype,cache,dim", [("f16", "same", 64), ("f16", "same", 128), ("f16", "same", 256), ("f16", "f8", 128),
                                             ("bf16", "same", 128)])
def test_many_small_weights(dtype, cache, dim, where, bits):
    import torch
    from kvx_b200 import ops
    dt, u = {"f16": (torch.float16, 2.0 ** -11), "bf16": (torch.bfloat16, 2.0 ** -8)}[dtype]
    total, n, seqs, bs = 131072, 160, 148, 64  # one tile of rows per share: contexts that are not cut
    store = torch.float8_e4m3fn if cache == "f8" else dt
    keys = torch.zeros((total // bs, bs, 1, dim), dtype=torch.float32, device="cuda")
    values = torch.ones_like(keys)
    keys[..., 0] = -16.0
    at = {"first": 0, "middle": total // 2, "late": total - 200}[where]
    keys[at // bs, at % bs] = 0.0
    values[at // bs, at % bs] = 0.0
    keys, values = keys.to(store), values.to(store)
    table = torch.arange(total // bs, device="cuda", dtype=torch.int32).repeat(seqs, 1)
    q = torch.zeros((n * seqs, 1, dim), dtype=dt, device="cuda")
    q[..., 0] = 1.0
    scale = torch.tensor(bits * math.log(2) / 16, dtype=torch.float32).item()
    one = torch.ones(1, device="cuda") if cache == "f8" else None
    out = ops.paged_attention_chunk(q, keys, values, table, torch.full((seqs,), total, dtype=torch.int32, device="cuda"),
                                    torch.arange(0, n * seqs + 1, n, device="cuda", dtype=torch.int32), scale,
                                    kv_cache_dtype="fp8" if cache == "f8" else "auto", k_scale=one, v_scale=one, num_kv_heads=1)
    p = torch.arange(total - n, total, device="cuda", dtype=torch.float64)  # others that new token i sees
    w = math.exp(-16 * scale)
    want = (p * w / (1 + p * w))[:, None].expand(n, dim)
    tol = want * (2 * u + p[:, None] / 16 * 2.0 ** -22 + 2.0 ** -13)
    if dtype == "f16":
        tol = tol + p[:, None] * 2.0 ** -32
    err = (out.double().view(seqs, n, dim) - want).abs() - tol
    worst = float(err.max())
    assert worst <= 0, (worst, float(want[0, 0]), float(out[0, 0, 0]))

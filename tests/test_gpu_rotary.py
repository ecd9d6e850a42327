"""Rotary positions (kvx_launch_rotary, kvx_launch_rotary_write_kv) against the formula in 64 bits.

Tolerance per element, from the arithmetic (u = 2^-8 bf16, 2^-11 f16, 2^-24 f32, half a unit in the
last place; X = the larger of |x1|, |x2|; f = |factor|):
  * the angle: reduced in f64, then half-turns as f32, off by at most 2^-24 (of half a turn), i.e.
    pi 2^-24 rad; sincospi within 2 ulp; factor as f32 and the product with it: 2 * 2^-24.
    Together below 8 * 2^-24 on cosine and sine;
  * y = fma(x1, c, -(x2 s)): two roundings below 2 * 2^-24 * 2 X f;
  * so |error| <= 2 X f * 10 * 2^-24 + the result's own rounding u * |y| (and the type's smallest
    step where y is tiny).
"""
import math

import pytest

pytestmark = pytest.mark.gpu

U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
TINY = {"bf16": 2.0 ** -133, "f16": 2.0 ** -24, "f32": 2.0 ** -149}


def _types():
    import torch
    return torch, {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def formula(x, positions, inv_freq, factor, interleaved, inverse, dtype):
    torch, _ = _types()
    half = inv_freq.numel()
    a = positions.double()[:, None] * inv_freq
    c, s = (a.cos() * factor)[:, None], (a.sin() * (-factor if inverse else factor))[:, None]
    z = x.double()
    out, tol = z.clone(), torch.zeros_like(z)
    i = torch.arange(half, device=x.device)
    i0, i1 = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    x1, x2 = z[..., i0], z[..., i1]
    out[..., i0], out[..., i1] = x1 * c - x2 * s, x2 * c + x1 * s
    big = torch.maximum(x1.abs(), x2.abs()) * abs(factor)
    for k in (i0, i1):
        tol[..., k] = 2 * big * 10 * 2.0 ** -24 + U[dtype] * out[..., k].abs() + TINY[dtype]
    return out, tol


def inputs(dtype, tokens, q_heads, k_heads, dim, pad=0, seed=0, far=100000, pos="i64", fused=False):
    torch, types = _types()
    g = torch.Generator(device="cuda").manual_seed(seed)
    heads = q_heads + k_heads * (2 if fused else 1)
    wide = torch.randn((tokens, heads * dim + pad), generator=g, device="cuda").to(types[dtype])
    rows = wide[:, :heads * dim].unflatten(1, (heads, dim))
    positions = torch.randint(-far // 10, far, (tokens,), generator=g, device="cuda")
    positions = positions.to(torch.int32) if pos == "i32" else positions
    return rows[:, :q_heads], rows[:, q_heads:q_heads + k_heads], rows[:, q_heads + k_heads:], positions


def close(got, exp, tol):
    err = ((got.double() - exp).abs() - tol).max()
    assert float(err) <= 0, float(err)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary_dim", [(128, 128), (64, 32), (80, 80), (96, 24), (40, 10), (7, 6), (256, 256), (128, 0), (32, 2)])
def test_formula(dtype, interleaved, dim, rotary_dim):
    """Both layouts, parts of the head, both tiers; Q and K; forward and inverse."""
    torch, _ = _types()
    from kvx_b200 import ops
    for i, (tokens, hq, hk, pad, pos) in enumerate([(1, 1, 1, 0, "i64"), (13, 7, 2, 0, "i32"), (200, 4, 4, 64, "i64"), (700, 3, 1, 3, "i64")]):
        q, k, _, positions = inputs(dtype, tokens, hq, hk, dim, pad, seed=i, pos=pos)
        freq, factor = (10000.0 ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / max(rotary_dim, 1))).cuda(), (1.0, 1.3)[i % 2]
        for inverse in (False, True):
            qo, ko = ops.rotary_embedding(q, k, positions, freq, interleaved=interleaved, factor=factor, inverse=inverse)
            close(qo, *formula(q, positions, freq, factor, interleaved, inverse, dtype))
            close(ko, *formula(k, positions, freq, factor, interleaved, inverse, dtype))


def test_in_place_outputs_and_no_key():
    torch, _ = _types()
    from kvx_b200 import ops
    q, k, _, positions = inputs("bf16", 300, 8, 2, 128, pad=40, seed=3)
    freq, _ = ops.rotary_inv_freq(64, device="cuda")
    qo, ko = ops.rotary_embedding(q, k, positions, freq)
    alone, none = ops.rotary_embedding(q, None, positions, freq)
    assert none is None and torch.equal(alone, qo)
    a, b = q.clone(), k.clone()
    ra, rb = ops.rotary_embedding(a, b, positions, freq, query_out=a, key_out=b)
    assert ra is a and torch.equal(a, qo) and torch.equal(b, ko)
    wide = torch.full((300, 8 * 128 + 9), 5.0, dtype=torch.bfloat16, device="cuda")
    view = wide[:, :8 * 128].unflatten(1, (8, 128))
    ops.rotary_embedding(q, None, positions, freq, query_out=view)
    assert torch.equal(view, qo) and bool((wide[:, 8 * 128:] == 5.0).all())


def test_inverse_undoes_and_is_the_gradient():
    """<R x, y> = <x, R^T y> (the inverse call is the transposed map), against differences too."""
    torch, _ = _types()
    from kvx_b200 import ops
    q, _, _, positions = inputs("f32", 50, 3, 1, 96, seed=4)
    freq, factor = ops.rotary_inv_freq(80, scaling="ramp", scale=4.0, high=32.0, device="cuda")
    for interleaved in (False, True):
        y = torch.randn_like(q.contiguous())
        fwd, _ = ops.rotary_embedding(q, None, positions, freq, interleaved, factor)
        grad, _ = ops.rotary_embedding(y, None, positions, freq, interleaved, factor, inverse=True)
        x64, y64 = q.double().clone().requires_grad_(True), y.double()
        out, _ = formula(x64.detach(), positions, freq, factor, interleaved, False, "f32")
        lhs, rhs = (fwd.double() * y64).sum(), (q.double() * grad.double()).sum()
        # both sums have q.numel() terms, each off by a few 2^-24 of its size
        size = (fwd.double() * y64).abs().sum()
        assert float((lhs - rhs).abs()) <= float(size) * 30 * 2.0 ** -24
        # the map is linear: a difference quotient is exact up to the roundings
        for (t, h, d) in ((0, 0, 0), (17, 2, 41), (49, 1, 95)):
            step = torch.zeros_like(x64.detach())
            step[t, h, d] = 1.0
            up, _ = formula(x64.detach() + step, positions, freq, factor, interleaved, False, "f32")
            assert abs(float(((up - out) * y64).sum()) - float(grad[t, h, d])) <= 1e-5 * (1 + abs(float(grad[t, h, d])))
        back, _ = ops.rotary_embedding(fwd, None, positions, freq, interleaved, 1.0 / factor, inverse=True)
        assert float((back - q).abs().max()) <= 40 * 2.0 ** -24 * float(q.abs().max())


def test_far_positions_keep_their_accuracy():
    torch, _ = _types()
    from kvx_b200 import ops
    q, _, _, _ = inputs("f32", 64, 2, 1, 64, seed=5)
    positions = torch.randint(2 ** 33, 2 ** 34, (64,), device="cuda")
    freq, _ = ops.rotary_inv_freq(64, device="cuda")
    out, _ = ops.rotary_embedding(q, None, positions, freq)
    exp, tol = formula(q, positions, freq, 1.0, False, False, "f32")
    # the f64 product of a position of 2^34 is off by 2^34 2^-52 rad, on both sides
    close(out, exp, tol + q.abs().max().double() * 4 * 2.0 ** -18)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("cache_dtype", ["auto", "fp8"])
@pytest.mark.parametrize("layout", ["nhd", "hnd", "view", "packed"])
def test_fused_write_equals_the_two_steps(dtype, cache_dtype, layout):
    """The pages hold the bits of rotary followed by the cache write; the query is turned, the key is
    not touched; padding, slots behind the pool, odd head dims and pages."""
    torch, types = _types()
    from kvx_b200 import ops
    for i, (tokens, hq, hk, dim, rd, bs, inter) in enumerate([(1, 4, 1, 128, 128, 16, False), (77, 8, 2, 64, 32, 16, True),
                                                              (300, 6, 3, 80, 80, 8, False), (65, 2, 2, 40, 20, 5, False),
                                                              (2500, 8, 8, 128, 64, 32, False)]):
        q, k, v, positions = inputs(dtype, tokens, hq, hk, dim, pad=16 * i, seed=i, fused=True)
        blocks = tokens // bs + 4
        g = torch.Generator(device="cuda").manual_seed(i)
        ct = torch.float8_e4m3fn if cache_dtype == "fp8" else types[dtype]
        shape = {"nhd": (blocks, bs, hk, dim), "hnd": (blocks, hk, bs, dim), "view": (blocks, hk, bs, dim),
                 "packed": (blocks, hk, dim // 8, bs, 8)}[layout]
        def pool():
            x = torch.zeros(shape, device="cuda").to(ct)
            return x.transpose(1, 2) if layout == "view" else x
        kc, vc, kc2, vc2 = pool(), pool(), pool(), pool()
        slots = torch.randperm(blocks * bs, generator=g, device="cuda")[:tokens]
        slots[::7] = -1
        if tokens > 20:
            slots[11] = blocks * bs + 3
        if i % 2:
            slots = slots.to(torch.int32)
        ks = vs = None
        if cache_dtype == "fp8":
            ks = torch.rand((hk,), generator=g, device="cuda") * 0.02 + 0.001
            vs = torch.rand((1,), generator=g, device="cuda") * 0.02 + 0.001
        freq, factor = ops.rotary_inv_freq(rd, scaling="bands", scale=8.0, device="cuda")
        before = k.clone()
        qo = ops.rotary_and_cache(q, k, v, positions, freq, kc, vc, slots, inter, factor, kv_cache_dtype=cache_dtype, k_scale=ks,
                                  v_scale=vs)
        q2, k2 = ops.rotary_embedding(q, k, positions, freq, inter, factor)
        ops.reshape_and_cache_flash_kvx(k2, v, kc2, vc2, slots, kv_cache_dtype=cache_dtype, k_scale=ks, v_scale=vs)
        torch.cuda.synchronize()
        assert torch.equal(k, before)
        same_q = torch.equal(qo, q2)
        assert same_q
        for a, b in ((kc, kc2), (vc, vc2)):
            same = torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
            assert same, (i, layout)


def test_no_tokens_and_graph_replay():
    torch, _ = _types()
    from kvx_b200 import ops
    freq, _ = ops.rotary_inv_freq(128, device="cuda")
    q, k, v, positions = inputs("bf16", 0, 4, 2, 128, fused=True)
    kc = torch.zeros((4, 16, 2, 128), dtype=torch.bfloat16, device="cuda")
    ops.rotary_embedding(q, k, positions, freq)
    ops.rotary_and_cache(q, k, v, positions, freq, kc, kc.clone(), positions)
    q, k, v, positions = inputs("bf16", 33, 4, 2, 128, seed=9, fused=True)
    vc, slots, out = kc.clone(), torch.arange(33, device="cuda"), torch.empty_like(q, memory_format=torch.contiguous_format)
    ops.rotary_and_cache(q, k, v, positions, freq, kc, vc, slots, query_out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rotary_and_cache(q, k, v, positions, freq, kc, vc, slots, query_out=out)
    positions.add_(17)
    slots.copy_(slots.flip(0).clone())
    graph.replay()
    torch.cuda.synchronize()
    close(out, *formula(q, positions, freq, 1.0, False, False, "bf16"))
    exp, tol = formula(k, positions, freq, 1.0, False, False, "bf16")
    close(kc.flatten(0, 1)[slots], exp, tol)
    assert torch.equal(vc.flatten(0, 1)[slots], v)


def test_frequencies_of_the_scalings():
    """Kept, divided and blended pairs where their definitions put them (no GPU work)."""
    torch, _ = _types()
    from kvx_b200 import ops
    plain, one = ops.rotary_inv_freq(128, base=500000.0)
    assert one == 1.0 and float(plain[0]) == 1.0 and math.isclose(float(plain[32]), 500000.0 ** -0.5, rel_tol=1e-14)
    lin, _ = ops.rotary_inv_freq(128, base=500000.0, scaling="linear", scale=8.0)
    assert torch.allclose(lin * 8, plain, rtol=1e-14)
    ntk, _ = ops.rotary_inv_freq(128, base=10000.0, scaling="ntk", scale=4.0)
    ref, _ = ops.rotary_inv_freq(128, base=10000.0)
    assert float(ntk[0]) == 1.0 and math.isclose(float(ntk[-1]) * 4, float(ref[-1]), rel_tol=1e-12)
    bands, one = ops.rotary_inv_freq(128, base=500000.0, scaling="bands", scale=8.0)
    turns = 8192 * plain / (2 * math.pi)
    assert one == 1.0 and torch.equal(bands[turns >= 4], plain[turns >= 4])
    assert torch.allclose(bands[turns <= 1] * 8, plain[turns <= 1], rtol=1e-14)
    mid = (turns > 1) & (turns < 4)
    keep = (turns[mid] - 1) / 3
    assert torch.allclose(bands[mid], plain[mid] * (keep + (1 - keep) / 8), rtol=1e-14)
    ramp, factor = ops.rotary_inv_freq(128, scaling="ramp", scale=4.0, original_length=4096, low=1.0, high=32.0)
    assert math.isclose(factor, 0.1 * math.log(4.0) + 1.0) and float(ramp[0]) == 1.0
    assert math.isclose(float(ramp[-1]) * 4, float(ref[-1]), rel_tol=1e-12)

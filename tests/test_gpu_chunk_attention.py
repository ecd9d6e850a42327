"""Attention of a chunk of new tokens over the paged cache (kvx_launch_paged_attention_chunk)
against the formula in 64 bits.

Tolerances, per element, from the arithmetic (u = half a unit in the last place, relative:
2^-8 bf16, 2^-11 f16, 2^-24 f32; V = the largest |v| of the row's K/V head):
  * rounding of the result: u * |out|;
  * tensor-core path: weights rounded to the type, each off by at most u relative, so the weighted
    mean moves by at most u * sum(w |v|) / sum(w) <= u * V; f32 path: none;
  * scores are sums of `dim` products in f32 (inputs are exact products): |error| <= (dim + 2) *
    2^-24 * scale * sum |q k| <= (dim + 2) * 2^-24 * scale * dim * Q * K, with Q, K the largest |q|,
    |k|; a score moved by e changes a weight by the factor exp(e), the mean by at most 2 (exp(e) - 1) V;
  * ex2 and the f32 sums: 2^-22 per weight and (tokens + 4) * 2^-24 for the sums, relative to V.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}


def _torch():
    import torch
    return torch, {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def make(dtype="bf16", cache="same", kv_heads=2, group=4, dim=128, block_size=16, layout="nhd", lens=((5, 40),), seed=0,
         index="i32", indptr="i32", bad_pages=0, extra_rows=0, q_pad=0, spread=1.0, k_scales="head"):
    """Pages, tables and queries of a batch; `lens` is (new tokens, cached tokens) per sequence."""
    torch, types = _torch()
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = types[dtype]
    need = [(n + block_size - 1) // block_size for _, n in lens]
    blocks = sum(need) + 3
    shape = {"nhd": (blocks, block_size, kv_heads, dim), "hnd": (blocks, kv_heads, block_size, dim),
             "packed": (blocks, kv_heads, dim // 8, block_size, 8)}[layout]
    pages = [torch.randn(shape, generator=g, device="cuda") for _ in range(2)]
    ks = vs = None
    if cache == "f8":
        pages = [(x * 50).to(torch.float8_e4m3fn) for x in pages]
        n = kv_heads if k_scales == "head" else 1
        ks = torch.rand((n,), generator=g, device="cuda") * 0.01 + 0.015
        vs = torch.rand((n,), generator=g, device="cuda") * 0.01 + 0.015
    else:
        pages = [x.to(dt) for x in pages]
    idx = torch.int32 if index == "i32" else torch.int64
    perm = torch.randperm(blocks, generator=g, device="cuda")
    table = torch.full((len(lens), max(max(need), 1) + 1), -1, dtype=idx, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = perm[at:at + n].to(idx)
        at += n
    if bad_pages:
        flat = table.view(-1)
        used = (flat >= 0).nonzero().view(-1)
        hit = used[torch.randperm(used.numel(), generator=g, device="cuda")[:bad_pages]]
        flat[hit] = torch.tensor([-1, blocks, -7, blocks + 1000], device="cuda", dtype=idx)[:bad_pages].repeat(bad_pages)[:bad_pages]
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    rows = starts[-1] + extra_rows
    wide = torch.randn((rows, kv_heads * group * dim + q_pad), generator=g, device="cuda") * spread
    q = wide.to(dt)[:, :kv_heads * group * dim].unflatten(1, (kv_heads * group, dim))
    return dict(q=q, kc=pages[0], vc=pages[1], table=table, lens=torch.tensor([n for _, n in lens], dtype=idx, device="cuda"),
                indptr=torch.tensor(starts, dtype=torch.int32 if indptr == "i32" else torch.int64, device="cuda"),
                ks=ks, vs=vs, dtype=dtype, layout=layout, block_size=block_size, kv_heads=kv_heads, group=group, dim=dim,
                host=list(lens), starts=starts)


def rows_of(c, cache, s, total, h, scale):
    """The cached tokens of one head of one sequence in 64 bits and which of them take part."""
    torch, _ = _torch()
    t = torch.arange(total, device="cuda")
    lb = t // c["block_size"]
    inside = lb < c["table"].shape[1]
    page = c["table"][s].long()[lb.clamp(max=c["table"].shape[1] - 1)]
    ok = inside & (page >= 0) & (page < cache.shape[0])
    page = torch.where(ok, page, 0)
    at = t % c["block_size"]
    src = cache.float() if cache.dtype == torch.float8_e4m3fn else cache
    if c["layout"] == "nhd":
        x = src[page, at, h]
    elif c["layout"] == "hnd":
        x = src[page, h, at]
    else:
        x = src[page, h, :, at].reshape(total, c["dim"])
    x = x.double()
    if scale is not None:
        x = x * scale[h if scale.numel() > 1 else 0].double()
    return x, ok


def expected(c, scale, causal=True, max_seq_len=None):
    """(out, tolerance) in 64 bits; NaN where no sequence owns the row."""
    torch, _ = _torch()
    H, G, D = c["kv_heads"], c["group"], c["dim"]
    out = torch.full((c["q"].shape[0], H * G, D), math.nan, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    u = U[c["dtype"]]
    for s, (n, total) in enumerate(c["host"]):
        if n == 0:
            continue
        seen = total if max_seq_len is None else min(total, max_seq_len)
        a = c["starts"][s]
        pos = torch.arange(total - n, total, device="cuda")
        for h in range(H):
            k, ok = rows_of(c, c["kc"], s, seen, h, c["ks"])
            v, _ = rows_of(c, c["vc"], s, seen, h, c["vs"])
            see = ok[None, :].expand(n, -1)
            if causal:
                see = see & (torch.arange(seen, device="cuda")[None, :] <= pos[:, None])
            for g in range(G):
                q = c["q"][a:a + n, h * G + g].double()
                sc = (q @ torch.where(ok[:, None], k, 0.0).t()) * scale if seen else q.new_zeros((n, 0))
                sc = torch.where(see, sc, -math.inf)
                m = sc.amax(-1, keepdim=True) if seen else sc.new_zeros((n, 1))
                w = torch.where(see, torch.exp(sc - torch.where(m.isinf(), 0.0, m)), 0.0)
                l = w.sum(-1, keepdim=True)
                vv = torch.where(ok[:, None], v, 0.0)
                # a token that is not seen is left out even where its V is not finite
                o = (w @ torch.nan_to_num(vv, nan=0.0, posinf=0.0, neginf=0.0)) if seen else q.new_zeros((n, D))
                if seen and not bool(torch.isfinite(vv).all()):  # a seen NaN gives NaN, infinities themselves
                    hit = lambda bad: (w > 0).double() @ bad.double() > 0
                    up, down, nan = hit(vv == math.inf), hit(vv == -math.inf), hit(vv.isnan())
                    o = torch.where(up, math.inf, torch.where(down, -math.inf, o))
                    o = torch.where(nan | (up & down), math.nan, o)
                o = torch.where(l > 0, o / l, 0.0)
                out[a:a + n, h * G + g] = o
                if seen:
                    big = lambda x: torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0).abs().amax()
                    V = big(vv)
                    e = (D + 2) * 2.0 ** -24 * abs(scale) * D * q.abs().amax() * big(torch.where(ok[:, None], k, 0.0))
                    t = u * o.abs() + V * (2 * (torch.exp(e) - 1) + 2.0 ** -22 + (seen + 4) * 2.0 ** -24)
                    if c["dtype"] != "f32":
                        t = t + u * V
                    tol[a:a + n, h * G + g] = t
    return out, tol


def run(c, scale, causal=True, max_seq_len=None, out=None, **kw):
    from kvx_b200 import ops
    fp8 = c["ks"] is not None
    return ops.paged_attention_chunk(c["q"], c["kc"], c["vc"], c["table"], c["lens"], c["indptr"], scale, causal=causal,
                                     max_seq_len=max_seq_len, out=out, kv_cache_dtype="fp8" if fp8 else "auto",
                                     k_scale=c["ks"], v_scale=c["vs"], num_kv_heads=c["kv_heads"], **kw)


def check(c, scale=None, causal=True, max_seq_len=None):
    torch, _ = _torch()
    import kvx_b200
    scale = c["dim"] ** -0.5 if scale is None else scale
    out = torch.full(c["q"].shape, 7.0, dtype=c["q"].dtype, device="cuda")
    run(c, scale, causal, max_seq_len, out=out)
    torch.cuda.synchronize()
    assert kvx_b200.lib().kvx_attention_device_error(0) == 0
    exp, tol = expected(c, scale, causal, max_seq_len)
    got = out.double()
    last = c["starts"][-1]
    assert bool((got[last:] == 7.0).all()), "rows behind the last sequence were written"
    got, exp, tol = got[:last], exp[:last], tol[:last]
    same_nan = torch.equal(got.isnan(), exp.isnan())
    assert same_nan
    err = torch.where(exp.isnan() | (got == exp), 0.0, (got - exp).abs() - tol)
    worst = float(err.max()) if err.numel() else 0.0
    assert worst <= 0, (worst, [int(i) for i in (err == err.max()).nonzero()[0]])
    return out


@pytest.mark.parametrize("layout", ["nhd", "hnd"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_one_tile(dtype, layout, dim):
    """Few rows, few tokens: one step of one stream, then two streams, then several steps."""
    for i, lens in enumerate([((1, 1),), ((5, 40),), ((17, 130),), ((32, 300), (1, 77), (3, 3))]):
        check(make(dtype=dtype, dim=dim, layout=layout, lens=lens, seed=i))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_wide_tiles(dim, causal):
    """More than one stream of rows, several tiles per head, tiles cut between CTAs, odd groups."""
    for i, (group, lens) in enumerate([(4, ((64, 64), (65, 200))), (3, ((500, 1000),)), (8, ((129, 129), (1, 900), (33, 2000))),
                                       (1, ((1000, 1500),)), (5, ((260, 260), (0, 50), (7, 4100)))]):
        check(make(dim=dim, group=group, lens=lens, seed=10 + i, spread=2.0), causal=causal)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_many_sequences_of_all_lengths(dtype):
    """Hundreds of sequences, with empty ones, ones longer in new tokens than in cached ones (rows at
    negative positions see nothing), and contexts around the edges of pages and tiles."""
    torch, _ = _torch()
    g = torch.Generator().manual_seed(3)
    n = torch.randint(0, 9, (300,), generator=g).tolist()
    t = [[0, 1, 2, 15, 16, 17, 127, 128, 129, 255, 256, 257, 300, 511, 640][i] for i in torch.randint(0, 15, (300,), generator=g).tolist()]
    check(make(dtype=dtype, lens=tuple(zip(n, t)), kv_heads=2, group=4, dim=64, seed=4))


def test_rows_that_see_nothing():
    check(make(lens=((20, 3), (5, 0), (300, 290), (2, 2)), seed=5))
    check(make(lens=((20, 3), (5, 0), (300, 290), (2, 2)), seed=5), causal=False)


@pytest.mark.parametrize("block_size,layout", [(8, "nhd"), (16, "hnd"), (24, "nhd"), (64, "nhd"), (128, "hnd"), (256, "nhd"),
                                               (1, "nhd"), (5, "nhd"), (12, "hnd"), (16, "packed"), (7, "packed")])
def test_page_sizes_and_layouts(block_size, layout):
    """Pages inside a tile, pages larger than a tile, pages TMA cannot read."""
    check(make(block_size=block_size, layout=layout, lens=((40, 300), (3, 129), (150, 150)), seed=block_size))


@pytest.mark.parametrize("dim", [8, 40, 72, 80, 96, 120, 160, 192, 248, 100, 65])
def test_head_dims(dim):
    """Head dims below the operand's width, down to ones without 16-byte rows."""
    check(make(dim=dim, lens=((40, 300), (3, 129), (200, 600)), seed=dim))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim,k_scales", [(64, "head"), (128, "tensor"), (128, "head"), (256, "head"), (80, "head")])
def test_fp8_cache(dtype, dim, k_scales):
    check(make(dtype=dtype, cache="f8", dim=dim, k_scales=k_scales, lens=((40, 300), (3, 1290), (150, 150), (1, 17)), seed=dim))
    check(make(dtype=dtype, cache="f8", dim=dim, k_scales=k_scales, block_size=64, layout="hnd", lens=((4, 300),), seed=dim))


@pytest.mark.parametrize("dim", [16, 64, 128, 200, 320, 600])
def test_f32(dim):
    check(make(dtype="f32", dim=dim, lens=((40, 300), (3, 1290), (70, 70), (1, 1), (2, 0)), seed=dim, group=3))
    check(make(dtype="f32", dim=dim, lens=((40, 300),), seed=dim, block_size=6, layout="hnd"), causal=False)


def test_wide_head_dim_in_16_bits():
    check(make(dtype="bf16", dim=320, lens=((40, 300), (3, 129)), seed=1))


def test_bad_pages():
    for i, (dt, bs) in enumerate([("bf16", 16), ("f16", 32), ("f32", 16), ("bf16", 6), ("bf16", 8)]):
        check(make(dtype=dt, block_size=bs, bad_pages=4, lens=((40, 300), (3, 1290), (150, 150)), seed=20 + i))


def test_index_types_strides_and_rows_without_a_sequence():
    """64-bit tables, 64-bit row numbers, query slices of a wider projection, rows behind the batch."""
    check(make(index="i64", indptr="i64", q_pad=512, extra_rows=9, lens=((40, 300), (3, 129)), seed=1))
    check(make(index="i64", q_pad=3, extra_rows=2, lens=((40, 300), (3, 129)), seed=2))
    check(make(dtype="f32", indptr="i64", q_pad=5, extra_rows=2, lens=((40, 300), (3, 129)), seed=3))


def test_max_seq_len_cuts_the_context():
    c = make(lens=((40, 300), (3, 1290), (150, 150)), seed=2)
    for n in (1, 100, 128, 290, 1000):
        check(c, max_seq_len=n)


def test_scales_of_every_sign():
    c = make(lens=((40, 300), (3, 129)), seed=6)
    for scale in (-0.1, 0.0, 1e-6, 0.7):
        check(c, scale=scale)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_long_context_is_cut_and_joined(dim):
    check(make(dim=dim, kv_heads=1, group=4, lens=((3, 20000),), seed=7))
    check(make(dim=dim, kv_heads=2, group=2, lens=((300, 9000), (1, 5000)), seed=8))


@pytest.mark.parametrize("dtype,cache", [("bf16", "same"), ("f32", "same"), ("f16", "f8")])
def test_values_behind_the_mask_do_not_matter(dtype, cache):
    """NaN and infinities in K and V where no row may look: behind the sequence in its last page, in
    pages the table does not name, and at later positions than a row's own -- the rows before
    that position keep their values, the rows that see it get the NaN."""
    torch, _ = _torch()
    c = make(dtype=dtype, cache=cache, lens=((40, 300), (3, 129), (150, 150)), seed=9, block_size=32)
    clean = check(c)
    bs = c["block_size"]
    used = torch.zeros(c["kc"].shape[0] * bs, dtype=torch.bool, device="cuda")
    for s, (_, total) in enumerate(c["host"]):
        t = torch.arange(total, device="cuda")
        used[c["table"][s].long()[t // bs] * bs + t % bs] = True
    for name in ("kc", "vc"):
        flat = c[name].view(torch.uint8).flatten(0, 1) if cache == "f8" else c[name].flatten(0, 1)
        flat[~used] = 0x7F if cache == "f8" else math.nan
    again = check(c)
    same = torch.equal(again, clean)
    assert same
    # the last prompt's token 70 turns bad in V: only rows from there on may change
    s, tok = 2, 70
    page = int(c["table"][s][tok // bs])
    if cache == "f8":
        c["vc"].view(torch.uint8)[page, tok % bs, 0, :5] = 0x7F
    else:
        c["vc"][page, tok % bs, 0, :5] = math.nan
        c["vc"][page, tok % bs, 1, :5] = math.inf
    check(c)
    first = c["starts"][s]
    # and in K, where the score decides
    if cache != "f8":
        c["kc"][page, tok % bs, 0, 3] = math.nan
        out = run(c, c["dim"] ** -0.5)
        assert bool(out[first:first + tok].isfinite().all())
        assert bool(out[first + tok:first + 150, :c["group"]].isnan().all())


def test_calls_are_repeatable_and_independent_of_scratch():
    """The same bits from call to call, whatever the scratch holds."""
    torch, _ = _torch()
    from kvx_b200 import ops
    c = make(lens=((500, 1000), (3, 5000), (1, 1)), seed=11)
    n = ops.chunk_attention_workspace_bytes(3, 504, 8, 2, 128, 5200)
    outs = []
    for fill in (0, 0xFF, 0x7F):
        ws = torch.full((n,), fill, dtype=torch.uint8, device="cuda")
        outs.append(run(c, 0.1, workspace=ws, max_seq_len=5200))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_one_new_token_agrees_with_decode_attention():
    """n = 1 is the decode step: both operators are within their tolerances of one formula."""
    torch, _ = _torch()
    from kvx_b200 import ops
    c = make(lens=tuple((1, n) for n in (1, 16, 100, 257, 411, 3000)), seed=12)
    out = check(c, scale=0.09)
    dec = ops.paged_attention_decode(c["q"].contiguous(), c["kc"], c["vc"], c["table"], c["lens"], 0.09, num_kv_heads=2)
    assert torch.allclose(out.float(), dec.float(), atol=1.5e-2, rtol=1.6e-2)


def test_graph_replay_with_new_lengths():
    """A captured call follows the lengths and tables it finds at replay."""
    torch, _ = _torch()
    from kvx_b200 import ops
    c = make(lens=((40, 300), (64, 2000)), seed=13)
    n = ops.chunk_attention_workspace_bytes(2, 104, 8, 2, 128, 2016)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    out = torch.zeros_like(c["q"], memory_format=torch.contiguous_format)
    run(c, 0.1, out=out, workspace=ws, max_seq_len=2016)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(c, 0.1, out=out, workspace=ws, max_seq_len=2016)
    for lens in (((40, 300), (64, 2000)), ((60, 200), (44, 1000)), ((0, 10), (104, 104))):
        c["host"] = list(lens)
        c["starts"] = [0, lens[0][0], lens[0][0] + lens[1][0]]
        c["lens"].copy_(torch.tensor([t for _, t in lens]))
        c["indptr"].copy_(torch.tensor(c["starts"]))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        exp, tol = expected(c, 0.1)
        assert float(((out.double() - exp).abs() - tol).max()) <= 0


def test_two_streams_with_scratch_of_their_own():
    torch, _ = _torch()
    a, b = make(lens=((500, 1000),), seed=14), make(lens=((300, 4000),), seed=15, group=2)
    ea, eb = run(a, 0.1), run(b, 0.1)
    torch.cuda.synchronize()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(sa):
            oa = run(a, 0.1)
        with torch.cuda.stream(sb):
            ob = run(b, 0.1)
        torch.cuda.synchronize()
        assert torch.equal(oa, ea) and torch.equal(ob, eb)


def test_more_sequences_than_the_plan_scans_at_once():
    torch, _ = _torch()
    g = torch.Generator().manual_seed(5)
    n = torch.randint(0, 3, (2500,), generator=g).tolist()
    t = torch.randint(0, 60, (2500,), generator=g).tolist()
    check(make(lens=tuple(zip(n, t)), kv_heads=1, group=2, dim=64, seed=6, block_size=32))


@pytest.mark.parametrize("cache", ["same", "f8"])
@pytest.mark.parametrize("layout", ["nhd", "hnd"])
@pytest.mark.parametrize("dim", [64, 80, 96, 128, 192, 256])
def test_heads_do_not_touch_each_other(dim, layout, cache):
    """NaN all over the K and V of every other head: the heads between keep their bits."""
    torch, _ = _torch()
    c = make(dim=dim, layout=layout, cache=cache, kv_heads=4, group=2, lens=((70, 300), (3, 40)), seed=15)
    clean = check(c)
    for name in ("kc", "vc"):
        x = c[name].view(torch.uint8) if cache == "f8" else c[name]
        for h in (1, 3):
            (x[:, :, h] if layout == "nhd" else x[:, h]).fill_(0x7F if cache == "f8" else math.nan)
    out = run(c, dim ** -0.5)
    kept, lost = out.unflatten(1, (4, 2))[:, [0, 2]], out.unflatten(1, (4, 2))[:, [1, 3]]
    same = torch.equal(kept, clean.unflatten(1, (4, 2))[:, [0, 2]])
    assert same
    all_nan = bool(lost.isnan().all())
    assert all_nan


def test_rows_behind_the_query_keep_their_positions():
    """query_indptr that names more rows than there are: those that exist are where they would be; the
    same for lengths beyond 32 bits that max_seq_len cuts."""
    torch, _ = _torch()
    c = make(lens=((9, 40), (20, 90)), seed=16, indptr="i64")
    full = check(c)
    c["q"] = c["q"][:17]
    out = run(c, c["dim"] ** -0.5)
    same = torch.equal(out, full[:17])
    assert same
    c["indptr"][2] = 2 ** 40  # the sequence's tokens lie far ahead of its length: none sees anything
    out = run(c, c["dim"] ** -0.5)
    assert torch.equal(out[:9], full[:9]) and not bool(out[9:].any())
    c = make(lens=((9, 40), (20, 90)), seed=16, index="i64")
    c["lens"][1] = 2 ** 40  # every new token is behind max_seq_len and sees all of it
    out = run(c, c["dim"] ** -0.5, max_seq_len=90)
    want, tol = expected(c, c["dim"] ** -0.5, causal=False)
    worst = float(((out[9:].double() - want[9:]).abs() - tol[9:]).max())
    assert worst <= 0


@pytest.mark.parametrize("layout", ["nhd", "hnd"])
@pytest.mark.parametrize("dim", [4, 60, 64, 100, 128, 192, 256])
def test_f32_tiles(dim, layout):
    """Full and ragged tiles of the f32 kernel, cut and whole, with pages that are missing."""
    for i, (group, lens, causal) in enumerate([(1, ((1, 1), (64, 64), (65, 130)), True), (5, ((13, 300), (1, 700)), True),
                                               (4, ((50, 200), (0, 9), (3, 2)), False)]):
        check(make(dtype="f32", dim=dim, layout=layout, group=group, lens=lens, seed=20 + i, bad_pages=i, block_size=(16, 8, 20)[i]),
              causal=causal)


@pytest.mark.parametrize("layout,cache,dim", [("packed", "same", 64), ("nhd", "f8", 128), ("nhd", "same", 66), ("hnd", "f8", 80)])
def test_f32_queries_over_other_pages(layout, cache, dim):
    """What the f32 kernel's copies cannot read goes element by element."""
    check(make(dtype="f32", cache=cache, dim=dim, layout=layout, group=2, lens=((40, 300), (1, 33)), seed=24))

"""Timed cases of the serving-step operators around the paged cache: rotary positions (alone and
fused with the cache write), attention of a chunk of new tokens over the pages, and the upkeep of
the pages themselves (copy, fork, free, compact).

``run`` computes a case in elementary torch operations, or through ``kvx_b200.ops`` when ``own``
is true.  Shapes follow the configurations of ``kvx_b200/workloads.py``: 8 KV heads of 128 with 4
query heads each and pages of 16 tokens (c2), 4 heads of 64 in half precision (c1), pages of 64
with an e4m3 cache (c5), contexts log-uniform up to 32 768 (c3).
"""
import math

import torch

own = False

TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4, "f8": 1}


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one decode step's positions and cache write of a middling batch: launch latency counts
        dict(name="rotary_cache_decode", op="rotary_cache", tokens=64, q_heads=32, kv_heads=8, dim=128, rotary_dim=128,
             interleaved=False, scaling="none", dtype="bf16", block_size=16, far=32768, padded=4),
        # one layer of a large prefill batch, long-context frequencies, a tenth of the slots padding
        dict(name="rotary_cache_prefill", op="rotary_cache", tokens=16384, q_heads=32, kv_heads=8, dim=128, rotary_dim=128,
             interleaved=False, scaling="bands", dtype="bf16", block_size=16, far=131072, padded=1638),
        # neighbouring pairs over half of each head, ragged token count, the transposed map (gradient)
        dict(name="rotary_interleaved_part", op="rotary", tokens=1021, q_heads=16, kv_heads=16, dim=128, rotary_dim=64,
             interleaved=True, scaling="ramp", dtype="f16", far=1000000, inverse=True),
        # a short prompt alone on the machine
        dict(name="chunk_short_prompt", op="chunk", dtype="f16", cache="f16", kv_heads=4, group=8, dim=64, block_size=16,
             layout="nhd", seqs=1, new_lo=17, new_hi=17, ctx_lo=53, ctx_hi=53, causal=True),
        # prefill of whole prompts, lengths of the c2 configuration
        dict(name="chunk_prefill", op="chunk", dtype="bf16", cache="bf16", kv_heads=8, group=4, dim=128, block_size=16,
             layout="nhd", seqs=16, new_lo=512, new_hi=4096, ctx_lo=0, ctx_hi=0, causal=True),
        # chunked prefill: the next 512 tokens of four long documents
        dict(name="chunk_long_context", op="chunk", dtype="bf16", cache="bf16", kv_heads=8, group=4, dim=128, block_size=16,
             layout="hnd", seqs=4, new_lo=512, new_hi=512, ctx_lo=30000, ctx_hi=32256, causal=True),
        # drafted tokens verified together: five new tokens on contexts of a decode batch
        dict(name="chunk_verify", op="chunk", dtype="bf16", cache="bf16", kv_heads=8, group=4, dim=128, block_size=32,
             layout="nhd", seqs=64, new_lo=5, new_hi=5, ctx_lo=1, ctx_hi=32768, causal=True),
        # mid-sized chunks over an e4m3 cache with one scale per head
        dict(name="chunk_fp8_cache", op="chunk", dtype="bf16", cache="f8", kv_heads=8, group=4, dim=128, block_size=64,
             layout="nhd", seqs=16, new_lo=100, new_hi=156, ctx_lo=1000, ctx_hi=4000, causal=True),
        # copy-on-write of a few pages through all layers of a model
        dict(name="pages_copy", op="copy", pairs=24, pages=256, layers=32, dtype="bf16", block_size=16, kv_heads=8, dim=128),
        # beam step: some sequences end, others fork with their last page duplicated
        dict(name="pages_fork", op="fork", seqs=96, ended=24, forks=48, max_len=400, pages=2048, layers=16, dtype="bf16",
             block_size=16, kv_heads=4, dim=128),
        # defragmentation of a pool that is a little over half full
        dict(name="pages_compact", op="compact", seqs=32, live=0.55, pages=2048, layers=8, dtype="bf16", block_size=16,
             kv_heads=8, dim=128),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "rotary_cache", "chunk", "chunk", "chunk", "copy", "fork", "compact"])
    if op in ("rotary", "rotary_cache"):
        kv_heads = rng.choice([1, 2, 4, 5, 8, 16])
        q_heads = kv_heads * rng.choice([1, 2, 4, 7, 8])
        dim = rng.choice([64, 80, 96, 128, 256])
        dtype = rng.choice(["bf16", "f16", "f32"])
        rotary_dim = rng.choice([dim, dim, dim // 2, dim // 4])
        most = min(16384, max(1, 16384 * 40 * 128 * 2 // ((q_heads + kv_heads) * dim * BYTES[dtype])))
        case = dict(op=op, tokens=_log_int(rng, 1, most), q_heads=q_heads, kv_heads=kv_heads, dim=dim,
                    rotary_dim=rotary_dim, interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "bands", "ramp"]),
                    dtype=dtype, far=_log_int(rng, 100, 1000000))
        if op == "rotary":
            case["inverse"] = rng.random() < 0.5
        else:
            case["block_size"] = rng.choice([8, 16, 32, 64])
            case["padded"] = rng.randrange(0, case["tokens"] // 4 + 1)
        return case
    if op == "chunk":
        dtype, cache = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f8"), ("f16", "f8"),
                                   ("f32", "f32")])
        dim = rng.choice([64, 64, 96, 128, 128, 256])
        kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
        new_hi, ctx_hi = _log_int(rng, 1, 4096), _log_int(rng, 1, 32768)
        cost = 4.0 * dim * kv_heads * group * new_hi * (ctx_hi + new_hi)  # one sequence at the largest lengths
        limit = 2e10 if dtype == "f32" else 8e11
        seqs = _log_int(rng, 1, 64)
        while new_hi > 1 and cost > limit:
            new_hi = (new_hi + 1) // 2
            cost = 4.0 * dim * kv_heads * group * new_hi * (ctx_hi + new_hi)
        seqs = max(1, min(seqs, int(limit // cost)))
        # the pool stays below 4 GB
        seqs = max(1, min(seqs, int(4e9 // ((ctx_hi + new_hi + 64) * kv_heads * dim * 2 * BYTES[cache]))))
        return dict(op="chunk", dtype=dtype, cache=cache, kv_heads=kv_heads, group=group, dim=dim,
                    block_size=rng.choice([8, 16, 16, 32, 64, 128]), layout=rng.choice(["nhd", "nhd", "hnd"]), seqs=seqs,
                    new_lo=rng.choice([1, max(1, new_hi // 4), new_hi]), new_hi=new_hi,
                    ctx_lo=rng.choice([0, ctx_hi // 2]), ctx_hi=ctx_hi,
                    causal=rng.random() < 0.85)
    shape = dict(dtype=rng.choice(["bf16", "f32", "f8"]), block_size=rng.choice([8, 16, 32]), kv_heads=rng.choice([1, 2, 4, 8]),
                 dim=rng.choice([64, 80, 128]), layers=_log_int(rng, 1, 16))
    if op == "copy":
        pages = _log_int(rng, 8, 1500)
        return dict(op="copy", pairs=rng.randrange(1, pages // 2 + 1), pages=pages, **_pool_cap(shape, pages))
    if op == "fork":
        seqs = _log_int(rng, 4, 128)
        max_len = _log_int(rng, 1, 300)
        pages = seqs * (max_len // shape["block_size"] + 2) + rng.randrange(0, 50)
        return dict(op="fork", seqs=seqs, ended=seqs // 4, forks=rng.randrange(1, seqs // 2 + 1), max_len=max_len, pages=pages,
                    **_pool_cap(shape, pages))
    pages = _log_int(rng, 64, 3000)
    return dict(op="compact", seqs=_log_int(rng, 1, 32), live=rng.uniform(0.1, 0.95), pages=pages, **_pool_cap(shape, pages))


def _pool_cap(shape, pages):
    """Fewer layers where the pool would pass 1 GB."""
    page = shape["block_size"] * shape["kv_heads"] * shape["dim"] * BYTES[shape["dtype"]]
    return dict(shape, layers=max(1, min(shape["layers"], int(1e9 // (2 * pages * page)))))


# ---------------------------------------------------------------- inputs

def _inv_freq(rotary_dim, scaling):
    """Frequencies of the rotated pairs in 64 bits, and the factor on the rotated values.  "bands"
    slows the low frequencies by 8 and blends a middle band; "ramp" blends by the pair's index
    and scales the result."""
    base = 10000.0 if scaling == "none" else 500000.0
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    f = base ** (-2.0 * i / rotary_dim)
    if scaling == "bands":
        turns = 8192 * f / (2 * math.pi)  # turns over the original context
        keep = ((turns - 1) / (4 - 1)).clamp(0, 1)
        return f * keep + f / 8 * (1 - keep), 1.0
    if scaling == "ramp":
        keep = (1 - (i - rotary_dim / 16) / (rotary_dim / 4)).clamp(0, 1)
        return f * keep + f / 4 * (1 - keep), 0.1 * math.log(4.0) + 1.0
    return f, 1.0


def _rotary_inputs(case, gen):
    dev, dt = "cuda", TORCH[case["dtype"]]
    T, hq, hk, D = case["tokens"], case["q_heads"], case["kv_heads"], case["dim"]
    # query, key and value are slices of one projection's output, as a model has them
    heads = hq + 2 * hk if case["op"] == "rotary_cache" else hq + hk
    qkv = torch.randn((T, heads, D), generator=gen, device=dev).to(dt)
    start = torch.randint(0, max(1, case["far"] - T), (1,), generator=gen, device=dev)
    jumps = torch.randint(0, max(1, case["far"]), (T,), generator=gen, device=dev)
    order = torch.arange(T, device=dev)
    pos = torch.where(order % 64 == 0, jumps, jumps[order // 64 * 64] + order % 64) if T <= 256 else start + order
    freq, factor = _inv_freq(case["rotary_dim"], case["scaling"])
    st = dict(case=case, query=qkv[:, :hq], key=qkv[:, hq:hq + hk], positions=pos.to(torch.int64).contiguous(),
              inv_freq=freq.to(dev), factor=factor, query_out=torch.empty((T, hq, D), dtype=dt, device=dev))
    if case["op"] == "rotary":
        st["key_out"] = torch.empty((T, hk, D), dtype=dt, device=dev)
        return st
    bs = case["block_size"]
    blocks = (T + bs - 1) // bs * 2 + 3
    perm = torch.randperm(blocks, generator=gen, device=dev)
    slots = perm[order // bs] * bs + order % bs
    if case["padded"]:
        slots[torch.randperm(T, generator=gen, device=dev)[:case["padded"]]] = -1
    st["value"] = qkv[:, hq + hk:]
    st["slots"] = slots
    st["key_cache"] = torch.randn((blocks, bs, hk, D), generator=gen, device=dev).to(dt)
    st["value_cache"] = torch.randn((blocks, bs, hk, D), generator=gen, device=dev).to(dt)
    return st


def _lengths(case, rng):
    """(new tokens, cached tokens in all) of every sequence; contexts spread over their logarithm
    when the range is wide."""
    out = []
    for _ in range(case["seqs"]):
        clo, chi = case["ctx_lo"], case["ctx_hi"]
        n = int(rng.integers(case["new_lo"], case["new_hi"] + 1))
        if clo > 0 and chi > 10 * clo:
            c = int(round(math.exp(rng.uniform(math.log(clo), math.log(chi)))))
        else:
            c = int(rng.integers(clo, chi + 1))
        out.append((n, c + n))
    return out


def _case_lengths(case):
    import numpy as np
    # the lengths belong to the case, not to the seed: work(case) counts them
    return _lengths(case, np.random.default_rng([case["new_lo"], case["new_hi"], case["ctx_lo"], case["ctx_hi"], case["seqs"]]))


def _chunk_inputs(case, gen):
    dev, dt = "cuda", TORCH[case["dtype"]]
    H, D, bs = case["kv_heads"], case["dim"], case["block_size"]
    lens = _case_lengths(case)
    need = [(n + bs - 1) // bs for _, n in lens]
    blocks = sum(need) + 5
    shape = (blocks, bs, H, D) if case["layout"] == "nhd" else (blocks, H, bs, D)
    st = dict(case=case, host_lens=lens, k_scale=None, v_scale=None)

    def pages():
        x = torch.empty(shape, dtype=torch.float32, device=dev).normal_(generator=gen)
        if case["cache"] == "f8":
            return (x * 60).to(torch.float8_e4m3fn)
        return x.to(TORCH[case["cache"]])

    st["key_cache"], st["value_cache"] = pages(), pages()
    if case["cache"] == "f8":
        st["k_scale"] = torch.rand((H,), generator=gen, device=dev) * 0.01 + 0.012
        st["v_scale"] = torch.rand((H,), generator=gen, device=dev) * 0.01 + 0.012
    perm = torch.randperm(blocks, generator=gen, device=dev).to(torch.int32)
    table = torch.full((case["seqs"], max(need) + 1), -1, dtype=torch.int32, device=dev)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = perm[at:at + n]
        at += n
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    rows = starts[-1]
    st["table"] = table
    st["lens"] = torch.tensor([n for _, n in lens], dtype=torch.int32, device=dev)
    st["indptr"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    st["host_starts"] = starts
    # scores a little wider than unit variance, as trained heads have them
    st["query"] = (torch.randn((rows, H * case["group"], D), generator=gen, device=dev) * 1.5).to(dt)
    st["out"] = torch.empty_like(st["query"])
    st["max_seq_len"] = max(n for _, n in lens)
    if own:
        from kvx_b200 import ops
        n = ops.chunk_attention_workspace_bytes(case["seqs"], rows, H * case["group"], H, D, st["max_seq_len"])
        st["workspace"] = torch.empty(max(n, 16), dtype=torch.uint8, device=dev)
    return st


def _pool(case, gen):
    dev = "cuda"
    shape = (case["pages"], case["block_size"], case["kv_heads"], case["dim"])

    def one():
        bits = torch.randint(0, 256, (math.prod(shape) * BYTES[case["dtype"]],), generator=gen, device=dev, dtype=torch.uint8)
        if case["dtype"] == "f8":
            return bits.view(shape)
        # clear the top exponent bit of every element: finite values only
        top = bits.view(-1, BYTES[case["dtype"]])[:, -1]
        top &= 0xBF
        return bits.view(TORCH[case["dtype"]]).view(shape)

    return [one() for _ in range(case["layers"])], [one() for _ in range(case["layers"])]


def _page_inputs(case, gen):
    dev = "cuda"
    keys, values = _pool(case, gen)
    st = dict(case=case, keys=keys, values=values)
    perm = torch.randperm(case["pages"], generator=gen, device=dev)
    if case["op"] == "copy":
        st["src"] = perm[:case["pairs"]].to(torch.int32)
        st["dst"] = perm[case["pairs"]:2 * case["pairs"]].to(torch.int32)
        return st
    bs, S = case["block_size"], case["seqs"]
    if case["op"] == "fork":
        lens = torch.randint(1, case["max_len"] + 1, (S,), generator=gen, device=dev)
        wide = (case["max_len"] + bs - 1) // bs
    else:
        per = max(1, int(case["pages"] * case["live"]) // S)
        lens = torch.full((S,), per * bs, device=dev)
        wide = per
    order = torch.randperm(S, generator=gen, device=dev)
    if case["op"] == "fork":
        # the first half of `order` lives on, the last rows are free for children
        lens[order[S - case["forks"]:]] = 0
    cols = torch.arange(wide, device=dev)
    used = cols[None, :] < ((lens + bs - 1) // bs)[:, None]
    ids = perm[(torch.cumsum(used.reshape(-1).long(), 0) - 1).clamp(min=0, max=case["pages"] - 1)].reshape(S, wide)
    st["table"] = torch.where(used, ids, -1).to(torch.int32).contiguous()
    st["lens"] = lens.to(torch.int32)
    refs = torch.zeros(case["pages"] + 1, dtype=torch.int32, device=dev)
    refs.index_add_(0, torch.where(used, ids, case["pages"]).reshape(-1), torch.ones(S * wide, dtype=torch.int32, device=dev))
    st["refs"] = refs[:-1].contiguous()
    if case["op"] == "fork":
        alive = S - case["forks"]
        st["ended"] = order[:min(case["ended"], alive - 1)].to(torch.int32)
        parents = order[min(case["ended"], alive - 1):alive]
        pick = torch.randint(0, parents.numel(), (case["forks"],), generator=gen, device=dev)
        st["parents"] = parents[pick].to(torch.int32)
        st["children"] = order[alive:].to(torch.int32)
    return st


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    if case["op"] in ("rotary", "rotary_cache"):
        return _rotary_inputs(case, gen)
    if case["op"] == "chunk":
        return _chunk_inputs(case, gen)
    return _page_inputs(case, gen)


# ---------------------------------------------------------------- plain forms

def _plain_rotate(x, positions, inv_freq, factor, interleaved, inverse=False):
    angle = positions.double()[:, None] * inv_freq[None, :]  # far positions need the 64 bits
    cos = (angle.cos() * factor).float()[:, None, :]
    sin = (angle.sin() * (-factor if inverse else factor)).float()[:, None, :]
    half = inv_freq.numel()
    r = x[..., :2 * half].float()
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = r[..., :half], r[..., half:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    out = x.clone()
    out[..., :2 * half] = turned.to(x.dtype)
    return out


def _plain_rotary(st):
    c = st["case"]
    rest = (st["positions"], st["inv_freq"], st["factor"], c["interleaved"])
    if c["op"] == "rotary":
        return (_plain_rotate(st["query"], *rest, c["inverse"]), _plain_rotate(st["key"], *rest, c["inverse"]))
    q, k = _plain_rotate(st["query"], *rest), _plain_rotate(st["key"], *rest)
    flat_k, flat_v = st["key_cache"].flatten(0, 1), st["value_cache"].flatten(0, 1)
    live = st["slots"] >= 0
    flat_k[st["slots"][live]] = k[live]
    flat_v[st["slots"][live]] = st["value"][live]
    return q, st["key_cache"], st["value_cache"]


def _plain_pages(cache, table_row, used, layout, scale):
    x = cache[table_row[:used].long()].float()
    x = x.flatten(0, 1) if layout == "nhd" else x.transpose(1, 2).flatten(0, 1)  # [tokens, heads, dim]
    return x if scale is None else x * scale[None, :, None]


def _plain_chunk(st):
    c = st["case"]
    H, G, D, bs = c["kv_heads"], c["group"], c["dim"], c["block_size"]
    out = torch.empty_like(st["query"])
    for s, (n, total) in enumerate(st["host_lens"]):
        used = (total + bs - 1) // bs
        k = _plain_pages(st["key_cache"], st["table"][s], used, c["layout"], st["k_scale"])[:total].transpose(0, 1)
        v = _plain_pages(st["value_cache"], st["table"][s], used, c["layout"], st["v_scale"])[:total].transpose(0, 1)
        step = max(1, int(2e9) // (H * G * total * 4))  # rows whose scores fit 2 GB
        for r0 in range(0, n, step):
            r1 = min(n, r0 + step)
            at = st["host_starts"][s]
            q = st["query"][at + r0:at + r1].float().view(r1 - r0, H, G, D).permute(1, 2, 0, 3)
            sc = torch.matmul(q, k.transpose(1, 2)[:, None]) * (D ** -0.5)  # [H, G, rows, total]
            if c["causal"]:
                pos = torch.arange(total - n + r0, total - n + r1, device=q.device)
                sc = sc.masked_fill(torch.arange(total, device=q.device)[None, :] > pos[:, None], -math.inf)
            p = torch.exp(sc - sc.amax(-1, keepdim=True))
            o = torch.matmul(p, v[:, None]) / p.sum(-1, keepdim=True)
            out[at + r0:at + r1] = o.permute(2, 0, 1, 3).reshape(r1 - r0, H * G, D).to(out.dtype)
    return out


def _plain_copy(keys, values, src, dst):
    ok = (src >= 0) & (dst >= 0)
    s, d = src[ok].long(), dst[ok].long()
    for t in keys + values:
        t[d] = t[s]


def _ranked(flags, ids, count):
    """ids of the set flags in order, as a list of `count` entries filled up with -1."""
    out = torch.full((count + 1,), -1, dtype=torch.int32, device=flags.device)
    rank = torch.cumsum(flags.long(), 0) - 1
    out.scatter_(0, torch.where(flags & (rank < count), rank, count), ids.to(torch.int32))
    return out[:count]


def _plain_fork(st):
    table, lens, refs = st["table"].clone(), st["lens"].clone(), st["refs"].clone()
    bs, pages = st["case"]["block_size"], st["refs"].numel()
    spare = torch.zeros(pages + 1, dtype=torch.int32, device=refs.device)  # the last entry takes what is not a page
    # free the sequences that ended
    rows = table[st["ended"].long()]
    gone = torch.where(rows >= 0, rows, pages).long().reshape(-1)
    refs -= spare.clone().index_add_(0, gone, torch.ones_like(gone, dtype=torch.int32))[:pages]
    table[st["ended"].long()] = -1
    lens[st["ended"].long()] = 0
    # fork: share the full pages, duplicate the one that is partly filled
    par, chi = st["parents"].long(), st["children"].long()
    plen = lens[par].long()
    cols = torch.arange(table.shape[1], device=table.device)[None, :]
    full = (plen // bs)[:, None]
    part = plen % bs != 0
    rows = torch.where(cols < full, table[par], -1)
    free_ids = _ranked(refs == 0, torch.arange(pages, device=refs.device), par.numel())
    rank = torch.cumsum(part.long(), 0) - 1
    last = table[par].gather(1, full.clamp(max=table.shape[1] - 1)).squeeze(1)
    src = torch.where(part, last, -1)
    dst = torch.where(part, free_ids[rank.clamp(min=0)], -1)
    rows = torch.where((cols == full) & part[:, None], dst[:, None], rows)
    table[chi] = rows
    lens[chi] = plen.to(torch.int32)
    named = torch.where(rows >= 0, rows, pages).long().reshape(-1)
    refs += spare.clone().index_add_(0, named, torch.ones_like(named, dtype=torch.int32))[:pages]
    _plain_copy(st["keys"], st["values"], src, dst)
    return [table, lens, refs, src, dst] + st["keys"] + st["values"]


def _plain_compact(st):
    table, refs = st["table"].clone(), st["refs"].clone()
    pages = refs.numel()
    ids = torch.arange(pages, device=refs.device)
    live = refs > 0
    count = live.sum()
    src = _ranked(live & (ids >= count), ids, pages // 2)
    dst = _ranked(~live & (ids < count), ids, pages // 2)
    moved = torch.cat((ids, ids[:1])).to(torch.int32)
    moved.scatter_(0, torch.where(src >= 0, src, pages).long(), dst)
    table = torch.where(table >= 0, moved[table.clamp(min=0).long()], table)
    kept = torch.cat((refs, refs[:1]))
    kept.scatter_(0, torch.where(src >= 0, dst, pages).long(), torch.cat((refs, refs[:1]))[src.long()])
    kept.scatter_(0, torch.where(src >= 0, src, pages).long(), torch.zeros_like(src))
    _plain_copy(st["keys"], st["values"], src, dst)
    return [table, kept[:pages], src, dst] + st["keys"] + st["values"]


# ---------------------------------------------------------------- the framework's calls

def _own_run(st):
    from kvx_b200 import ops
    c = st["case"]
    if c["op"] == "rotary":
        return ops.rotary_embedding(st["query"], st["key"], st["positions"], st["inv_freq"], interleaved=c["interleaved"],
                                    factor=st["factor"], inverse=c["inverse"], query_out=st["query_out"], key_out=st["key_out"])
    if c["op"] == "rotary_cache":
        q = ops.rotary_and_cache(st["query"], st["key"], st["value"], st["positions"], st["inv_freq"], st["key_cache"],
                                 st["value_cache"], st["slots"], interleaved=c["interleaved"], factor=st["factor"],
                                 query_out=st["query_out"])
        return q, st["key_cache"], st["value_cache"]
    if c["op"] == "chunk":
        return ops.paged_attention_chunk(st["query"], st["key_cache"], st["value_cache"], st["table"], st["lens"], st["indptr"],
                                         c["dim"] ** -0.5, causal=c["causal"], max_seq_len=st["max_seq_len"], out=st["out"],
                                         workspace=st.get("workspace"), kv_cache_dtype="fp8" if c["cache"] == "f8" else "auto",
                                         k_scale=st["k_scale"], v_scale=st["v_scale"], num_kv_heads=c["kv_heads"])
    if c["op"] == "copy":
        ops.copy_pages(st["keys"], st["values"], st["src"], st["dst"])
        return st["keys"] + st["values"]
    table, refs = st["table"].clone(), st["refs"].clone()
    if c["op"] == "fork":
        lens = st["lens"].clone()
        ops.free_sequences(table, lens, refs, st["ended"])
        src, dst = ops.fork_sequences(table, lens, refs, st["parents"], st["children"], c["block_size"])
        ops.copy_pages(st["keys"], st["values"], src, dst)
        return [table, lens, refs, src, dst] + st["keys"] + st["values"]
    src, dst = ops.compact_pages(table, refs)
    ops.copy_pages(st["keys"], st["values"], src, dst)
    return [table, refs, src, dst] + st["keys"] + st["values"]


def run(state):
    if own:
        return _own_run(state)
    op = state["case"]["op"]
    if op in ("rotary", "rotary_cache"):
        return _plain_rotary(state)
    if op == "chunk":
        return _plain_chunk(state)
    if op == "copy":
        _plain_copy(state["keys"], state["values"], state["src"], state["dst"])
        return state["keys"] + state["values"]
    return _plain_fork(state) if op == "fork" else _plain_compact(state)


# ---------------------------------------------------------------- bytes and operations

def work(case):
    if case["op"] in ("rotary", "rotary_cache"):
        e, T = BYTES[case["dtype"]], case["tokens"]
        turned = T * (case["q_heads"] + case["kv_heads"]) * case["rotary_dim"]
        if case["op"] == "rotary":
            return {"bytes": 2 * T * (case["q_heads"] + case["kv_heads"]) * case["dim"] * e + 8 * T, "flops": 3 * turned}
        live = T - case["padded"]
        rows = 2 * T * case["q_heads"] + 4 * live * case["kv_heads"]
        return {"bytes": rows * case["dim"] * e + 16 * T, "flops": 3 * turned}
    if case["op"] == "chunk":
        H, G, D = case["kv_heads"], case["group"], case["dim"]
        tokens = pairs = rows = 0
        for n, total in _case_lengths(case):
            rows += n
            tokens += total
            pairs += n * (total - n) + n * (n + 1) // 2 if case["causal"] else n * total
        return {"bytes": 2 * rows * H * G * D * BYTES[case["dtype"]] + 2 * tokens * H * D * BYTES[case["cache"]],
                "flops": 4 * pairs * H * G * D}
    page = case["block_size"] * case["kv_heads"] * case["dim"] * BYTES[case["dtype"]]
    if case["op"] == "copy":
        moved = case["pairs"]
    elif case["op"] == "fork":
        moved = case["forks"] * (case["block_size"] - 1) // case["block_size"]  # parents with a partly filled page
    else:
        per = max(1, int(case["pages"] * case["live"]) // case["seqs"]) * case["seqs"]
        moved = per * (case["pages"] - per) // case["pages"]  # live pages beyond the live count, on average
    return {"bytes": 4 * moved * page * case["layers"], "flops": 0}


# ---------------------------------------------------------------- the definition in 64 bits

def _exact_turn(x, positions, inv_freq, factor, interleaved, inverse):
    half = inv_freq.numel()
    z = x.double()
    r = z[..., :2 * half]
    pair = torch.complex(r[..., 0::2], r[..., 1::2]) if interleaved else torch.complex(r[..., :half], r[..., half:])
    phase = torch.polar(torch.full_like(inv_freq, factor)[None].expand(positions.numel(), -1),
                        (-1.0 if inverse else 1.0) * positions.double()[:, None] * inv_freq)
    turned = pair * phase[:, None, :]
    both = torch.view_as_real(turned).flatten(-2) if interleaved else torch.cat((turned.real, turned.imag), -1)
    return torch.cat((both, z[..., 2 * half:]), -1)


def exact(case, seed):
    if case["op"] in ("copy", "fork", "compact"):
        return None  # whole numbers and copied bits
    st = prepare(case, seed)
    if case["op"] in ("rotary", "rotary_cache"):
        args = (st["positions"], st["inv_freq"], st["factor"], case["interleaved"], case.get("inverse", False))
        q, k = _exact_turn(st["query"], *args), _exact_turn(st["key"], *args)
        if case["op"] == "rotary":
            return q, k
        caches = []
        for cache, rows in ((st["key_cache"], k), (st["value_cache"], st["value"].double())):
            c = cache.double().reshape(-1, case["kv_heads"], case["dim"])
            for_slot = st["slots"].clamp(min=0)
            keep = st["slots"] >= 0
            c.index_copy_(0, for_slot[keep], rows[keep])
            caches.append(c.view(cache.shape))
        return q, caches[0], caches[1]
    H, G, D, bs = case["kv_heads"], case["group"], case["dim"], case["block_size"]
    if sum(n * t for n, t in st["host_lens"]) * H * G * D > 4e12:
        return None
    out = torch.zeros(st["query"].shape, dtype=torch.float64, device="cuda")
    for s, (n, total) in enumerate(st["host_lens"]):
        token = torch.arange(total, device="cuda")
        page, at = st["table"][s].long()[token // bs], token % bs
        r0 = st["host_starts"][s]
        for h in range(H):
            k, v = ((c[page, at, h] if case["layout"] == "nhd" else c[page, h, at]).double()
                    for c in ((st["key_cache"], st["value_cache"]) if case["cache"] != "f8" else
                              (st["key_cache"].float(), st["value_cache"].float())))
            if case["cache"] == "f8":
                k, v = k * st["k_scale"][h].double(), v * st["v_scale"][h].double()
            for g in range(G):
                for a in range(0, n, 1024):
                    b = min(n, a + 1024)
                    logits = st["query"][r0 + a:r0 + b, h * G + g].double() @ k.t() / math.sqrt(D)
                    if case["causal"]:
                        late = token[None, :] - (total - n) > torch.arange(a, b, device="cuda")[:, None]
                        logits[late] = -math.inf
                    out[r0 + a:r0 + b, h * G + g] = torch.softmax(logits, -1) @ v
    return out

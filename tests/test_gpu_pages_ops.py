"""Upkeep of the page pool (include/kvx_pages_ops.h) against plain loops on the host: whole numbers
and copied bits, so everything is equal, bit for bit."""
import random

import pytest

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


# ---------------------------------------------------------------- plain restatements

def plain_pairs(src, dst, blocks):
    """The pairs that take part."""
    ok = lambda a, b: 0 <= a < blocks and 0 <= b < blocks and a != b
    live = [(i, a, b) for i, (a, b) in enumerate(zip(src, dst)) if ok(a, b)]
    targets = {b for _, _, b in live}
    last = {b: i for i, _, b in live}
    return [(a, b) for i, a, b in live if last[b] == i and a not in targets]


def plain_free(table, lens, refs, rows):
    for r in dict.fromkeys(rows):
        if 0 <= r < len(table):
            for b, page in enumerate(table[r]):
                if 0 <= page < len(refs):
                    refs[page] = max(0, refs[page] - 1)
                table[r][b] = -1
            lens[r] = 0


def plain_fork(table, lens, refs, parents, children, bs):
    old_table, old_lens, n = [list(r) for r in table], list(lens), len(parents)
    spare = [b for b, x in enumerate(refs) if x == 0]
    src, dst, width = [-2] * n, [-2] * n, len(table[0]) if table else 0
    for i, (a, c) in enumerate(zip(parents, children)):
        if not (0 <= a < len(table) and 0 <= c < len(table)) or a == c or c in children[:i] or a in children:
            continue
        length = max(0, old_lens[a])
        full, page = length // bs, -1
        if length % bs and full < width and 0 <= old_table[a][full] < len(refs):
            if not spare:
                continue
            page = spare.pop(0)
            src[i], dst[i] = old_table[a][full], page
        else:
            src[i] = dst[i] = -1
        for b in range(width):
            x = old_table[a][b] if b < full else page if b == full else -1
            table[c][b] = x
            if 0 <= x < len(refs):
                refs[x] += 1
        lens[c] = length
    return src, dst


def plain_compact(table, refs):
    blocks = len(refs)
    live = [b for b in range(blocks) if refs[b] > 0]
    n = len(live)
    movers, holes = [b for b in live if b >= n], [b for b in range(n) if refs[b] <= 0]
    name = dict(zip(movers, holes))
    for a, b in name.items():
        refs[b], refs[a] = refs[a], 0
    for row in table:
        row[:] = [name.get(x, x) for x in row]
    cap = max(1, blocks // 2)
    return movers + [-1] * (cap - n_moves(movers, holes)), holes + [-1] * (cap - len(holes))


def n_moves(movers, holes):
    assert len(movers) == len(holes)
    return len(movers)


# ---------------------------------------------------------------- copy

def pools(layers, blocks, shape, dtype, seed=0, view=None):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(seed)
    size = {torch.bfloat16: 2, torch.float16: 2, torch.float32: 4}.get(dtype, 1)
    out = []
    for _ in range(layers):
        n = blocks
        for x in shape:
            n *= x
        t = torch.randint(0, 256, (n * size,), generator=g, device="cuda", dtype=torch.uint8).view(dtype).view((blocks,) + shape)
        out.append(t if view is None else view(t))
    return out


def check_copy(keys, values, src, dst, index):
    torch = _torch()
    from kvx_b200 import ops
    want = [t.clone() for t in keys + values]
    blocks = keys[0].shape[0]
    for a, b in plain_pairs(src, dst, blocks):
        for t in want:
            t[b] = t[a].clone()
    ops.copy_pages(keys, values, torch.tensor(src, dtype=index, device="cuda"), torch.tensor(dst, dtype=index, device="cuda"))
    torch.cuda.synchronize()
    for i, (got, exp) in enumerate(zip(keys + values, want)):
        same = torch.equal(got.contiguous().view(torch.uint8), exp.contiguous().view(torch.uint8))
        assert same, i


@pytest.mark.parametrize("index", ["int32", "int64"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32", "float8_e4m3fn", "uint8"])
def test_copy_every_layer_and_type(dtype, index):
    torch = _torch()
    index, dtype = getattr(torch, index), getattr(torch, dtype)
    rng = random.Random(1)
    for layers, blocks, shape, pairs in [(1, 8, (16, 8, 128), 1), (3, 60, (16, 2, 64), 20), (70, 12, (8, 2, 64), 5), (2, 50, (3, 1, 5), 20),
                                         (2, 30, (4, 2, 8, 16, 8), 9), (1, 4, (256, 8, 128), 2)]:
        if len(shape) == 5:
            shape = (2, 8, 16, 8)  # HND_PACKED
        ids = rng.sample(range(blocks), 2 * pairs)
        check_copy(pools(layers, blocks, shape, dtype, 1), pools(layers, blocks, shape, dtype, 2), ids[:pairs], ids[pairs:], index)


def test_copy_pages_with_gaps_and_views():
    """K and V interleaved in one allocation, permuted views, padded rows, misaligned bases."""
    torch = _torch()
    both = pools(1, 40, (2, 16, 4, 64), torch.bfloat16, 3)[0]
    check_copy([both[:, 0]], [both[:, 1]], [1, 2, 3], [10, 11, 12], torch.int32)
    k, v = (pools(2, 40, (4, 16, 64), torch.float16, s, lambda t: t.transpose(1, 2)) for s in (4, 5))
    check_copy(k, v, [1, 2, 3], [10, 11, 12], torch.int64)
    k, v = (pools(2, 40, (16, 4, 72), torch.bfloat16, s, lambda t: t[..., :64]) for s in (6, 7))
    check_copy(k, v, [1, 2, 3], [10, 11, 12], torch.int32)
    k, v = (pools(1, 40, (16, 2, 64), torch.uint8, s) for s in (8, 9))
    odd = [torch.cat((torch.zeros(3, dtype=torch.uint8, device="cuda"), t.flatten()))[3:].view(t.shape) for t in k]
    check_copy(odd, v, [1, 2, 3], [10, 11, 12], torch.int32)


@pytest.mark.parametrize("n", [5, 200, 257, 3000])
def test_copy_leaves_out_pairs_that_clash(n):
    """Numbers outside the pool, a page copied to itself, destinations named twice, chains -- both
    where the copying warps check and where a kernel ahead does."""
    torch = _torch()
    rng = random.Random(n)
    blocks = max(8, n)
    src = [rng.randrange(-2, blocks + 2) for _ in range(n)]
    dst = [rng.randrange(-2, blocks + 2) if rng.random() < 0.4 else -1 for _ in range(n)]
    check_copy(pools(2, blocks, (8, 1, 64), torch.bfloat16, 1), pools(2, blocks, (8, 1, 64), torch.bfloat16, 2), src, dst, torch.int32)
    # a sparse list: most destinations unused
    src = [rng.randrange(blocks // 2) for _ in range(n)]
    dst = [-1] * n
    for i in rng.sample(range(n), max(1, n // 50)):
        dst[i] = blocks // 2 + rng.randrange(blocks // 2)
    check_copy(pools(1, blocks, (8, 1, 64), torch.bfloat16, 3), pools(1, blocks, (8, 1, 64), torch.bfloat16, 4), src, dst, torch.int64)


# ---------------------------------------------------------------- tables

def state(rng, rows, blocks, bs, width, shared=0.3):
    """A consistent table: some pages shared between rows."""
    free = list(range(blocks))
    rng.shuffle(free)
    refs, table, lens = [0] * blocks, [], []
    for _ in range(rows):
        length = rng.choice([0, 1, bs - 1, bs, bs + 1, rng.randrange(0, width * bs + 1)])
        length = min(length, width * bs)
        row = []
        for b in range((length + bs - 1) // bs):
            donor = rng.choice(table) if table and rng.random() < shared else None
            if donor and b < len(donor) and donor[b] >= 0 and (b + 1) * bs <= length:
                page = donor[b]
            elif free:
                page = free.pop()
            else:
                length = b * bs
                break
            refs[page] += 1
            row.append(page)
        table.append(row + [-1] * (width - len(row)))
        lens.append(length)
    return table, lens, refs


def on_gpu(index, *lists):
    torch = _torch()
    return [torch.tensor(x, dtype=index, device="cuda") for x in lists]


def equal(got, exp):
    return got.cpu().tolist() == exp


@pytest.mark.parametrize("index", ["int32", "int64"])
@pytest.mark.parametrize("seed", range(6))
def test_free_fork_compact_in_sequence(index, seed):
    """A run of them, as a beam search uses them; then odd row numbers, repeated and clashing ones."""
    torch = _torch()
    from kvx_b200 import ops
    index = getattr(torch, index)
    rng = random.Random(seed)
    rows, bs, width = rng.choice([(1, 16, 3), (9, 1, 7), (40, 16, 12), (300, 8, 20), (1500, 16, 4), (30, 7, 200)])
    blocks = rng.choice([rows * width, rows * width // 2 + 3, rows * width // 8 + 2])
    table, lens, refs = state(rng, rows, blocks, bs, width)
    t, l = on_gpu(index, table, lens)
    r = torch.tensor(refs, dtype=torch.int32, device="cuda")
    for turn in range(3):
        pick = lambda n: [rng.randrange(-1, rows + 1) if rng.random() < 0.1 else rng.randrange(rows) for _ in range(n)]
        gone = pick(rng.randrange(0, rows // 2 + 2))
        ops.free_sequences(t, l, r, *on_gpu(index, gone))
        plain_free(table, lens, refs, gone)
        assert equal(t, table) and equal(l, lens) and equal(r, refs), ("free", turn)
        n = rng.randrange(0, rows // 2 + 2)
        if turn == 0:  # proper pairs: children are empty rows
            empty = [i for i in range(rows) if lens[i] == 0]
            full = [i for i in range(rows) if lens[i] > 0]
            children = empty[:n] if full else []
            parents = [rng.choice(full) for _ in children]
        else:
            parents, children = pick(n), pick(n)
        src, dst = ops.fork_sequences(t, l, r, *on_gpu(index, parents, children), bs)
        esrc, edst = plain_fork(table, lens, refs, parents, children, bs)
        assert equal(src, esrc) and equal(dst, edst), ("fork pairs", turn)
        assert equal(t, table) and equal(l, lens) and equal(r, refs), ("fork", turn)
        src, dst = ops.compact_pages(t, r)
        esrc, edst = plain_compact(table, refs)
        assert equal(src, esrc) and equal(dst, edst), ("compact pairs", turn)
        assert equal(t, table) and equal(r, refs), ("compact", turn)


def test_large_pool():
    torch = _torch()
    from kvx_b200 import ops
    rng = random.Random(5)
    blocks = 100003
    refs = [rng.choice([0, 0, 1, 2, 3]) for _ in range(blocks)]
    table = [[rng.randrange(-1, blocks + 1) for _ in range(300)] for _ in range(100)]
    t, = on_gpu(torch.int32, table)
    r = torch.tensor(refs, dtype=torch.int32, device="cuda")
    src, dst = ops.compact_pages(t, r)
    esrc, edst = plain_compact(table, refs)
    assert equal(src, esrc) and equal(dst, edst) and equal(t, table) and equal(r, refs)
    n = sum(x > 0 for x in refs)
    assert all(x > 0 for x in refs[:n]) and not any(refs[n:])


def test_counts_never_fall_below_zero():
    torch = _torch()
    from kvx_b200 import ops
    table, lens, refs = [[0, 0, 1, 9, -1], [0, 1, 1, 1, 2]], [80, 80], [1, 2, 0, 5]
    t, l = on_gpu(torch.int32, table, lens)
    r = torch.tensor(refs, dtype=torch.int32, device="cuda")
    ops.free_sequences(t, l, r, *on_gpu(torch.int32, [0, 1, 0]))
    plain_free(table, lens, refs, [0, 1, 0])
    assert equal(t, table) and equal(l, lens) and equal(r, refs) and refs == [0, 0, 0, 5]


def test_empty_calls():
    torch = _torch()
    from kvx_b200 import ops
    t, l = on_gpu(torch.int32, [[0, 1]], [20])
    r = torch.tensor([1, 1, 0, 0], dtype=torch.int32, device="cuda")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    ops.free_sequences(t, l, r, none)
    src, dst = ops.fork_sequences(t, l, r, none, none, 16)
    assert src.numel() == 0 and dst.numel() == 0
    k = pools(1, 4, (16, 2, 64), torch.bfloat16)
    ops.copy_pages(k, [k[0].clone()], none, none)
    one = torch.tensor([1], dtype=torch.int32, device="cuda")
    t1 = torch.empty((0, 3), dtype=torch.int32, device="cuda")
    src, dst = ops.compact_pages(t1, one)
    assert src.tolist() == [-1] and dst.tolist() == [-1]


def test_compacting_and_copying_keeps_what_sequences_read():
    """Pages written, shared, forked, compacted and copied: every sequence gathers the same tokens as
    before, a fork those of its parent."""
    torch = _torch()
    from kvx_b200 import ops
    rng = random.Random(7)
    bs, width, blocks, heads, dim, layers = 16, 12, 300, 2, 64, 3
    table, lens, refs = state(rng, 24, blocks, bs, width, shared=0.4)
    for s in range(0, 24, 3):  # some rows end before the fork
        plain_free(table, lens, refs, [s])
    t, l = on_gpu(torch.int32, table, lens)
    r = torch.tensor(refs, dtype=torch.int32, device="cuda")
    keys, values = pools(layers, blocks, (bs, heads, dim), torch.bfloat16, 1), pools(layers, blocks, (bs, heads, dim), torch.bfloat16, 2)

    def read():
        out = []
        for k, v in zip(keys, values):
            gk = torch.zeros((24, width * bs, heads, dim), dtype=torch.bfloat16, device="cuda")
            gv = torch.zeros_like(gk)
            ops.gather_kv(k, v, t, l, gk, gv)
            out += [gk, gv]
        return out

    before = read()
    parents, children = [1, 1, 2, 4], [0, 3, 6, 9]
    src, dst = ops.fork_sequences(t, l, r, *on_gpu(torch.int32, parents, children), bs)
    ops.copy_pages(keys, values, src, dst)
    forked = read()
    src, dst = ops.compact_pages(t, r)
    ops.copy_pages(keys, values, src, dst)
    after = read()
    torch.cuda.synchronize()
    for a, b, c in zip(before, forked, after):
        want = a.clone()
        for p, ch in zip(parents, children):
            want[ch] = a[p]
        same = torch.equal(b.view(torch.int16), want.view(torch.int16)) and torch.equal(c.view(torch.int16), want.view(torch.int16))
        assert same


def test_graph_replay():
    """Fork and copy captured together: a replay follows the rows it finds."""
    torch = _torch()
    from kvx_b200 import ops
    rng = random.Random(8)
    table, lens, refs = state(rng, 10, 60, 16, 6, shared=0.0)
    plain_free(table, lens, refs, [7, 8, 9])
    keys, values = pools(2, 60, (16, 2, 64), torch.bfloat16, 1), pools(2, 60, (16, 2, 64), torch.bfloat16, 2)
    t, l = on_gpu(torch.int32, table, lens)
    r = torch.tensor(refs, dtype=torch.int32, device="cuda")
    parents, children = on_gpu(torch.int32, [0, 1], [7, 8])
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):  # warm up on copies of the state
        src, dst = ops.fork_sequences(t.clone(), l.clone(), r.clone(), parents, children, 16)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        src, dst = ops.fork_sequences(t, l, r, parents, children, 16)
        ops.copy_pages(keys, values, src, dst)
    parents.copy_(torch.tensor([2, 2]))
    children.copy_(torch.tensor([9, 7]))
    want = [x.clone() for x in keys + values]
    graph.replay()
    torch.cuda.synchronize()
    esrc, edst = plain_fork(table, lens, refs, [2, 2], [9, 7], 16)
    assert equal(src, esrc) and equal(dst, edst) and equal(t, table) and equal(l, lens) and equal(r, refs)
    for a, b in plain_pairs(esrc, edst, 60):
        for x in want:
            x[b] = x[a].clone()
    for got, exp in zip(keys + values, want):
        same = torch.equal(got.view(torch.int16), exp.view(torch.int16))
        assert same

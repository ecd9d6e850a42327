"""The operators of a serving step run together, as a scheduler would: prompts, decode steps, a fork
with its page copies, drafted tokens of several lengths, rows that are freed, a compaction, and the
same step captured and replayed.

The oracle keeps every sequence's tokens in lists of its own and never looks at the tables, so a
page that was lost, shared wrongly or copied too late shows.  Turned keys are read back where
they were written and held against the formula (tolerance of the rotary tests: 2 X f 10 * 2^-24 +
u |y|); the oracle then keeps the stored bits, so that the attention is held to the tolerance of
the chunk tests alone: u |out| + V (u + 2 (exp(e) - 1) + 2^-22 + (tokens + 4) 2^-24) with
e = (dim + 2) 2^-24 * scale * dim * Q * K and u = 2^-8 (bf16)."""
import pytest

pytestmark = pytest.mark.gpu

H, G, D, BS, ROWS, MAXB, POOL, LAYERS = 2, 4, 64, 16, 8, 12, 64, 2
U = 2.0 ** -8


class Server:
    def __init__(self, index):
        import torch
        from kvx_b200 import ops
        self.torch, self.ops = torch, ops
        self.g = torch.Generator(device="cuda").manual_seed(3)
        self.idx = index
        self.kc = [torch.randn((POOL, BS, H, D), generator=self.g, device="cuda").bfloat16() for _ in range(LAYERS)]
        self.vc = [torch.randn((POOL, BS, H, D), generator=self.g, device="cuda").bfloat16() for _ in range(LAYERS)]
        self.table = torch.full((ROWS, MAXB), -1, dtype=index, device="cuda")
        self.lens = torch.zeros(ROWS, dtype=index, device="cuda")
        self.refs = torch.zeros(POOL, dtype=torch.int32, device="cuda")
        self.inv, self.factor = ops.rotary_inv_freq(D, base=500000.0, scaling="bands", scale=8.0, device="cuda")
        none = torch.zeros((0, H, D), dtype=torch.float64, device="cuda")
        self.seen = [[(none, none) for _ in range(ROWS)] for _ in range(LAYERS)]  # the oracle's K, V

    def numbers(self, xs):
        return self.torch.tensor(xs, dtype=self.idx, device="cuda")

    def grow(self, new):
        """Pages for `new[row]` more tokens per row; returns their slots, positions and rows' starts."""
        table, lens, refs = self.table.cpu(), self.lens.cpu(), self.refs.cpu()
        slots, positions, starts = [], [], [0]
        for row in range(ROWS):
            for _ in range(new.get(row, 0)):
                at = int(lens[row])
                if at % BS == 0:
                    page = int((refs == 0).nonzero()[0])
                    table[row, at // BS] = page
                    refs[page] = 1
                page = int(table[row, at // BS])
                assert int(refs[page]) == 1  # a page that is written belongs to this row alone
                slots.append(page * BS + at % BS)
                positions.append(at)
                lens[row] += 1
            starts.append(len(slots))
        self.table.copy_(table)
        self.lens.copy_(lens)
        self.refs.copy_(refs)
        return self.numbers(slots), self.numbers(positions), self.numbers(starts)

    def inputs(self, tokens):
        draw = lambda heads: self.torch.randn((tokens, heads, D), generator=self.g, device="cuda").bfloat16()
        return draw(H * G), draw(H), draw(H)

    def launch(self, layer, q, k, v, slots, positions, indptr, **kw):
        turned = self.ops.rotary_and_cache(q, k, v, positions, self.inv, self.kc[layer], self.vc[layer], slots, factor=self.factor)
        out = self.ops.paged_attention_chunk(turned, self.kc[layer], self.vc[layer], self.table, self.lens, indptr, D ** -0.5, **kw)
        return turned, out

    def turned(self, x, positions):
        a = positions.double()[:, None] * self.inv
        c, s = a.cos()[:, None] * self.factor, a.sin()[:, None] * self.factor
        x1, x2 = x.double().chunk(2, -1)
        y = self.torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], -1)
        big = self.torch.maximum(x1.abs(), x2.abs()).repeat(1, 1, 2) * self.factor
        return y, 2 * big * 10 * 2.0 ** -24 + U * y.abs() + 2.0 ** -133

    def close(self, got, want, tol):
        assert bool(self.torch.isfinite(got).all())
        assert float(((got.double() - want).abs() - tol).max()) <= 0

    def check(self, layer, new, q, k, v, slots, positions, turned, out):
        """Takes the new tokens into the oracle's lists and holds the step's results against them."""
        torch = self.torch
        self.close(turned, *self.turned(q, positions))
        stored_k = self.kc[layer].view(-1, H, D)[slots.long()]
        stored_v = self.vc[layer].view(-1, H, D)[slots.long()]
        self.close(stored_k, *self.turned(k, positions))
        assert bool((stored_v == v).all())
        a = 0
        for row in range(ROWS):
            n = new.get(row, 0)
            if n == 0:
                continue
            K, V = self.seen[layer][row]
            K, V = torch.cat([K, stored_k[a:a + n].double()]), torch.cat([V, stored_v[a:a + n].double()])
            self.seen[layer][row] = K, V
            Q = turned[a:a + n].double().view(n, H, G, D)
            total = K.shape[0]
            sc = torch.einsum("nhgd,thd->hgnt", Q, K) * D ** -0.5
            pos = torch.arange(total - n, total, device="cuda")
            sc = sc.masked_fill(torch.arange(total, device="cuda")[None, :] > pos[:, None], float("-inf"))
            want = torch.einsum("hgnt,thd->nhgd", sc.softmax(-1), V).reshape(n, H * G, D)
            e = (D + 2) * 2.0 ** -24 * D ** -0.5 * D * Q.abs().amax() * K.abs().amax()
            tol = U * want.abs() + V.abs().amax() * (U + 2 * (torch.exp(e) - 1) + 2.0 ** -22 + (total + 4) * 2.0 ** -24)
            self.close(out[a:a + n], want, tol)
            a += n

    def step(self, new):
        slots, positions, indptr = self.grow(new)
        for layer in range(LAYERS):
            q, k, v = self.inputs(slots.numel())
            turned, out = self.launch(layer, q, k, v, slots, positions, indptr)
            self.check(layer, new, q, k, v, slots, positions, turned, out)
            if all(new.get(r, 0) <= 1 for r in range(ROWS)):  # a decode step may go either way
                rows = [r for r in range(ROWS) if new.get(r, 0) == 1]
                t, n = self.table[rows].contiguous(), self.lens[rows].contiguous()
                single = self.ops.paged_attention_decode(turned, self.kc[layer], self.vc[layer], t, n, D ** -0.5)
                # each is within u |out| + u V + 2 (exp(e) - 1) V < 3 u V of the formula (e < 1e-3 here)
                big = self.vc[layer].abs().amax().double()
                assert float((single.double() - out.double()).abs().max()) <= float(6 * U * big)

    def fork(self, pairs):
        src, dst = self.ops.fork_sequences(self.table, self.lens, self.refs, self.numbers([a for a, _ in pairs]),
                                           self.numbers([c for _, c in pairs]), BS)
        self.ops.copy_pages(self.kc, self.vc, src, dst)
        for layer in self.seen:
            for a, c in pairs:
                layer[c] = layer[a]

    def free(self, rows):
        self.ops.free_sequences(self.table, self.lens, self.refs, self.numbers(rows))
        for layer in self.seen:
            for r in rows:
                layer[r] = layer[r][0][:0], layer[r][1][:0]

    def compact(self):
        src, dst = self.ops.compact_pages(self.table, self.refs)
        self.ops.copy_pages(self.kc, self.vc, src, dst)
        live = int((self.refs > 0).sum())
        assert bool((self.refs[:live] > 0).all()) and int(self.table.max()) < live


def life(s):
    s.step({0: 37, 1: 16, 2: 1, 3: 50})
    s.step({0: 1, 1: 1, 2: 1, 3: 1})
    s.fork([(0, 4), (0, 5), (1, 6)])
    s.step({0: 3, 2: 1, 3: 1, 4: 1, 5: 17, 6: 2})
    s.free([0, 3])
    s.compact()
    s.step({1: 1, 2: 1, 4: 1, 5: 1, 6: 1})
    s.step({0: 20, 1: 4, 2: 40, 6: 1})


@pytest.mark.parametrize("index", ["int32", "int64"])
def test_a_life_of_the_pool(index):
    import torch
    s = Server(getattr(torch, index))
    life(s)
    assert s.ops.lib().kvx_attention_device_error(0) == 0


def test_on_another_stream():
    """The whole life on a side stream, with work pending on the default one."""
    import torch
    side = torch.cuda.Stream()
    busy = torch.randn((4096, 4096), device="cuda")
    s = Server(torch.int32)
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        busy = busy @ busy * 1e-4
    with torch.cuda.stream(side):
        life(s)
    torch.cuda.synchronize()


def test_captured_and_replayed():
    """A decode step of every row captured once; each replay sees the lengths, slots and tables that
    are in its inputs then, and rows that stopped (no new token) are left as they were."""
    import torch
    s = Server(torch.int32)
    s.step({r: 5 + 9 * r for r in range(ROWS)})
    slots, positions, indptr = (torch.zeros(n, dtype=s.idx, device="cuda") for n in (ROWS, ROWS, ROWS + 1))
    fixed = s.inputs(ROWS)
    slots.fill_(-1)  # the runs ahead of the first replay cache nothing
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        s.launch(0, *fixed, slots, positions, indptr)
    torch.cuda.current_stream().wait_stream(warm)
    out = torch.full((ROWS, H * G, D), 7.0, dtype=torch.bfloat16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        turned, _ = s.launch(0, *fixed, slots, positions, indptr, out=out)
    for live in (range(ROWS), [0, 2, 3, 7], [5], range(ROWS)):
        new = {r: 1 for r in live}
        a, b, c = s.grow(new)
        n = a.numel()
        out.fill_(7.0)
        slots.fill_(-1)
        positions.zero_()
        slots[:n], positions[:n] = a, b
        indptr.copy_(c)
        for x, y in zip(fixed, s.inputs(ROWS)):
            x.copy_(y)
        graph.replay()
        s.check(0, new, *(x[:n] for x in fixed), a, b, turned[:n], out[:n])
        assert bool((out[n:] == 7.0).all())

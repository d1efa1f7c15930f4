"""GPU: attention over the paged pool against the 64-bit form: one query a
sequence to long chunks, groups with a shared prefix, every cache type, with
what no query may see (slots behind a length, free blocks) set to NaN."""
import pytest

torch = pytest.importorskip("torch")

import paged_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def ints(values, cuda):
    return torch.tensor(values, dtype=torch.int32, device=cuda)


class Step:
    """A batch over a pool: sequences of `lengths` tokens, the last `counts` of
    them queries; the sequences [a, b) of a group share their first tokens."""

    def __init__(self, kvx, cuda, counts, lengths, q_heads, heads, dim, block, dtype, cache,
                 groups=(), seed=0, spread=1.0):
        gen = torch.Generator(device=cuda).manual_seed(seed + dim + sum(counts))
        self.counts, self.lengths, self.groups, self.cuda = counts, lengths, groups, cuda
        self.starts = [0]
        for n in counts:
            self.starts.append(self.starts[-1] + n)
        self.dtype, self.scale = dtype, dim ** -0.5
        self.width = max([1] + [(n + block - 1) // block for n in lengths])
        need = [(n + block - 1) // block for n in lengths]
        blocks = sum(need) + 5
        ids = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).tolist()
        self.tables, at = [], 0
        for n in need:
            self.tables.append(ids[at:at + n])
            at += n
        for a, b, prefix in groups:
            for s in range(a + 1, b):
                self.tables[s][:prefix // block] = self.tables[a][:prefix // block]
        used = torch.zeros(blocks, block, dtype=torch.bool)
        for s, n in enumerate(lengths):
            for p in range(n):
                used[self.tables[s][p // block], p % block] = True
        shape = (blocks, block, heads, dim)
        x = [torch.randn(shape, device=cuda, generator=gen) * spread for _ in range(2)]
        hole = ~used.to(cuda)[:, :, None, None].expand(shape)
        self.scales, kw = [None, None], {}
        if cache == FP8:
            self.scales = [torch.rand(blocks, heads, device=cuda, generator=gen) * 0.01 + 0.002
                           for _ in range(2)]
            x = [(c / s[:, None, :, None]).clamp(-448, 448) for c, s in zip(x, self.scales)]
            kw = dict(scale_tables=self.scales)
        self.caches = [c.masked_fill(hole, float("nan")).to(cache) for c in x]
        self.mgr = kvx.KVCacheManager(self.caches, host_blocks_to_allocate=1, **kw)
        self.q = torch.randn(self.starts[-1], q_heads, dim, device=cuda,
                             generator=gen).to(dtype)
        self.product = BF16 if cache == FP8 else dtype

    def args(self):
        pad = [t + [-1] * (self.width - len(t)) for t in self.tables]
        return ints(pad, self.cuda), ints(self.lengths, self.cuda)

    def kw(self):
        kw = {}
        if self.counts != [1] * len(self.counts):
            kw["starts"] = ints(self.starts, self.cuda)
        if self.groups:
            bounds = [self.groups[0][0]] + [b for _, b, _ in self.groups]
            kw["group_starts"] = ints(bounds, self.cuda)
            kw["prefix_lengths"] = ints([p for _, _, p in self.groups], self.cuda)
        return kw

    def run(self, **kw):
        return self.mgr.attend(0, 1, self.q, *self.args(), **{**self.kw(), **kw})

    def check(self, out, lse=None, causal=True, scale=None):
        caches = [c.cpu() for c in self.caches]
        scales = [s.cpu() if s is not None else None for s in self.scales]
        for s, n in enumerate(self.counts):
            rows = slice(self.starts[s], self.starts[s + 1])
            k, v = (ref.gather(c, f, self.tables[s], self.lengths[s])
                    for c, f in zip(caches, scales))
            last = torch.arange(self.lengths[s] - n, self.lengths[s])
            if not causal:
                last = torch.full_like(last, self.lengths[s])
            visible = torch.arange(self.lengths[s])[None] <= last[:, None]
            want, want_lse, slack = ref.attend(self.q[rows].cpu(), k, v, visible,
                                               scale or self.scale, self.dtype, self.product)
            ref.assert_rounded(out[rows], want, slack, self.dtype)
            if lse is not None and n > 0:
                got = lse[rows].double().cpu()
                none = torch.isneginf(want_lse)
                assert torch.equal(torch.isneginf(got), none)
                off = (got - want_lse)[~none].abs()
                size = (self.q[rows].cpu().double().abs().amax() * k.abs().sum(-1).amax()
                        if k.numel() else 0)
                room = (self.q.shape[-1] * size * self.scale + self.lengths[s] + 128) * ref.U32
                assert (off <= room).all()
        return out


ONE = [  # one query a sequence: counts come from lengths
    ([1], 4, 1, 128, 16), ([7, 0, 129, 300], 8, 2, 128, 16), ([33] * 5, 8, 8, 64, 16),
    ([513, 15, 16, 17], 32, 8, 128, 16), ([100, 31], 20, 4, 80, 7), ([260], 16, 1, 96, 32),
    ([90, 4], 48, 1, 128, 8), ([140, 1], 6, 3, 256, 64), ([40], 5, 5, 16, 1),
    ([2500, 12], 64, 2, 128, 16), ([64, 200], 2, 2, 104, 48), ([0, 0], 4, 4, 64, 16)]


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, F16), (BF16, FP8), (F16, FP8)])
@pytest.mark.parametrize("lengths,hq,hk,dim,block", ONE)
def test_one_query_a_sequence(kvx, cuda, dtype, cache, lengths, hq, hk, dim, block):
    step = Step(kvx, cuda, [1] * len(lengths), lengths, hq, hk, dim, block, dtype, cache)
    out, lse = step.run(return_lse=True)
    step.check(out, lse)
    assert torch.equal(step.run(), out)  # the same bytes again
    step.mgr.close()


MANY = [  # (new tokens, lengths)
    ([5, 0, 1], [5, 9, 30], 8, 2, 128, 16), ([64], [64], 4, 4, 64, 16),
    ([130, 3, 1], [130, 400, 257], 8, 1, 128, 16), ([200], [777], 6, 2, 96, 8),
    ([33, 40], [33, 150], 16, 1, 80, 32), ([70], [70], 4, 2, 256, 16),
    ([9, 300], [4, 300], 4, 1, 128, 16),  # more queries than tokens: the first see nothing
    ([2, 2, 2], [64, 128, 1000], 32, 2, 128, 16), ([257], [1500], 10, 2, 64, 24),
    ([20], [1100], 40, 1, 128, 16)]


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, F16), (BF16, FP8)])
@pytest.mark.parametrize("counts,lengths,hq,hk,dim,block", MANY)
def test_chunks(kvx, cuda, dtype, cache, counts, lengths, hq, hk, dim, block):
    step = Step(kvx, cuda, counts, lengths, hq, hk, dim, block, dtype, cache)
    out, lse = step.run(return_lse=True)
    step.check(out, lse)
    step.check(step.run(causal=False), causal=False)
    step.mgr.close()


GROUPED = [  # (new tokens, lengths, groups as (first, end, prefix))
    ([1] * 4, [70, 65, 99, 64], 8, 2, 128, 16, [(0, 4, 64)]),
    ([1] * 40, [700 + i for i in range(40)], 16, 2, 128, 16, [(0, 40, 640)]),
    ([1] * 6, [50, 200, 220, 90, 100, 33], 4, 4, 64, 16, [(1, 3, 192), (3, 5, 80)]),
    ([1] * 3, [300, 310, 305], 48, 1, 128, 16, [(0, 3, 288)]),
    ([3, 1, 40], [150, 160, 190], 8, 2, 128, 16, [(0, 3, 128)]),
    ([2, 2], [96, 96], 6, 2, 96, 32, [(0, 2, 96)]),  # a prefix into the new tokens: masked
    ([1] * 2, [64, 64], 4, 2, 256, 16, [(0, 2, 64)]),  # nothing of their own
    ([1] * 5, [0, 80, 80, 81, 0], 8, 8, 80, 8, [(1, 4, 72)])]


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, FP8)])
@pytest.mark.parametrize("counts,lengths,hq,hk,dim,block,groups", GROUPED)
def test_shared_prefixes(kvx, cuda, dtype, cache, counts, lengths, hq, hk, dim, block, groups):
    step = Step(kvx, cuda, counts, lengths, hq, hk, dim, block, dtype, cache, groups)
    out, lse = step.run(return_lse=True)
    step.check(out, lse)
    assert torch.equal(step.run(), out)
    step.mgr.close()


def test_wide_scores_and_scales(kvx, cuda):
    """Scores of hundreds, so that the running maximum keeps moving."""
    for counts, lengths in (([1, 1], [900, 77]), ([90], [300])):
        step = Step(kvx, cuda, counts, lengths, 8, 2, 128, 16, BF16, BF16, spread=12.0)
        step.q *= 4
        step.check(step.run(scale=0.3), scale=0.3)
        step.mgr.close()


def test_ids_outside_the_pool_are_not_seen(kvx, cuda):
    for counts in ([1, 1], [40, 3]):
        step = Step(kvx, cuda, counts, [100, 90], 8, 2, 64, 16, BF16, BF16)
        tables, lengths = step.args()
        for bad in (-1, 10**6, -2**31):
            tables[0, 2] = bad
            out = step.mgr.attend(0, 1, step.q, tables, lengths, **step.kw())
            caches = [c.cpu() for c in step.caches]
            k, v = (ref.gather(c, None, step.tables[0], 100) for c in caches)
            n = counts[0]
            visible = torch.arange(100)[None] <= torch.arange(100 - n, 100)[:, None]
            visible[:, 32:48] = False
            want, _, slack = ref.attend(step.q[:n].cpu(), k, v, visible, step.scale, BF16, BF16)
            ref.assert_rounded(out[:n], want, slack, BF16)
        # Every block bad, a length past the table.
        tables[0] = -1
        out, lse = step.mgr.attend(0, 1, step.q, tables, lengths, return_lse=True, **step.kw())
        assert bool((out[:counts[0]] == 0).all()) and bool(torch.isneginf(lse[:counts[0]]).all())
        tables, _ = step.args()
        out = step.mgr.attend(0, 1, step.q, tables, ints([2**31 - 1, 90], cuda), **step.kw())
        assert bool(torch.isfinite(out[counts[0]:]).all())
        step.mgr.close()


def test_rows_behind_the_last_sequence_stay(kvx, cuda):
    step = Step(kvx, cuda, [3, 50], [60, 90], 8, 2, 128, 16, BF16, BF16)
    q = torch.cat([step.q, torch.full_like(step.q[:4], float("nan"))])
    out, tables = torch.full_like(q, 5.0), step.args()
    step.mgr.attend(0, 1, q, *tables, out=out, **step.kw())
    step.check(out[:53])
    assert bool((out[53:] == 5).all())
    # Starts out of order and out of range: nothing outside is touched.
    for starts in ([60, 3, -5], [-9, 2**31 - 1, 40], [0, 0, 0]):
        step.mgr.attend(0, 1, q, *tables, out=out, starts=ints(starts, cuda))
    torch.cuda.synchronize()
    step.mgr.close()


def test_strides_in_place_and_streams(kvx, cuda):
    step = Step(kvx, cuda, [2, 60, 1], [40, 160, 300], 8, 2, 96, 16, F16, F16)
    want = step.run()
    tables, lengths = step.args()
    q = step.q
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.zeros(q.numel() + 1, dtype=F16, device=cuda)[1:].view(q.shape)
    odd.copy_(q)
    wide = torch.zeros(q.shape[0], 24, 96, dtype=F16, device=cuda)
    wide[:, 8:16] = q
    side = torch.cuda.Stream(cuda)
    torch.cuda.synchronize()
    for x in (heads_first, odd, wide[:, 8:16]):
        assert torch.equal(step.mgr.attend(0, 1, x, tables, lengths, **step.kw()), want)
    for stream in (side, side.cuda_stream):
        got = step.run(stream=stream)
        side.synchronize()
        assert torch.equal(got, want)
    out = torch.zeros_like(wide)
    step.mgr.attend(0, 1, q, tables, lengths, out=out[:, 8:16], **step.kw())
    assert torch.equal(out[:, 8:16], want) and bool((out[:, :8] == 0).all())
    assert bool((out[:, 16:] == 0).all())
    own = wide[:, 8:16]
    assert step.mgr.attend(0, 1, own, tables, lengths, out=own, **step.kw()) is own
    assert torch.equal(own, want) and bool((wide[:, :8] == 0).all())
    padded = torch.full((3, tables.shape[1] + 9), 2**31 - 1, dtype=torch.int32, device=cuda)
    padded[:, :tables.shape[1]] = tables
    assert torch.equal(step.mgr.attend(0, 1, q, padded[:, :tables.shape[1]], lengths,
                                       **step.kw()), want)
    step.mgr.close()


def test_many_sequences(kvx, cuda):
    lengths = [(7 * s) % 50 for s in range(1500)]
    step = Step(kvx, cuda, [1] * 1500, lengths, 4, 2, 64, 16, BF16, BF16)
    step.check(step.run())
    step.mgr.close()
    step = Step(kvx, cuda, [s % 3 for s in range(400)], [s % 41 + 2 for s in range(400)], 4, 2, 64,
                16, BF16, BF16, groups=[(10, 12, 16)])
    for s in (10, 11):
        assert step.lengths[s] >= 12
    step.groups = ()
    step.check(step.run())
    step.mgr.close()


def test_nothing_to_do(kvx, cuda):
    step = Step(kvx, cuda, [1], [5], 4, 2, 64, 16, BF16, BF16)
    none = torch.empty(0, dtype=torch.int32, device=cuda)
    q = step.q[:0]
    assert step.mgr.attend(0, 1, q, none.view(0, 3), none).shape == (0, 4, 64)
    # Tokens, but no sequence that owns them.
    out = torch.full_like(step.q, 3.0)
    step.mgr.attend(0, 1, step.q, none.view(0, 1), none, starts=ints([0], cuda), out=out)
    assert bool((out == 3).all())
    # A table without blocks.
    out = step.mgr.attend(0, 1, step.q, torch.empty(1, 0, dtype=torch.int32, device=cuda),
                          ints([5], cuda))
    assert bool((out == 0).all())
    step.mgr.close()


def test_captured_steps_follow_their_lengths(kvx, cuda):
    """norm_rope, append_kv and attend of a decode loop, captured once each in
    two graphs and replayed in turn, against the eager calls."""
    gen = torch.Generator(device=cuda).manual_seed(3)
    S, Hq, Hk, D, B, W = 6, 8, 2, 128, 16, 20
    inv = (10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)).float().to(cuda)
    w = torch.randn(D, device=cuda, generator=gen).to(BF16)

    def new():
        caches = [torch.zeros(S * W, B, Hk, D, dtype=BF16, device=cuda) for _ in range(2)]
        return kvx.KVCacheManager(caches, host_blocks_to_allocate=1), caches

    tables = torch.randperm(S * W, generator=torch.Generator().manual_seed(4)).int().view(S, W)
    tables = tables.to(cuda)

    def step(mgr, qkv, lengths):
        pos = lengths - 1
        q, _ = kvx.norm_rope(qkv[:, :Hq], None, pos, inv, q_weight=w)
        mgr.append_kv(0, 1, qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:], tables, lengths, inv_freq=inv,
                      k_weight=w)
        return mgr.attend(0, 1, q, tables, lengths)

    (eager, eager_caches), (a, a_caches), (b, b_caches) = new(), new(), new()
    first = torch.tensor([0, 15, 127, 130, 200, 255], dtype=torch.int32, device=cuda)
    for caches in (a_caches, b_caches):
        for c, e in zip(caches, eager_caches):
            if caches is a_caches:
                e.normal_(generator=gen)
            c.copy_(e)
    graphs = []
    for mgr in (a, b):
        qkv = torch.zeros(S, Hq + 2 * Hk, D, dtype=BF16, device=cuda)
        lengths = torch.zeros(S, dtype=torch.int32, device=cuda)
        side = torch.cuda.Stream(cuda)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(mgr, qkv, lengths)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(mgr, qkv, lengths)
        graphs.append((graph, qkv, lengths, out))
    for i in range(5):
        x = torch.randn(S, Hq + 2 * Hk, D, device=cuda, generator=gen).to(BF16)
        lengths = first + 1 + i
        want = step(eager, x, lengths)
        for graph, qkv, held, _ in graphs:
            qkv.copy_(x)
            held.copy_(lengths)
            graph.replay()
        torch.cuda.synchronize()
        for _, _, _, out in graphs:
            assert torch.equal(out, want)
    for c, d, e in zip(a_caches, b_caches, eager_caches):
        assert torch.equal(c, e) and torch.equal(d, e)
    for m in (eager, a, b):
        m.close()


@pytest.mark.parametrize("cache", [BF16, FP8])
def test_prefill_decode_offload_reload(kvx, cuda, cache):
    """A served sequence's life: prefill in chunks, single tokens, its blocks
    to the host tier and back into other ones, and on; every output against
    attention over what the cache holds."""
    gen = torch.Generator(device=cuda).manual_seed(8)
    Hq, Hk, D, B, blocks = 8, 2, 128, 16, 40
    caches = [torch.zeros(blocks, B, Hk, D, dtype=BF16, device=cuda).to(cache) for _ in range(4)]
    scales = [torch.zeros(blocks, Hk, device=cuda) for _ in range(4)] if cache == FP8 else []
    mgr = kvx.KVCacheManager(caches, host_blocks_to_allocate=16, scale_tables=scales)
    inv = (10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)).float().to(cuda)
    ids = [31, 4, 17, 9, 22, 0, 38, 12]
    length = 0
    for turn, n in enumerate([50, 1, 20, 1, 1]):
        if turn == 3:  # the sequence leaves the pool and comes back elsewhere
            stream = torch.cuda.current_stream()
            mgr.d2h(ids, list(range(8)), stream=stream).Await()
            for c in caches:
                c.view(torch.uint8).zero_()
            other = [1, 2, 3, 5, 6, 7, 8, 10]
            back = mgr.h2d(list(range(8)), other, stream=stream)
            back.wait_on_stream()
            ids = other
        length += n
        qkv = torch.randn(n, Hq + 2 * Hk, D, device=cuda, generator=gen).to(BF16)
        pos = torch.arange(length - n, length, device=cuda)
        tables, lengths, starts = ints([ids], cuda), ints([length], cuda), ints([0, n], cuda)
        for layer in (0, 2):
            q, _ = kvx.norm_rope(qkv[:, :Hq], None, pos, inv)
            mgr.append_kv(layer, layer + 1, qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:], tables, lengths,
                          starts=starts, inv_freq=inv)
            out = mgr.attend(layer, layer + 1, q, tables, lengths, starts=starts)
            k, v = (ref.gather(caches[i].cpu(), scales[i].cpu() if scales else None, ids, length)
                    for i in (layer, layer + 1))
            visible = torch.arange(length)[None] <= torch.arange(length - n, length)[:, None]
            want, _, slack = ref.attend(q.cpu(), k, v, visible, D ** -0.5, BF16, BF16)
            ref.assert_rounded(out, want, slack, BF16)
    mgr.close()

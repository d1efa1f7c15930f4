"""GPU: weigh, choose_kept and compact against plain forms, every entry that the
call does not own left as it was, and a served loop that evicts."""
import pytest

torch = pytest.importorskip("torch")

import fp4_reference as fp4  # noqa: E402
import paged_reference as ref  # noqa: E402
from test_gpu_append_kv import freqs, ints  # noqa: E402
from test_gpu_attend import Step  # noqa: E402
from test_gpu_fp4_pool import Step4  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
INF, NAN = float("inf"), float("nan")


def make(kvx, cuda, counts, lengths, hq, hk, dim, block, dtype, cache, **kw):
    if cache == "fp4":
        return Step4(kvx, cuda, counts, lengths, hq, hk, dim, block, dtype, **kw)
    return Step(kvx, cuda, counts, lengths, hq, hk, dim, block, dtype, cache, **kw)


def keys_of(step, s):
    if step.caches[0].dtype == fp4.FP4:
        return fp4.gather(step.caches[0], step.scales[0], step.tables[s], step.lengths[s])
    scales = step.scales[0].cpu() if step.scales[0] is not None else None
    return ref.gather(step.caches[0].cpu(), scales, step.tables[s], step.lengths[s])


def check_weights(step, before, after, lse, begins, decay, causal=True, scale=None):
    """after: before, but for the entries of the sequences' tokens. Of an
    exponential, the score is off by 2 (D + 8) half steps of sum |q k| scale, the
    log by 4 of its size, both also by being moved into powers of two, and the
    exponential by 32; its sum by one a row and 16, the decayed part by 2."""
    block, dim = before.shape[2], step.q.shape[2]
    want, room = before.double().cpu(), torch.zeros(before.shape, dtype=torch.float64)
    group, scale = step.q.shape[1] // before.shape[1], scale or step.scale
    for s, n in enumerate(step.counts):
        length = step.lengths[s]
        begin = begins[s] if begins else 0
        if n == 0 or begin >= length:
            continue
        k = keys_of(step, s)
        rows = slice(step.starts[s], step.starts[s + 1])
        q, of = step.q[rows].double().cpu(), lse[rows].double().cpu()
        j = torch.arange(length)
        last = torch.arange(length - n, length) if causal else torch.full((n,), length)
        visible = (j[None] <= last[:, None])
        place = torch.tensor(step.tables[s])[j // block][begin:], (j % block)[begin:]
        for h in range(before.shape[1]):
            got, slack = torch.zeros(length).double(), torch.zeros(length).double()
            for g in range(h * group, h * group + group):
                p = (q[:, g] @ k[:, h].t() * scale - of[:, g:g + 1]).exp()
                p = torch.where(visible, p, 0.0)
                size = q[:, g].abs() @ k[:, h].abs().t() * scale
                rel = 2 * (dim + 8) * size + 4 * of[:, g:g + 1].abs().nan_to_num(0, 0, 0) + 128
                got += p.sum(0)
                slack += torch.where(visible, p * rel, 0.0).sum(0)
            slack += got * (n * group + 16)
            old = torch.zeros(length).double()
            old[begin:] = before.double().cpu()[place[0], h, place[1]]
            old = torch.where(j < length - n, old * decay, 0.0) if decay else old * 0
            want[place[0], h, place[1]] = (got + old)[begin:]
            room[place[0], h, place[1]] = ((slack + 4 * (got + old).abs()) * ref.U32)[begin:]
    off = (after.double().cpu() - want).abs()
    assert bool((off <= room).all()), float((off / room.clamp_min(1e-300)).max())


WEIGH = [  # (new tokens, lengths, q heads, heads, dim, block)
    ([1], [1], 4, 1, 128, 16), ([1] * 4, [7, 0, 129, 300], 8, 2, 128, 16),
    ([1] * 3, [513, 15, 33], 32, 8, 128, 16), ([1] * 2, [100, 31], 20, 4, 96, 7),
    ([1] * 2, [90, 4], 48, 1, 128, 8), ([1] * 2, [140, 1], 6, 3, 256, 64),
    ([1], [40], 5, 5, 32, 1), ([1] * 2, [2500, 12], 64, 2, 128, 16), ([1], [77], 17, 1, 64, 16),
    ([5, 0, 1], [5, 9, 30], 8, 2, 128, 16), ([64], [64], 4, 4, 64, 16),
    ([130, 3, 1], [130, 400, 257], 8, 1, 128, 16), ([200], [777], 6, 2, 96, 8),
    ([33, 40], [33, 150], 16, 1, 64, 32), ([70], [370], 4, 2, 256, 16),
    ([9, 300], [4, 300], 4, 1, 128, 16),  # more queries than tokens: the first see nothing
    ([20], [1100], 40, 1, 160, 16), ([600, 3], [900, 700], 8, 2, 128, 16)]


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, F16), (BF16, FP8), (F16, FP8),
                                         (BF16, "fp4"), (F16, "fp4")])
@pytest.mark.parametrize("counts,lengths,hq,hk,dim,block", WEIGH)
def test_weigh(kvx, cuda, dtype, cache, counts, lengths, hq, hk, dim, block):
    step = make(kvx, cuda, counts, lengths, hq, hk, dim, block, dtype, cache)
    _, lse = step.run(return_lse=True)
    blocks = step.caches[0].shape[0]
    before = torch.rand(blocks, hk, block, device=cuda)
    # What new tokens find in their place is not theirs.
    for s, n in enumerate(counts):
        for p in range(max(lengths[s] - n, 0), lengths[s]):
            before[step.tables[s][p // block], :, p % block] = NAN
    begins = [n // 3 for n in lengths]
    for decay, skip, causal in ((1.0, False, True), (0.0, True, True), (0.5, True, False)):
        after = before.clone()
        if not causal:
            _, lse = step.run(return_lse=True, causal=False)
        kw = dict(begins=ints(begins, cuda) if skip else None, decay=decay, causal=causal,
                  **step.kw())
        step.mgr.weigh(0, step.q, *step.args(), lse, after, **kw)
        again = before.clone()
        step.mgr.weigh(0, step.q, *step.args(), lse, again, **kw)
        assert torch.equal(again.view(torch.int32), after.view(torch.int32))
        clean = before.nan_to_num(0)
        # Entries of new tokens before `begins` keep what they hold.
        check_weights(step, clean, torch.where(after.isnan(), clean, after), lse,
                      begins if skip else None, decay, causal)
        owned = torch.zeros_like(before, dtype=torch.bool)
        for s, n in enumerate(counts):
            for p in range(begins[s] if skip else 0, lengths[s] if n else 0):
                owned[step.tables[s][p // block], :, p % block] = True
        assert not bool(after[owned].isnan().any())
        assert torch.equal(after[~owned].view(torch.int32), before[~owned].view(torch.int32))
    step.mgr.close()


def test_weights_of_a_row_add_up_to_one(kvx, cuda):
    for counts, lengths in (([1] * 3, [50, 600, 7]), ([100, 40], [100, 900])):
        for cache in (BF16, FP8, "fp4"):
            step = make(kvx, cuda, counts, lengths, 8, 2, 128, 16, BF16, cache)
            _, lse = step.run(return_lse=True)
            table = torch.zeros(step.caches[0].shape[0], 2, 16, device=cuda)
            step.mgr.weigh(0, step.q, *step.args(), lse, table, decay=0.0, **step.kw())
            for s, n in enumerate(counts):
                got = table[torch.tensor(step.tables[s], device=cuda).long()].sum((0, 2))
                # Each row's weights add up to 1 but for what lse and they are off by.
                assert bool(((got - n * 4).abs() <= n * 4 * 2e-4).all())
            step.mgr.close()


def test_weigh_of_places_strides_and_streams(kvx, cuda):
    for counts in ([1, 1], [40, 3]):
        step = Step(kvx, cuda, counts, [100, 90], 8, 2, 64, 16, BF16, BF16)
        tables, lengths = step.args()
        _, lse = step.run(return_lse=True)
        table = torch.ones(step.caches[0].shape[0], 2, 16, device=cuda)
        want = table.clone()
        step.mgr.weigh(0, step.q, tables, lengths, lse, want, **step.kw())
        for bad in (-1, 10**6, -2**31):  # blocks outside the pool are skipped
            tables[0, 2] = bad
            got = table.clone()
            step.mgr.weigh(0, step.q, tables, lengths, lse, got, **step.kw())
            hole = want.clone()
            hole[step.tables[0][2]] = 1
            assert torch.equal(got, hole)
        tables, _ = step.args()
        side = torch.cuda.Stream(cuda)
        odd = torch.zeros(step.q.numel() + 1, dtype=BF16, device=cuda)[1:].view(step.q.shape)
        odd.copy_(step.q)
        wide = torch.zeros(step.q.shape[0], 20, 64, dtype=BF16, device=cuda)
        wide[:, 4:12] = step.q
        larger = torch.ones(table.shape[0] + 3, 2, 16, device=cuda)
        torch.cuda.synchronize()
        for q, stream in ((odd, side), (wide[:, 4:12], side.cuda_stream),
                          (step.q.transpose(0, 1).contiguous().transpose(0, 1), None)):
            got = larger.clone()
            torch.cuda.synchronize()
            step.mgr.weigh(0, q, tables, lengths, lse, got, stream=stream, **step.kw())
            torch.cuda.synchronize()
            assert torch.equal(got[:len(want)], want) and bool((got[len(want):] == 1).all())
        # Lengths past the table, of zero and below, begins of any kind, starts out of order.
        for bad in ([2**31 - 1, 90], [0, -7]):
            step.mgr.weigh(0, step.q, tables, ints(bad, cuda), lse, got,
                           begins=ints([-5, 2**31 - 1], cuda), **step.kw())
        if len(step.q) > 2:
            for starts in ([60, 3, -5], [-9, 2**31 - 1, 40], [0, 0, 0]):
                step.mgr.weigh(0, step.q, tables, lengths, lse, got, starts=ints(starts, cuda))
        torch.cuda.synchronize()
        step.mgr.close()


# -- choose_kept ------------------------------------------------------------------

def plain_choice(weights, budget, recent, begin):
    """Positions that stay, of a list of weights."""
    n = len(weights)
    if n <= budget:
        return list(range(n))
    first = min(begin, budget)
    recent = min(recent, budget - first)
    middle = range(first, n - recent)
    nan = [w != w for w in weights]  # less than any number, -infinity among them
    order = sorted(middle, key=lambda p: (nan[p], 0.0 if nan[p] else -weights[p], p))
    return sorted(list(range(first)) + order[:budget - first - recent]
                  + list(range(n - recent, n)))


CHOICES = [  # (lengths, heads, block, budget, recent, begins)
    ([5000], 8, 16, 1024, 128, [4]), ([1, 0, 40, 41, 39], 2, 16, 40, 3, None),
    ([300] * 5, 1, 7, 1, 0, None), ([300, 20, 64], 3, 1, 64, 64, [0, 50, 3]),
    ([100, 100, 100, 100], 2, 32, 50, 20, [0, 49, 50, 1000]), ([2049], 2, 64, 2048, 1, None),
    ([3000, 2900], 4, 8, 1023, 0, [-3, 7]), ([9], 5, 16, 0, 0, None), ([70], 2, 16, 69, 69, None),
    ([40000, 50000], 1, 64, 7000, 500, None)]


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "odd"])
@pytest.mark.parametrize("lengths,heads,block,budget,recent,begins", CHOICES)
def test_choose(kvx, cuda, kind, lengths, heads, block, budget, recent, begins):
    gen = torch.Generator().manual_seed(budget + len(lengths))
    need = [(n + block - 1) // block for n in lengths]
    blocks = sum(need) + 4
    if kind == "spread":
        w = torch.randn(blocks, heads, block, generator=gen).mul(3).exp()
    elif kind == "ties":
        w = torch.randint(0, 5, (blocks, heads, block), generator=gen).float()
    elif kind == "equal":
        w = torch.zeros(blocks, heads, block)
    else:
        w = torch.randn(blocks, heads, block, generator=gen)
        pick = torch.rand(w.shape, generator=gen)
        for i, x in enumerate([INF, -INF, NAN, 0.0, -0.0, 1e-40, -1e-40, 3e38]):
            w[(pick > i / 20) & (pick < (i + 1) / 20)] = x
    ids, tables, at = torch.randperm(blocks, generator=gen).tolist(), [], 0
    for n in need:
        tables.append(ids[at:at + n])
        at += n
    width = max(need) + 1
    args = (w.to(cuda), ints([t + [-1] * (width - len(t)) for t in tables], cuda),
            ints(lengths, cuda), budget)
    kw = dict(recent=recent, begins=ints(begins, cuda) if begins else None)
    kept, cut = kvx.choose_kept(*args, **kw)
    assert cut.tolist() == [min(n, budget) for n in lengths]
    for s, n in enumerate(lengths):
        for h in range(heads):
            x = [float(v) for v in torch.cat([w[b, h] for b in tables[s]] or [w[0, 0, :0]])[:n]]
            want = plain_choice(x, budget, recent, max(begins[s], 0) if begins else 0)
            assert kept[s, h].tolist() == want + [-1] * (budget - len(want))
    assert torch.equal(kvx.choose_kept(*args, **kw)[0], kept)


def test_choose_of_bad_tables(kvx, cuda):
    w = torch.rand(9, 2, 16, device=cuda) + 1
    tables = ints([[3, -1, 5, 2**31 - 1, 6], [0, 1, 2, 7, -2**31]], cuda)
    kept, cut = kvx.choose_kept(w, tables, ints([2**31 - 1, 70], cuda), 40)
    assert cut.tolist() == [40, 40]
    # Tokens that have a place come first, then the earliest without one.
    assert kept[0, 0].tolist() == plain_choice(
        sum(([float(v) for v in w[b, 0]] if 0 <= b < 9 else [NAN] * 16
             for b in tables[0].tolist()), []), 40, 0, 0)
    kept, cut = kvx.choose_kept(w, tables, ints([-4, 0], cuda), 40)
    assert cut.tolist() == [0, 0] and bool((kept == -1).all())
    none = torch.empty(0, 5, dtype=torch.int32, device=cuda)
    kept, cut = kvx.choose_kept(w, none, none[:, 0], 7)
    assert kept.shape == (0, 2, 7) and cut.shape == (0,)
    side = torch.cuda.Stream(cuda)
    torch.cuda.synchronize()
    want = kvx.choose_kept(w, tables[1:], ints([70], cuda), 20)[0]
    got = kvx.choose_kept(w, tables[1:], ints([70], cuda), 20, stream=side)[0]
    torch.cuda.synchronize()
    assert torch.equal(got, want)


# -- compact ----------------------------------------------------------------------

def raw(t):
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()]).cpu().clone()


def storages(cuda, cache, blocks, block, heads, dim, seed):
    gen = torch.Generator().manual_seed(seed)
    if cache == "fp4":
        pairs = [fp4.storage(torch.randn(blocks, heads, block, dim, generator=gen), BF16, cuda)
                 for _ in range(2)]
        return [list(x) for x in zip(*pairs)]
    x = [torch.randn(blocks, block, heads, dim, generator=gen) for _ in range(2)]
    if cache == FP8:
        # Scales up to 2^6 apart, so that codes are rounded again.
        scales = [torch.rand(blocks, heads, generator=gen).mul(6).exp2() for _ in range(2)]
        return [(c * 60).to(FP8).to(cuda) for c in x], [s.to(cuda) for s in scales]
    return [c.to(cache).to(cuda) for c in x], []


COMPACTS = [  # (sequences, heads, dim, block, held, budget, prefix)
    (1, 8, 128, 16, 500, 100, 4), (5, 2, 64, 16, 200, 130, 0), (3, 1, 96, 7, 90, 45, 20),
    (2, 3, 256, 64, 400, 399, 0), (9, 4, 128, 8, 64, 1, 0), (2, 2, 32, 1, 50, 25, 3),
    (40, 8, 128, 16, 300, 200, 0), (2, 1, 64, 200, 900, 500, 0), (1, 2, 160, 24, 3000, 2000, 9),
    (1, 1, 128, 300, 1000, 700, 0), (1, 2, 64, 600, 1900, 1500, 5), (33, 8, 32, 300, 400, 350, 0),
    (33, 8, 64, 16, 700, 600, 0)]


@pytest.mark.parametrize("cache", [BF16, F16, FP8, "fp4"])
@pytest.mark.parametrize("sequences,heads,dim,block,held,budget,prefix", COMPACTS)
def test_compact(kvx, cuda, cache, sequences, heads, dim, block, held, budget, prefix):
    need = (held + block - 1) // block
    blocks = sequences * need + 3
    caches, scales = storages(cuda, cache, blocks, block, heads, dim, budget)
    mgr = kvx.KVCacheManager(caches, host_blocks_to_allocate=1, scale_tables=scales)
    gen = torch.Generator().manual_seed(held)
    tables = torch.randperm(blocks, generator=gen)[:sequences * need].view(sequences, need)
    kept = torch.full((sequences, heads, budget), -1, dtype=torch.int32)
    for s in range(sequences):
        for h in range(heads):
            n = budget if s % 3 != 2 else budget // 2  # some keep fewer
            rest = torch.randperm(held - prefix, generator=gen)[:n - min(prefix, n)] + prefix
            both = torch.cat([torch.arange(min(prefix, n)), rest]).sort().values
            if s % 4 == 3:
                both = torch.arange(n)  # nothing moves
            kept[s, h, :n] = both.int()
    weights = torch.rand(blocks, heads, block, device=cuda)
    old = [raw(t) for t in caches + scales + [weights]]
    want = [t.clone() for t in old]
    head_major = cache == "fp4"
    for s in range(sequences):
        for h in range(heads):
            p = kept[s, h][kept[s, h] >= 0].long()
            i = torch.arange(len(p))
            moved = p != i
            p_of, i_of = tables[s][p // block], tables[s][i // block]
            for c in range(2):
                if cache == FP8:
                    f = scales[c].cpu()
                    values = old[c].view(FP8)[p_of, p % block, h].double()
                    for b in (i // block).unique().tolist():
                        mine = i // block == b
                        if not moved[mine].any():
                            continue
                        top = f[p_of[mine], h].max()
                        want[2 + c].view(torch.float32)[tables[s][b], h] = top
                        # Through fp32, as the ratio is.
                        again = (values[mine].float() * (f[p_of[mine], h] / top)[:, None]).to(FP8)
                        same = (f[p_of[mine], h] == top)[:, None]
                        again = torch.where(same, old[c][p_of[mine], (p % block)[mine], h],
                                            again.view(torch.uint8))
                        want[c][tables[s][b], (i % block)[mine], h] = again
                elif head_major:
                    for t in (c, 2 + c):
                        want[t][i_of[moved], h, (i % block)[moved]] = \
                            old[t][p_of[moved], h, (p % block)[moved]]
                else:
                    want[c][i_of[moved], (i % block)[moved], h] = \
                        old[c][p_of[moved], (p % block)[moved], h]
            want[-1][i_of[moved], h, (i % block)[moved]] = old[-1][p_of[moved], h, (p % block)[moved]]
    for table in (weights, None):
        for t, o in zip(caches + scales + [weights], old):
            t.view(o.dtype).copy_(o)
        mgr.compact(0, 1, kept.to(cuda), tables.int().to(cuda), weights=table)
        got = [raw(t) for t in caches + scales + [weights]]
        for n, (g, w) in enumerate(zip(got, want[:-1] + [want[-1] if table is not None else old[-1]])):
            assert torch.equal(g, w), n
    mgr.close()


@pytest.mark.parametrize("cache", [BF16, FP8, "fp4"])
def test_compact_stays_inside(kvx, cuda, cache):
    """Places and positions without a block, and positions that do not ascend."""
    caches, scales = storages(cuda, cache, 12, 16, 2, 64, 1)
    mgr = kvx.KVCacheManager(caches, host_blocks_to_allocate=1, scale_tables=scales)
    weights = torch.rand(12, 2, 16, device=cuda)
    spare = [raw(t)[9:] for t in caches + scales + [weights]]
    tables = ints([[0, 1, -1, 3], [4, 2**31 - 1, 6, -2**31]], cuda)
    gen = torch.Generator().manual_seed(2)
    for low, high in ((-5, 70), (-2**31, 2**31 - 1), (0, 64)):
        kept = torch.randint(low, high, (2, 2, 90), generator=gen, dtype=torch.int64).int()
        mgr.compact(0, 1, kept.to(cuda), tables, weights=weights)
    # In order, what has no place moves nothing.
    old = [raw(t) for t in caches]
    kept = torch.arange(10, 40, dtype=torch.int32)[None, None].expand(2, 2, 30).contiguous()
    mgr.compact(0, 1, kept.to(cuda), tables, weights=weights)
    if cache == BF16:
        got = raw(caches[0])
        assert torch.equal(got[0, 0], old[0][0, 10]) and torch.equal(got[1, 5], old[0][1, 15])
        assert torch.equal(got[1, 6], old[0][1, 6])  # position 32 is in no block
    for t, o in zip(caches + scales + [weights], spare):
        assert torch.equal(raw(t)[9:], o)
    mgr.compact(0, 1, torch.empty(0, 2, 5, dtype=torch.int32, device=cuda), tables[:0])
    mgr.compact(0, 1, torch.empty(2, 2, 0, dtype=torch.int32, device=cuda), tables)
    torch.cuda.synchronize()
    mgr.close()


def test_compact_of_scales_far_apart(kvx, cuda):
    """Quotients of scales below fp32's least number: the rows become zeros."""
    gen = torch.Generator(device=cuda).manual_seed(5)
    caches = [torch.randn(4, 16, 1, 64, device=cuda, generator=gen).to(FP8) for _ in range(2)]
    old = [c.float() for c in caches]
    scales = [torch.tensor([1e-30, 1e20, 0.0, 1.0], device=cuda)[:, None].contiguous() for _ in range(2)]
    mgr = kvx.KVCacheManager(caches, host_blocks_to_allocate=1, scale_tables=scales)
    positions = list(range(3, 9)) + [17, 20, 33]
    mgr.compact(0, 1, ints([[positions]], cuda), ints([[0, 1, 2]], cuda))
    for c, o, f in zip(caches, old, scales):
        assert torch.equal(f[:, 0], torch.tensor([1e20, 1e20, 0.0, 1.0], device=cuda))
        for i, p in enumerate(positions):
            want = o[1, p - 16, 0] if 16 <= p < 32 else torch.zeros(64, device=cuda)
            assert torch.equal(c.float()[0, i, 0], want), p
    mgr.close()


# -- together ---------------------------------------------------------------------

@pytest.mark.parametrize("cache", [BF16, FP8, "fp4"])
def test_a_loop_that_evicts(kvx, cuda, cache):
    """Prefill, decode steps that weigh, and a cut to a budget whenever a sequence
    has grown over it, against attention over what the cache holds; the tokens that
    stay are those of the largest weights."""
    gen = torch.Generator(device=cuda).manual_seed(4)
    S, Hq, Hk, D, B, W = 3, 8, 2, 128, 16, 8
    caches, scales = storages(cuda, cache, S * W + 2, B, Hk, D, 3)
    mgr = kvx.KVCacheManager(caches, host_blocks_to_allocate=1, scale_tables=scales)
    weights = torch.full((S * W + 2, Hk, B), NAN, device=cuda)
    tables = torch.randperm(S * W, generator=torch.Generator().manual_seed(4)).view(S, W)
    inv, on = freqs(D // 2, cuda), tables.int().to(cuda)
    lengths, written = ints([0] * S, cuda), [0] * S
    begins = ints([0, 2, 40], cuda)

    def held(s, n):
        out = []
        for c in range(2):
            if cache == "fp4":
                out.append(fp4.gather(caches[c], scales[c], tables[s].tolist(), n))
            else:
                out.append(ref.gather(caches[c].cpu(), scales[c].cpu() if scales else None,
                                      tables[s].tolist(), n))
        return out

    for turn in range(6):
        counts = [60, 3, 45] if turn == 0 else [1] * S
        T = sum(counts)
        starts = ints([0] + torch.tensor(counts).cumsum(0).tolist(), cuda)
        lengths = (lengths + torch.tensor(counts, device=cuda)).int()
        qkv = torch.randn(T, Hq + 2 * Hk, D, device=cuda, generator=gen).to(BF16)
        pos = torch.cat([torch.arange(written[s], written[s] + n) for s, n in enumerate(counts)])
        pos = pos.to(cuda)
        written = [w + n for w, n in zip(written, counts)]
        q, _ = kvx.norm_rope(qkv[:, :Hq], None, pos, inv)
        mgr.append_kv(0, 1, qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:], on, lengths, starts=starts,
                      inv_freq=inv, positions=pos)
        out, lse = mgr.attend(0, 1, q, on, lengths, starts=starts, return_lse=True)
        mgr.weigh(0, q, on, lengths, lse, weights, starts=starts)
        first = 0
        for s, n in enumerate(counts):
            L = int(lengths[s])
            k, v = held(s, L)
            visible = torch.arange(L)[None] <= torch.arange(L - n, L)[:, None]
            want, _, slack = ref.attend(q[first:first + n].cpu(), k, v, visible, D ** -0.5, BF16,
                                        BF16)
            ref.assert_rounded(out[first:first + n], want, slack, BF16)
            first += n
        if turn % 2 == 0:
            before = [held(s, int(lengths[s])) for s in range(S)]
            w = weights.cpu()
            was, lengths = lengths.tolist(), mgr.evict(0, 1, weights, on, lengths, 37, recent=5,
                                                       begins=begins)
            assert lengths.tolist() == [min(n, 37) for n in was]
            for s in range(S):
                now = held(s, int(lengths[s]))
                got = weights.cpu()
                for h in range(Hk):
                    x = torch.cat([w[b, h] for b in tables[s]])[:was[s]]
                    stay = plain_choice(x.tolist(), 37, 5, int(begins[s]))
                    new = torch.cat([got[b, h] for b in tables[s]])[:len(stay)]
                    assert torch.equal(new, x[stay])
                    for c in range(2):
                        if cache != FP8:
                            assert torch.equal(now[c][:, h], before[s][c][stay, h])
                        else:
                            # Half a step of e4m3 under the block's scale.
                            top = scales[c].cpu()[tables[s][torch.arange(len(stay)) // B], h]
                            room = now[c][:, h].abs() / 16 + top.double()[:, None] * 2.0**-9
                            assert bool(((now[c][:, h] - before[s][c][stay, h]).abs() <= room).all())
    mgr.close()


@pytest.mark.parametrize("each", [1, 30])
def test_captured_eviction_follows_lengths(kvx, cuda, each):
    """weigh and evict captured once in two graphs that are replayed in turn,
    against the eager calls."""
    gen = torch.Generator(device=cuda).manual_seed(3)
    S, Hq, Hk, D, B, W = 4, 8, 2, 64, 16, 12
    start, none = storages(cuda, BF16, S * W, B, Hk, D, 3)
    tables = torch.randperm(S * W, generator=torch.Generator().manual_seed(4)).int().view(S, W)
    tables = tables.to(cuda)
    table = torch.rand(S * W, Hk, B, device=cuda, generator=gen)
    starts = ints([n * each for n in range(S + 1)], cuda)

    def step(mgr, q, lengths, weights):
        kw = dict(starts=starts) if each > 1 else {}
        _, lse = mgr.attend(0, 1, q, tables, lengths, return_lse=True, **kw)
        mgr.weigh(0, q, tables, lengths, lse, weights, **kw)
        return mgr.evict(0, 1, weights, tables, lengths, 50, recent=8)

    sides = []
    for captured in (False, True, True):
        caches, weights = [c.clone() for c in start], table.clone()
        mgr = kvx.KVCacheManager(caches, host_blocks_to_allocate=1)
        q = torch.zeros(S * each, Hq, D, dtype=BF16, device=cuda)
        lengths = torch.zeros(S, dtype=torch.int32, device=cuda)
        graph = out = None
        if captured:
            side = torch.cuda.Stream(cuda)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step(mgr, q, lengths, weights)
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step(mgr, q, lengths, weights)
        sides.append((mgr, caches, weights, q, lengths, graph, out))
    for i in range(4):
        x = torch.randn(S * each, Hq, D, device=cuda, generator=gen).to(BF16)
        now = ints([0, 30 + 10 * i, 51 + i, 190 - 30 * i], cuda)
        cuts = []
        for mgr, _, weights, q, lengths, graph, out in sides:
            q.copy_(x)
            lengths.copy_(now)
            if graph is None:
                cuts.append(step(mgr, q, lengths, weights))
            else:
                graph.replay()
                cuts.append(out)
        torch.cuda.synchronize()
        assert all(torch.equal(c, cuts[0]) for c in cuts)
        for _, caches, weights, *_ in sides[1:]:
            assert all(torch.equal(a, b) for a, b in zip(caches, sides[0][1]))
            assert torch.equal(weights, sides[0][2])
    for mgr, *_ in sides:
        mgr.close()


def test_kept_at_any_strides(kvx, cuda):
    caches, _ = storages(cuda, BF16, 40, 16, 2, 64, 1)
    mgr = kvx.KVCacheManager(caches, host_blocks_to_allocate=1)
    tables = torch.arange(40, dtype=torch.int32, device=cuda).view(2, 20)
    gen = torch.Generator().manual_seed(1)
    kept = torch.stack([torch.randperm(320, generator=gen)[:100].sort().values
                        for _ in range(4)]).view(2, 2, 100).int().to(cuda)
    old = [c.clone() for c in caches]
    mgr.compact(0, 1, kept, tables)
    want = [c.clone() for c in caches]
    wide = torch.full((2, 2, 300), -7, dtype=torch.int32, device=cuda)
    wide[:, :, 2::3] = kept
    for other in (kept.transpose(0, 2).contiguous().transpose(0, 2),
                  kept.transpose(1, 2).contiguous().transpose(1, 2), wide[:, :, 2::3]):
        for c, o in zip(caches, old):
            c.copy_(o)
        mgr.compact(0, 1, other, tables)
        assert all(torch.equal(c, w) for c, w in zip(caches, want))
    # One list for all sequences and heads.
    for c, o in zip(caches, old):
        c.copy_(o)
    mgr.compact(0, 1, kept[:1, :1].expand(2, 2, 100), tables)
    one = [c.clone() for c in caches]
    for c, o in zip(caches, old):
        c.copy_(o)
    mgr.compact(0, 1, kept[:1, :1].expand(2, 2, 100).contiguous(), tables)
    assert all(torch.equal(c, w) for c, w in zip(caches, one))
    mgr.close()


def test_two_calls_at_once(kvx, cuda):
    """Layers of one pool evicted on two streams, chunks weighed on both: as in turn."""
    gen = torch.Generator(device=cuda).manual_seed(3)
    S, Hq, Hk, D, B, W = 3, 8, 2, 128, 16, 40
    start = [torch.randn(S * W, B, Hk, D, device=cuda, generator=gen).to(BF16) for _ in range(4)]
    tables = torch.randperm(S * W, generator=torch.Generator().manual_seed(4)).int().view(S, W)
    tables, lengths = tables.to(cuda), ints([600, 77, 431], cuda)
    starts = ints([0, 150, 170, 300], cuda)
    q = [torch.randn(300, Hq, D, device=cuda, generator=gen).to(BF16) for _ in range(2)]
    results = []
    for at_once in (False, True):
        caches = [c.clone() for c in start]
        mgr = kvx.KVCacheManager(caches, host_blocks_to_allocate=1)
        tabs = [torch.zeros(S * W, Hk, B, device=cuda) for _ in range(2)]
        streams = [torch.cuda.Stream(cuda) for _ in range(2)]
        lse = [mgr.attend(2 * i, 2 * i + 1, q[i], tables, lengths, starts=starts,
                          return_lse=True)[1] for i in range(2)]
        torch.cuda.synchronize()
        cuts = []
        for i in range(2):
            for _ in range(3):
                mgr.weigh(2 * i, q[i], tables, lengths, lse[i], tabs[i], starts=starts, decay=0.5,
                          stream=streams[i])
            cuts.append(mgr.evict(2 * i, 2 * i + 1, tabs[i], tables, lengths, 100, recent=9,
                                  stream=streams[i]))
            if not at_once:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        results.append(caches + tabs + cuts)
        mgr.close()
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("cache", [BF16, FP8, "fp4"])
def test_blocks_past_32_bits(kvx, cuda, cache):
    """A step and an eviction in the last blocks of storages of over 4 GiB (and of over
    2^31 weights), against the same in a small pool."""
    S, Hq, Hk, D, B, W = 2, 16, 8, 128, 16, 12
    each = {BF16: 32768, FP8: 16384, "fp4": 8192}[cache]
    far = (4 << 30) // each + 1000
    small, scales = storages(cuda, cache, S * W, B, Hk, D, 7)
    gen = torch.Generator(device=cuda).manual_seed(3)
    q = torch.randn(40, Hq, D, device=cuda, generator=gen).to(BF16)
    k, v = (torch.randn(40, Hk, D, device=cuda, generator=gen).to(BF16) for _ in range(2))
    starts, lengths = ints([0, 39, 40], cuda), ints([180, 100], cuda)
    results = []
    for blocks in (S * W, far):
        def grown(t):
            if blocks == S * W:
                return t.clone()
            big = torch.zeros((blocks,) + tuple(t.shape[1:]), device=cuda,
                              dtype=torch.uint8 if t.element_size() == 1 else t.dtype)
            big = big.view(t.dtype)
            big.view(torch.uint8)[-S * W:] = t.view(torch.uint8)
            return big
        caches, tabs = [grown(c) for c in small], [grown(t) for t in scales]
        table_blocks = blocks if blocks == S * W else (1 << 31) // (Hk * B) + 1000
        if table_blocks < blocks:
            table_blocks = blocks
        weights = torch.zeros(table_blocks, Hk, B, device=cuda)
        mgr = kvx.KVCacheManager(caches, host_blocks_to_allocate=1, scale_tables=tabs)
        tables = torch.arange(S * W, dtype=torch.int32, device=cuda).view(S, W) + (blocks - S * W)
        mgr.append_kv(0, 1, k, v, tables, lengths, starts=starts)
        out, lse = mgr.attend(0, 1, q, tables, lengths, starts=starts, return_lse=True)
        one = mgr.attend(0, 1, q[:2], tables, lengths)
        mgr.weigh(0, q, tables, lengths, lse, weights, starts=starts)
        mgr.weigh(0, q[:2], tables, lengths, lse[:2].contiguous(), weights)
        last = weights[blocks - S * W:blocks]
        got = last.clone()
        cut = mgr.evict(0, 1, weights, tables, lengths, 70, recent=4)
        results.append([out, one, got, cut, last.clone()]
                       + [t.view(torch.uint8)[-S * W:].clone() for t in caches + tabs])
        mgr.close()
        del caches, tabs, weights, last
        torch.cuda.empty_cache()
    assert all(torch.equal(a, b) for a, b in zip(*results))
    # Weights past 2^31 entries.
    blocks = (1 << 31) // (Hk * B) + 50
    big = torch.zeros(blocks, Hk, B, device=cuda)
    few = torch.rand(20, Hk, B, device=cuda)
    big[-20:] = few
    tables = torch.arange(20, dtype=torch.int32, device=cuda)[None]
    kept, _ = kvx.choose_kept(few, tables, ints([320], cuda), 100)
    assert torch.equal(kvx.choose_kept(big, tables + (blocks - 20), ints([320], cuda), 100)[0], kept)


def test_many_sequences(kvx, cuda):
    for counts, lengths in (([1] * 1500, [(7 * s) % 50 for s in range(1500)]),
                            ([s % 12 for s in range(400)], [s % 41 + 12 for s in range(400)])):
        step = Step(kvx, cuda, counts, lengths, 8, 2, 64, 16, BF16, BF16)
        _, lse = step.run(return_lse=True)
        before = torch.rand(step.caches[0].shape[0], 2, 16, device=cuda)
        after = before.clone()
        step.mgr.weigh(0, step.q, *step.args(), lse, after, decay=0.5, **step.kw())
        check_weights(step, before, after, lse, None, 0.5)
        w, (tables, held) = before.cpu(), step.args()
        kept, cut = kvx.choose_kept(before, tables, held, 13, recent=2)
        for s, n in enumerate(lengths):
            x = torch.cat([w[b, 1] for b in step.tables[s]] or [w[0, 0, :0]])[:n].tolist()
            want = plain_choice(x, 13, 2, 0)
            assert kept[s, 1].tolist() == want + [-1] * (13 - len(want)) and int(cut[s]) == min(n, 13)
        step.mgr.close()

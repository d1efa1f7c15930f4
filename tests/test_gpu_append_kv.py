"""GPU: new keys and values into the paged pool against the 64-bit form, every
byte that no token has a place in left as it was."""
import pytest

torch = pytest.importorskip("torch")

import paged_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def freqs(n, cuda):
    return (10000.0 ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))).float().to(cuda)


def ints(values, cuda):
    return torch.tensor(values, dtype=torch.int32, device=cuda)


def build(kvx, cuda, gen, blocks, block, heads, dim, dtype):
    """A manager over one K and one V storage with random contents."""
    shape, kw = (blocks, block, heads, dim), {}
    caches = [torch.randn(shape, device=cuda, generator=gen) for _ in range(2)]
    if dtype == FP8:
        scales = [torch.rand(blocks, heads, device=cuda, generator=gen) * 0.01 + 0.002
                  for _ in range(2)]
        caches = [(c / s[:, None, :, None]).clamp(-448, 448).to(FP8)
                  for c, s in zip(caches, scales)]
        kw = dict(scale_tables=scales)
    else:
        caches = [c.to(dtype) for c in caches]
        scales = [None, None]
    mgr = kvx.KVCacheManager(caches, host_blocks_to_allocate=1, **kw)
    return mgr, caches, scales


def bits(t):
    return t.view(torch.uint8 if t.dtype == FP8 else torch.int16).cpu()


def slots(where, tables, block, blocks):
    """{token: (block id, slot)} of the tokens that have a place."""
    out = {}
    for t, s, p in where:
        if 0 <= p < len(tables[s]) * block and 0 <= tables[s][p // block] < blocks:
            out[t] = (tables[s][p // block], p % block)
    return out


def sequences_of(counts):
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    return starts


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("counts,lengths,block,heads,dim,rotary,norm,inter", [
    ([1, 1, 1], [1, 17, 40], 16, 8, 128, 128, False, False),
    ([5, 0, 33, 1], [5, 9, 60, 1], 16, 2, 128, 128, True, False),
    ([40], [47], 8, 1, 64, 64, True, False),
    ([3, 20], [3, 90], 7, 3, 80, 32, False, True),
    ([9, 1], [30, 64], 64, 2, 96, 0, True, False),
    ([2, 2], [6, 2], 1, 1, 20, 6, True, False),
    ([4], [4], 32, 2, 256, 256, True, True),
    ([700, 800], [700, 1000], 16, 1, 64, 64, False, False)])
def test_16_bit_pool(kvx, cuda, dtype, counts, lengths, block, heads, dim, rotary, norm, inter):
    gen = torch.Generator(device=cuda).manual_seed(sum(counts) + dim)
    width = max((n + block - 1) // block for n in lengths) + 1
    blocks = width * len(counts) + 3
    mgr, caches, _ = build(kvx, cuda, gen, blocks, block, heads, dim, dtype)
    perm = torch.randperm(blocks, generator=torch.Generator().manual_seed(1)).tolist()
    tables = [perm[s * width:(s + 1) * width] for s in range(len(counts))]
    starts = sequences_of(counts)
    tokens = starts[-1] + 3  # the last three belong to no sequence
    single = counts == [1] * len(counts)
    if single:
        tokens = len(counts)
    fused = torch.randn(tokens, 4 * heads, dim, device=cuda, generator=gen).to(dtype)
    k, v = fused[:, heads:2 * heads], fused[:, 3 * heads:]
    inv = freqs(rotary // 2, cuda) if rotary else None
    w = torch.randn(dim, device=cuda, generator=gen).to(dtype) if norm else None
    before = [bits(c) for c in caches]
    mgr.append_kv(0, 1, k, v, ints(tables, cuda), ints(lengths, cuda),
                  starts=None if single else ints(starts, cuda), inv_freq=inv, k_weight=w,
                  interleaved=inter)
    where = ref.places(starts, lengths, tokens, len(counts))
    place = slots(where, tables, block, blocks)
    assert len(place) == sum(counts)
    positions = torch.zeros(tokens, dtype=torch.int64)
    for t, _, p in where:
        positions[t] = p
    want, slack = ref.norm_rope(k, w, positions, inv, 1e-6, inter)
    after = [c.cpu() for c in caches]
    ids = list(place)
    at = [place[t] for t in ids]
    got = torch.stack([after[0][b, s] for b, s in at])
    ref.assert_rounded(got, want[ids], slack[ids], dtype)
    assert torch.equal(torch.stack([after[1][b, s] for b, s in at]), v.cpu()[ids])
    for c, old in zip(caches, before):
        now = bits(c)
        for b, s in at:
            old[b, s] = now[b, s]
        assert torch.equal(now, old)
    mgr.close()


def test_tokens_without_a_place_are_dropped(kvx, cuda):
    gen = torch.Generator(device=cuda).manual_seed(5)
    for dtype in (BF16, FP8):
        mgr, caches, scales = build(kvx, cuda, gen, 9, 16, 2, 64, dtype)
        k = torch.randn(8, 2, 64, device=cuda, generator=gen).to(BF16)
        before = [bits(c) for c in caches]
        old_scales = [s.clone() for s in scales if s is not None]
        # Ids outside the pool, a length past the table, of zero and below.
        tables = ints([[-1, 3], [9, 3], [2**31 - 1, 3], [-2**31, 3], [0, 1], [0, 1], [0, 1],
                       [0, 1]], cuda)
        lengths = ints([5, 16, 1, 7, 33, 0, -4, 2**31 - 1], cuda)
        mgr.append_kv(0, 1, k, k, tables, lengths, inv_freq=freqs(32, cuda))
        # One sequence with more new tokens than it is long, starts out of order
        # and out of range.
        mgr.append_kv(0, 1, k, k, tables[:4], ints([2, 0, 0, 0], cuda),
                      starts=ints([8, 3, -5, 8, 2**31 - 1], cuda))
        torch.cuda.synchronize()
        assert all(torch.equal(bits(c), b) for c, b in zip(caches, before))
        assert all(torch.equal(s, o) for s, o in zip([s for s in scales if s is not None],
                                                     old_scales))
        # Of four new tokens of a sequence of two the last two have a place.
        mgr.append_kv(0, 1, k[:4], k[:4], ints([[4]], cuda), ints([2], cuda),
                      starts=ints([0, 4], cuda))
        if dtype == BF16:
            assert torch.equal(caches[1][4, :2], k[2:4])
            before[1][4, :2] = bits(caches[1])[4, :2]
            assert torch.equal(bits(caches[1]), before[1])
        mgr.close()


def test_positions_strides_and_other_streams(kvx, cuda):
    gen = torch.Generator(device=cuda).manual_seed(6)
    mgr, caches, _ = build(kvx, cuda, gen, 12, 16, 2, 128, BF16)
    k = torch.randn(5, 2, 128, device=cuda, generator=gen).to(BF16)
    v = torch.randn(2, 5, 128, device=cuda, generator=gen).to(BF16).transpose(0, 1)
    odd = torch.zeros(5 * 2 * 128 + 1, dtype=BF16, device=cuda)[1:].view(5, 2, 128)
    odd.copy_(k)
    inv = freqs(64, cuda)
    tables = ints([[1, 2, 0], [7, 8, 0]], cuda)[:, :2]  # rows apart
    lengths, starts = ints([18, 2], cuda), ints([0, 3, 5], cuda)
    pos = torch.tensor([900, 2, 2**33, 0, 5], device=cuda)
    at = [(1, 15), (2, 0), (2, 1), (7, 0), (7, 1)]
    want, slack = ref.norm_rope(k, None, pos, inv)
    side = torch.cuda.Stream(cuda)
    for keys, stream in ((k, None), (odd, side), (k, side.cuda_stream)):
        for c in caches:
            c.zero_()
        torch.cuda.synchronize()
        mgr.append_kv(0, 1, keys, v, tables, lengths, starts=starts, inv_freq=inv, positions=pos,
                      stream=stream)
        torch.cuda.synchronize()
        ref.assert_rounded(torch.stack([caches[0][b, s] for b, s in at]), want, slack, BF16)
        assert torch.equal(torch.stack([caches[1][b, s] for b, s in at]), v)
    small = pos.clamp(max=1000).int()
    mgr.append_kv(0, 1, k, v, tables, lengths, starts=starts, inv_freq=inv, positions=small)
    want, slack = ref.norm_rope(k, None, small, inv)
    ref.assert_rounded(torch.stack([caches[0][b, s] for b, s in at]), want, slack, BF16)
    mgr.close()


def e4m3_bound(value, scale, slack=0.0):
    """Half a step of e4m3 around value under scale."""
    return value.abs() * ref.half(FP8) * (1 + 2.0 ** -10) + ref.tiny(FP8) * scale + slack


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("counts,lengths,block,heads,dim,rotary,gain", [
    ([1, 1, 1, 1], [1, 17, 40, 32], 16, 8, 128, 128, 1.0),   # scales stay or grow a little
    ([1, 1], [20, 35], 16, 2, 64, 64, 30.0),                 # scales grow
    ([1, 1], [20, 35], 16, 2, 64, 64, 0.01),                 # scales stay
    ([50, 7, 0], [50, 90, 4], 16, 3, 80, 80, 2.0),
    ([100], [130], 48, 1, 96, 32, 1.0),                      # more tokens than one pass
    ([5, 6], [5, 9], 7, 2, 20, 0, 3.0),
    ([300], [300], 32, 2, 256, 256, 1.0)])
def test_e4m3_pool(kvx, cuda, dtype, counts, lengths, block, heads, dim, rotary, gain):
    gen = torch.Generator(device=cuda).manual_seed(sum(counts) + dim)
    width = max((n + block - 1) // block for n in lengths)
    blocks = width * len(counts) + 3
    mgr, caches, scales = build(kvx, cuda, gen, blocks, block, heads, dim, FP8)
    perm = torch.randperm(blocks, generator=torch.Generator().manual_seed(2)).tolist()
    tables = [perm[s * width:(s + 1) * width] for s in range(len(counts))]
    starts = sequences_of(counts)
    tokens = starts[-1]
    k, v = ((torch.randn(tokens, heads, dim, device=cuda, generator=gen) * gain).to(dtype)
            for _ in range(2))
    v[0, 0] = 0
    inv = freqs(rotary // 2, cuda) if rotary else None
    before = [(c.cpu(), bits(c), s.double().cpu()) for c, s in zip(caches, scales)]
    mgr.append_kv(0, 1, k, v, ints(tables, cuda), ints(lengths, cuda),
                  starts=None if counts == [1] * len(counts) else ints(starts, cuda),
                  inv_freq=inv)
    where = ref.places(starts, lengths, tokens, len(counts))
    place = slots(where, tables, block, blocks)
    positions = torch.zeros(tokens, dtype=torch.int64)
    for t, _, p in where:
        positions[t] = p
    key, key_slack = ref.norm_rope(k, None, positions, inv)
    touched = {}
    for t, (b, s) in place.items():
        touched.setdefault(b, []).append((s, t))
    for n, (x, slack) in enumerate(((key, key_slack), (v.double().cpu(), torch.zeros_like(key)))):
        old, old_bits, old_scales = before[n]
        got, got_bits = caches[n].cpu(), bits(caches[n])
        new_scales = scales[n].double().cpu()
        for b in range(blocks):
            if b not in touched:
                assert torch.equal(got_bits[b], old_bits[b])
                assert torch.equal(new_scales[b], old_scales[b])
                continue
            rows = sorted(touched[b])
            first = rows[0][0]
            values = torch.stack([x[t] for _, t in rows])
            room = torch.stack([slack[t] for _, t in rows])
            held = old_scales[b] if first > 0 else torch.zeros(heads, dtype=torch.float64)
            want = torch.maximum(held, values.abs().amax((0, 2)) / 448)
            # amax to its slack, one rounding of the quotient.
            assert ((new_scales[b] - want).abs()
                    <= room.amax((0, 2)) / 448 + want * 2 * ref.U32).all()
            sc = new_scales[b][None, :, None]
            back = torch.stack([got[b, s].double() for s, _ in rows]) * sc
            assert ((back - values).abs() <= e4m3_bound(values, sc, room)).all()
            grown = (new_scales[b] > held)[None, :, None]
            kept = old[b, :first].double() * held[None, :, None]
            now = got[b, :first].double() * sc
            same = got_bits[b, :first] == old_bits[b, :first]
            assert (grown | same).all()
            assert ((now - kept).abs() <= e4m3_bound(kept, sc)).all()
            after = rows[-1][0] + 1
            assert torch.equal(got_bits[b, after:], old_bits[b, after:])
    mgr.close()


def test_e4m3_of_values_that_are_not_finite(kvx, cuda):
    gen = torch.Generator(device=cuda).manual_seed(9)
    mgr, caches, scales = build(kvx, cuda, gen, 4, 16, 1, 64, FP8)
    x = torch.randn(3, 1, 64, device=cuda, generator=gen).to(BF16)
    x[0, 0, 1], x[1, 0, 2], x[2, 0, 3] = float("nan"), float("inf"), float("-inf")
    x[0, 0, 0] = 56.0
    mgr.append_kv(0, 1, x, x, ints([[2]], cuda), ints([3], cuda), starts=ints([0, 3], cuda))
    for c, s in zip(caches, scales):
        assert float(s[2, 0]) == 0.125  # 56 / 448
        got = c[2, :3, 0].float()
        assert bool(torch.isnan(got[0, 1])) and int(torch.isnan(got).sum()) == 1
        assert float(got[1, 2]) == 448 and float(got[2, 3]) == -448 and float(got[0, 0]) == 448
    # Zeros only: a scale of zero, and no NaN from dividing by it.
    zero = torch.zeros(1, 1, 64, dtype=BF16, device=cuda)
    mgr.append_kv(0, 1, zero, zero, ints([[1]], cuda), ints([1], cuda))
    assert float(scales[0][1, 0]) == 0 and bool((caches[0][1, 0].float() == 0).all())
    # A scale that is not a number counts as none.
    scales[0][3, 0] = float("nan")
    mgr.append_kv(0, 1, x[:1].nan_to_num(0), x[:1].nan_to_num(0), ints([[3]], cuda),
                  ints([5], cuda))
    assert float(scales[0][3, 0]) == 0.125
    mgr.close()


def test_storages_behind_four_gib(kvx, cuda):
    """Block offsets pass 2^32 elements."""
    blocks, block, heads, dim = 262200, 16, 8, 128  # 4.3e9 elements a storage
    caches = [torch.empty(blocks, block, heads, dim, dtype=BF16, device=cuda) for _ in range(2)]
    mgr = kvx.KVCacheManager(caches, host_blocks_to_allocate=1)
    k = torch.randn(40, heads, dim, device=cuda).to(BF16)
    ids = [blocks - 1, 5, blocks - 3]
    for c in caches:
        c[torch.tensor(ids, device=cuda)] = 0
    mgr.append_kv(0, 1, k, -k, ints([ids], cuda), ints([40], cuda), starts=ints([0, 40], cuda))
    got = [torch.cat([c[i] for i in ids])[:40] for c in caches]
    assert torch.equal(got[0], k) and torch.equal(got[1], -k)
    q = torch.randn(1, 32, dim, device=cuda).to(BF16)
    out = mgr.attend(0, 1, q, ints([ids], cuda), ints([40], cuda))
    want, _, slack = ref.attend(q.cpu(), k.double().cpu(), -k.double().cpu(),
                                torch.ones(1, 40, dtype=torch.bool), dim ** -0.5, BF16, BF16)
    ref.assert_rounded(out, want, slack, BF16)
    mgr.close()

"""GPU: append_kv into and attend over a pool in 4 bits against the 64-bit form,
with every byte that no token has a place in left as it was, and every slot that
no query may see set to NaN."""
import pytest

torch = pytest.importorskip("torch")

import fp4_reference as fp4  # noqa: E402
import paged_reference as ref  # noqa: E402
from test_gpu_append_kv import freqs, ints, sequences_of, slots  # noqa: E402
from test_gpu_attend import Step  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def build(kvx, cuda, seed, blocks, block, heads, dim, layers=2):
    """A manager over random storages."""
    gen = torch.Generator().manual_seed(seed)
    shape = (blocks, heads, block, dim)
    pairs = [fp4.storage(torch.randn(shape, generator=gen), BF16, cuda) for _ in range(layers)]
    caches, scales = [list(x) for x in zip(*pairs)]
    mgr = kvx.KVCacheManager(caches, host_blocks_to_allocate=max(8, blocks // 2),
                             scale_tables=scales)
    return mgr, caches, scales


def check_rows(codes, scales, want, slack, dtype):
    """Stored rows [n, heads, ...] against values [n, heads, dim] that are off by
    `slack` before they are stored."""
    groups, room = want.unflatten(-1, (-1, 32)), slack.unflatten(-1, (-1, 32))
    # The scale: that of a largest value within the slack.
    largest = groups.abs().amax(-1)
    spare = room.amax(-1)
    code = scales.long()
    assert bool((code >= fp4.scale_code((largest - spare).clamp_min(0), dtype)).all())
    assert bool((code <= fp4.scale_code(largest + spare, dtype)).all())
    # The values: within half a step, which is exact, of what they may have been;
    # those that the scale's bound cuts are the largest code.
    s = fp4.scale_values(scales)[..., None]
    got = fp4.values(codes).unflatten(-1, (-1, 32)) * s
    most = 7 * s
    size = groups.abs().clamp_max(most.expand_as(groups))
    step = fp4.half_step((size + room) / s) * s
    off = (got.abs() - size).abs()
    assert bool((off <= step + room).all()), float((off - step - room).amax())
    assert bool((torch.sign(got) * torch.sign(groups) >= 0).logical_or(groups.abs() <= room).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("counts,lengths,block,heads,dim,rotary,norm,inter", [
    ([1, 1, 1], [1, 17, 40], 16, 8, 128, 128, False, False),
    ([5, 0, 33, 1], [5, 9, 60, 1], 16, 2, 128, 128, True, False),
    ([40], [47], 8, 1, 64, 64, True, False),
    ([3, 20], [3, 90], 7, 3, 96, 32, False, True),
    ([9, 1], [30, 64], 64, 2, 96, 0, True, False),
    ([2, 2], [6, 2], 1, 1, 32, 6, True, False),
    ([4], [4], 32, 2, 256, 256, True, True),
    ([6], [9], 5, 1, 160, 64, False, False),
    ([700, 800], [700, 1000], 16, 1, 64, 64, False, False)])
def test_append(kvx, cuda, dtype, counts, lengths, block, heads, dim, rotary, norm, inter):
    gen = torch.Generator(device=cuda).manual_seed(sum(counts) + dim)
    width = max((n + block - 1) // block for n in lengths) + 1
    blocks = width * len(counts) + 3
    mgr, caches, scales = build(kvx, cuda, dim, blocks, block, heads, dim)
    perm = torch.randperm(blocks, generator=torch.Generator().manual_seed(1)).tolist()
    tables = [perm[s * width:(s + 1) * width] for s in range(len(counts))]
    starts = sequences_of(counts)
    single = counts == [1] * len(counts)
    tokens = starts[-1] + (0 if single else 3)  # the last three belong to no sequence
    fused = torch.randn(tokens, 4 * heads, dim, device=cuda, generator=gen).to(dtype)
    # Exact quotients in the middle between two codes, zeros of both signs, groups of
    # zeros, and magnitudes far apart.
    fused[:, 3 * heads:, :32] = fused[:, 3 * heads:, :32].mul(4).round().div(4)
    fused[0, 3 * heads:, 1] = -0.0
    fused[:, 3 * heads, :32] *= torch.logspace(-4, 4, tokens, base=2, device=cuda).to(dtype)[:, None]
    fused[tokens // 2, 3 * heads:, :32] = 0
    k, v = fused[:, heads:2 * heads], fused[:, 3 * heads:]
    inv = freqs(rotary // 2, cuda) if rotary else None
    w = torch.randn(dim, device=cuda, generator=gen).to(dtype) if norm else None
    before = [fp4.raw(t) for t in caches + scales]
    # Odd addresses and strides take another path, with the same result.
    odd = torch.zeros(fused.numel() + 1, dtype=dtype, device=cuda)[1:].view(fused.shape)
    odd.copy_(fused)
    results = []
    for keys, vals in ((k, v), (odd[:, heads:2 * heads], odd[:, 3 * heads:])):
        for t, old in zip(caches + scales, before):
            t.view(torch.uint8).copy_(old)
        mgr.append_kv(0, 1, keys, vals, ints(tables, cuda), ints(lengths, cuda),
                      starts=None if single else ints(starts, cuda), inv_freq=inv, k_weight=w,
                      interleaved=inter)
        results.append([fp4.raw(t) for t in caches + scales])
    where = ref.places(starts, lengths, tokens, len(counts))
    place = slots(where, tables, block, blocks)
    assert len(place) == sum(counts)
    positions = torch.zeros(tokens, dtype=torch.int64)
    for t, _, p in where:
        positions[t] = p
    ids = list(place)
    b, s = torch.tensor([place[t] for t in ids]).t()
    if inv is None and w is None:
        want, slack = k.double().cpu(), torch.zeros(k.shape, dtype=torch.float64)
    else:
        want, slack = ref.norm_rope(k, w, positions, inv, 1e-6, inter)
    for now in results:
        check_rows(now[0][b, :, s], now[2][b, :, s], want[ids], slack[ids], dtype)
        codes, sizes = fp4.encode(v.cpu()[ids], dtype)
        assert torch.equal(now[1][b, :, s], codes) and torch.equal(now[3][b, :, s], sizes)
        for new, old in zip(now, before):
            new[b, :, s] = old[b, :, s]
            assert torch.equal(new, old)
    mgr.close()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_append_of_values_at_the_ends(kvx, cuda, dtype):
    """Infinities, NaN, the largest and the smallest values of the type, and every
    mantissa around the border between two scales."""
    mgr, caches, scales = build(kvx, cuda, 3, 40, 16, 2, 64)
    info, n = torch.finfo(dtype), 512
    x = torch.randn(n, 2, 64, generator=torch.Generator().manual_seed(9)).to(dtype)
    x[0, 0, 3], x[0, 1, 5] = float("inf"), -float("inf")
    x[1, 0, 40], x[1, 0, 41] = float("nan"), float("inf")
    x[2], x[3] = info.max, -info.max
    x[4], x[5], x[6] = info.tiny, info.smallest_normal / 4, 0
    x[7] = float("inf")
    x[8, :, :32] = 0
    x[8, 0, 7] = -float("inf")
    x[9, :, :32] = float("nan")
    for i in range(256):  # largest values around 7 x 2^e
        x[16 + i] = 0
        x[16 + i, :, i % 64] = (7.0 + (i - 128) / 32) * 2.0 ** (i % 8 - 4)
    tables, lengths = ints([list(range(32))], cuda), ints([n], cuda)
    mgr.append_kv(0, 1, x.to(cuda), x.to(cuda), tables, lengths, starts=ints([0, n], cuda))
    codes, sizes = fp4.encode(x, dtype)
    # Codes under a scale of NaN mean nothing.
    keep = (sizes != 255).repeat_interleave(16, -1)
    for t, s in zip(caches, scales):
        got = fp4.raw(t)[:32].transpose(1, 2).reshape(n, 2, 32)
        assert torch.equal(fp4.raw(s)[:32].transpose(1, 2).reshape(n, 2, 2), sizes)
        assert torch.equal(got[keep], codes[keep])
    assert int((sizes == 255).sum()) == 3
    back = fp4.decode(codes, sizes)
    assert bool(torch.isfinite(back.to(dtype))[sizes.repeat_interleave(32, -1) != 255].all())
    mgr.close()


def test_tokens_without_a_place_are_dropped(kvx, cuda):
    mgr, caches, scales = build(kvx, cuda, 4, 9, 16, 2, 64)
    k = torch.randn(8, 2, 64, device=cuda).to(BF16)
    before = [fp4.raw(c) for c in caches + scales]
    tables = ints([[-1, 3], [9, 3], [2**31 - 1, 3], [-2**31, 3], [0, 1], [0, 1], [0, 1], [0, 1]],
                  cuda)
    mgr.append_kv(0, 1, k, k, tables, ints([5, 16, 1, 7, 33, 0, -4, 2**31 - 1], cuda),
                  inv_freq=freqs(32, cuda))
    mgr.append_kv(0, 1, k, k, tables[:4], ints([2, 0, 0, 0], cuda),
                  starts=ints([8, 3, -5, 8, 2**31 - 1], cuda))
    torch.cuda.synchronize()
    assert all(torch.equal(fp4.raw(c), b) for c, b in zip(caches + scales, before))
    # Of four new tokens of a sequence of two the last two have a place.
    mgr.append_kv(0, 1, k[:4], k[:4], ints([[4]], cuda), ints([2], cuda),
                  starts=ints([0, 4], cuda))
    codes, _ = fp4.encode(k[2:4].cpu(), BF16)
    assert torch.equal(fp4.raw(caches[1])[4].transpose(0, 1)[:2], codes)
    mgr.close()


class Step4(Step):
    """A batch over a 4-bit pool."""

    def __init__(self, kvx, cuda, counts, lengths, q_heads, heads, dim, block, dtype, groups=(),
                 seed=0, spread=1.0):
        super().__init__(kvx, cuda, counts, lengths, q_heads, heads, dim, block, dtype, dtype,
                         groups, seed, spread)
        self.mgr.close()
        self.caches, self.scales = [list(x) for x in zip(*(
            fp4.storage(c.transpose(1, 2).float(), dtype, cuda) for c in self.caches))]
        # (Unused slots hold NaN, so their scales are that.)
        self.mgr = kvx.KVCacheManager(self.caches, host_blocks_to_allocate=1,
                                      scale_tables=self.scales)

    def check(self, out, lse=None, causal=True, scale=None):
        # The plain form takes gathered tokens: decode them all, in its layout.
        caches, scales = self.caches, self.scales
        self.caches = [fp4.decode(c, s).transpose(1, 2) for c, s in zip(caches, scales)]
        self.scales = [None, None]
        try:
            return super().check(out, lse, causal, scale)
        finally:
            self.caches, self.scales = caches, scales


ONE = [([1], 4, 1, 128, 16), ([7, 0, 129, 300], 8, 2, 128, 16), ([33] * 5, 8, 8, 64, 16),
       ([513, 15, 16, 17], 32, 8, 128, 16), ([100, 31], 20, 4, 96, 7), ([260], 16, 1, 96, 32),
       ([90, 4], 48, 1, 128, 8), ([140, 1], 6, 3, 256, 64), ([40], 5, 5, 32, 1),
       ([2500, 12], 64, 2, 128, 16), ([64, 200], 2, 2, 160, 48), ([0, 0], 4, 4, 64, 16),
       ([95, 33], 20, 1, 64, 5), ([77], 12, 2, 224, 16), ([70, 71], 17, 1, 256, 16)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lengths,hq,hk,dim,block", ONE)
def test_one_query_a_sequence(kvx, cuda, dtype, lengths, hq, hk, dim, block):
    step = Step4(kvx, cuda, [1] * len(lengths), lengths, hq, hk, dim, block, dtype)
    out, lse = step.run(return_lse=True)
    step.check(out, lse)
    assert torch.equal(step.run(), out)  # the same bytes again
    step.mgr.close()


MANY = [([5, 0, 1], [5, 9, 30], 8, 2, 128, 16), ([64], [64], 4, 4, 64, 16),
        ([130, 3, 1], [130, 400, 257], 8, 1, 128, 16), ([200], [777], 6, 2, 96, 8),
        ([33, 40], [33, 150], 16, 1, 32, 32), ([70], [70], 4, 2, 256, 16),
        ([9, 300], [4, 300], 4, 1, 128, 16), ([2, 2, 2], [64, 128, 1000], 32, 2, 128, 16),
        ([257], [1500], 10, 2, 64, 24), ([20], [1100], 40, 1, 160, 16)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("counts,lengths,hq,hk,dim,block", MANY)
def test_chunks(kvx, cuda, dtype, counts, lengths, hq, hk, dim, block):
    step = Step4(kvx, cuda, counts, lengths, hq, hk, dim, block, dtype)
    out, lse = step.run(return_lse=True)
    step.check(out, lse)
    step.check(step.run(causal=False), causal=False)
    step.mgr.close()


GROUPED = [([1] * 4, [70, 65, 99, 64], 8, 2, 128, 16, [(0, 4, 64)]),
           ([1] * 40, [700 + i for i in range(40)], 16, 2, 128, 16, [(0, 40, 640)]),
           ([1] * 6, [50, 200, 220, 90, 100, 33], 4, 4, 64, 16, [(1, 3, 192), (3, 5, 80)]),
           ([3, 1, 40], [150, 160, 190], 8, 2, 128, 16, [(0, 3, 128)]),
           ([2, 2], [96, 96], 6, 2, 96, 32, [(0, 2, 96)]),
           ([1] * 2, [64, 64], 4, 2, 256, 16, [(0, 2, 64)])]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("counts,lengths,hq,hk,dim,block,groups", GROUPED)
def test_shared_prefixes(kvx, cuda, dtype, counts, lengths, hq, hk, dim, block, groups):
    step = Step4(kvx, cuda, counts, lengths, hq, hk, dim, block, dtype, groups)
    out, lse = step.run(return_lse=True)
    step.check(out, lse)
    assert torch.equal(step.run(), out)
    step.mgr.close()


def test_scales_from_end_to_end(kvx, cuda):
    """Tokens whose scales are powers of two apart: bf16 takes all that are stored,
    fp16 those up to 2^13."""
    for dtype, spread in ((BF16, 40), (F16, 12)):
        for counts, lengths in (([1, 1], [90, 300]), ([70], [200])):
            step = Step4(kvx, cuda, counts, lengths, 8, 2, 64, 16, dtype)
            gen = torch.Generator().manual_seed(spread)
            for i, s in enumerate(step.scales):
                old = fp4.raw(s)
                new = 127 + torch.randint(-spread, 1 if i == 0 else spread + 1, old.shape,
                                          generator=gen)
                s.view(torch.uint8).copy_(torch.where(old == 255, 255, new).to(torch.uint8))
            if dtype == F16:
                # Results stay in the type's range.
                s.view(torch.uint8)[s.view(torch.uint8).ne(255)] -= 2
            step.check(step.run())
            step.mgr.close()


def test_large_scales_in_fp16_are_bounded(kvx, cuda):
    step = Step4(kvx, cuda, [1], [40], 4, 1, 64, 16, F16)
    v = step.scales[1].view(torch.uint8)
    v[v.ne(255)] = 150
    out = step.run()
    v[v.ne(255)] = 140
    assert torch.equal(step.run(), out) and bool(torch.isfinite(out).all())
    step.mgr.close()


def test_ids_outside_the_pool_and_lengths_past_the_table(kvx, cuda):
    for counts in ([1, 1], [40, 3]):
        step = Step4(kvx, cuda, counts, [100, 90], 8, 2, 64, 16, BF16)
        tables, lengths = step.args()
        n = counts[0]
        for bad in (-1, 10**6, -2**31):
            tables[0, 2] = bad
            out = step.mgr.attend(0, 1, step.q, tables, lengths, **step.kw())
            k, v = (fp4.gather(c, s, step.tables[0], 100)
                    for c, s in zip(step.caches, step.scales))
            visible = torch.arange(100)[None] <= torch.arange(100 - n, 100)[:, None]
            visible[:, 32:48] = False
            want, _, slack = ref.attend(step.q[:n].cpu(), k, v, visible, step.scale, BF16, BF16)
            ref.assert_rounded(out[:n], want, slack, BF16)
        tables[0] = -1
        out, lse = step.mgr.attend(0, 1, step.q, tables, lengths, return_lse=True, **step.kw())
        assert bool((out[:n] == 0).all()) and bool(torch.isneginf(lse[:n]).all())
        tables, _ = step.args()
        out = step.mgr.attend(0, 1, step.q, tables, ints([2**31 - 1, 90], cuda), **step.kw())
        assert bool(torch.isfinite(out[n:]).all())
        step.mgr.close()


def test_prefill_decode_offload_reload(kvx, cuda):
    """A served sequence's life in 4 bits: prefill in chunks, single tokens, its
    blocks and scales to the host tier and back into other ones, and on."""
    gen = torch.Generator(device=cuda).manual_seed(8)
    Hq, Hk, D, B = 8, 2, 128, 16
    mgr, caches, scales = build(kvx, cuda, 5, 40, B, Hk, D, layers=4)
    inv = freqs(64, cuda)
    ids = [31, 4, 17, 9, 22, 0, 38, 12]
    length = 0
    for turn, n in enumerate([50, 1, 20, 1, 1]):
        if turn == 3:  # the sequence leaves the pool and comes back elsewhere
            stream = torch.cuda.current_stream()
            mgr.d2h(ids, list(range(8)), stream=stream).Await()
            for c in caches + scales:
                c.view(torch.uint8).zero_()
            ids = [1, 2, 3, 5, 6, 7, 8, 10]
            mgr.h2d(list(range(8)), ids, stream=stream).wait_on_stream()
        length += n
        qkv = torch.randn(n, Hq + 2 * Hk, D, device=cuda, generator=gen).to(BF16)
        pos = torch.arange(length - n, length, device=cuda)
        tables, lengths, starts = ints([ids], cuda), ints([length], cuda), ints([0, n], cuda)
        for layer in (0, 2):
            q, _ = kvx.norm_rope(qkv[:, :Hq], None, pos, inv)
            mgr.append_kv(layer, layer + 1, qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:], tables, lengths,
                          starts=starts, inv_freq=inv)
            out = mgr.attend(layer, layer + 1, q, tables, lengths, starts=starts)
            k, v = (fp4.gather(caches[i], scales[i], ids, length) for i in (layer, layer + 1))
            visible = torch.arange(length)[None] <= torch.arange(length - n, length)[:, None]
            want, _, slack = ref.attend(q.cpu(), k, v, visible, D ** -0.5, BF16, BF16)
            ref.assert_rounded(out, want, slack, BF16)
    mgr.close()

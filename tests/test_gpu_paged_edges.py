"""GPU: calls on the paged pool that other tests do not make: the same call on its
own result, starts that are out of order, interleaved heads, inputs that are
differentiated, tables without a column, queries that see nothing beside values
that are not finite, rows of nothing but infinities, thousands of sequences around
64 KiB of LDS, one token far above thousands."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_attend import BF16, F16, FP8, ints  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("counts,block,dim", [([1, 1], 16, 64), ([7, 30], 16, 128),
                                              ([300, 9], 256, 128), ([5, 4], 8, 80)])
def test_append_again_stores_the_same_codes(kvx, cuda, dtype, counts, block, dim):
    """An e4m3 block that holds earlier tokens: the new ones come from the largest
    value's exact quotient, by the call that raises the scale and by the same call
    (a replay, a step that is taken back) after it. The largest value is 31 / 4 and
    the others 93 / 2^n, so 448 x / largest = 21 x 2^(8 - n) is the middle between
    two codes; by the scale, 31 / 1792 rounded down in its last bit, the quotient
    is the next number above it."""
    gen = torch.Generator(device=cuda).manual_seed(dim)
    before = 3  # tokens of each sequence's first block, not of these calls
    blocks = sum((before + n + block - 1) // block for n in counts)
    caches = [torch.ones(blocks, block, 2, dim, device=cuda).to(FP8) for _ in range(2)]
    scales = [torch.full((blocks, 2), 1 / 1024, device=cuda) for _ in range(2)]
    mgr = kvx.KVCacheManager(caches, host_blocks_to_allocate=1, scale_tables=scales)
    tokens, table, starts, at = sum(counts), [], [0], 0
    width = max((before + n + block - 1) // block for n in counts)
    for n in counts:
        need = (before + n + block - 1) // block
        table.append(list(range(at, at + need)) + [-1] * (width - need))
        at += need
        starts.append(starts[-1] + n)
    n = torch.randint(4, 13, (tokens, 2, dim), device=cuda, generator=gen)
    x = 93 * torch.pow(2.0, -n) * (1 - 2 * (n % 2))
    x[:, :, 0] = 31 / 4
    k, v = x.to(dtype), (-x).to(dtype)
    assert torch.equal(k.float(), x)
    args = (ints(table, cuda), ints([before + n for n in counts], cuda))
    held = []
    for _ in range(3):
        mgr.append_kv(0, 1, k, v, *args, starts=ints(starts, cuda))
        held.append([c.view(torch.uint8).clone() for c in caches] + [s.clone() for s in scales])
    for again in held[1:]:
        assert all(torch.equal(a, b) for a, b in zip(held[0], again))
    want = (x.double() * 1792 / 31).to(FP8).view(torch.uint8)
    for s, count in enumerate(counts):
        rows = [caches[0][table[s][p // block], p % block]
                for p in range(before, before + count)]
        assert torch.equal(torch.stack(rows).view(torch.uint8), want[starts[s]:starts[s + 1]])
    mgr.close()


def test_append_to_e4m3_with_starts_out_of_order(kvx, cuda):
    """Starts that give each of 2048 sequences the same 2099200 tokens, a block each,
    over 2^32 blocks in all: each block is written once, by the first sequence."""
    tokens, sequences = 2**21 + 2048, 4096
    caches = [torch.zeros(tokens, 1, 1, 8, device=cuda).to(FP8) for _ in range(2)]
    scales = [torch.zeros(tokens, 1, device=cuda) for _ in range(2)]
    mgr = kvx.KVCacheManager(caches, host_blocks_to_allocate=1, scale_tables=scales)
    gen = torch.Generator(device=cuda).manual_seed(1)
    k = torch.randn(tokens, 1, 8, device=cuda, generator=gen).to(BF16)
    ids = torch.randperm(tokens, device=cuda, generator=gen).to(torch.int32)
    back = torch.tensor([0, tokens] * (sequences // 2) + [0], dtype=torch.int32, device=cuda)
    held = []
    for n, starts in ((sequences, back), (1, ints([0, tokens], cuda))):
        for t in caches + scales:
            t.view(torch.uint8).zero_()
        mgr.append_kv(0, 1, k, -k, ids[None].expand(n, tokens),
                      torch.full((n,), tokens, dtype=torch.int32, device=cuda), starts=starts)
        held.append([t.view(torch.uint8).clone() for t in caches + scales])
    assert all(torch.equal(a, b) for a, b in zip(*held))
    assert bool((scales[0] > 0).all())
    mgr.close()


@pytest.mark.parametrize("dim", [64, 80, 5])
def test_norm_rope_in_place_of_interleaved_heads(kvx, cuda, dim):
    """A projection that lies as [tokens, heads, (q, k, v), head_dim]."""
    gen = torch.Generator(device=cuda).manual_seed(dim)
    qkv = torch.randn(33, 6, 3, dim, device=cuda, generator=gen).to(BF16)
    held, pos = qkv.clone(), torch.arange(33, device=cuda) * 100
    inv = torch.rand(dim // 2, device=cuda, generator=gen)
    w = torch.rand(dim, device=cuda, generator=gen).to(BF16)
    q, k = qkv[:, :, 0], qkv[:, :, 1]
    want = kvx.norm_rope(q, k, pos, inv, q_weight=w, k_weight=w)
    kvx.norm_rope(q, k, pos, inv, q_weight=w, k_weight=w, out_q=q, out_k=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(qkv[:, :, 2], held[:, :, 2])


def test_inputs_that_are_differentiated_are_refused(kvx, cuda):
    from torch.autograd import forward_ad
    caches = [torch.zeros(4, 16, 2, 64, device=cuda).to(BF16) for _ in range(2)]
    mgr = kvx.KVCacheManager(caches, host_blocks_to_allocate=1)
    pos, args = ints([0, 1, 2], cuda), (ints([[0, 1, 2, 3]], cuda), ints([3], cuda))
    good = dict(x=torch.ones(3, 2, 64, device=cuda).to(BF16), inv=torch.ones(32, device=cuda),
                w=torch.ones(64, device=cuda))

    def calls(x, inv, w):
        kw = dict(starts=ints([0, 3], cuda))
        yield lambda: kvx.norm_rope(x, None, pos, inv, q_weight=w)
        yield lambda: mgr.append_kv(0, 1, x, x, *args, inv_freq=inv, k_weight=w, **kw)
        if inv is good["inv"] and w is good["w"]:
            yield lambda: mgr.attend(0, 1, x, *args, **kw)

    for call in calls(**good):
        call()
    for name, t in good.items():
        leaf = t.clone().requires_grad_()
        for call in calls(**{**good, name: leaf}):
            with pytest.raises(ValueError, match="requires gradients"):
                call()
            with torch.no_grad():
                call()
        with forward_ad.dual_level():
            for call in calls(**{**good, name: forward_ad.make_dual(t, torch.ones_like(t))}):
                with pytest.raises(ValueError, match="has a tangent"):
                    call()
            for call in calls(**good):
                call()
    mgr.close()


@pytest.mark.parametrize("cache", [BF16, FP8])
@pytest.mark.parametrize("counts", [[1, 1, 1], [3, 0, 40], [200]])
def test_tables_without_a_column(kvx, cuda, cache, counts):
    """No token has a place: nothing is stored, and every query sees nothing."""
    caches = [torch.full((4, 16, 2, 64), 7.0, device=cuda).to(cache) for _ in range(2)]
    kw = {}
    if cache == FP8:
        kw = dict(scale_tables=[torch.ones(4, 2, device=cuda) for _ in range(2)])
    mgr = kvx.KVCacheManager(caches, host_blocks_to_allocate=1, **kw)
    n, tokens = len(counts), sum(counts)
    starts = ints([sum(counts[:i]) for i in range(n + 1)], cuda)
    args = (torch.empty((n, 0), dtype=torch.int32, device=cuda), ints(counts, cuda))
    k = torch.ones(tokens, 2, 64, device=cuda).to(BF16)
    mgr.append_kv(0, 1, k, k, *args, starts=starts)
    assert all(bool((c.float() == 7).all()) for c in caches)
    out, lse = mgr.attend(0, 1, torch.ones(tokens, 8, 64, device=cuda).to(BF16), *args,
                          starts=starts, return_lse=True)
    assert bool((out == 0).all()) and bool(torch.isneginf(lse).all())
    mgr.close()


@pytest.mark.parametrize("cache", [BF16, FP8])
@pytest.mark.parametrize("counts,lengths,prefix", [
    ([1, 1, 1], [90, 0, 70], 64),  # padded with an empty sequence, within a group
    ([1] * 40, [5000] + [0] * 38 + [4992], 4992),  # cut into many parts
    ([2, 3, 2], [66, 0, 65], 64),
    ([4], [2], 0),  # the first two of a chunk are before its sequence
    ([40], [3], 0), ([50, 300], [20, 200], 0)])
def test_queries_that_see_nothing_beside_infinities(kvx, cuda, cache, counts, lengths, prefix):
    """Zeros and an lse of -inf, whatever values are masked."""
    gen = torch.Generator(device=cuda).manual_seed(1)
    blocks = [(n + 15) // 16 for n in lengths]
    width = max(blocks)
    caches = [torch.randn(sum(blocks) + 1, 16, 2, 64, device=cuda, generator=gen) for _ in range(2)]
    caches[1][:, 1] = float("nan") if cache == FP8 else float("inf")
    kw = {}
    if cache == FP8:
        kw = dict(scale_tables=[torch.ones(sum(blocks) + 1, 2, device=cuda) for _ in range(2)])
    mgr = kvx.KVCacheManager([c.to(cache) for c in caches], host_blocks_to_allocate=1, **kw)
    tables, at = [], 0
    for n in blocks:
        tables.append(list(range(at, at + n)) + [-1] * (width - n))
        at += n
    call = dict(starts=ints([sum(counts[:i]) for i in range(len(counts) + 1)], cuda))
    if prefix:
        for t, n in zip(tables[1:], lengths[1:]):
            if n:
                t[:prefix // 16] = tables[0][:prefix // 16]
        call.update(group_starts=ints([0, len(counts)], cuda),
                    prefix_lengths=ints([prefix], cuda))
    q = torch.randn(sum(counts), 8, 64, device=cuda, generator=gen).to(BF16)
    out, lse = mgr.attend(0, 1, q, ints(tables, cuda), ints(lengths, cuda), return_lse=True, **call)
    first = 0
    for count, n in zip(counts, lengths):
        none = slice(first, first + max(count - n, 0))
        assert bool((out[none] == 0).all()) and bool(torch.isneginf(lse[none]).all())
        seen = slice(none.stop, first + count)
        assert bool(torch.isfinite(lse[seen]).all())
        first += count
    mgr.close()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("count,dim", [(1, 64), (16, 128), (40, 80), (3, 5)])
def test_append_of_infinities_alone(kvx, cuda, dtype, count, dim):
    """No finite value but 0 gives a scale of 0 and infinities are clamped to 448
    scales: their codes are +-448, which stand for 0, and not NaN."""
    block, blocks = 16, (count + 15) // 16
    caches = [torch.ones(blocks, block, 2, dim, device=cuda).to(FP8) for _ in range(2)]
    scales = [torch.ones(blocks, 2, device=cuda) for _ in range(2)]
    mgr = kvx.KVCacheManager(caches, host_blocks_to_allocate=1, scale_tables=scales)
    x = torch.zeros(count, 2, dim, device=cuda)
    x[:, 0, 1], x[:, 0, 3], x[:, 1, 2] = float("inf"), float("-inf"), float("nan")
    mgr.append_kv(0, 1, x.to(dtype), (-x).to(dtype), ints([list(range(blocks))], cuda),
                  ints([count], cuda), starts=ints([0, count], cuda))
    for cache, table, sign in zip(caches, scales, (1, -1)):
        assert bool((table == 0).all())
        got = cache.reshape(-1, 2, dim)[:count].float()
        want = (x * sign).clamp(-448, 448)
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(0), want.nan_to_num(0))
    mgr.close()


@pytest.mark.parametrize("sequences", [2130, 2250, 2340])
def test_sequences_whose_plan_and_arrays_pass_64_kib(kvx, cuda, sequences):
    """28 bytes a sequence are under 64 KiB of LDS, with the joining kernel's own
    6 KiB over it."""
    gen = torch.Generator(device=cuda).manual_seed(1)
    caches = [torch.randn(40, 16, 1, 64, device=cuda, generator=gen).to(BF16) for _ in range(2)]
    mgr = kvx.KVCacheManager(caches, host_blocks_to_allocate=1)
    tables = torch.randint(0, 40, (sequences, 8), device=cuda, dtype=torch.int32, generator=gen)
    lengths = torch.randint(1, 129, (sequences,), device=cuda, dtype=torch.int32, generator=gen)
    q = torch.randn(sequences, 2, 64, device=cuda, generator=gen).to(BF16)
    out = mgr.attend(0, 1, q, tables, lengths)
    for s in range(0, sequences, 97):
        one = mgr.attend(0, 1, q[s:s + 1], tables[s:s + 1], lengths[s:s + 1])
        # Two roundings of the same sums, which parts of other sizes add up.
        assert bool(((out[s] - one[0]).float().abs() <= 2.0**-6 * one[0].float().abs() + 0.01).all())
    mgr.close()


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, F16), (BF16, FP8), (F16, FP8)])
@pytest.mark.parametrize("count,sequences", [(1, 1100), (40, 600)])
@pytest.mark.parametrize("drop", [8.0, 12.0, 14.0])
def test_many_tokens_far_below_the_largest(kvx, cuda, dtype, cache, count, sequences, drop):
    """One token's score is `drop` above those of 16383 others, whose exponentials
    are then 2^-11 to 2^-20 of its own (below fp16's normal numbers) and add up to 5
    to 1 % of it. They have the values 1, it has 0: the result is their share.
    So many sequences over the same blocks that one worker goes through each."""
    n, dim, block = 16384, 64, 64
    code = 16 if cache == FP8 else 1  # the value 1 at a scale of 1 / code
    k, v = torch.zeros(n, dim, device=cuda), torch.full((n, dim), float(code), device=cuda)
    k[0, 0], v[0] = drop * code, 0.0
    pool = [x.reshape(n // block, block, 1, dim).to(cache) for x in (k, v)]
    assert all(torch.equal(x.float().reshape(n, dim), y) for x, y in zip(pool, (k, v)))
    kw = {}
    if cache == FP8:
        kw = dict(scale_tables=[torch.full((n // block, 1), 1 / code, device=cuda)
                                for _ in range(2)])
    mgr = kvx.KVCacheManager(pool, host_blocks_to_allocate=1, **kw)
    q = torch.zeros(count * sequences, 1, dim, device=cuda)
    q[:, 0, 0] = 1.0
    table = torch.arange(n // block, dtype=torch.int32, device=cuda)
    out = mgr.attend(0, 1, q.to(dtype), table[None].expand(sequences, -1),
                     torch.full((sequences,), n, dtype=torch.int32, device=cuda), scale=1.0,
                     starts=torch.arange(sequences + 1, dtype=torch.int32, device=cuda) * count)
    others = torch.arange(n - count, n, device=cuda).double()[None, :, None, None]
    size = torch.exp(torch.tensor(-drop, dtype=torch.float64)).item()
    want = others * size / (1 + others * size)
    # Each exponential is off by half a step of its type, in fp16 by up to 2^-25 of
    # the largest; in fp32 its exponent by 64 half steps and its sums by n. The
    # result has half a step of its own.
    half = torch.finfo(dtype).eps / 2
    low = others * 2.0**-25 if dtype == F16 else 0.0
    room = want * (2 * half + (n + 128) * 2.0**-24) + low
    off = (out.double().reshape(sequences, count, 1, dim) - want).abs()
    assert bool((off <= room).all()), f"{float((off / want).max())} off"
    mgr.close()

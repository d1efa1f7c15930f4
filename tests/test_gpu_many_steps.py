"""GPU: weigh, and attend over a 4-bit pool, where every worker has several steps,
heads, sequences or tiles in turn and tiles are cut and joined, against the 64-bit
form on the same device. A grid is never larger than what the GPU holds at once, so
work of three times that many units gives some worker three of them or more,
whatever a call's grid is."""
import pytest

torch = pytest.importorskip("torch")

import fp4_reference as fp4  # noqa: E402
import paged_reference as ref  # noqa: E402
from test_gpu_append_kv import ints  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
MOST_GROUPS = 256 * 8  # workgroups of 256 threads that 256 CUs hold
MOST_WAVES = MOST_GROUPS * 4
NAN = float("nan")


class Pool:
    """A batch of sequences over a pool of any kind, with NaN in the slots behind them."""

    def __init__(self, kvx, cuda, counts, lengths, hq, hk, dim, block, dtype, cache, seed=0):
        gen = torch.Generator(device=cuda).manual_seed(seed + dim)
        self.counts, self.lengths, self.scale, self.dtype = counts, lengths, dim ** -0.5, dtype
        self.cache, self.product = cache, BF16 if cache == FP8 else dtype
        self.starts = [0] + torch.tensor(counts).cumsum(0).tolist()
        need = [(n + block - 1) // block for n in lengths]
        blocks, width = sum(need) + 3, max(need)
        ids = torch.randperm(blocks, device=cuda, generator=gen).int()
        self.tables = torch.full((len(counts), width), -1, dtype=torch.int32, device=cuda)
        used, at = torch.zeros(blocks, block, dtype=torch.bool, device=cuda), 0
        for s, n in enumerate(need):
            mine = ids[at:at + n]
            self.tables[s, :n] = mine
            used[mine.long()] = (torch.arange(n * block, device=cuda) < lengths[s]).view(n, block)
            at += n
        self.storages, self.scales = [], []
        for _ in range(2):
            if cache == "fp4":
                codes = torch.randint(0, 256, (blocks, hk, block, dim // 2), device=cuda,
                                      generator=gen, dtype=torch.uint8)
                sizes = torch.randint(124, 127, (blocks, hk, block, dim // 32), device=cuda,
                                      generator=gen, dtype=torch.uint8)
                sizes[~used[:, None].expand(-1, hk, -1)] = 255
                self.storages.append(codes.view(fp4.FP4))
                self.scales.append(sizes.view(fp4.E8M0))
                continue
            x = torch.randn(blocks, block, hk, dim, device=cuda, generator=gen)
            if cache == FP8:
                self.scales.append(torch.rand(blocks, hk, device=cuda, generator=gen) * 0.02 + 0.005)
                x = x * 60
            x[~used] = NAN
            self.storages.append(x.to(cache))
        self.mgr = kvx.KVCacheManager(self.storages, host_blocks_to_allocate=1,
                                      scale_tables=self.scales)
        self.q = torch.randn(self.starts[-1], hq, dim, device=cuda, generator=gen).to(dtype)
        self.held = ints(lengths, cuda)
        self.kw = {} if counts == [1] * len(counts) else dict(starts=ints(self.starts, cuda))

    def tokens(self, which, s):
        """A sequence's keys or values, [length, heads, dim] in 64 bits."""
        block = self.storages[0].shape[2 if self.cache == "fp4" else 1]
        ids = self.tables[s, :(self.lengths[s] + block - 1) // block].long()
        if self.cache == "fp4":
            b = self.storages[which].view(torch.uint8)[ids].long()
            e = self.scales[which].view(torch.uint8)[ids].double()
            x = fp4.CODES.to(b.device)[torch.stack((b & 15, b >> 4), -1).flatten(-2)]
            x = x * torch.where(e == 255, NAN, 2.0 ** (e - 127)).repeat_interleave(32, -1)
            x = x.transpose(1, 2)
        else:
            x = self.storages[which][ids].double()
            if self.scales:
                x = x * self.scales[which][ids].double()[:, None, :, None]
        return x.flatten(0, 1)[:self.lengths[s]]

    def visible(self, s, causal=True):
        n, length = self.counts[s], self.lengths[s]
        j = torch.arange(length, device=self.q.device)
        last = j[length - n:] if causal else torch.full((n,), length, device=self.q.device)
        return j[None] <= last[:, None]

    def rows(self, s):
        return slice(self.starts[s], self.starts[s + 1])


def check_weights(pool, before, after, lse, begins, decay, causal=True):
    """As in test_gpu_eviction: of an exponential, the score is off by 2 (D + 8) half
    steps of sum |q k| scale, the log by 4 of its size, both also by being moved into
    powers of two, and the exponential by 32; its sum by one a row and 16, the decayed
    part by 2."""
    hk, block = before.shape[1:]
    group, dim = pool.q.shape[1] // hk, pool.q.shape[2]
    want, room = before.double(), torch.zeros(before.shape, dtype=torch.float64,
                                              device=before.device)
    for s, n in enumerate(pool.counts):
        length, begin = pool.lengths[s], begins[s] if begins else 0
        if n == 0 or begin >= length:
            continue
        k, visible = pool.tokens(0, s), pool.visible(s, causal)
        q, of = pool.q[pool.rows(s)].double(), lse[pool.rows(s)].double()
        j = torch.arange(length, device=before.device)
        block_of, slot = pool.tables[s].long()[j // block][begin:], (j % block)[begin:]
        for h in range(hk):
            got = torch.zeros(length, dtype=torch.float64, device=before.device)
            slack, keys = got.clone(), k[:, h].t().contiguous()
            for g in range(h * group, h * group + group):
                p = (q[:, g].contiguous() @ keys * pool.scale - of[:, g:g + 1]).exp()
                p = torch.where(visible, p, 0.0)
                size = q[:, g].abs().contiguous() @ keys.abs() * pool.scale
                rel = 2 * (dim + 8) * size + 4 * of[:, g:g + 1].abs() + 128
                got += p.sum(0)
                slack += (p * rel).sum(0)
            slack += got * (n * group + 16)
            old = torch.zeros_like(got)
            old[begin:] = before.double()[block_of, h, slot]
            old = torch.where(j < length - n, old * decay, 0.0)
            want[block_of, h, slot] = (got + old)[begin:]
            room[block_of, h, slot] = ((slack + 4 * (got + old)) * ref.U32)[begin:]
    off = (after.double() - want).abs()
    assert bool((off <= room).all()), float((off / room.clamp_min(1e-300)).max())


def log_sums(pool, causal=True):
    """lse of the 64-bit form, rounded."""
    out = torch.empty(pool.q.shape[:2], dtype=torch.float64, device=pool.q.device)
    group = pool.q.shape[1] // pool.storages[0].shape[1 if pool.cache == "fp4" else 2]
    for s in range(len(pool.counts)):
        k, visible = pool.tokens(0, s), pool.visible(s, causal)
        for g in range(pool.q.shape[1]):
            score = (pool.q[pool.rows(s), g].double().contiguous()
                     @ k[:, g // group].t().contiguous() * pool.scale)
            out[pool.rows(s), g] = score.masked_fill(~visible, -float("inf")).logsumexp(-1)
    return out.float()


def weigh_and_check(kvx, pool, lse, begins, decay, causal=True):
    blocks, hk = pool.storages[0].shape[0], pool.storages[0].shape[1 if pool.cache == "fp4" else 2]
    block = pool.storages[0].shape[2 if pool.cache == "fp4" else 1]
    before = torch.rand(blocks, hk, block, device=pool.q.device)
    tables = []
    for _ in range(2):
        after = before.clone()
        pool.mgr.weigh(0, pool.q, pool.tables, pool.held, lse, after, decay=decay, causal=causal,
                       begins=ints(begins, pool.q.device) if begins else None, **pool.kw)
        tables.append(after)
    assert torch.equal(*tables)  # the same bytes again
    check_weights(pool, before, tables[0], lse, begins, decay, causal)


def few_steps(lengths, begins=None):
    """Steps of 32 tokens of one head."""
    return sum((n - b + 31) // 32 for n, b in zip(lengths, begins or [0] * len(lengths)))


def lengths_of(n, longest, seed):
    """Mixed lengths, the borders of steps and blocks among them."""
    gen = torch.Generator().manual_seed(seed)
    return [1, 31, 32, 33, 65] + torch.randint(2, longest, (n - 5,), generator=gen).tolist()


FEW = [  # (sequences, longest, q heads, heads, dim, block)
    (64, 8000, 32, 8, 128, 16), (48, 9000, 40, 8, 96, 7), (40, 7000, 12, 12, 64, 32),
    (44, 8000, 48, 8, 256, 16), (64, 8000, 136, 8, 64, 16), (40, 9000, 20, 10, 160, 48)]


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, F16), (BF16, FP8), (F16, FP8),
                                         (BF16, "fp4"), (F16, "fp4")])
@pytest.mark.parametrize("sequences,longest,hq,hk,dim,block", FEW)
def test_single_tokens(kvx, cuda, dtype, cache, sequences, longest, hq, hk, dim, block):
    lengths = lengths_of(sequences, longest, dim)
    begins = [n // 5 for n in lengths]
    assert few_steps(lengths, begins) * hk >= 3 * MOST_WAVES
    pool = Pool(kvx, cuda, [1] * sequences, lengths, hq, hk, dim, block, dtype, cache)
    out, lse = pool.mgr.attend(0, 1, pool.q, pool.tables, pool.held, return_lse=True)
    if cache == "fp4":
        for s, n in enumerate(lengths):
            k, v = pool.tokens(0, s), pool.tokens(1, s)
            want, want_lse, slack = ref.attend(pool.q[s:s + 1], k, v, pool.visible(s), pool.scale,
                                               dtype, pool.product)
            ref.assert_rounded(out[s:s + 1], want, slack, dtype)
            size = pool.q[s].double().abs().amax() * k.abs().sum(-1).amax()
            room = (dim * float(size) * pool.scale + n + 128) * ref.U32
            assert bool(((lse[s].double().cpu() - want_lse[0]).abs() <= room).all())
        again = pool.mgr.attend(0, 1, pool.q, pool.tables, pool.held)
        assert torch.equal(again, out)
    weigh_and_check(kvx, pool, lse, None, 1.0)
    weigh_and_check(kvx, pool, lse, begins, 0.5)
    pool.mgr.close()


def many_stages(counts, lengths, group, dim, causal, begins=None):
    """Stages of 64 rows over all tiles of one head."""
    tile, all_stages = 256 if dim <= 128 else 128, []
    for s, (n, length) in enumerate(zip(counts, lengths)):
        if n * group <= 32:
            continue
        for first in range(begins[s] if begins else 0, length, tile):
            hidden = max(first - (length - n), 0) * group // 64 if causal else 0
            all_stages.append((n * group + 63) // 64 - hidden)
    return all_stages


MANY = [  # (new tokens, lengths, q heads, heads, dim, block): parts of a tile
    ([1000, 700, 351], [7700, 2500, 4000], 24, 8, 128, 16),
    ([1000, 700, 351], [7700, 2500, 4000], 20, 4, 64, 16),
    ([600, 401], [3700, 2900], 80, 2, 128, 16), ([300, 201], [3000, 2500], 160, 2, 96, 7),
    ([1900, 2, 151], [1900, 2500, 6000], 32, 8, 256, 32),
    # whole tiles, several of them a workgroup, beside sequences with few rows
    ([15, 33, 9, 1, 60] * 8, [8000, 7000, 5000, 6000, 2001] * 8, 32, 8, 128, 16),
    ([15, 33, 9, 3, 60] * 10, [8000, 7000, 5000, 6000, 2001] * 10, 20, 4, 64, 24)]


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, FP8), (BF16, "fp4")])
@pytest.mark.parametrize("counts,lengths,hq,hk,dim,block", MANY)
def test_chunks(kvx, cuda, dtype, cache, counts, lengths, hq, hk, dim, block):
    pool = Pool(kvx, cuda, counts, lengths, hq, hk, dim, block, dtype, cache)
    begins = [length // 7 for length in lengths]
    for causal, begin, decay in ((True, None, 1.0), (True, begins, 0.5), (False, None, 0.0)):
        stages = many_stages(counts, lengths, hq // hk, dim, causal, begin)
        assert sum(stages) * hk >= 3 * MOST_GROUPS
        weigh_and_check(kvx, pool, log_sums(pool, causal), begin, decay, causal)
    pool.mgr.close()


def test_single_tokens_do_not_depend_on_the_batch(kvx, cuda):
    """A single token's weights are the same bytes beside other sequences."""
    lengths = lengths_of(64, 8000, 1)
    pool = Pool(kvx, cuda, [1] * 64, lengths, 32, 8, 128, 16, BF16, BF16)
    _, lse = pool.mgr.attend(0, 1, pool.q, pool.tables, pool.held, return_lse=True)
    before = torch.rand(pool.storages[0].shape[0], 8, 16, device=cuda)
    together, alone = before.clone(), before.clone()
    pool.mgr.weigh(0, pool.q, pool.tables, pool.held, lse, together)
    for s in range(64):
        one = slice(s, s + 1)
        pool.mgr.weigh(0, pool.q[one], pool.tables[one], pool.held[one], lse[one], alone)
    assert torch.equal(together, alone)
    pool.mgr.close()

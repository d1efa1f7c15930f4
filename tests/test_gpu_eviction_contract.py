"""GPU: tables of weights over a sequence's life: beside its blocks on the host, and
over steps that are not weighed."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_append_kv import ints  # noqa: E402
from test_gpu_eviction import storages  # noqa: E402
from test_gpu_many_steps import Pool  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn
NAN = float("nan")


@pytest.mark.parametrize("cache", [BF16, FP8, "fp4"])
def test_weights_travel_with_their_blocks(kvx, cuda, cache):
    """A sequence that goes to the host and comes back into other blocks is cut as one
    that stayed."""
    Hq, Hk, D, B, n = 8, 2, 64, 16, 100
    results = []
    for moves in (False, True):
        gen = torch.Generator(device=cuda).manual_seed(6)
        caches, scales = storages(cuda, cache, 20, B, Hk, D, 5)
        weights = torch.rand(20, Hk, B, device=cuda, generator=gen)
        mgr = kvx.KVCacheManager(caches, host_blocks_to_allocate=8,
                                 scale_tables=scales + [weights])
        ids = [3, 17, 0, 9, 12, 5, 8]
        q = torch.randn(1, Hq, D, device=cuda, generator=gen).to(BF16)
        lengths = ints([n], cuda)
        _, lse = mgr.attend(0, 1, q, ints([ids], cuda), lengths, return_lse=True)
        mgr.weigh(0, q, ints([ids], cuda), lengths, lse, weights)
        if moves:
            stream, host = torch.cuda.current_stream(), list(range(len(ids)))
            mgr.d2h(ids, host, stream=stream).Await()
            for t in caches + scales + [weights]:
                t.view(torch.uint8).zero_()
            ids = [1, 2, 4, 6, 7, 10, 11]
            mgr.h2d(host, ids, stream=stream).wait_on_stream()
        cut = mgr.evict(0, 1, weights, ints([ids], cuda), lengths, 40, recent=5)
        kept = [t.view(torch.uint8)[ids[:3]].cpu() for t in caches + scales + [weights]]
        results.append([cut.cpu()] + kept)
        mgr.close()
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("cache", [BF16, FP8, "fp4"])
@pytest.mark.parametrize("counts", [[1, 1, 1], [40, 1, 70]])
def test_tokens_that_have_not_been_weighed_start_from_nothing(kvx, cuda, cache, counts):
    """The same as over a table whose entries of such tokens have been cleared."""
    pool = Pool(kvx, cuda, counts, [700, 45, 1100], 8, 2, 64, 16, BF16, cache)
    _, lse = pool.mgr.attend(0, 1, pool.q, pool.tables, pool.held, return_lse=True, **pool.kw)
    before = torch.rand(pool.storages[0].shape[0], 2, 16, device=cuda)

    def weigh(table, **kw):
        pool.mgr.weigh(0, pool.q, pool.tables, pool.held, lse, table, decay=0.5, **kw, **pool.kw)
        return table

    plain = weigh(before.clone())
    for weighed in ([650, 0, 3], [-5, 44, 1029], [2**31 - 1, -2**31, 1100], [0, 0, 0]):
        clear, stale = before.clone(), before.clone()
        for s, n in enumerate(pool.lengths):
            p = torch.arange(min(max(weighed[s], 0), n), n, device=cuda)
            at = pool.tables[s].long()[p // 16]
            clear[at, :, p % 16] = 0
            stale[at, :, p % 16] = NAN
        assert torch.equal(weigh(stale, weighed=ints(weighed, cuda)), weigh(clear))
    # More than there are: all but the call's own, as without the argument.
    assert torch.equal(weigh(before.clone(), weighed=ints([2**31 - 1] * 3, cuda)), plain)
    with pytest.raises(kvx.KvxError, match="weights: overlaps weighed"):
        table = before.clone()
        weigh(table, weighed=table.view(torch.int32).flatten()[8:11])
    pool.mgr.close()


def test_a_loop_that_weighs_every_third_step(kvx, cuda):
    """Slots that an eviction frees are filled again in steps that are not weighed; what
    the tokens get is what the weighed steps gave them."""
    gen = torch.Generator(device=cuda).manual_seed(1)
    S, Hq, Hk, D, B, W = 2, 8, 2, 64, 16, 8
    caches, _ = storages(cuda, BF16, S * W, B, Hk, D, 3)
    mgr = kvx.KVCacheManager(caches, host_blocks_to_allocate=1)
    tables = torch.randperm(S * W, generator=torch.Generator().manual_seed(4)).int().view(S, W)
    tables = tables.to(cuda)
    weights = torch.full((S * W, Hk, B), NAN, device=cuda)
    # What each place should hold, [sequences, heads, places], and how many places do.
    want = torch.zeros(S, Hk, W * B, device=cuda)
    length, weighed = 0, 0

    def held():
        return weights[tables.long()].transpose(1, 2).flatten(2)

    for step in range(24):
        n = 41 if step == 0 else 1
        length += n
        k, v = (torch.randn(S * n, Hk, D, device=cuda, generator=gen).to(BF16) for _ in range(2))
        q = torch.randn(S * n, Hq, D, device=cuda, generator=gen).to(BF16)
        lengths = ints([length] * S, cuda)
        kw = dict(starts=ints([n * s for s in range(S + 1)], cuda))
        mgr.append_kv(0, 1, k, v, tables, lengths, **kw)
        _, lse = mgr.attend(0, 1, q, tables, lengths, return_lse=True, **kw)
        if step % 3 == 1:
            alone = torch.zeros_like(weights)
            mgr.weigh(0, q, tables, lengths, lse, alone, decay=0.0, **kw)
            mgr.weigh(0, q, tables, lengths, lse, weights, weighed=ints([weighed] * S, cuda), **kw)
            weighed = length
            got = alone[tables.long()].transpose(1, 2).flatten(2)
            want[..., :length] += got[..., :length]
            assert torch.equal(held()[..., :length], want[..., :length])
        if step % 6 == 5:
            assert length - weighed < 10 and length > 30  # the others are among the recent
            kept, _ = kvx.choose_kept(weights, tables, lengths, 30, recent=10)
            mgr.evict(0, 1, weights, tables, lengths, 30, recent=10)
            weighed -= length - 30
            length = 30
            want[..., :weighed] = want.gather(2, kept.long())[..., :weighed]
            want[..., weighed:] = 0
    mgr.close()

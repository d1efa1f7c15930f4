"""GPU: tables of weights over a sequence's life: beside its blocks on the host, and
over steps that are not weighed."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_append_kv import ints  # noqa: E402
from test_gpu_eviction import storages  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn


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

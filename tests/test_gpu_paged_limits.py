"""GPU: the paged operators where their kernels change hands: axes cut into many
parts, the largest numbers of sequences and groups, calls at once from several
threads and streams, and e4m3 roundings that have to be exact."""
import threading

import pytest

torch = pytest.importorskip("torch")

import paged_reference as ref  # noqa: E402
from test_gpu_attend import BF16, F16, FP8, Step, ints  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, FP8)])
@pytest.mark.parametrize("counts,lengths,hq,hk,dim,block,groups", [
    ([1], [30011], 4, 1, 128, 16, ()),  # one head's tokens over every wave
    ([1, 1, 1], [9001, 3, 8000], 16, 2, 80, 24, ()),
    ([70], [9000], 4, 2, 128, 16, ()),  # few tiles, cut many times
    ([150, 2, 140], [4000, 4100, 150], 6, 2, 64, 8, ()),  # tiles and waves in one call
    ([40], [2600], 4, 1, 256, 32, ()),
    ([1, 1, 3, 1], [9000, 9100, 8800, 8801], 8, 2, 128, 16, ((0, 4, 8736),)),
    ([1] * 3, [5000, 5000, 700], 4, 1, 256, 16, ((0, 2, 4992),))])
def test_long_axes(kvx, cuda, dtype, cache, counts, lengths, hq, hk, dim, block, groups):
    step = Step(kvx, cuda, counts, lengths, hq, hk, dim, block, dtype, cache, groups)
    out, lse = step.run(return_lse=True)
    step.check(out, lse)
    assert torch.equal(step.run(), out)
    step.mgr.close()


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_ends_of_chunks_meet_ends_of_steps(kvx, cuda, dim):
    """Lengths and counts around 32, 64 and 128: the first and last halves."""
    counts = [33, 31, 64, 65, 32, 127, 129, 1]
    lengths = [33, 32, 64, 129, 95, 128, 191, 63]
    step = Step(kvx, cuda, counts, lengths, 4, 2, dim, 16, BF16, BF16)
    step.check(step.run())
    step.check(step.run(causal=False), causal=False)
    step.mgr.close()


def test_most_sequences_and_groups(kvx, cuda):
    lengths = [(11 * s) % 37 + 16 for s in range(4096)]
    step = Step(kvx, cuda, [1] * 4096, lengths, 2, 1, 256, 16, BF16, BF16)
    step.check(step.run())
    step.groups = tuple((16 * g, 16 * g + 16, 16) for g in range(256))
    for a, b, _ in step.groups:
        for s in range(a, b):
            step.tables[s][0] = step.tables[a][0]
    step.check(step.run())
    step.mgr.close()


def test_threads_and_streams_at_once(kvx, cuda):
    """Calls of several host threads, each on a stream of its own."""
    cases = [Step(kvx, cuda, [1] * 20, [300 + 9 * s for s in range(20)], 16, 2, 128, 16, BF16,
                  BF16),
             Step(kvx, cuda, [130, 5], [700, 90], 8, 2, 96, 16, F16, FP8),
             Step(kvx, cuda, [1] * 6, [800 + s for s in range(6)], 16, 2, 64, 16, BF16, BF16,
                  [(0, 6, 784)])]
    want = [c.run() for c in cases]
    streams = [torch.cuda.Stream(cuda) for _ in range(4)]
    torch.cuda.synchronize()
    wrong = []

    def calls(i):
        try:
            with torch.cuda.stream(streams[i]):
                outs = [(n, cases[n].run()) for r in range(6) for n in ((i + r) % 3, i % 3)]
            streams[i].synchronize()
            wrong.extend(n for n, out in outs if not torch.equal(out, want[n]))
        except Exception as e:  # noqa: BLE001 - reported by the assertion
            wrong.append(repr(e))

    threads = [threading.Thread(target=calls, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == []
    for c in cases:
        c.mgr.close()


def test_fp16_on_e4m3_rounds_once(kvx, cuda):
    """With fp16 queries an e4m3 value stays exact, whatever its scale: a product
    is off by the half step of its fp16 exponential and no more."""
    for counts, lengths in (([1, 1], [400, 33]), ([90], [300])):
        step = Step(kvx, cuda, counts, lengths, 8, 2, 128, 16, F16, FP8)
        step.product = F16
        step.scales[1].mul_(2.0 ** torch.randint(-4, 3, step.scales[1].shape, device=cuda))
        step.check(step.run())
        step.mgr.close()


@pytest.mark.parametrize("count", [1, 40])
@pytest.mark.parametrize("code,scale", [(2.0**-9, 2.0**-15), (448.0, 2.0**7), (1.125, 2.0**13),
                                        (2.0**-9, 2.0**13), (-13.0, 0.0)])
def test_fp16_on_e4m3_of_extreme_scales(kvx, cuda, count, code, scale):
    """A constant value comes out as it is, the smallest and largest included."""
    gen = torch.Generator(device=cuda).manual_seed(1)
    k = torch.randn(4, 16, 2, 64, device=cuda, generator=gen).to(FP8)
    v = torch.full((4, 16, 2, 64), code, device=cuda).to(FP8)
    tables = [torch.ones(4, 2, device=cuda), torch.full((4, 2), scale, device=cuda)]
    mgr = kvx.KVCacheManager([k, v], host_blocks_to_allocate=1, scale_tables=tables)
    q = torch.randn(count, 8, 64, device=cuda, generator=gen).to(F16)
    out = mgr.attend(0, 1, q, ints([[3, 0, 2, 1]], cuda), ints([64], cuda),
                     starts=ints([0, count], cuda))
    # 64 exponentials, each off by 2^-11 of itself, the result by 2^-11 and 2^-25.
    off = (out.double() - code * scale).abs()
    assert bool((off <= abs(code * scale) * 2.0**-10 * 1.01 + 2.0**-25).all())
    mgr.close()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("count,block,dim", [(1, 16, 128), (37, 16, 64), (300, 64, 128),
                                             (90, 32, 80), (130, 64, 256)])
def test_e4m3_codes_of_values_are_exact(kvx, cuda, dtype, count, block, dim):
    """Values have few bits, so 448 x / largest is often the very middle between
    two codes: every code is the one of the exact quotient, also there."""
    gen = torch.Generator(device=cuda).manual_seed(count)
    blocks = (count + block - 1) // block + 1
    caches = [torch.zeros(blocks, block, 2, dim, device=cuda).to(FP8) for _ in range(2)]
    scales = [torch.zeros(blocks, 2, device=cuda) for _ in range(2)]
    mgr = kvx.KVCacheManager(caches, host_blocks_to_allocate=1, scale_tables=scales)
    # Eighths up to 56 / 8: with a largest value of 7 the codes' middles are met.
    v = torch.randint(-56, 57, (count, 2, dim), device=cuda, generator=gen).div(8).to(dtype)
    ids = list(range(blocks))[::-1]
    mgr.append_kv(0, 1, v, v * 3, ints([ids], cuda), ints([count], cuda),
                  starts=ints([0, count], cuda))
    for cache, x in zip(caches, (v, v * 3)):
        for j in range(0, count, block):
            rows = x[j:j + block].double()
            largest = rows.abs().amax((0, 2))
            want = (rows * 448 / largest[None, :, None]).nan_to_num(0).to(FP8)
            got = cache[ids[j // block], :rows.shape[0]]
            assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))
    mgr.close()


def test_starts_and_groups_out_of_order(kvx, cuda):
    """Starts that give the same tokens to thousands of sequences, and groups that
    overlap: the work stays what the sizes allow, and nothing outside is touched."""
    T, S, width = 4096, 4096, 64
    caches = [torch.randn(70, 16, 1, 64, device=cuda).to(BF16) for _ in range(2)]
    mgr = kvx.KVCacheManager(caches, host_blocks_to_allocate=1)
    room = torch.full((T + 64, 8, 64), 5.0, device=cuda).to(BF16)
    q = torch.randn(T, 8, 64, device=cuda).to(BF16)
    tables = torch.randint(0, 70, (S, width), device=cuda, dtype=torch.int32)
    lengths = torch.full((S,), 2**31 - 1, device=cuda, dtype=torch.int32)
    back = torch.tensor([0, T] * (S // 2) + [0], device=cuda, dtype=torch.int32)
    groups = torch.tensor([0, S] * 128 + [0], device=cuda, dtype=torch.int32)
    prefixes = torch.full((256,), 2**31 - 1, device=cuda, dtype=torch.int32)
    one = torch.arange(S + 1, device=cuda, dtype=torch.int32)
    for starts, kw in ((back, {}), (one, dict(group_starts=groups, prefix_lengths=prefixes)),
                       (back, dict(group_starts=groups, prefix_lengths=prefixes))):
        mgr.attend(0, 1, q, tables, lengths, starts=starts, out=room[32:32 + T], **kw)
        torch.cuda.synchronize()
        assert bool((room[:32] == 5).all()) and bool((room[32 + T:] == 5).all())
    # A valid call after it, through the same manager.
    few = mgr.attend(0, 1, q[:2], tables[:2], ints([100, 30], cuda))
    assert bool(torch.isfinite(few).all())
    mgr.close()


def test_captured_chunks_that_share_memory(kvx, cuda):
    """Chunks, and sequences on a shared prefix, captured in two graphs that take
    their workspaces from one pool, replayed in turn between eager calls."""
    steps = [Step(kvx, cuda, [40, 3, 150], [500, 90, 150], 8, 2, 128, 16, BF16, BF16),
             Step(kvx, cuda, [1] * 8, [700 + s for s in range(8)], 8, 2, 128, 16, F16, FP8,
                  [(0, 8, 640)])]
    graphs, pool = [], None
    for step in steps:
        args, kw = step.args(), step.kw()
        want = step.mgr.attend(0, 1, step.q, *args, **kw)
        held = torch.zeros_like(step.q)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            held.copy_(step.mgr.attend(0, 1, step.q, *args, **kw))
        pool = graph.pool()
        graphs.append((graph, held, want, args, kw))
    for i in range(4):
        for step, (graph, held, want, args, kw) in zip(steps, graphs):
            graph.replay()
            eager = step.mgr.attend(0, 1, step.q, *args, **kw)
            if i % 2:
                torch.cuda.synchronize()
            assert torch.equal(held, want) and torch.equal(eager, want)
            held.zero_()
    del graphs, graph
    for step in steps:
        step.mgr.close()

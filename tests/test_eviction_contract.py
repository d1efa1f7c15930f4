"""What the eviction operators say of themselves, on the CPU."""
import textwrap

import pytest

torch = pytest.importorskip("torch")

from fake_device import FakeDeviceTensor  # noqa: E402
from test_eviction_checks import Manager, bytes_as  # noqa: E402
from test_paged_attention_checks import fake, refused  # noqa: E402


def example(doc):
    """The indented part of a docstring."""
    lines = doc.splitlines()
    return textwrap.dedent("\n".join(x for x in lines[1:] if x.startswith("    ") or not x))


def test_the_documented_loop_cuts_every_layer_from_the_same_lengths(kvx):
    class Manager:
        def __init__(self):
            self.attended, self.weighed, self.evicted = {}, {}, {}

        def attend(self, k, v, q, tables, lengths, **kw):
            self.attended[k, v] = lengths
            return "out", "lse"

        def weigh(self, k, q, tables, lengths, lse, weights):
            self.weighed[k] = lengths, weights

        def evict(self, k, v, weights, tables, lengths, budget, **kw):
            self.evicted[k, v] = lengths, weights
            return min(lengths, budget)

    mgr = Manager()
    names = dict(mgr=mgr, layers=3, i=0, q="q", tables="tables", lengths=5000, weights=["a", "b", "c"])
    exec(example(kvx.eviction.__doc__), names)
    pairs = [(0, 1), (2, 3), (4, 5)]
    assert mgr.attended == {p: 5000 for p in pairs}
    assert mgr.weighed == {p[0]: (5000, w) for p, w in zip(pairs, "abc")}
    assert mgr.evicted == {p: (5000, w) for p, w in zip(pairs, "abc")}
    assert names["lengths"] == 2048


def test_side_tables_may_follow_the_scales(kvx):
    fp8, fp4, e8m0 = torch.float8_e4m3fn, torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
    weights = [fake((9, 2, 16), torch.float32)]
    for storage, scale in ((FakeDeviceTensor(torch.zeros(9, 16, 2, 64).to(fp8)),
                            fake((9, 2), torch.float32)),
                           (bytes_as((9, 2, 16, 32), fp4), bytes_as((9, 2, 16, 2), e8m0))):
        for more in ([], weights, weights * 2):
            mgr = Manager(kvx, [storage] * 2, [scale] * 2 + more)
            # The cache is taken, so the refusal is that of the next argument.
            refused("kept must be", mgr.compact, 0, 1, fake((3, 4, 5), torch.int32),
                    fake((3, 4), torch.int32), stream=0)
        refused("one scale table", Manager(kvx, [storage] * 2, [scale]).compact, 0, 1,
                fake((3, 2, 5), torch.int32), fake((3, 4), torch.int32), stream=0)


def test_weigh_refuses_other_counts_of_weighed_tokens(kvx):
    mgr = Manager(kvx, [fake((9, 16, 2, 64)), fake((9, 16, 2, 64))])
    args = (0, fake((3, 8, 64)), fake((3, 4), torch.int32), fake((3,), torch.int32),
            fake((3, 8), torch.float32), fake((9, 2, 16), torch.float32))
    refused("weighed must be", mgr.weigh, *args, weighed=fake((2,), torch.int32), stream=0)
    refused("weighed must be one of", mgr.weigh, *args, weighed=fake((3,), torch.int64), stream=0)
    refused("weighed is on device 1", mgr.weigh, *args, weighed=fake((3,), torch.int32, 1), stream=0)
    refused("HIP device", mgr.weigh, *args, weighed=torch.zeros(3, dtype=torch.int32), stream=0)

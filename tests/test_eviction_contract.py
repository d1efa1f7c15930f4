"""What the eviction operators say of themselves, on the CPU."""
import textwrap

import pytest

pytest.importorskip("torch")


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

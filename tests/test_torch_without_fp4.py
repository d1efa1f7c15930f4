"""A torch that lacks the 4-bit types runs the operators on the other pools (CPU:
the argument handling up to its last refusals)."""
import sys

import pytest

torch = pytest.importorskip("torch")

from fake_device import FakeDeviceTensor  # noqa: E402
from test_paged_attention_checks import FakeManager, fake, refused  # noqa: E402


class OlderTorch:
    def __getattr__(self, name):
        if name in ("float4_e2m1fn_x2", "float8_e8m0fnu"):
            raise AttributeError(f"module 'torch' has no attribute '{name}'")
        return getattr(torch, name)


def test_other_pools_do_not_need_the_4_bit_types(kvx, monkeypatch):
    base = kvx.paged_attention
    monkeypatch.setitem(sys.modules, "torch", OlderTorch())
    for name, value in (("_torch", None), ("_TYPES", {}), ("_FP4", None)):
        monkeypatch.setattr(base, name, value, raising=False)
    refused("positions are needed", kvx.norm_rope, fake((3, 4, 64)), None, None,
            fake((32,), torch.float32), stream=0)
    tables, lengths = fake((3, 4), torch.int32), fake((3,), torch.int32)
    fp8 = [FakeDeviceTensor(torch.zeros(9, 16, 2, 64).to(torch.float8_e4m3fn)) for _ in range(2)]
    for mgr in (FakeManager(kvx, [fake((9, 16, 2, 64))] * 2),
                FakeManager(kvx, fp8, [fake((9, 2), torch.float32)] * 2)):
        refused("head_dim", mgr.attend, 0, 1, fake((3, 8, 32)), tables,
                lengths, stream=0)
    kept = fake((3, 4, 5), torch.int32)
    mgr.compact = kvx.KVCacheManager.compact.__get__(mgr)
    refused("kept must be", mgr.compact, 0, 1, kept, tables, stream=0)
    refused("the cache must be", FakeManager(kvx, [fake((9, 16, 2, 64), torch.int8)] * 2).attend, 0,
            1, fake((3, 8, 64)), tables, lengths, stream=0)

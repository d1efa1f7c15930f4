"""Refusals of weigh, choose_kept, compact and of 4-bit caches, on the CPU: the
library's checks driven from C++, and the Python boundary's with tensors that only
claim to be on a device."""
import os
import shutil
import subprocess

import pytest

torch = pytest.importorskip("torch")

from fake_device import FakeDeviceTensor  # noqa: E402
from test_paged_attention_checks import FakeManager, fake, refused  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
FP4, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


def test_library_refuses_bad_arguments(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    libdir = os.path.join(ROOT, "tpu-sync_amd")
    if cxx is None or not os.path.exists(os.path.join(libdir, "libkvx.so")):
        pytest.skip("no C++ compiler or libkvx.so not built")
    exe = tmp_path / "eviction_args_check"
    env = {k: v for k, v in os.environ.items() if k != "LD_PRELOAD"}
    env.update(HIP_VISIBLE_DEVICES="-1", ROCR_VISIBLE_DEVICES="-1")
    r = subprocess.run([cxx, "-O1", "-std=c++17", "-Wall", "-Werror", "-D__HIP_PLATFORM_AMD__",
                        "-I/opt/rocm/include", "-I", os.path.join(ROOT, "include"),
                        "-I", os.path.join(ROOT, "tpu-sync_amd", "csrc", "host"),
                        os.path.join(ROOT, "tests", "eviction_args_check.cc"), "-o", str(exe),
                        "-L", libdir, "-lkvx", f"-Wl,-rpath,{libdir}"],
                       capture_output=True, text=True, env=env)
    assert r.returncode == 0, r.stdout + r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120, env=env)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "all passed" in r.stdout


def test_null_arguments(kvx):
    lib = kvx._capi.load()
    assert lib.kvx_manager_weigh(None, None, None) == 3
    assert lib.kvx_manager_weigh_workspace(None, None, None) == 3
    assert lib.kvx_choose_kept(None, None) == 3
    assert lib.kvx_manager_compact(None, None, None) == 3


def bytes_as(shape, dtype):
    return FakeDeviceTensor(torch.zeros(shape, dtype=torch.uint8).view(dtype))


class Manager(FakeManager):
    def __init__(self, kvx, kv, scales=()):
        super().__init__(kvx, kv, scales)
        for name in ("weigh", "compact", "evict"):
            setattr(self, name, getattr(kvx.KVCacheManager, name).__get__(self))


def test_a_4_bit_cache_refuses(kvx):
    codes, scales = (9, 2, 16, 32), (9, 2, 16, 2)
    q, k = fake((3, 8, 64)), fake((3, 2, 64))
    tables, lengths = fake((3, 4), I32), fake((3,), I32)
    for match, kv, tabs in (
            ("one scale table", [bytes_as(codes, FP4)] * 2, [bytes_as(scales, E8M0)]),
            ("float8_e8m0fnu", [bytes_as(codes, FP4)] * 2, [fake((9, 2), F32)] * 2),
            # As many bytes in the 16-bit pools' order.
            ("float8_e8m0fnu", [bytes_as(codes, FP4)] * 2, [bytes_as((9, 16, 2, 2), E8M0)] * 2),
            ("same type", [bytes_as(codes, FP4), bytes_as((9, 16, 2, 32), FP4)],
             [bytes_as(scales, E8M0)] * 2)):
        mgr = Manager(kvx, kv, tabs)
        refused(match, mgr.attend, 0, 1, q, tables, lengths, stream=0)
        refused(match, mgr.append_kv, 0, 1, k, k, tables, lengths, stream=0)
        refused(match, mgr.compact, 0, 1, fake((3, 2, 5), I32), tables, stream=0)


def test_weigh_refuses(kvx):
    mgr = Manager(kvx, [fake((9, 16, 2, 64)), fake((9, 16, 2, 64))])
    q, tables, lengths = fake((3, 8, 64)), fake((3, 4), I32), fake((3,), I32)
    lse, w = fake((3, 8), F32), fake((9, 2, 16), F32)

    def call(match, q=q, tables=tables, lengths=lengths, lse=lse, w=w, **kw):
        refused(match, mgr.weigh, 0, q, tables, lengths, lse, w, stream=0, **kw)

    call("HIP device", q=torch.zeros(3, 8, 64, dtype=BF16))
    call("head_dim", q=fake((3, 8, 32)))
    call("lse must be", lse=fake((3, 4), F32))
    call("lse must be", lse=fake((3, 8), BF16))
    call("lse is on device 1", lse=fake((3, 8), F32, 1))
    call("lse must be", lse=FakeDeviceTensor(torch.zeros(8, 3).t()))
    call("weights must be", w=fake((9, 2, 16), BF16))
    call("weights must be", w=fake((9, 16, 2), F32))
    call("weights must be", w=fake((8, 2, 16), F32))
    call("weights must be", w=fake((9, 32), F32))
    call("weights must be", w=FakeDeviceTensor(torch.zeros(9, 16, 2).transpose(1, 2)))
    call("no backward", w=FakeDeviceTensor(torch.zeros(9, 2, 16, requires_grad=True)))
    call("begins must be", begins=fake((2,), I32))
    call("begins must be one of", begins=fake((3,), torch.int64))
    call("without starts", tables=fake((2, 4), I32), lengths=fake((2,), I32))
    with pytest.raises(kvx.KvxError, match="out of range"):
        mgr.weigh(2, q, tables, lengths, lse, w, stream=0)


def test_choose_kept_refuses(kvx):
    w, tables, lengths = fake((9, 2, 16), F32), fake((3, 4), I32), fake((3,), I32)
    fn = kvx.choose_kept
    refused("HIP device", fn, torch.zeros(9, 2, 16), tables, lengths, 5, stream=0)
    refused("weights must be", fn, fake((9, 2, 16)), tables, lengths, 5, stream=0)
    refused("weights must be", fn, fake((9, 32), F32), tables, lengths, 5, stream=0)
    refused("tables must be", fn, w, fake((3, 4), torch.int64), lengths, 5, stream=0)
    refused("tables must be", fn, w, fake((12,), I32), lengths, 5, stream=0)
    refused("tables must be", fn, w, [[0, 1, 2]], lengths, 5, stream=0)
    refused("lengths must be", fn, w, tables, fake((2,), I32), 5, stream=0)
    refused("begins must be", fn, w, tables, lengths, 5, begins=fake((4,), I32), stream=0)
    for bad in (-1, 1 << 31, 2.5, True, None):
        refused("budget must be", fn, w, tables, lengths, bad, stream=0)
        refused("recent must be", fn, w, tables, lengths, 5, recent=bad, stream=0)


def test_compact_refuses(kvx):
    mgr = Manager(kvx, [fake((9, 16, 2, 64)), fake((9, 16, 2, 64))])
    kept, tables = fake((3, 2, 5), I32), fake((3, 4), I32)

    def call(match, kept=kept, tables=tables, **kw):
        refused(match, mgr.compact, 0, 1, kept, tables, stream=0, **kw)

    call("HIP device", kept=torch.zeros(3, 2, 5, dtype=I32))
    call("kept must be", kept=fake((3, 2, 5), torch.int64))
    call("kept must be", kept=fake((3, 4, 5), I32))
    call("kept must be", kept=fake((3, 10), I32))
    call("tables must have 3", tables=fake((2, 4), I32))
    call("tables must be", tables=fake((3, 4), torch.int64))
    call("weights must be", weights=fake((9, 16, 2), F32))
    call("weights is on device 1", weights=fake((9, 2, 16), F32, 1))
    refused("the cache must be", Manager(kvx, [fake((9, 16, 2, 64), F32)] * 2).compact, 0, 1, kept,
            tables, stream=0)


def test_a_host_only_manager_has_no_cache(kvx):
    mgr = kvx.KVCacheManager.create_host_only_for_testing(num_layers=2, slice_byte_size=64,
                                                          host_blocks=4)
    with pytest.raises(kvx.KvxError, match="device-backed") as e:
        mgr.compact(0, 1, fake((3, 2, 5), I32), fake((3, 4), I32), stream=0)
    assert e.value.code == 9
    lib = kvx._capi.load()
    assert lib.kvx_manager_weigh(mgr._h, kvx._capi.WeighArgs(), None) == 9
    assert lib.kvx_manager_compact(mgr._h, kvx._capi.CompactArgs(), None) == 9
    mgr.close()

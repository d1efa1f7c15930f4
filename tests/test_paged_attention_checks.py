"""Refusals of norm_rope, append_kv and attend, on the CPU: the library's checks
driven from C++ with a pool and addresses of its own making, and the Python
boundary's with tensors that only claim to be on a device."""
import os
import shutil
import subprocess

import pytest

torch = pytest.importorskip("torch")

from fake_device import FakeDeviceTensor  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16 = torch.bfloat16


def test_library_refuses_bad_arguments(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    libdir = os.path.join(ROOT, "tpu-sync_amd")
    if cxx is None or not os.path.exists(os.path.join(libdir, "libkvx.so")):
        pytest.skip("no C++ compiler or libkvx.so not built")
    exe = tmp_path / "attention_args_check"
    env = {k: v for k, v in os.environ.items() if k != "LD_PRELOAD"}
    env.update(HIP_VISIBLE_DEVICES="-1", ROCR_VISIBLE_DEVICES="-1")
    r = subprocess.run([cxx, "-O1", "-std=c++17", "-Wall", "-Werror", "-D__HIP_PLATFORM_AMD__",
                        "-I/opt/rocm/include", "-I", os.path.join(ROOT, "include"),
                        "-I", os.path.join(ROOT, "tpu-sync_amd", "csrc", "host"),
                        os.path.join(ROOT, "tests", "attention_args_check.cc"), "-o", str(exe),
                        "-L", libdir, "-lkvx", f"-Wl,-rpath,{libdir}"],
                       capture_output=True, text=True, env=env)
    assert r.returncode == 0, r.stdout + r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120, env=env)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "all passed" in r.stdout


def test_null_arguments(kvx):
    lib = kvx._capi.load()
    assert lib.kvx_norm_rope(None, None) == 3
    assert lib.kvx_manager_append_kv(None, None, None) == 3
    assert lib.kvx_manager_attend(None, None, None) == 3
    assert lib.kvx_manager_attend_workspace(None, None, None) == 3


def fake(shape, dtype=BF16, index=0):
    return FakeDeviceTensor(torch.zeros(shape, dtype=dtype), index)


def refused(match, fn, *args, **kw):
    with pytest.raises(ValueError, match=match):
        fn(*args, **kw)


def test_norm_rope_refuses(kvx):
    q, k, pos = fake((3, 4, 64)), fake((3, 2, 64)), fake((3,), torch.int64)
    inv = fake((32,), torch.float32)
    fn = kvx.norm_rope
    refused("HIP device", fn, torch.zeros(3, 4, 64), None, pos, inv, stream=0)
    refused(r"\[tokens, heads, head_dim\]", fn, fake((3, 64)), None, pos, inv, stream=0)
    refused("float16 or float32", fn, fake((3, 4, 64), torch.float64), None, pos, inv, stream=0)
    refused("last dimension", fn, FakeDeviceTensor(torch.zeros(3, 64, 4, dtype=BF16)
                                                   .transpose(1, 2)), None, pos, inv, stream=0)
    refused("k must be", fn, q, fake((2, 2, 64)), pos, inv, stream=0)
    refused("k must be", fn, q, fake((3, 2, 64), torch.float16), pos, inv, stream=0)
    refused("device 1", fn, q, fake((3, 2, 64), index=1), pos, inv, stream=0)
    refused("positions must be a contiguous tensor of 3", fn, q, k, fake((4,), torch.int64), inv,
            stream=0)
    refused("positions must be one of", fn, q, k, fake((3,), torch.int16), inv, stream=0)
    refused("positions are needed", fn, q, k, None, inv, stream=0)
    refused("inv_freq", fn, q, k, pos, fake((33,), torch.float32), stream=0)
    refused("inv_freq", fn, q, k, pos, fake((32,), torch.float64), stream=0)
    refused("q_weight", fn, q, k, pos, inv, q_weight=fake((63,)), stream=0)
    refused("q_weight", fn, q, k, pos, inv, q_weight=fake((64,), torch.float16), stream=0)
    refused("same dtype", fn, q, k, pos, inv, q_weight=fake((64,)),
            k_weight=fake((64,), torch.float32), stream=0)
    refused("out_k without k", fn, q, None, pos, inv, out_k=k, stream=0)
    grad = FakeDeviceTensor(torch.zeros(3, 4, 64, dtype=BF16, requires_grad=True))
    refused("no backward", fn, grad, None, pos, inv, stream=0)
    refused("no backward", fn, q, None, pos, inv, stream=0, q_weight=FakeDeviceTensor(
        torch.zeros(64, dtype=BF16, requires_grad=True)))


class FakeManager:
    """What the argument handling reads of a manager: its tensors and device.
    A call that passed every check would fail on the missing handle."""

    def __init__(self, kvx, kv, scales=()):
        self._tensors = [[t] for t in list(kv) + list(scales)]
        self.num_kv_layers, self._device, self._h = len(kv), 0, None
        self.append_kv = kvx.KVCacheManager.append_kv.__get__(self)
        self.attend = kvx.KVCacheManager.attend.__get__(self)


def test_append_and_attend_refuse(kvx):
    fp8 = torch.float8_e4m3fn
    mgr = FakeManager(kvx, [fake((9, 16, 2, 64)), fake((9, 16, 2, 64))])
    k, q = fake((3, 2, 64)), fake((3, 8, 64))
    tables, lengths = fake((3, 4), torch.int32), fake((3,), torch.int32)
    for fn, x in ((lambda *a, **kw: mgr.append_kv(a[0], a[1], a[2], a[2], *a[3:], stream=0, **kw), k),
                  (lambda *a, **kw: mgr.attend(*a, stream=0, **kw), q)):
        refused("HIP device", fn, 0, 1, torch.zeros(3, 2, 64, dtype=BF16), tables, lengths)
        refused("the cache must be", fn, 0, 1, FakeDeviceTensor(x._t.half()), tables, lengths)
        refused("head_dim|must be \\(3, 2, 64\\)", fn, 0, 1, fake((3, x.shape[1], 32)), tables,
                lengths)
        refused("tables must be an int32", fn, 0, 1, x, fake((3, 4), torch.int64), lengths)
        refused("tables must be an int32", fn, 0, 1, x, fake((12,), torch.int32), lengths)
        refused("tables must be contiguous", fn, 0, 1, x,
                FakeDeviceTensor(torch.zeros(4, 3, dtype=torch.int32).t()), lengths)
        refused("lengths must be", fn, 0, 1, x, tables, fake((4,), torch.int32))
        refused("lengths must be one of", fn, 0, 1, x, tables, fake((3,), torch.int64))
        refused("starts must be", fn, 0, 1, x, tables, lengths, starts=fake((3,), torch.int32))
        refused("without starts", fn, 0, 1, x, fake((2, 4), torch.int32), fake((2,), torch.int32))
        refused("device 1", fn, 0, 1, x, fake((3, 4), torch.int32, 1), lengths)
        refused("no backward", fn, 0, 1, FakeDeviceTensor(x._t.clone().requires_grad_()), tables,
                lengths)
        for layer, shard in ((2, 0), (-1, 0), (0, 1)):
            with pytest.raises(kvx.KvxError, match="out of range") as e:
                fn(layer, 1, x, tables, lengths, shard_idx=shard)
            assert e.value.code == 11
    refused("v must be", mgr.append_kv, 0, 1, k, fake((3, 2, 32)), tables, lengths, stream=0)
    refused("positions without", mgr.append_kv, 0, 1, k, k, tables, lengths, stream=0,
            positions=fake((3,), torch.int32))
    refused("go together", mgr.attend, 0, 1, q, tables, lengths, stream=0,
            group_starts=fake((2,), torch.int32))
    refused("group_starts must be", mgr.attend, 0, 1, q, tables, lengths, stream=0,
            group_starts=fake((3,), torch.int32), prefix_lengths=fake((1,), torch.int32))
    flat = FakeManager(kvx, [fake((9, 2048)), fake((9, 2048))])
    refused("storages must be", flat.attend, 0, 1, q, tables, lengths, stream=0)
    mixed = FakeManager(kvx, [fake((9, 16, 2, 64)), fake((9, 32, 2, 64))])
    refused("same type and block shape", mixed.attend, 0, 1, q, tables, lengths, stream=0)
    pair = [FakeDeviceTensor(torch.zeros(9, 16, 2, 64).to(fp8)) for _ in range(2)]
    refused("one scale table", FakeManager(kvx, pair, [fake((9, 2), torch.float32)]).attend, 0, 1,
            q, tables, lengths, stream=0)
    refused("float32", FakeManager(kvx, pair, [fake((9, 2), torch.int32)] * 2).attend, 0, 1, q,
            tables, lengths, stream=0)


def test_a_host_only_manager_has_no_cache(kvx):
    mgr = kvx.KVCacheManager.create_host_only_for_testing(num_layers=2, slice_byte_size=64,
                                                          host_blocks=4)
    tables, lengths = fake((3, 4), torch.int32), fake((3,), torch.int32)
    with pytest.raises(kvx.KvxError, match="device-backed") as e:
        mgr.attend(0, 1, fake((3, 8, 64)), tables, lengths, stream=0)
    assert e.value.code == 9
    args = kvx._capi.AttendArgs()
    assert kvx._capi.load().kvx_manager_attend(mgr._h, args, None) == 9
    mgr.close()

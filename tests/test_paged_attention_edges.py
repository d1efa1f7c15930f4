"""The paged operators' checks and arithmetic on the CPU where calls are unusual:
programs of their own that include the library's sources' headers."""
import glob
import os
import re
import shutil
import subprocess

import pytest

torch = pytest.importorskip("torch")

from fake_device import FakeDeviceTensor  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run_check(name, tmp_path, library):
    """Builds tests/<name>.cc, runs it without a GPU and returns what it prints."""
    cxx = shutil.which("g++") or shutil.which("c++")
    csrc = os.path.join(ROOT, "tpu-sync_amd", "csrc")
    libdir = os.path.join(ROOT, "tpu-sync_amd")
    if cxx is None or (library and not os.path.exists(os.path.join(libdir, "libkvx.so"))):
        pytest.skip("no C++ compiler or libkvx.so not built")
    exe = tmp_path / name
    env = {k: v for k, v in os.environ.items() if k != "LD_PRELOAD"}
    env.update(HIP_VISIBLE_DEVICES="-1", ROCR_VISIBLE_DEVICES="-1")
    link = ["-L", libdir, "-lkvx", f"-Wl,-rpath,{libdir}"] if library else []
    r = subprocess.run([cxx, "-O1", "-std=c++17", "-Wall", "-Werror", "-D__HIP_PLATFORM_AMD__",
                        "-I/opt/rocm/include", "-I", os.path.join(ROOT, "include"),
                        "-I", os.path.join(csrc, "host"), "-I", os.path.join(csrc, "kernels"),
                        os.path.join(ROOT, "tests", name + ".cc"), "-o", str(exe)] + link,
                       capture_output=True, text=True, env=env)
    assert r.returncode == 0, r.stdout + r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120, env=env)
    assert r.returncode == 0, r.stdout + r.stderr
    return r.stdout


def test_sums_of_work_do_not_wrap(tmp_path):
    assert "all passed" in run_check("paged_sums_check", tmp_path, library=False)


def test_arguments_in_one_buffer(tmp_path):
    assert "all passed" in run_check("attention_overlap_check", tmp_path, library=True)


def test_frequencies_that_require_gradients_are_refused(kvx):
    def fake(*shape, dtype=torch.bfloat16, **kw):
        return FakeDeviceTensor(torch.zeros(shape, dtype=dtype, **kw))

    q, pos = fake(3, 4, 64), fake(3, dtype=torch.int64)
    inv = fake(32, dtype=torch.float32, requires_grad=True)
    with pytest.raises(ValueError, match="inv_freq requires gradients: there is no backward"):
        kvx.norm_rope(q, None, pos, inv, out_q=fake(3, 4, 64), stream=0)


def test_tangents_are_refused(kvx):
    from torch.autograd import forward_ad
    module = __import__(kvx.__name__ + ".paged_attention", fromlist=["paged_attention"])
    module._load_torch()
    x = torch.ones(4)
    module._refuse_gradients(x, "x")
    with forward_ad.dual_level():
        module._refuse_gradients(x, "x")
        with pytest.raises(ValueError, match="x has a tangent"):
            module._refuse_gradients(forward_ad.make_dual(x, torch.ones(4)), "x")
    module._refuse_gradients(x, "x")


def test_inline_assembly_does_not_write_m0():
    """The compiler uses m0 too and reserves it, so that a clobber says nothing: a
    load into LDS gets its address by an operand that the compiler puts there."""
    kernels = os.path.join(ROOT, "tpu-sync_amd", "csrc", "kernels")
    found = 0
    for path in glob.glob(os.path.join(kernels, "*")):
        with open(path) as f:
            for statement in re.findall(r"asm volatile\((.*?)\);", f.read(), re.S):
                code, operands = statement.split(":", 1)
                assert "m0" not in code, f"{path}: {statement}"
                if "_lds_" in code:
                    found += 1
                    assert '"{m0}"' in operands, f"{path}: {statement}"
    assert found > 0

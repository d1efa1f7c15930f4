"""The paged operators' checks and arithmetic on the CPU where calls are unusual:
programs of their own that include the library's sources' headers."""
import os
import shutil
import subprocess

import pytest

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

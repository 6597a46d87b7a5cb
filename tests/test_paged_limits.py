"""Limits of the operators over a paged cache (CPU only): tests/cpp/paged_limits.cpp, built against the library
and run."""
import os
import subprocess

from mvlm_amd import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_limits(tmp_path):
    exe = str(tmp_path / "paged_limits")
    src = os.path.join(ROOT, "tests", "cpp", "paged_limits.cpp")
    r = subprocess.run([build.HIPCC, f"--offload-arch={build.ARCH}", *build.COMMON, "-O1", src, "-o", exe,
                        f"-L{build.LIBDIR}", "-lmvlm_hip", f"-Wl,-rpath,{build.LIBDIR}", "-Wl,-rpath,/opt/rocm/lib"],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr

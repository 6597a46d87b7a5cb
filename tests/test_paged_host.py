"""Host side of the operators over a paged cache (CPU only): tests/cpp/paged_host.cpp,
built against the library's sources and run."""
import os
import subprocess

from mvlm_amd import build
from test_abi import declared_functions

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_indexes_and_refusals(tmp_path):
    exe = str(tmp_path / "paged_host")
    src = os.path.join(ROOT, "tests", "cpp", "paged_host.cpp")
    r = subprocess.run([build.HIPCC, f"--offload-arch={build.ARCH}", *build.COMMON, "-O1", src, "-o", exe,
                        f"-L{build.LIBDIR}", "-lmvlm_hip", f"-Wl,-rpath,{build.LIBDIR}", "-Wl,-rpath,/opt/rocm/lib"],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


def test_entry_points_have_plan_entries():
    names = declared_functions()
    for op in ("kv_append_paged", "attention_paged", "logits_process"):
        assert f"mvlm_{op}" in names and f"mvlm_plan_add_{op}" in names

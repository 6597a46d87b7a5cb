"""Host side of the 8-bit paged cache and the token draw (CPU only): tests/cpp/paged_8bit_host.cpp, built against the
library's sources and run."""
import os
import subprocess

import pytest

import mvlm_amd as m
from mvlm_amd import build
from test_abi import declared_functions

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_rules_and_refusals(tmp_path):
    exe = str(tmp_path / "paged_8bit_host")
    src = os.path.join(ROOT, "tests", "cpp", "paged_8bit_host.cpp")
    r = subprocess.run([build.HIPCC, f"--offload-arch={build.ARCH}", *build.COMMON, "-O1", src, "-o", exe,
                        f"-L{build.LIBDIR}", "-lmvlm_hip", f"-Wl,-rpath,{build.LIBDIR}", "-Wl,-rpath,/opt/rocm/lib"],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


def test_entry_points_have_plan_entries():
    names = declared_functions()
    for op in ("kv_append_paged_ex", "kv_read_paged", "sample"):
        assert f"mvlm_{op}" in names and f"mvlm_plan_add_{op}" in names


def test_sizes_through_the_binding():
    assert m.paged_kv_bytes(m.MXFP8, 3, 5, 7, 24) == 2528 + 420
    assert m.paged_kv_bytes(m.F16, 3, 5, 7, 24) == 2 * 105 * 24
    with pytest.raises(m.MvlmError):
        m.paged_kv_bytes(m.F32, 3, 5, 7, 24)

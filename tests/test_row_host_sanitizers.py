"""The host code of the operators on rows and of the 8-bit products under AddressSanitizer and UBSan: all sources are
rebuilt with the sanitizers on the host side (-Xarch_host; the device code as usual), and tests/host_fuzz_rows.cpp calls
their entry points with seeded random and edge-case sizes, never far enough to launch. CPU only: skipped where a GPU is
present."""
from __future__ import annotations

import concurrent.futures
import os
import pathlib
import subprocess

import pytest

from conftest import ROOT
from test_dense_host_sanitizers import PKG, SAN, _hipcc


@pytest.mark.skipif(_hipcc() is None, reason="hipcc is not installed")
@pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="CPU-only test: a GPU is present")
def test_row_host_code_under_asan_and_ubsan(tmp_path: pathlib.Path):
    hipcc = _hipcc()
    flags = ["--offload-arch=gfx950", "-O1", "-g", "-std=c++17", "-fPIC", "-Xclang", "-target-feature", "-Xclang",
             "-packed-fp32-ops", *SAN, f"-I{ROOT / 'include'}", f"-I{PKG / 'csrc'}"]
    sources = sorted((PKG / "csrc").glob("*.hip")) + sorted((PKG / "csrc").glob("*.cpp"))

    def compile_one(src: pathlib.Path) -> pathlib.Path:
        obj = tmp_path / (src.name + ".o")
        lang = ["-x", "hip"] if src.suffix == ".hip" else []
        res = subprocess.run([hipcc, *flags, *lang, "-c", str(src), "-o", str(obj)], capture_output=True, text=True)
        assert res.returncode == 0, res.stderr[-3000:]
        return obj

    with concurrent.futures.ThreadPoolExecutor(max_workers=8) as pool:
        objs = list(pool.map(compile_one, sources))
    res = subprocess.run([hipcc, "-x", "c++", "-O1", "-g", "-std=c++17", *SAN, f"-I{ROOT / 'include'}", "-c",
                          str(ROOT / "tests" / "host_fuzz_rows.cpp"), "-o", str(tmp_path / "fuzz.o")],
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-3000:]
    exe = tmp_path / "host_fuzz_rows"
    res = subprocess.run([hipcc, "--offload-arch=gfx950", *SAN[:4], *map(str, objs), str(tmp_path / "fuzz.o"), "-o",
                          str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-3000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:halt_on_error=1", UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1")
    res = subprocess.run([str(exe), "200000"], capture_output=True, text=True, env=env, timeout=600)
    assert res.returncode == 0, (res.stdout[-3000:], res.stderr[-3000:])

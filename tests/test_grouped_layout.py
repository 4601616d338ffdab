"""CPU check of the grouped product's work list, carve-up and index arithmetic
(tests/grouped_layout_host.cu; nvcc builds it for sm_100a, it runs on the CPU)."""

from __future__ import annotations

import subprocess

import pytest

from test_kernel_layout import CSRC, ROOT, _nvcc


def test_grouped_index_arithmetic(tmp_path):
    nvcc = _nvcc()
    if nvcc is None:
        pytest.skip("nvcc not found")
    exe = tmp_path / "grouped_layout_host"
    build = subprocess.run(
        [nvcc, "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a",
         "-I", str(CSRC), "-I", str(ROOT / "include"),
         str(ROOT / "tests" / "grouped_layout_host.cu"), "-o", str(exe)],
        capture_output=True, text=True, timeout=600)
    assert build.returncode == 0, build.stderr[-4000:]
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout[-4000:]
    assert run.stdout.startswith("grouped layout checks ok ("), run.stdout

"""The C++ entries of the experts' products (kiwi/gemm/fp8_gemm.hpp and its
neighbours) refuse bad arguments before they touch a device, so this runs
without a GPU: tests/native/product_args.cpp makes the calls."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NVCC = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
SOURCES = ["csrc/fp8_gemm.cu", "csrc/fp8_few_rows.cu", "csrc/grouped_linear.cu", "csrc/swiglu_gpu.cu", "csrc/tensor_map.cpp", "src/p2p/driver.cpp",
           "tests/native/product_args.cpp"]


@pytest.fixture(scope="module")
def refusals(tmp_path_factory):
    if not os.path.exists(NVCC):
        pytest.skip("needs nvcc")
    out = tmp_path_factory.mktemp("args")
    # Optimised code is not needed, and the device code never runs.
    flags = ["-gencode", "arch=compute_100a,code=sm_100a", "-O1", "-std=c++17", "--expt-relaxed-constexpr",
             "-I" + os.path.join(ROOT, "include")]
    jobs = [(src, str(out / (os.path.basename(src) + ".o"))) for src in SOURCES]
    procs = [subprocess.Popen([NVCC, *flags, "-c", os.path.join(ROOT, s), "-o", o], stderr=subprocess.PIPE, text=True)
             for s, o in jobs]
    for p in procs:
        err = p.communicate(timeout=600)[1]
        assert p.returncode == 0, err[-3000:]
    binary = str(out / "product_args")
    r = subprocess.run([NVCC, *flags, *(o for _, o in jobs), "-o", binary], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([binary], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, (r.returncode, r.stderr)
    return dict(line.split(": ", 1) for line in r.stdout.splitlines())


@pytest.mark.parametrize("case,words", [
    ("fp8 groups without counts", "counts"),
    ("fp8 no groups", "1..1024 groups"),
    ("fp8 no output", "missing operands or output"),
    ("fp8 k", "multiple of 16"),
    ("fp8 large k", "2^31"),
    ("forward large k", "2^31"),
    ("dgrad large k", "2^31"),
    ("wgrad large k", "2^31"),
    ("forward unaligned rows", "16-byte boundaries"),
    ("wgrad unaligned rows", "16-byte boundaries"),
    ("swiglu columns", "multiple of 128"),
    ("swiglu no columns", "multiple of 128"),
    ("swiglu row stride", "16-byte boundaries"),
    ("swiglu short rows", "row stride"),
    ("swiglu input base", "16-byte boundaries"),
    ("swiglu output base", "16-byte boundaries"),
    ("swiglu missing input", "missing"),
    ("swiglu missing output", "missing"),
])
def test_refused_before_a_device_is_touched(refusals, case, words):
    assert words in refusals[case], refusals[case]
    if case.startswith("swiglu"):
        assert words in refusals[case + " backward"], refusals[case + " backward"]

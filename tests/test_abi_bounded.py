"""The argument validation of windowed attention, caches cut by weight and drafted tokens under
AddressSanitizer and UBSan (CPU only): tests/abi_bounded.cpp, built as test_abi_sanitized.py
builds its driver, against the sources that hold these entry points; and the refusals of their
Python methods."""
import os
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from crucible_amd import _build
from crucible_amd._lib import CrucibleError
from crucible_amd.gpu import Gpu
from crucible_amd.paged import PagePool, SequencePages

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
OUT = os.path.join(HERE, "_build", "sanitized", "bounded")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
SOURCES = ("attn_span.hip", "cache_weights.hip", "verify.hip", "abi_common.cpp", "paging.cpp")
HOST_SAN = ["-Xarch_host", "-fsanitize=address", "-Xarch_host", "-fsanitize=undefined",
            "-Xarch_host", "-fno-sanitize-recover=all", "-Xarch_host", "-fno-omit-frame-pointer"]


def _build_driver() -> str:
    hipcc = os.path.join(ROCM, "bin", "hipcc")
    clang = os.path.join(ROCM, "llvm", "bin", "clang++")
    if not (os.path.exists(hipcc) and os.path.exists(clang)):
        pytest.skip("ROCm's hipcc and clang++ are needed to build the sanitized library")
    os.makedirs(OUT, exist_ok=True)
    sources = [os.path.join(_build.CSRC, s) for s in SOURCES]
    objs = [os.path.join(OUT, os.path.splitext(s)[0] + ".o") for s in SOURCES]
    headers = [os.path.join(_build.CSRC, f) for f in os.listdir(_build.CSRC) if f.endswith(".hpp")]
    headers.append(os.path.join(ROOT, "include", "crucible_attn.h"))
    newest = max(map(os.path.getmtime, headers))
    flags = ["-O1", "-g", "-std=c++17", "-fPIC", f"--offload-arch={_build.ARCH}",
             "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
             "-I", _build.CSRC, "-I", os.path.join(ROOT, "include")]
    jobs = [[hipcc, *flags, *HOST_SAN, "-x", "hip", "-c", s, "-o", o] for s, o in zip(sources, objs)
            if not os.path.exists(o) or os.path.getmtime(o) < max(newest, os.path.getmtime(s))]
    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:
        for proc in pool.map(lambda c: subprocess.run(c, capture_output=True, text=True), jobs):
            assert proc.returncode == 0, proc.stderr[-3000:]
    exe = os.path.join(OUT, "abi_bounded")
    proc = subprocess.run([clang, "-O1", "-g", "-std=c++17", "-D__HIP_PLATFORM_AMD__",
                           "-I", os.path.join(ROCM, "include"),
                           "-I", os.path.join(ROOT, "include"),
                           "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                           os.path.join(HERE, "abi_bounded.cpp"),
                           os.path.join(HERE, "hip_stub.cpp"), *objs, "-o", exe],
                          capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr[-3000:]
    return exe


@pytest.mark.timeout(600)
def test_validation_under_sanitizers():
    exe = _build_driver()
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:halt_on_error=1",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    proc = subprocess.run([exe], capture_output=True, text=True, timeout=300, env=env)
    out = proc.stdout + proc.stderr
    assert proc.returncode == 0, out[-6000:]
    assert "AddressSanitizer" not in out and "runtime error" not in out, out[-6000:]
    assert " 0 failed;" in proc.stdout, proc.stdout[-3000:]


def test_shrink_from_python():
    pool, s = PagePool(8, 12, 192), SequencePages()
    s.grow(pool, 100)
    first = s.pages().tolist()
    s.shrink(pool, 40)
    assert len(s) == 40 and s.pages().tolist() == first[:3] and pool.free_pages() == 5
    with pytest.raises(CrucibleError, match="shrink"):
        s.shrink(pool, 41)
    s.grow(pool, 70)
    assert len(s) == 110 and s.n_pages() == 7
    s.release(pool)
    assert pool.free_pages() == 8


def test_methods_refuse_host_tensors_and_wrong_types():
    gpu = Gpu(0)
    x = torch.zeros(4096)
    i = torch.zeros(4096, dtype=torch.int32)
    h = torch.zeros(4096, dtype=torch.float16)
    with pytest.raises(CrucibleError, match="q must be a device tensor"):
        gpu.attention_decode_window_paged(x, h, h, x, i, i, 1, 2, 1, 64, 4, 1, 0, 64, 64, 9, 0)
    with pytest.raises(CrucibleError, match="device tensor"):
        gpu.attention_prefill_window_tiled(x, h, h, x, i, i, 1, 4, 4, 2, 1, 64, 1, 0, 64, 9, 0)
    with pytest.raises(CrucibleError, match="q is required"):
        gpu.attention_decode_weigh_paged(None, h, h, x, i, x, i, i, i, 1, 2, 1, 64, 4, 1, 0, 64, 64)
    with pytest.raises(CrucibleError, match="device tensor"):
        gpu.cache_weigh_tiled(x, h, x, i, i, i, i, 1, 4, 4, 2, 1, 64, 1, 0, 64, 8)
    with pytest.raises(CrucibleError, match="device tensor"):
        gpu.cache_evict_paged(h, h, x, i, i, i, i, 1, 1, 64, 4, 1, 64, 64, 16, 0, 4)
    with pytest.raises(CrucibleError, match="target must be a device tensor"):
        gpu.verify_drafts(x, None, i, i, x, x, i, i, 1, 2, 100)

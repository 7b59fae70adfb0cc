"""Out-of-bounds regression (round 6).  Round 5's intermittent "Memory access fault by GPU" was `conv_wgrad_tr`'s masked units reading
their (unclamped) channel piece at the clamped pixel 0: up to 32 bytes past the END of a 512-byte activation of the legacy U-Nets'
1 x 1 stage -- harmless unless torch's caching allocator had put that tensor at the very end of a segment, so no functional test can
see it.  This one can: the offending tests run in a child process whose every device tensor ENDS at an unmapped page
(tools/dbg/guard_alloc.cpp as torch's pluggable allocator, GUARD_ALLOC_END=1 GUARD_ALLOC_LEAK=1); an access >= 16 bytes past the end of
any buffer aborts the child."""
import ctypes
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = "/opt/rocm/bin/hipcc"


def _guard_lib(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc on this box: the guard allocator is built where it runs")
    so = str(tmp_path_factory.mktemp("guard") / "libguard_alloc.so")
    r = subprocess.run([HIPCC, "-O2", "-w", "-shared", "-fPIC", "-o", so, os.path.join(ROOT, "tools", "dbg", "guard_alloc.cpp")],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    return so


def test_guard_allocator_places_every_tensor_at_the_end_of_its_mapping(tmp_path_factory):
    """The arithmetic of tools/dbg/guard_alloc.cpp, on the host: what is mapped holds the tensor, the tensor begins at a multiple of 16 bytes and
    ends at most 15 bytes before the end of what is mapped -- so an access 16 bytes past the tensor's end lies outside of it.  (No test
    makes that access: a fault takes the GPU away from everything else that runs on it.)"""
    lib = ctypes.CDLL(_guard_lib(tmp_path_factory))
    lib.guard_place.restype = ctypes.c_size_t
    lib.guard_place.argtypes = [ctypes.c_size_t, ctypes.c_size_t, ctypes.c_int, ctypes.POINTER(ctypes.c_size_t)]
    for gran in (4096, 65536, 2 << 20):
        for size in (1, 2, 15, 16, 17, 100, 12000, gran - 1, gran, gran + 1, 3 * gran - 17, 3 * gran, (1 << 33) + 5):
            mapped = ctypes.c_size_t()
            at = lib.guard_place(size, gran, 1, ctypes.byref(mapped))
            assert mapped.value % gran == 0 and size <= mapped.value < size + gran, (size, gran)
            assert at % 16 == 0 and 0 <= mapped.value - (at + size) <= 15, (size, gran)
            assert lib.guard_place(size, gran, 0, ctypes.byref(mapped)) == 0


@pytest.mark.gpu
def test_guard_allocator_is_sound(tmp_path_factory):
    """The tool itself: torch fills, copies and kernels are right under it."""
    so = _guard_lib(tmp_path_factory)
    env = dict(os.environ, GUARD_ALLOC_END="1", GUARD_ALLOC_LEAK="1")
    ok = ("import torch\n"
          "a = torch.cuda.memory.CUDAPluggableAllocator(%r, 'guard_malloc', 'guard_free')\n"
          "torch.cuda.memory.change_current_allocator(a)\n"
          "x = torch.arange(3000, dtype=torch.float32).cuda()\n"
          "assert bool(((x * 2).cpu() == torch.arange(3000) * 2.0).all())\n" % so)
    r = subprocess.run([sys.executable, "-c", ok], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.gpu
def test_no_kernel_reads_past_the_end_of_a_buffer_legacy_backward(tmp_path_factory):
    so = _guard_lib(tmp_path_factory)
    env = dict(os.environ, FDGAN_TEST_GUARD_ALLOC=so, GUARD_ALLOC_END="1", GUARD_ALLOC_LEAK="1", FDGAN_TEST_HYGIENE="none")
    env.pop("FDGAN_TEST_MEMTRACE", None)
    r = subprocess.run([sys.executable, "-m", "pytest", os.path.join(ROOT, "tests", "test_hip_models.py"), "-m", "gpu", "-q", "-x",
                        "-p", "no:cacheprovider", "-k", "legacy_unets_backward or legacy_dehaze_backward or dehaze22_d_backward"],
                       env=env, capture_output=True, text=True, timeout=1500, cwd=ROOT)
    tail = (r.stdout[-1500:] + "\n" + r.stderr[-1500:])
    assert r.returncode == 0 and "passed" in r.stdout, tail

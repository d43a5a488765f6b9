"""A plan of shared-prefix attention is complete on the device when its C entry returns: kernels on any
stream may read its lists at once.  Shown without a GPU: the library runs in a child process over
stand-ins of the few runtime calls that a plan makes.  A copy from pageable host memory may return
once the source is staged, before the bytes are on the device; the stand-in therefore writes them
only when the copy's stream is waited for, and counts those still under way."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

from ane import _abi

STAND_IN = r"""
#include <stdlib.h>
#include <string.h>
typedef struct { void* dst; void* src; size_t n; void* stream; } copy_t;
static copy_t copies[64];
static int n_copies, allocations, fail_copy;
int fake_pending(void) { return n_copies; }
int fake_allocations(void) { return allocations; }
void fake_fail_copies(int on) { fail_copy = on; }
static void land(void* stream, int all) {
  int kept = 0;
  for (int i = 0; i < n_copies; ++i) {
    if (all || copies[i].stream == stream) memcpy(copies[i].dst, copies[i].src, copies[i].n), free(copies[i].src);
    else copies[kept++] = copies[i];
  }
  n_copies = kept;
}
static void* legacy(void* s) { return s == (void*)1 ? NULL : s; } /* cudaStreamLegacy is the null stream */
int cudaGetDevice(int* d) { return *d = 0, 0; }
int cudaSetDevice(int d) { return 0; }
int cudaFuncSetAttribute(const void* f, int a, int v) { return 0; }
static int last; /* launches fail for want of a device */
int cudaLaunchKernel(const void* f, ...) { return last = 100; }
int cudaLaunchKernelExC(const void* c, const void* f, void** a) { return last = 100; }
int cudaGetLastError(void) { int e = last; last = 0; return e; }
int cudaMalloc(void** p, size_t n) { *p = calloc(n ? n : 1, 1); ++allocations; return *p ? 0 : 2; }
int cudaFree(void* p) { if (p) --allocations; free(p); return 0; }
int cudaMemcpyAsync(void* d, const void* s, size_t n, int kind, void* stream) {
  if (fail_copy) return 1;
  if (n_copies == 64) return 1;
  copy_t c = {d, malloc(n), n, legacy(stream)};
  memcpy(c.src, s, n);
  copies[n_copies++] = c;
  return 0;
}
int cudaMemcpy(void* d, const void* s, size_t n, int kind) { return cudaMemcpyAsync(d, s, n, kind, NULL); }
int cudaStreamSynchronize(void* s) { return land(legacy(s), 0), 0; }
int cudaDeviceSynchronize(void) { return land(NULL, 1), 0; }
"""

CHILD = r"""
import ctypes as C, sys
fake, L = C.CDLL(sys.argv[1]), C.CDLL(sys.argv[2])
fail = int(sys.argv[3])
i32 = lambda *a: (C.c_int32 * len(a))(*a)
h = C.c_void_p()
fake.fake_fail_copies(fail)
for rows, n in (((1, 1), 2), ((300, 0), 2), ((0, 0), 2), ((5,) * 64, 64)):
    rc = L.llm_prefix_plan_create(0, 1, 8, 2, 64, i32(*range(n)), i32(*rows), n, i32(n), i32(32), 1, 4096, C.byref(h))
    if fail:
        assert rc != 0 and not h.value and fake.fake_allocations() == 0, (rc, h.value)
        continue
    assert rc == 0 and fake.fake_allocations() == 1, rc
    assert fake.fake_pending() == 0, f"{fake.fake_pending()} copies still under way"
    assert L.llm_prefix_plan_destroy(h) == 0 and fake.fake_allocations() == 0
print("complete")
"""


@pytest.mark.parametrize("fail", [0, 1])
def test_a_new_plan_is_on_the_device(tmp_path, fail):
    src, so, child = tmp_path / "runtime.c", tmp_path / "runtime.so", tmp_path / "child.py"
    src.write_text(STAND_IN)
    child.write_text(CHILD)
    subprocess.run(["cc", "-shared", "-fPIC", "-w", "-o", str(so), str(src)], check=True)
    r = subprocess.run([sys.executable, str(child), str(so), str(Path(_abi.LIB_PATH)), str(fail)], capture_output=True, text=True,
                       timeout=120, env={**os.environ, "LD_PRELOAD": str(so), "CUDA_VISIBLE_DEVICES": ""})
    assert r.returncode == 0 and "complete" in r.stdout, r.stdout + r.stderr

"""The library's host side without a GPU: the HIP calls it makes answered by a small
C library that stands in front of the runtime, in a process of its own.  Allocations
are counted and never touched, launches are counted and run nothing."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

_SOURCE = r"""
#include <stddef.h>
#include <stdint.h>
typedef struct { unsigned x, y, z; } dim3;
static int last, launches, fail_at = -1;
static size_t bytes;
static uintptr_t next = 1ul << 40;
int fake_launches(void) { return launches; }
size_t fake_bytes(void) { return bytes; }
/* the n-th launch from now on (0: the next) fails, the ones around it succeed */
void fake_fail(int n) { fail_at = launches + n; }

int hipGetDeviceCount(int* n) { *n = 1; return 0; }
int hipGetDevice(int* d) { *d = 0; return 0; }
int hipSetDevice(int d) { return 0; }
int hipDeviceGetAttribute(int* v, int a, int d) { *v = 256; return 0; }
int hipFuncSetAttribute(const void* f, int a, int v) { return 0; }
int hipOccupancyMaxActiveBlocksPerMultiprocessor(int* n, const void* f, int b, size_t s) {
  *n = 2;
  return 0;
}
int hipGetSymbolAddress(void** p, const void* s) { *p = (void*)next; return 0; }
int hipMalloc(void** p, size_t n) {
  bytes += n;
  *p = (void*)next;
  next += (n + 4095) & ~(size_t)4095;
  return 0;
}
int hipFree(void* p) { return 0; }
int hipMemset(void* p, int v, size_t n) { return 0; }
int hipMemcpy(void* d, const void* s, size_t n, int k) { return 0; }
int hipStreamIsCapturing(void* s, int* state) { *state = 0; return 0; }
int hipStreamSynchronize(void* s) { return 0; }
int __hipPushCallConfiguration(dim3 g, dim3 b, size_t m, void* s) { return 0; }
int __hipPopCallConfiguration(dim3* g, dim3* b, size_t* m, void** s) {
  *g = *b = (dim3){1, 1, 1};
  *m = 0;
  *s = 0;
  return 0;
}
/* the error of the last call, as a runtime has it whose successful calls clear it */
int hipLaunchKernel(const void* f, dim3 g, dim3 b, void** args, size_t m, void* s) {
  last = launches++ == fail_at ? 719 : 0;
  return last;
}
int hipGetLastError(void) { const int e = last; last = 0; return e; }
"""

_PRELUDE = """
import ctypes, sys
fake = ctypes.CDLL({lib!r}, mode=ctypes.RTLD_GLOBAL)
fake.fake_bytes.restype = ctypes.c_size_t
from aiimage_amd import _abi
lib = _abi.load()
ctx = ctypes.c_void_p()
assert lib.aexq_create(0, None, ctypes.byref(ctx)) == 0, lib.aexq_last_error()
PTR = 1 << 20    # a device address as far as the host can tell
def paged(**over):
    d = dict(k=PTR, v=PTR, pages=64, page_size=64, heads_kv=2, head_dim=128, table=PTR,
             lengths=PTR, sequences=3, table_width=40)
    d.update(over)
    return _abi.PagedKv(**d)
"""


def run(tmp_path, body):
    """Runs `body` after the prelude above."""
    src, lib = tmp_path / "fake_hip.c", tmp_path / "libfake_hip.so"
    src.write_text(_SOURCE)
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(lib), str(src)], check=True)
    done = subprocess.run([sys.executable, "-c", _PRELUDE.format(lib=str(lib)) + body], cwd=ROOT,
                          capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stdout + done.stderr
    return done.stdout

"""The pinned memory that a cache stages its records in (no GPU: the runtime's
allocations are stood in for, in a process of its own)."""
import subprocess
import sys
from pathlib import Path

import pytest

from mi50grad_amd._lib import LIB_PATH

ROOT = Path(__file__).resolve().parent.parent
pytestmark = pytest.mark.skipif(LIB_PATH.name == "libkvattn_san.so", reason="the sanitizer's library links its own")

# libkvattn's calls go to the first of these names that the process knows.
RUNTIME = """
#include <cstdio>
#include <cstdlib>
extern "C" {
int hipHostMalloc(void **p, size_t n, unsigned flags) {
    std::printf("%08x\\n", flags);
    std::fflush(stdout);
    *p = std::calloc(1, n);
    return *p ? 0 : 2;
}
int hipHostFree(void *p) { std::free(p); return 0; }
int hipMalloc(void **p, size_t) { *p = std::malloc(16); return 0; }
int hipFree(void *p) { std::free(p); return 0; }
int hipMemset(void *, int, size_t) { return 0; }
int hipMemcpy(void *, const void *, size_t, int) { return 0; }
int hipGetDevice(int *d) { *d = 0; return 0; }
int hipDeviceGetAttribute(int *v, int, int) { *v = 256; return 0; }
int hipDeviceSynchronize() { return 0; }
int hipEventCreateWithFlags(void **e, unsigned) { *e = std::malloc(1); return 0; }
int hipEventDestroy(void *e) { std::free(e); return 0; }
}
"""

SCRIPT = """
import ctypes, sys
ctypes.CDLL(sys.argv[1], ctypes.RTLD_GLOBAL)
from mi50grad_amd.kv_cache import PagedKVCache
for bits in (8, 16):
    PagedKVCache(n_layers=1, max_seqs=2, max_blocks=8, max_blocks_per_seq=4, max_step_tokens=64, kv_bits=bits).destroy()
"""


def test_staging_memory_is_coherent(tmp_path):
    """A kernel reads an eviction's records from it directly, and its addresses
    are used again: it has to be coherent whatever the environment says."""
    (tmp_path / "runtime.cpp").write_text(RUNTIME)
    lib = tmp_path / "runtime.so"
    subprocess.run(["g++", "-shared", "-fPIC", "-o", str(lib), str(tmp_path / "runtime.cpp")], check=True)
    r = subprocess.run([sys.executable, "-c", SCRIPT, str(lib)], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stderr
    flags = [int(x, 16) for x in r.stdout.split()]
    assert flags and all(f & 0x40000000 for f in flags), r.stdout  # hipHostMallocCoherent

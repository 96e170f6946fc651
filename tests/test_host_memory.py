"""Calls that run out of host memory answer with an error and change nothing
(host-only caches, in a process whose allocator fails when told to)."""
import subprocess
import sys
from pathlib import Path

import pytest

from mi50grad_amd._lib import LIB_PATH

ROOT = Path(__file__).resolve().parent.parent
pytestmark = pytest.mark.skipif(LIB_PATH.name == "libkvattn_san.so", reason="the sanitizer has an allocator of its own")

# Allocations in libkvattn go to the first operator new that the process knows.
ALLOCATOR = """
#include <cstdlib>
#include <new>
static long left = -1;  // allocations that succeed before one (forever: all) fails; -1: none does
static bool forever = false;
extern "C" void fail_at(long n, bool all) { left = n, forever = all; }
void *operator new(std::size_t n) {
    if (left == 0) {
        if (!forever) left = -1;
        throw std::bad_alloc();
    }
    if (left > 0) --left;
    if (void *p = std::malloc(n ? n : 1)) return p;
    throw std::bad_alloc();
}
void operator delete(void *p) noexcept { std::free(p); }
void operator delete(void *p, std::size_t) noexcept { std::free(p); }
"""

SCRIPT = """
import ctypes, sys
alloc = ctypes.CDLL(sys.argv[1], ctypes.RTLD_GLOBAL)
alloc.fail_at.argtypes = [ctypes.c_long, ctypes.c_bool]
from mi50grad_amd._lib import KvaError
from mi50grad_amd.kv_cache import PagedKVCache

def make(bits):
    c = PagedKVCache(n_layers=2, max_seqs=40, max_blocks=400, max_blocks_per_seq=40, max_step_tokens=4096,
                     host_only=True, kv_bits=bits)
    c.reserve(0, 30)
    c.begin_step([0, 1], [40, 70])
    c.begin_step([1, 0], [1, 3])
    c.set_len(1, 50)
    return c

def state(c):
    return [(c.seq_len(s), c.blocks(s)) for s in range(40)], c.free_block_count()

def failing(bits, call):
    \"\"\"`call` with its first, second, ... allocation refused, it alone or all from
    there on: an error that leaves the cache as it was, and the call works afterwards.\"\"\"
    whole = make(bits)
    call(whole)
    n = 0
    while True:
        c = make(bits)
        before = state(c)
        alloc.fail_at(n // 2, n % 2 == 1)
        try:
            call(c)
        except KvaError as e:
            alloc.fail_at(-1, False)
            assert e.code == -5 and "out of host memory" in str(e), e
            assert state(c) == before, f"allocation {n // 2}"
            call(c)
        else:
            alloc.fail_at(-1, False)
            print(n, flush=True)
            assert n > 1, "no allocation was refused"
            return
        assert state(c) == state(whole)
        c.destroy()
        n += 1

"""

CALLS = {
    "begin_step": "lambda c: c.begin_step(list(range(30)), [5 * b for b in range(30)])",
    "begin_step of tokens": "lambda c: c.begin_step(list(range(40)), [1] * 40)",
    "reserve": "lambda c: c.reserve(5, 640)",
    "set_blocks": "lambda c: c.set_blocks(0, list(range(300, 340)))",
    "rollback": "lambda c: c.rollback([0, 1], [20, 30], {8: [[0, 1], [0]], 16: [[0, 2, 5], [3, 4]]}[c.kv_bits])",
}


@pytest.fixture(scope="module")
def allocator(tmp_path_factory):
    d = tmp_path_factory.mktemp("allocator")
    (d / "alloc.cpp").write_text(ALLOCATOR)
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-o", str(d / "alloc.so"), str(d / "alloc.cpp")], check=True)
    return d / "alloc.so"


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("name", CALLS)
def test_a_refused_allocation_changes_nothing(allocator, name, bits):
    script = SCRIPT + f"failing({bits}, {CALLS[name]})\n"
    r = subprocess.run([sys.executable, "-c", script, str(allocator)], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout + r.stderr

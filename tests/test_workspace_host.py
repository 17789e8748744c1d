"""Growth of a context's workspace (csrc/workspace.h) with an allocator of a fixed budget, on the host."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MIB = 1 << 20
SOURCE = """
#include "workspace.h"
#include <map>
static size_t budget, used, calls;
static std::map<void*, size_t> live;
static void* ws;
static size_t have;
static void* take(size_t n) {
    ++calls;
    if (n > budget - used) return nullptr;
    void* p = reinterpret_cast<void*>((calls << 12));
    live[p] = n;
    used += n;
    return p;
}
static void give(void* p) { used -= live.at(p); live.erase(p); }
extern "C" void start(size_t total, size_t first) {
    live.clear(); used = calls = 0; budget = total; ws = first ? take(first) : nullptr; have = first;
}
extern "C" int grow(size_t need) { return need <= have || ws_grow(&ws, &have, need, take, give); }
extern "C" size_t size() { return have; }
extern "C" int sound() { return live.size() == (ws ? 1u : 0u) && used == have && (!ws || live.at(ws) == have); }
extern "C" void set_budget(size_t total) { budget = total; }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("workspace")
    (d / "w.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(ROOT, "tramp_amd", "csrc"), str(d / "w.cpp"),
                    "-o", str(d / "w.so")], check=True)
    lib = C.CDLL(str(d / "w.so"))
    lib.size.restype = C.c_size_t
    for f in (lib.grow, lib.set_budget):
        f.argtypes = [C.c_size_t]
    lib.start.argtypes = [C.c_size_t, C.c_size_t]
    return lib


def test_it_doubles(lib):
    lib.start(1 << 40, 4 * MIB)
    for need, size in ((4 * MIB, 4), (4 * MIB + 1, 8), (9 * MIB, 16), (100 * MIB, 128), (3, 128)):
        assert lib.grow(need) and lib.size() == size * MIB and lib.sound()


def test_a_size_that_fits_only_exactly(lib):
    lib.start(100 * MIB, 4 * MIB)
    assert lib.grow(70 * MIB) and lib.size() == 70 * MIB and lib.sound()


@pytest.mark.timeout(20)
def test_a_failure_leaves_the_context_usable(lib):
    lib.start(100 * MIB, 4 * MIB)
    assert lib.grow(20 * MIB) and lib.size() == 32 * MIB
    assert not lib.grow(101 * MIB) and lib.size() == 32 * MIB and lib.sound()
    assert lib.grow(1 * MIB) and lib.grow(50 * MIB) and lib.size() == 64 * MIB and lib.sound()


@pytest.mark.timeout(20)
def test_nothing_left_and_memory_that_comes_back(lib):
    lib.start(8 * MIB, 4 * MIB)
    lib.set_budget(1 * MIB)                                        # somebody else has taken the rest
    assert not lib.grow(8 * MIB) and lib.size() == 0 and lib.sound()
    assert not lib.grow(2 * MIB) and lib.size() == 0               # from a size of 0, an end all the same
    assert lib.grow(1) and lib.size() == 1 and lib.sound()         # exactly the need fits
    lib.set_budget(8 * MIB)
    assert lib.grow(2) and lib.size() == 4 * MIB and lib.sound()
    assert not lib.grow((1 << 64) - 1) and lib.size() == 4 * MIB and lib.sound()

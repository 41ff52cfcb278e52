"""What kernels have been opted in to (csrc/opt_in.h, compiled alone): on the CPU, against a stand-in for the runtime that keeps, as it does, the last limit that it was given."""

import ctypes as C
import os
import subprocess

import pytest

from yule_b200 import _lib

SOURCE = r"""
#include <map>
#include "opt_in.h"
static yule::OptIns all;
static std::map<std::pair<const void *, int>, size_t> limit;
static int calls;
extern "C" {
// An opt-in of `kernel` on `device`; `error` is what the runtime says.
int ask(size_t kernel, int device, size_t smem, int clusters, int error) {
    const void *k = reinterpret_cast<const void *>(kernel);
    return all.take(k, device, smem, clusters != 0, [&](size_t n) { return calls++, error ? error : (limit[{k, device}] = n, 0); }, [&] { return calls++, error; }, 2);
}
size_t has(size_t kernel, int device) { return limit[{reinterpret_cast<const void *>(kernel), device}]; }
int made() { return calls; }
}
"""


@pytest.fixture()
def runtime(tmp_path):
    (tmp_path / "opt.cpp").write_text(SOURCE)
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(_lib.HERE, "csrc"), "-o", str(tmp_path / "opt.so"),
                           str(tmp_path / "opt.cpp")])
    lib = C.CDLL(str(tmp_path / "opt.so"))
    lib.ask.argtypes, lib.has.argtypes, lib.has.restype = [C.c_size_t, C.c_int, C.c_size_t, C.c_int, C.c_int], [C.c_size_t, C.c_int], C.c_size_t
    return lib


def test_a_smaller_call_takes_nothing_away_however_many_kernels_and_devices_there_are(runtime):
    places = [(k, d) for d in range(16) for k in range(1, 41)]
    for k, d in places:
        assert runtime.ask(k, d, 100000 + k, 0, 0) == 0
    for k, d in places:
        assert runtime.ask(k, d, 30000, 0, 0) == 0
    assert all(runtime.has(k, d) == 100000 + k for k, d in places)


def test_what_has_been_asked_for_is_not_asked_again(runtime):
    for smem, clusters, made in [(0, 0, 0), (50000, 0, 1), (50000, 0, 1), (60000, 1, 3), (60000, 1, 3), (0, 1, 3), (0, 0, 3)]:
        assert runtime.ask(1, 0, smem, clusters, 0) == 0 and runtime.made() == made


def test_what_was_refused_is_asked_again(runtime):
    assert runtime.ask(1, 0, 50000, 0, 7) == 7 and runtime.ask(1, 0, 0, 1, 7) == 7
    assert runtime.ask(1, 0, 50000, 1, 0) == 0 and runtime.made() == 4 and runtime.has(1, 0) == 50000

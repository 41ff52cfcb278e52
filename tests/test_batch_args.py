"""What the entry points for a batch served together refuse, and the bytes they ask of each buffer (csrc/batch_args.h, compiled alone): on the CPU."""

import ctypes as C
import subprocess

import pytest

from yule_b200 import _lib

INVALID, UNSUPPORTED = 1, 4
SOURCE = r"""
#include <cstdarg>
#include <cstdio>
#include "batch_args.h"
static char text[512];
namespace yule {
int32_t fail(int32_t code, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof(text), fmt, ap);
    va_end(ap);
    return code;
}
}
extern "C" {
const char *said() { return text; }
int32_t prefix(const yule_prefix_attention *s, size_t *n) { return yule::check_prefix_attention(s, reinterpret_cast<yule::PrefixNeeds *>(n)); }
int32_t adapters(const yule_adapters *s, size_t *n) { return yule::check_adapters(s, reinterpret_cast<yule::AdapterNeeds *>(n)); }
int32_t verification(const yule_verification *s, int32_t draft, size_t *n) { return yule::check_verification(s, draft != 0, reinterpret_cast<yule::VerifyNeeds *>(n)); }
}
"""


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    import os
    here = tmp_path_factory.mktemp("args")
    (here / "args.cpp").write_text(SOURCE)
    csrc = os.path.join(_lib.HERE, "csrc")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", csrc, "-o", str(here / "args.so"), str(here / "args.cpp")])
    lib = C.CDLL(str(here / "args.so"))
    lib.said.restype = C.c_char_p
    return lib


def asked(checks, kind, shape, draft=1):
    need = (C.c_size_t * 8)()
    args = [C.byref(shape) if shape is not None else None] + ([draft] if kind == "verification" else []) + [need]
    rc = getattr(checks, kind)(*args)
    return rc, list(need), checks.said().decode()


def prefix(**over):
    return _lib.PrefixAttention(**{**dict(head_dim=128, n_heads=32, n_kv_heads=8, prefix_len=100, n_seqs=3, n_query=2, tail_capacity=40, q_stride=4096, out_stride=4100,
                                          prefix_stride=1024, tail_stride=1028), **over})


def adapters(**over):
    return _lib.Adapters(**{**dict(gguf_type=1, n_adapters=3, max_rank=16, n_rows=100, n_cols=64, batch=5, x_stride=68, out_stride=101), **over})


def verification(**over):
    return _lib.Verification(**{**dict(vocab_size=1000, n_seqs=3, n_draft=4, target_stride=1001, draft_stride=1002, temperature=0.7, greedy=0), **over})


def test_bytes_of_prefix_attention(checks):
    rc, need, _ = asked(checks, "prefix", prefix())
    assert rc == 0 and need[:5] == [4 * 6 * 4096, 4 * (5 * 4100 + 4096), 4 * 100 * 1024, 4 * (119 * 1028 + 1024), 12]
    rc, need, _ = asked(checks, "prefix", prefix(prefix_len=0, tail_capacity=0, prefix_stride=0, tail_stride=0))
    assert rc == 0 and need[2:5] == [0, 0, 0]


@pytest.mark.parametrize("over,word", [
    (dict(n_heads=0), "shape"), (dict(n_kv_heads=0), "shape"), (dict(n_heads=30), "shape"), (dict(n_seqs=0), "shape"), (dict(head_dim=0), "head_dim"),
    (dict(head_dim=130), "head_dim"), (dict(head_dim=260), "head_dim"), (dict(n_query=0), "query"), (dict(n_query=65), "query"), (dict(q_stride=4092), "strides"),
    (dict(out_stride=4092), "strides"), (dict(prefix_stride=1020), "strides"), (dict(tail_stride=1020), "strides"), (dict(q_stride=4097), "strides"),
    (dict(out_stride=4098), "strides"), (dict(prefix_stride=1025), "strides"), (dict(tail_stride=1030), "strides"), (dict(n_seqs=0xFFFFFFFF), "positions"), (dict(n_seqs=0xFFFFFFFF, tail_capacity=0), "rows"),
    (dict(prefix_len=0x80000000), "positions"), (dict(tail_capacity=0xFFFFFFFF), "positions")])
def test_refusals_of_prefix_attention(checks, over, word):
    rc, _, said = asked(checks, "prefix", prefix(**over))
    assert rc == INVALID and word in said


def test_products_do_not_come_out_small(checks):
    for kind, shape in (("prefix", prefix(n_seqs=1 << 12, n_heads=8, tail_capacity=0x7FFFF, tail_stride=0xFFFFFFFC)), ("adapters", adapters(n_adapters=0xFFFFFFFF, n_cols=0xFFFFFFFC, x_stride=0xFFFFFFFC)),
                        ("verification", verification(target_stride=0xFFFFFFFF, n_seqs=65536, n_draft=256))):
        rc, need, _ = asked(checks, kind, shape)
        assert rc == 0 and max(need) >= 1 << 56


def test_bytes_of_adapters(checks):
    rc, need, _ = asked(checks, "adapters", adapters())
    assert rc == 0 and need[:6] == [2 * 48 * 64, 2 * 300 * 16, 12, 20, 4 * (4 * 68 + 64), 4 * (4 * 101 + 100)]
    assert asked(checks, "adapters", adapters(gguf_type=0))[1][:2] == [4 * 48 * 64, 4 * 300 * 16]


@pytest.mark.parametrize("over,code", [
    (dict(gguf_type=12), UNSUPPORTED), (dict(gguf_type=30), UNSUPPORTED), (dict(n_adapters=0), INVALID), (dict(max_rank=0), INVALID), (dict(max_rank=257), INVALID),
    (dict(n_cols=0, x_stride=0), INVALID), (dict(n_cols=62), INVALID), (dict(n_rows=0), INVALID), (dict(n_rows=(1 << 23) + 1, out_stride=1 << 24), INVALID), (dict(batch=0), INVALID),
    (dict(batch=0xFFFFFFFF), INVALID), (dict(x_stride=60), INVALID), (dict(x_stride=66), INVALID), (dict(out_stride=99), INVALID)])
def test_refusals_of_adapters(checks, over, code):
    assert asked(checks, "adapters", adapters(**over))[0] == code


def test_bytes_of_verification(checks):
    rc, need, _ = asked(checks, "verification", verification())
    assert rc == 0 and need[:5] == [4 * (14 * 1001 + 1000), 4 * (11 * 1002 + 1000), 48, 60, 12]
    assert asked(checks, "verification", verification(), draft=0)[1][1] == 0
    assert asked(checks, "verification", verification(greedy=1, temperature=0.0))[:2] == (0, [4 * (14 * 1001 + 1000), 0, 48, 60, 12, 0, 0, 0])
    assert asked(checks, "verification", verification(draft_stride=0), draft=0)[0] == 0


@pytest.mark.parametrize("over", [dict(vocab_size=0), dict(vocab_size=(1 << 24) + 1, target_stride=1 << 25, draft_stride=1 << 25), dict(n_seqs=0), dict(n_seqs=65537), dict(n_draft=0),
                                  dict(n_draft=257), dict(target_stride=999), dict(draft_stride=999), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=1e-7),
                                  dict(temperature=float("nan")), dict(temperature=float("inf"))])
def test_refusals_of_verification(checks, over):
    rc, _, said = asked(checks, "verification", verification(**over))
    assert rc == INVALID and said


@pytest.mark.parametrize("kind", ["prefix", "adapters", "verification"])
def test_no_shape_is_refused(checks, kind):
    assert asked(checks, kind, None)[0] == INVALID


def test_entry_points_without_a_context(native_libs):
    lib = _lib.cuda_lib()
    assert lib.yule_cuda_prefix_attention(None, 1, 1, 1, 1, 1, 1, 1, C.byref(prefix())) == INVALID
    assert lib.yule_cuda_adapter_matmul_batched(None, 1, 1, 1, 1, 1, 1, 1, 1, C.byref(adapters())) == INVALID
    assert lib.yule_cuda_verify_drafts(None, 1, 1, 1, 1, 1, 1, 1, C.byref(verification())) == INVALID
    assert lib.yule_cuda_buffer_address(None, 1, C.byref(C.c_uint64())) == INVALID

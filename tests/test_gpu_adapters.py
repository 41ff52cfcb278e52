"""Low-rank adapters beside a projection (csrc/adapters.cu) against their formula in 64 bits.

Tolerance.  A product of fp32 numbers is off by at most 2^-20 of its size on the tensor core, a sum of some tens of products in 24 bits by less than 2^-19 of the sum of
their sizes, and there are two such sums one behind the other: 2^-17 of Σ_k |up| Σ_c |down| |x| · |scale|, and half a step of the output."""

import os
import subprocess
import sys

import numpy as np
import pytest

from yule_b200 import CudaB200Backend, DType, YuleGpuError, synth

pytestmark = pytest.mark.gpu
NONE = 0xFFFFFFFF


class Call:
    def __init__(self, batch=5, rows=64, cols=128, adapters=3, rank=16, dtype=DType.F16, ids=None, ranks=None, seed=0, pad_x=0, pad_out=0, in_place=False):
        r = np.random.default_rng(seed)
        self.n = dict(batch=batch, rows=rows, cols=cols, adapters=adapters, rank=rank)
        self.dtype, self.pad_x, self.pad_out, self.in_place = dtype, pad_x, pad_out, in_place
        t = np.float16 if dtype == DType.F16 else np.float32
        f = lambda *s: r.standard_normal(s).astype(np.float32)  # noqa: E731
        self.down, self.up = (f(adapters, rank, cols) / np.sqrt(cols)).astype(t), f(adapters, rows, rank).astype(t)
        self.scales, self.x, self.base = f(adapters), f(batch, cols), f(batch, rows)
        self.ranks = np.asarray(ranks if ranks is not None else r.integers(0, rank + 1, adapters), np.uint32)
        self.ids = np.asarray(ids if ids is not None else np.where(r.random(batch) < 0.2, NONE, r.integers(0, adapters, batch)), np.uint32)

    def upload(self, b):
        def wide(a, pad, fill):
            return np.concatenate([a, np.full((len(a), pad), fill, np.float32)], 1)

        self.h = {n: b.upload(getattr(self, n)) for n in ("down", "up", "ranks", "scales", "ids")}
        self.h["x"] = b.upload(wide(self.x, self.pad_x, np.nan))
        self.h["base"] = b.upload(np.append(wide(self.base, self.pad_out, 7.0), np.full(64, 7.0, np.float32)))
        self.h["out"] = self.h["base"] if self.in_place else b.upload(np.full(self.base.size + self.pad_out * len(self.base) + 64, 7.0, np.float32))
        return self

    def run(self, b):
        n, h = self.n, self.h
        b.adapter_matmul_batched(h["down"], h["up"], h["ranks"], h["scales"], h["ids"], h["x"], h["base"], h["out"], n["rows"], n["cols"], self.dtype, n["adapters"], n["rank"],
                                 n["batch"], x_stride=n["cols"] + self.pad_x, out_stride=n["rows"] + self.pad_out)

    def got(self, b):
        n, width = self.n, self.n["rows"] + self.pad_out
        a = b.download(self.h["out"], n["batch"] * width + 64)
        assert (a[n["batch"] * width:] == 7).all()
        a = a[:n["batch"] * width].reshape(n["batch"], width)
        assert (a[:, n["rows"]:] == 7).all()
        return a[:, :n["rows"]]

    def reference(self):
        out, tol = self.base.astype(np.float64), np.zeros(self.base.shape)
        for i, a in enumerate(self.ids):
            if a < self.n["adapters"]:
                r = min(int(self.ranks[a]), self.n["rank"])
                d, u, x, s = self.down[a, :r].astype(np.float64), self.up[a, :, :r].astype(np.float64), self.x[i].astype(np.float64), float(self.scales[a])
                out[i] += s * (u @ (d @ x))
                tol[i] = 2.0 ** -17 * abs(s) * (np.abs(u) @ (np.abs(d) @ np.abs(x)))
        return out, tol + 2.0 ** -23 * np.abs(out)

    def check(self, b):
        got, (out, tol) = self.got(b), self.reference()
        assert np.isfinite(got).all() and (np.abs(got - out) <= tol).all(), np.abs(got - out).max()
        none = self.ids >= self.n["adapters"]
        assert (got[none] == self.base[none]).all()

    def free(self, b):
        for h in {h.id: h for h in self.h.values()}.values():
            b.free(h)


def go(b, **kw):
    c = Call(**kw).upload(b)
    c.run(b)
    c.check(b)
    c.free(b)


BOTH = pytest.mark.parametrize("dtype", [DType.F16, DType.F32])


@BOTH
@pytest.mark.parametrize("rank", [1, 3, 4, 7, 8, 12, 16, 17, 32, 50, 64, 65, 128, 256])
def test_ranks(backend, dtype, rank):
    go(backend, dtype=dtype, rank=rank, seed=rank)
    go(backend, dtype=dtype, rank=rank, batch=134, rows=33, seed=rank, ranks=[rank, max(1, rank - 1), (rank + 1) // 2])


@BOTH
@pytest.mark.parametrize("rows,cols", [(1, 4), (3, 8), (31, 12), (32, 60), (33, 64), (128, 68), (129, 256), (130, 260), (1000, 2560), (2048, 5632)])
def test_projections(backend, dtype, rows, cols):
    go(backend, dtype=dtype, rows=rows, cols=cols, seed=rows)
    go(backend, dtype=dtype, rows=rows, cols=cols, batch=129, seed=rows)


@BOTH
@pytest.mark.parametrize("batch", [1, 2, 7, 8, 9, 31, 32, 33, 64, 65, 127, 128, 129, 159, 160, 161, 257])
def test_batches(backend, dtype, batch):
    go(backend, dtype=dtype, batch=batch, adapters=40, seed=batch)
    go(backend, dtype=dtype, batch=batch, adapters=2, seed=batch, in_place=True)


@pytest.mark.parametrize("batch", [1100, 1700, 2500, 4800])
def test_long_prompts(backend, batch):
    """As many CTAs to a tile as are there at once: from eight down to one; rows of an adapter in runs, and mixed ones at the start."""
    ids = np.arange(batch) * 7 // batch
    ids[:50] = np.arange(50) % 8
    go(backend, batch=batch, rows=260, cols=320, adapters=7, rank=20, ids=ids, seed=batch)


@BOTH
def test_large_adapters_of_few_requests(backend, dtype):
    go(backend, dtype=dtype, batch=12, rows=4100, cols=4096, adapters=9, rank=64)


@pytest.mark.parametrize("batch", [6, 164])
def test_order_of_the_rows_does_not_matter(backend, batch):
    """Neighbours of one adapter, all of one, all different, none at all."""
    for ids in (np.zeros(batch), np.arange(batch) % 50, np.full(batch, NONE), np.arange(batch) // 3, np.where(np.arange(batch) % 2, 49, 50), (np.arange(batch) * 7) % 51):
        go(backend, batch=batch, adapters=50, ids=ids)
        go(backend, batch=batch, adapters=50, ids=ids, in_place=True)


@pytest.mark.parametrize("batch", [5, 141])
def test_strides(backend, batch):
    """Rows of x, base and output further apart than they are long (vectors of four or not), NaN and marks between them."""
    for pad_out in (0, 1, 4, 6):
        go(backend, batch=batch, pad_x=8, pad_out=pad_out, rows=60)
        go(backend, batch=batch, pad_x=4, pad_out=pad_out, rows=61, in_place=True)


@BOTH
@pytest.mark.parametrize("batch", [5, 141])
def test_what_lies_beyond_a_rank_does_not_count(backend, dtype, batch):
    for rank in (16, 18):
        c = Call(batch=batch, dtype=dtype, rank=rank, ranks=[0, 5, 14], adapters=3)
        for a, r in enumerate(c.ranks):
            c.down[a, r:], c.up[a, :, r:] = np.nan, np.inf
        c.upload(backend).run(backend)
        c.check(backend)
        c.free(backend)


@pytest.mark.parametrize("batch", [5, 141])
def test_a_row_that_is_not_finite_stays_by_itself(backend, batch):
    c = Call(batch=batch, ids=np.arange(batch) % 3, ranks=[16, 16, 16])
    clean = c.reference()
    c.x[3, 7] = np.nan
    c.x[4, 100] = np.inf
    c.upload(backend).run(backend)
    got = c.got(backend)
    rest = np.setdiff1d(np.arange(batch), [3, 4])
    assert not np.isfinite(got[3]).any() and not np.isfinite(got[4]).any()
    assert (np.abs(got - clean[0]) <= clean[1])[rest].all()


@BOTH
def test_sizes(backend, dtype):
    """Inputs of very different sizes in one batch, and within a row."""
    for batch in (5, 141):
        c = Call(batch=batch, dtype=dtype, cols=512)
        c.x *= (10.0 ** np.linspace(-25, 25, batch)).astype(np.float32)[:, None]
        c.x[:, ::3] *= np.float32(2.0 ** -12)
        c.base[:] = 0
        c.upload(backend).run(backend)
        c.check(backend)
        c.free(backend)


@BOTH
@pytest.mark.parametrize("batch", [5, 141])
def test_sizes_within_a_rank(backend, dtype, batch):
    """Rows of `down` of very different sizes against columns of `up` that bring their products back to one size, in some adapters and some rows only."""
    c = Call(batch=batch, dtype=dtype, rank=40, ranks=[40, 33, 40], cols=256)
    size = (2.0 ** np.linspace(-11, 11, 40)).astype(np.float32)
    for a in (0, 1):
        c.down[a] = (c.down[a].astype(np.float32) * size[:, None]).astype(c.down.dtype)
        c.up[a] = (c.up[a].astype(np.float32) / size[None]).astype(c.up.dtype)
    c.x[::3, :] = 0
    c.x[::3, 5] = 1
    c.base[:] = 0
    c.upload(backend).run(backend)
    c.check(backend)
    c.free(backend)


@BOTH
@pytest.mark.parametrize("batch", [9, 200])
def test_errors_have_no_sign(backend, dtype, batch):
    """Two products one behind the other.  A sum on the tensor core is cut off at most eight times, by 2^-24 of what it has by then in the mean, two thirds of the whole: 2^-21.6 in each product,
    2^-20.6 in both, and what is rounded on either side adds up in squares.  Products that were all short by 2^-22 (F32: twice that) would leave as much in every output."""
    c = Call(batch=batch, rows=512, cols=4096, rank=64, ranks=[64, 64, 64], dtype=dtype, ids=np.arange(batch) % 3)
    c.base[:] = 0
    c.upload(backend).run(backend)
    out, _ = c.reference()
    assert np.linalg.norm(c.got(backend) - out) <= 2.0 ** -20.5 * np.linalg.norm(out)
    c.free(backend)


def test_ranks_beyond_the_largest_count_as_it(backend):
    go(backend, ranks=[17, NONE, 16])


def test_same_bits_again(backend):
    for batch in (9, 214):
        c = Call(batch=batch, rows=500, cols=1024).upload(backend)
        c.run(backend)
        first = c.got(backend)
        for _ in range(4):
            c.run(backend)
            assert (c.got(backend) == first).all()


def test_captured_and_replayed_with_other_adapters(backend):
    c = Call(batch=6, in_place=False).upload(backend)
    c.run(backend)
    backend.graph_begin()
    c.run(backend)
    g = backend.graph_end()
    for ids in ([0, 1, 2, 0, 1, 2], [NONE, 2, 2, 2, 1, NONE]):
        c.ids = np.array(ids, np.uint32)
        backend.copy_to_device(c.ids, c.h["ids"])
        backend.graph_launch(g)
        c.check(backend)
    backend.graph_destroy(g)


def test_beside_a_quantised_projection(backend):
    """The projection's output is the base, in place, in the chain of launches; then another projection reads the sum."""
    rows, cols, batch = 256, 256, 3
    w = synth.random_blocks(DType.Q8_0, 3, rows * cols // 32, 0.02)
    c = Call(batch=batch, rows=rows, cols=cols, in_place=True, ids=[0, NONE, 2])
    wh, y2 = backend.upload(w), backend.allocate(batch * rows * 4)
    c.upload(backend)
    plain, deq = backend.allocate(batch * rows * 4), backend.allocate(rows * cols * 4)
    backend.dequantize(wh, DType.Q8_0, rows * cols // 32, deq)
    W = backend.download(deq, rows * cols).reshape(rows, cols).astype(np.float64)
    for _ in range(20):
        backend.quantized_matmul_batched(wh, c.h["x"], plain, rows, cols, DType.Q8_0, batch)
        backend.copy_buffer(plain, c.h["out"], batch * rows * 4)
        c.run(backend)
        backend.quantized_matmul_batched(wh, c.h["out"], y2, rows, cols, DType.Q8_0, batch)
    c.base = backend.download(plain, batch * rows).reshape(batch, rows)
    out, tol = c.reference()
    got = c.got(backend)
    assert (np.abs(got - out) <= tol).all()
    second = backend.download(y2, batch * rows).reshape(batch, rows)
    assert np.abs(second - got.astype(np.float64) @ W.T).max() <= 1e-5 * (np.abs(got) @ np.abs(W).T).max()


def test_a_small_call_does_not_take_room_from_a_larger_one():
    """The first calls of a process: sixteen CTAs with little shared memory, then eight with more."""
    code = ("import sys; sys.path[:0] = [{!r}, {!r}]\nfrom test_gpu_adapters import CudaB200Backend, go\nb = CudaB200Backend(0)\n"
            "for n, rank in ((1, 1), (91, 16), (1, 17), (91, 50), (8, 256), (100, 256)):\n    go(b, batch=n, rank=rank, adapters=12)\n")
    here = os.path.dirname(os.path.abspath(__file__))
    subprocess.run([sys.executable, "-c", code.format(here, os.path.dirname(here))], check=True, timeout=300)


def test_refusals(backend):
    c = Call().upload(backend)
    good = [c.h["down"], c.h["up"], c.h["ranks"], c.h["scales"], c.h["ids"], c.h["x"], c.h["base"], c.h["out"], 64, 128, DType.F16, 3, 16, 5]
    small = backend.allocate(4)

    def refused(code, at, value):
        args = list(good)
        args[at] = value
        with pytest.raises(YuleGpuError) as e:
            backend.adapter_matmul_batched(*args)
        assert e.value.code == code

    for at in range(8):
        refused(3, at, small)
    for at in range(6):
        refused(1, at, c.h["out"])
    refused(4, 10, DType.Q4_K)
    refused(3, 10, DType.F32)
    refused(1, 12, 300)
    refused(1, 13, 0)
    c.run(backend)
    c.check(backend)


def test_a_capture_cannot_grow_the_scratch():
    b = CudaB200Backend(0)
    c = Call(batch=134).upload(b)
    b.graph_begin()
    with pytest.raises(YuleGpuError, match="outside the capture"):
        c.run(b)
    b.graph_destroy(b.graph_end())
    c.run(b)
    c.check(b)
    b.close()

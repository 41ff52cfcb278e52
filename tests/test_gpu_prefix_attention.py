"""Attention of a batch behind a shared prefix (csrc/prefix_attention.cu) against its formula in 64 bits.

Tolerance.  A product of fp32 numbers is off by at most 2^-20 of its size on the tensor core (hi and lo of 11 bits each), and sums of some tens of products in 24 bits by
less than 2^-19 of the sum of their sizes.  So a score is off by at most ds = 2^-18 · Σ|q_i k_i| / sqrt(hd), a probability by 2 ds of itself and the
soft-max's own rounding, 2^-20 in all, and an output by (4 ds + 2^-18) of the largest |v| that its row sees."""

import numpy as np
import pytest

from yule_b200 import CudaB200Backend, YuleGpuError

pytestmark = pytest.mark.gpu


# Which kernels: by the rules, parts of prefix and own positions, all of a sequence in a CTA (where there is one query token), the prefix on the tensor core behind or before the
# sequences' own positions.
ROUTES = {"rules": {}, "parts": {"YULE_PREFIX_TC": "0", "YULE_PREFIX_SINGLE": "0"}, "single": {"YULE_PREFIX_TC": "0", "YULE_PREFIX_SINGLE": "1"}, "own first": {"YULE_PREFIX_TC": "1", "YULE_PREFIX_OWN_FIRST": "1"}, "own last": {"YULE_PREFIX_TC": "1", "YULE_PREFIX_OWN_FIRST": "0"}}


@pytest.fixture(autouse=True, params=ROUTES)
def route(request, monkeypatch):
    for name, value in ROUTES[request.param].items():
        monkeypatch.setenv(name, value)
    return request.param


def reference(q, pk, pv, tk, tv, lens):
    """q [B][T][H][hd], pk, pv [P][kv][hd], tk, tv [B][C][kv][hd] → (out, tolerance) [B][T][H][hd], [B][T][H]."""
    q, pk, pv, tk, tv = (np.asarray(a, np.float64) for a in (q, pk, pv, tk, tv))
    B, T, H, hd = q.shape
    group = H // pk.shape[1]
    out, tol = np.zeros(q.shape), np.zeros(q.shape[:3])
    for b in range(B):
        for t in range(T):
            n = max(0, min(int(lens[b]), tk.shape[1]) - (T - 1 - t))
            k, v = np.concatenate([pk, tk[b, :n]]), np.concatenate([pv, tv[b, :n]])
            if not len(k):
                continue
            x = q[b, t].reshape(-1, group, hd)
            s = np.einsum("kgd,jkd->kgj", x, k) / np.sqrt(hd)
            size = np.einsum("kgd,jkd->kgj", np.abs(x), np.abs(k)).max(-1).reshape(H) / np.sqrt(hd)
            e = np.exp(s - s.max(-1, keepdims=True))
            out[b, t] = np.einsum("kgj,jkd->kgd", e / e.sum(-1, keepdims=True), v).reshape(H, hd)
            tol[b, t] = (4 * 2.0 ** -18 * size + 2.0 ** -18) * np.abs(v).max(axis=(0, 2)).repeat(group)
    return out, tol


class Call:
    def __init__(self, B=3, T=1, H=8, kv=2, hd=64, P=70, C=50, lens=None, seed=0, spread=1.0, pad=0):
        r = np.random.default_rng(seed)
        self.n = dict(B=B, T=T, H=H, kv=kv, hd=hd, P=P, C=C)
        self.pad = pad  # floats between rows
        f = lambda *s: r.standard_normal(s).astype(np.float32)  # noqa: E731
        self.q, self.pk, self.pv, self.tk, self.tv = f(B, T, H, hd) * np.float32(spread), f(P, kv, hd), f(P, kv, hd), f(B, C, kv, hd), f(B, C, kv, hd)
        self.lens = np.asarray(lens if lens is not None else r.integers(0, C + 1, B), np.uint32)

    def padded(self, a, rows):
        a = a.reshape(rows, -1)
        return np.concatenate([a, np.full((rows, self.pad), np.nan, np.float32)], 1) if self.pad else a

    def upload(self, b):
        n = self.n
        rows = dict(q=n["B"] * n["T"], pk=n["P"], pv=n["P"], tk=n["B"] * n["C"], tv=n["B"] * n["C"])
        self.h = {k: b.upload(self.padded(getattr(self, k), r)) if r and getattr(self, k).size else None for k, r in rows.items()}
        self.h["lens"] = b.upload(self.lens)
        self.out_floats = n["B"] * n["T"] * (n["H"] * n["hd"] + self.pad)
        self.h["out"] = b.upload(np.full(self.out_floats + 64, 7.0, np.float32))
        return self

    def run(self, b):
        n, h, pad = self.n, self.h, self.pad
        b.prefix_attention(h["q"], h["pk"], h["pv"], h["tk"], h["tv"], h["lens"], h["out"], n["hd"], n["H"], n["kv"], n["P"], n["B"], n["C"], n_query=n["T"],
                           q_stride=n["H"] * n["hd"] + pad, out_stride=n["H"] * n["hd"] + pad, prefix_stride=n["kv"] * n["hd"] + pad, tail_stride=n["kv"] * n["hd"] + pad)

    def got(self, b):
        """The output; what lies between its rows and behind them has to be as it was."""
        n = self.n
        a = b.download(self.h["out"], self.out_floats + 64)
        assert (a[self.out_floats:] == 7).all()
        a = a[:self.out_floats].reshape(n["B"] * n["T"], -1)
        assert (a[:, n["H"] * n["hd"]:] == 7).all()
        return a[:, :n["H"] * n["hd"]].reshape(n["B"], n["T"], n["H"], n["hd"])

    def check(self, b):
        out, tol = reference(self.q, self.pk, self.pv, self.tk, self.tv, self.lens)
        got = self.got(b)
        assert np.isfinite(got).all()
        assert (np.abs(got - out).max(-1) <= tol).all(), np.abs(got - out).max()

    def free(self, b):
        for h in self.h.values():
            if h:
                b.free(h)


def go(b, **kw):
    c = Call(**kw).upload(b)
    c.run(b)
    c.check(b)
    c.free(b)


@pytest.mark.parametrize("H,kv,hd", [(4, 4, 32), (8, 2, 64), (32, 4, 64), (20, 5, 96), (12, 2, 80), (32, 8, 128), (64, 8, 128), (3, 1, 4), (7, 1, 36), (8, 2, 160), (6, 3, 256)])
def test_head_layouts(backend, H, kv, hd):
    go(backend, H=H, kv=kv, hd=hd, B=3, P=77, C=33, lens=[33, 0, 17])
    go(backend, H=H, kv=kv, hd=hd, B=2, T=3, P=130, C=70, lens=[70, 2])


@pytest.mark.parametrize("P,C", [(0, 1), (1, 0), (1, 1), (15, 16), (16, 17), (63, 64), (64, 65), (65, 127), (0, 300), (1000, 0), (2049, 129)])
def test_lengths(backend, P, C):
    go(backend, B=2, P=P, C=C, lens=[C, C // 2], seed=P + C)
    go(backend, B=1, T=4, P=P, C=C, lens=[C], seed=P + C)


@pytest.mark.parametrize("T", [1, 2, 5, 8, 17, 64])
def test_query_tokens(backend, T):
    """Rows of drafts see what came before them; sequences shorter than their query tokens have rows that see nothing of their own."""
    go(backend, B=5, T=T, P=40, C=90, lens=[0, 1, min(T, 90), min(T + 1, 90), 90], seed=T)
    go(backend, B=5, T=T, P=0, C=90, lens=[0, 1, min(T, 90), min(T + 1, 90), 90], seed=T)


@pytest.mark.parametrize("B", [1, 2, 7, 16, 33, 64, 130])
def test_batches(backend, B):
    go(backend, B=B, H=8, kv=2, hd=64, P=300, C=40, seed=B)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("P", [64, 65, 95, 96, 97, 127, 128, 129, 200, 777, 4097, 20000])
def test_many_rows(backend, hd, P):
    """Enough query rows for 128 at a time: one tile of positions, several, a last one of few; rows that do not fill their 128."""
    go(backend, B=11, T=1, H=8, kv=2, hd=hd, P=P, C=20, seed=P)
    go(backend, B=45, T=2, H=3, kv=1, hd=hd, P=P, C=0, lens=np.zeros(45), seed=P)


@pytest.mark.parametrize("where", ["pk", "pv"])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_a_prefix_that_is_not_finite(backend, where, value):
    """Every row sees it: what is not finite in K makes no row finite, in V no row's dimension, and other KV heads are as they were."""
    c = Call(B=20, H=8, kv=2, hd=128, P=300, C=20)
    clean = reference(c.q, c.pk, c.pv, c.tk, c.tv, c.lens)
    getattr(c, where)[150, 0, 5] = value
    c.upload(backend).run(backend)
    got = c.got(backend)
    assert not np.isfinite(got[:, :, :4]).all(-1).any()
    assert (np.abs(got - clean[0]).max(-1) <= clean[1])[:, :, 4:].all()
    if where == "pv":
        assert not np.isfinite(got[:, :, :4, 5]).any()


@pytest.mark.parametrize("where", ["tk", "tv"])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("T,hd", [(1, 64), (4, 64), (5, 96), (3, 160)])
def test_own_positions_that_are_not_finite(backend, where, value, T, hd):
    """One that all of a sequence's query tokens see, and each of the newest ones: the rows that see it are not finite (K: no number of them, whatever the sign of the query's
    element), the others as they were."""
    n = 40
    c = Call(B=2, T=T, H=8, kv=2, hd=hd, P=30, C=50, lens=[n, 20])
    c.q[:, :, ::2, 5], c.q[:, :, 1::2, 5] = 1.5, -1.5  # (of either sign against the position's element)
    clean = reference(c.q, c.pk, c.pv, c.tk, c.tv, c.lens)
    c.upload(backend)
    for j in [3] + list(range(n - T, n)):
        bad = getattr(c, where).copy()
        bad[0, j, 0, 5] = value
        backend.copy_to_device(bad, c.h[where])
        c.run(backend)
        got = c.got(backend)
        sees = max(0, j - (n - T))  # the first query token that does
        rows = got[0, sees:, :4]
        assert not np.isfinite(rows if where == "tk" else rows[..., 5]).any()
        rest = np.ones(got.shape[:3], bool)
        rest[0, sees:, :4] = False
        assert (np.abs(got - clean[0]).max(-1) <= clean[1])[rest].all()
    c.free(backend)


def test_larger(backend):
    go(backend, B=32, H=32, kv=8, hd=128, P=2048, C=200, seed=1)
    go(backend, B=40, T=3, H=16, kv=2, hd=128, P=1111, C=99, seed=2)


@pytest.mark.parametrize("T,hd", [(1, 128), (1, 96), (3, 64), (8, 128)])
def test_errors_have_no_sign(backend, T, hd):
    """Over many positions.  Rounded terms are off by up to 2^-22 of a product on either side, a score of up to 16 in 32 bits by 2^-21: 2^-20 of the output's norm, where products that
    are all short by 2^-22 would add 2^-22 times the score of 8 to 16 to every probability on one side."""
    c = Call(B=2, T=T, H=8, kv=2, hd=hd, P=5000, C=300, lens=[300, 150], spread=1.3, seed=T)
    c.pk += np.random.default_rng(9).standard_normal(c.pk.shape[1:]).astype(np.float32)
    c.upload(backend).run(backend)
    out, _ = reference(c.q, c.pk, c.pv, c.tk, c.tv, c.lens)
    assert np.linalg.norm(c.got(backend) - out) <= 2.0 ** -20 * np.linalg.norm(out)
    c.free(backend)


def test_strides(backend):
    """Rows of all tensors further apart than they are long, with NaN between them."""
    go(backend, pad=12, B=3, T=2, P=100, C=40)
    go(backend, pad=4, H=32, kv=8, hd=128, B=16, T=2, P=300, C=40)


def test_rows_that_see_nothing_are_zero(backend):
    c = Call(B=4, T=3, P=0, C=20, lens=[0, 1, 2, 20]).upload(backend)
    c.run(backend)
    c.check(backend)
    got = c.got(backend)
    assert (got[0] == 0).all() and (got[1, :2] == 0).all() and (got[2, :1] == 0).all() and (got[1, 2] != 0).any()
    c = Call(B=2, T=2, P=0, C=0, lens=[0, 0]).upload(backend)
    c.run(backend)
    assert (c.got(backend) == 0).all()


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf, 3e38, -3e38])
def test_what_is_hidden_does_not_count(backend, value):
    """Positions behind a sequence's length, and drafts that a query token does not see, hold anything."""
    c = Call(B=3, T=4, H=32, kv=8, hd=128, P=66, C=70, lens=[60, 3, 33])
    clean = reference(c.q, c.pk, c.pv, c.tk, c.tv, c.lens)
    for b, n in enumerate(c.lens):
        c.tk[b, n:] = value
        c.tv[b, n:] = value
        c.tv[b, n - 1], c.tk[b, n - 1] = value, value  # the last token's own position
    c.upload(backend).run(backend)
    got = c.got(backend)
    assert (np.abs(got - clean[0]).max(-1) <= clean[1])[:, :3].all()


def test_scores_that_lie_far_apart(backend):
    go(backend, spread=30.0, B=4, P=200, C=60)
    go(backend, spread=1e-3, B=4, P=200, C=60)


@pytest.mark.parametrize("k,v", [(1e-20, 1.0), (1e15, 1e-20), (1.0, 1e25), (1.0, 1e-30)])
def test_sizes(backend, k, v):
    """Numbers of any size, and rows of very different ones."""
    c = Call(B=17, T=1, H=32, kv=8, hd=128, P=333, C=40)
    for a, f in ((c.pk, k), (c.tk, k), (c.pv, v), (c.tv, v)):
        a *= np.float32(f)
    c.q /= np.float32(k)
    c.pv[::3] *= np.float32(2.0 ** -18)
    c.pk[::5] *= np.float32(2.0 ** -18)
    c.upload(backend).run(backend)
    c.check(backend)


@pytest.mark.parametrize("hd", [64, 128])
def test_dimensions_of_very_different_sizes(backend, hd, route):
    """Per dimension of V: its error goes by the dimension's own largest |v|, and on the tensor core, where the numbers of 64 positions of V share a scale that leaves their largest at 2^13 or
    more beside terms of fp16's 2^-24, by half a step of that: 2^-38 of the largest of all."""
    c = Call(B=20, H=8, kv=2, hd=hd, P=300, C=30)
    size = (2.0 ** -np.arange(hd)[::-1].clip(0, 26)).astype(np.float32)
    c.pv *= size
    c.tv *= size
    out, _ = reference(c.q, c.pk, c.pv, c.tk, c.tv, c.lens)
    _, of_one = reference(c.q, c.pk, np.ones_like(c.pv), c.tk, np.ones_like(c.tv), c.lens)  # tolerance where the largest is 1
    largest = np.maximum(np.abs(c.pv).max((0, 1)), np.abs(c.tv).max((0, 1, 2))).astype(np.float64)  # of a dimension
    tol = of_one[..., None] * largest + (0 if route in ("parts", "single") else 2.0 ** -38 * largest.max())
    c.upload(backend).run(backend)
    assert (np.abs(c.got(backend) - out) <= tol).all()
    c.free(backend)


def test_lengths_beyond_the_capacity(backend):
    a = Call(B=2, P=20, C=30, lens=[30, 30]).upload(backend)
    c = Call(B=2, P=20, C=30, lens=[31, 0xFFFFFFFF]).upload(backend)
    a.run(backend), c.run(backend)
    assert (a.got(backend) == c.got(backend)).all()


def test_same_bits_again_and_for_the_same_row(backend):
    c = Call(B=9, T=2, P=700, C=300, H=32, kv=8, hd=128).upload(backend)
    c.run(backend)
    first = c.got(backend)
    for _ in range(5):
        c.run(backend)
        assert (c.got(backend) == first).all()


def test_captured_and_replayed_with_other_lengths(backend):
    c = Call(B=3, T=2, P=100, C=80, lens=[10, 20, 30]).upload(backend)
    c.run(backend)
    backend.graph_begin()
    c.run(backend)
    c.run(backend)
    g = backend.graph_end()
    for lens in ([80, 1, 0], [5, 79, 42]):
        c.lens = np.array(lens, np.uint32)
        backend.copy_to_device(c.lens, c.h["lens"])
        backend.graph_launch(g)
        c.check(backend)
    backend.graph_destroy(g)


def test_graphs_captured_before_and_after_the_scratch_grew(route):
    """One replays in the scratch that it was captured with, the other in the larger one, eager calls between them."""
    b = CudaB200Backend(0)
    small, large = Call(B=3, T=2, P=100, C=80).upload(b), Call(B=33, T=2, P=600, C=200).upload(b)
    graphs = []
    for c in (small, large):
        c.run(b)
        b.graph_begin()
        c.run(b)
        graphs.append(b.graph_end())
    for first, second in ((0, 1), (1, 0)):
        for c in (small, large):
            b.copy_to_device(np.full(c.out_floats, 7.0, np.float32), c.h["out"])
        b.graph_launch(graphs[first])
        b.graph_launch(graphs[second])
        small.check(b), large.check(b)
        small.run(b), large.run(b)
    for g in graphs:
        b.graph_destroy(g)
    b.close()


def test_a_capture_cannot_grow_the_scratch(route):
    if route == "single":
        pytest.skip("no scratch")
    b = CudaB200Backend(0)
    c = Call(B=3, P=100, C=80).upload(b)
    b.graph_begin()
    with pytest.raises(YuleGpuError, match="outside the capture"):
        c.run(b)
    b.graph_destroy(b.graph_end())
    c.run(b)
    c.check(b)
    b.close()


def test_offsets_beyond_32_bits(backend):
    """Own caches of 2^33 bytes and more each: the last sequence's rows lie behind 2^31 floats."""
    B, C, kv, hd = 3, 1 << 18, 32, 128
    rng = np.random.default_rng(5)
    q = rng.standard_normal((B, 1, kv, hd)).astype(np.float32)
    lens = np.array([1, 2, 40], np.uint32)
    bytes_ = B * C * kv * hd * 4
    tk, tv = backend.allocate(bytes_), backend.allocate(bytes_)
    rows = rng.standard_normal((2, B, 40, kv, hd)).astype(np.float32)
    small = [backend.upload(rows[i, b]) for i in range(2) for b in range(B)]
    for i, to in enumerate((tk, tv)):
        for b in range(B):
            backend.copy_buffer_offset(small[i * B + b], to, 0, b * C * kv * hd * 4, 40 * kv * hd * 4)
    h = [backend.upload(q), backend.upload(lens), backend.allocate(q.nbytes)]
    backend.prefix_attention(h[0], None, None, tk, tv, h[1], h[2], hd, kv, kv, 0, B, C)
    out, tol = reference(q, np.zeros((0, kv, hd)), np.zeros((0, kv, hd)), rows[0], rows[1], lens)
    assert (np.abs(backend.download(h[2], q.size).reshape(q.shape) - out).max(-1) <= tol).all()
    for x in [tk, tv] + small + h:
        backend.free(x)


def test_a_prefix_whose_operands_come_in_pieces(backend, route):
    """70000 positions of 16 heads of 64: 573 MB as the tensor core reads them, of which 512 are in memory at a time."""
    if not route.startswith("own"):
        pytest.skip("no operands")
    go(backend, B=2, H=16, kv=16, hd=64, P=70000, C=10)


def test_more_rows_than_one_grid_of_the_tensor_core_takes(backend, route):
    """8392704 query rows of a KV head, 2.1 GB: zeros (every output is the mean of V) but for some rows."""
    if route not in ("rules", "own first"):
        pytest.skip("the same kernels")
    B, T, H, hd, P = 2049, 64, 64, 64, 3
    rng = np.random.default_rng(6)
    pk, pv = (rng.standard_normal((P, 1, hd)).astype(np.float32) for _ in range(2))
    rows, floats = B * T * H, B * T * H * hd
    q, out = backend.allocate(floats * 4), backend.allocate(floats * 4)
    at = [0, 8388480 - 8, 8388480, rows - 8]  # eights of rows
    x = rng.standard_normal((len(at), 8, hd)).astype(np.float32)
    small = backend.upload(x)
    for i, row in enumerate(at):
        backend.copy_buffer_offset(small, q, i * 8 * hd * 4, row * hd * 4, 8 * hd * 4)
    h = [backend.upload(pk), backend.upload(pv)]
    backend.prefix_attention(q, h[0], h[1], None, None, None, out, hd, H, 1, P, B, 0, n_query=T)
    want, tol = reference(x.reshape(len(at), 1, 8, hd), pk, pv, np.zeros((len(at), 0, 1, hd)), np.zeros((len(at), 0, 1, hd)), np.zeros(len(at)))
    mean, around = reference(np.zeros((1, 1, 1, hd)), pk, pv, np.zeros((1, 0, 1, hd)), np.zeros((1, 0, 1, hd)), [0])
    piece = 16 * hd
    for i, row in enumerate(at):
        backend.copy_buffer_offset(out, small, row * hd * 4, 0, 8 * hd * 4)
        assert (np.abs(backend.download(small, 8 * hd).reshape(8, hd) - want[i, 0]).max(-1) <= tol[i, 0]).all()
    for row in (8, 1 << 20, 8388480 - 24, 8388480 + 8, rows - 24):
        backend.copy_buffer_offset(out, small, row * hd * 4, 0, piece * 4)
        assert (np.abs(backend.download(small, piece).reshape(16, hd) - mean[0, 0]).max(-1) <= around[0, 0]).all()
    for b in [q, out, small] + h:
        backend.free(b)


def test_handles_that_are_not_looked_at(backend):
    """Those of caches without positions may be anything, the output's among them."""
    c = Call(B=2, P=0, C=30, lens=[30, 11]).upload(backend)
    c.h["pk"] = c.h["pv"] = c.h["out"]
    c.run(backend)
    c.check(backend)
    c = Call(B=2, P=40, C=0, lens=[0, 0]).upload(backend)
    c.h["tk"] = c.h["tv"] = c.h["lens"] = c.h["out"]
    c.run(backend)
    c.check(backend)


def test_refusals(backend):
    c = Call().upload(backend)
    good = [c.h["q"], c.h["pk"], c.h["pv"], c.h["tk"], c.h["tv"], c.h["lens"], c.h["out"], 64, 8, 2, 70, 3, 50]
    small = backend.allocate(16)

    def refused(code, at, value):
        args = list(good)
        args[at] = value
        with pytest.raises(YuleGpuError) as e:
            backend.prefix_attention(*args)
        assert e.value.code == code

    for at in range(7):
        refused(3, at, small) if at != 5 else refused(3, 5, backend.allocate(4))
    for at in (0, 1, 2, 3, 4, 5):
        refused(1, at, c.h["out"])
    refused(1, 7, 66)
    refused(1, 8, 7)
    refused(3, 10, 10 ** 6)
    refused(2, 1, None)
    refused(2, 5, None)
    c.run(backend)
    c.check(backend)

"""One step of speculative decoding of a batch as a server runs it: projection with the requests' adapters, attention behind their shared prefix, logits with adapters,
verification of the drafts.  Each stage is held against its definition in 64 bits on the inputs that it had; tolerances are those of the operators' own
tests, and 1e-5 of Σ |w| |x| for the quantised projections."""

import threading

import numpy as np
import pytest

from test_gpu_prefix_attention import reference as attention_reference
from test_gpu_verify_drafts import reference as verify_reference
from yule_b200 import CudaB200Backend, DType, synth

pytestmark = pytest.mark.gpu
NONE = 0xFFFFFFFF
DIM, HEADS, KV, HD, VOCAB, ADAPTERS, RANK = 256, 4, 2, 64, 512, 5, 12


class Adapters:
    def __init__(self, r, rows, cols):
        f = lambda *s: r.standard_normal(s).astype(np.float32)  # noqa: E731
        self.rows, self.cols = rows, cols
        self.down, self.up = (f(ADAPTERS, RANK, cols) / np.sqrt(cols)).astype(np.float16), (f(ADAPTERS, rows, RANK) * 0.1).astype(np.float16)
        self.ranks, self.scales = np.array([12, 4, 0, 7, 12], np.uint32), f(ADAPTERS)

    def upload(self, b):
        self.h = [b.upload(a) for a in (self.down, self.up, self.ranks, self.scales)]

    def add(self, ids, base, x):
        out, tol = base.astype(np.float64), np.zeros(base.shape)
        for i, a in enumerate(ids):
            if a < ADAPTERS:
                n = int(self.ranks[a])
                d, u, v, s = self.down[a, :n].astype(np.float64), self.up[a, :, :n].astype(np.float64), x[i].astype(np.float64), float(self.scales[a])
                out[i] += s * (u @ (d @ v))
                tol[i] = 2.0 ** -17 * abs(s) * (np.abs(u) @ (np.abs(d) @ np.abs(v)))
        return out, tol + 2.0 ** -23 * np.abs(out)


class Step:
    """What a server holds for B sequences with K drafts each; the state of a step is the adapters of its rows, the lengths, the drafts and the random numbers."""

    def __init__(self, b, B, K, P, C, seed=0):
        r = np.random.default_rng(seed)
        f = lambda *s: r.standard_normal(s).astype(np.float32)  # noqa: E731
        self.B, self.K, self.T, self.P, self.C, self.V, self.temperature, self.greedy = B, K, K + 1, P, C, VOCAB, 0.8, False
        self.rows = B * self.T
        blocks = {"q": synth.random_blocks(DType.Q8_0, seed + 1, HEADS * HD * DIM // 32, 0.002), "l": synth.random_blocks(DType.Q8_0, seed + 2, VOCAB * HEADS * HD // 32, 0.002)}
        self.w = {n: b.upload(a) for n, a in blocks.items()}
        self.W = {}
        for n, (rows, cols) in {"q": (HEADS * HD, DIM), "l": (VOCAB, HEADS * HD)}.items():
            out = b.allocate(rows * cols * 4)
            b.dequantize(self.w[n], DType.Q8_0, rows * cols // 32, out)
            self.W[n] = b.download(out, rows * cols).reshape(rows, cols).astype(np.float64)
        self.of_q, self.of_l = Adapters(r, HEADS * HD, DIM), Adapters(r, VOCAB, HEADS * HD)
        self.of_q.upload(b), self.of_l.upload(b)
        self.x, self.pk, self.pv, self.tk, self.tv = f(self.rows, DIM), f(P, KV, HD), f(P, KV, HD), f(B, C, KV, HD), f(B, C, KV, HD)
        self.draft = f(B, K, VOCAB)
        self.h = {n: b.upload(getattr(self, n)) for n in ("x", "pk", "pv", "tk", "tv", "draft")}
        self.h |= {n: b.allocate(c * 4) for n, c in {"q": self.rows * HEADS * HD, "att": self.rows * HEADS * HD, "logits": self.rows * VOCAB, "tokens": self.rows, "accepted": B}.items()}
        self.h |= {n: b.allocate(c * 4) for n, c in {"ids": self.rows, "seen": B, "drafts": B * K, "lens": B, "random": self.rows}.items()}
        self.state(b, seed)

    def state(self, b, seed):
        r = np.random.default_rng(1000 + seed)
        self.ids = np.repeat(np.where(r.random(self.B) < 0.2, NONE, r.integers(0, ADAPTERS, self.B)), self.T).astype(np.uint32)
        self.seen = r.integers(self.T, self.C + 1, self.B).astype(np.uint32)
        self.drafts = r.integers(0, VOCAB, (self.B, self.K)).astype(np.uint32)
        self.lens = r.integers(0, self.K + 1, self.B).astype(np.uint32)
        self.random = r.random((self.B, self.T)).astype(np.float32) * np.float32(0.99)
        for n in ("ids", "seen", "drafts", "lens", "random"):
            b.copy_to_device(getattr(self, n), self.h[n])

    def run(self, b):
        h = self.h
        b.quantized_matmul_batched(self.w["q"], h["x"], h["q"], HEADS * HD, DIM, DType.Q8_0, self.rows)
        b.adapter_matmul_batched(*self.of_q.h, h["ids"], h["x"], h["q"], h["q"], HEADS * HD, DIM, DType.F16, ADAPTERS, RANK, self.rows)
        b.prefix_attention(h["q"], h["pk"], h["pv"], h["tk"], h["tv"], h["seen"], h["att"], HD, HEADS, KV, self.P, self.B, self.C, n_query=self.T)
        b.quantized_matmul_batched(self.w["l"], h["att"], h["logits"], VOCAB, HEADS * HD, DType.Q8_0, self.rows)
        b.adapter_matmul_batched(*self.of_l.h, h["ids"], h["att"], h["logits"], h["logits"], VOCAB, HEADS * HD, DType.F16, ADAPTERS, RANK, self.rows)
        b.verify_drafts(h["logits"], h["draft"], h["drafts"], h["lens"], h["random"], h["tokens"], h["accepted"], VOCAB, self.B, self.K, temperature=self.temperature)

    def results(self, b):
        out = {n: b.download(self.h[n], self.rows * c).reshape(self.rows, c) for n, c in {"q": HEADS * HD, "att": HEADS * HD, "logits": VOCAB}.items()}
        return out | {"tokens": b.download(self.h["tokens"], self.rows, np.uint32).reshape(self.B, self.T), "accepted": b.download(self.h["accepted"], self.B, np.uint32)}

    def check(self, got):
        def projected(w, adapters, x, out):
            ref, tol = adapters.add(self.ids, x.astype(np.float64) @ w.T, x)
            assert (np.abs(out - ref) <= tol + 1e-5 * (np.abs(x).astype(np.float64) @ np.abs(w).T)).all()

        projected(self.W["q"], self.of_q, self.x, got["q"])
        ref, tol = attention_reference(got["q"].reshape(self.B, self.T, HEADS, HD), self.pk, self.pv, self.tk, self.tv, self.seen)
        assert (np.abs(got["att"].reshape(ref.shape) - ref) <= tol[..., None]).all()
        projected(self.W["l"], self.of_l, got["att"], got["logits"])
        self.target = got["logits"].reshape(self.B, self.T, VOCAB)
        tokens, accepted, close = verify_reference(self)
        assert close > 2.0 ** -29
        assert (got["tokens"] == tokens).all() and (got["accepted"] == accepted).all()


def same(a, b):
    return all((a[n] == b[n]).all() for n in a)


# (both ways of each operator: few rows and many, a prefix for the tensor core's 128 rows and one that is too short for it)
@pytest.mark.parametrize("B,K,P,C", [(1, 1, 5, 9), (3, 4, 70, 40), (8, 3, 300, 33), (64, 3, 1100, 50)])
def test_a_step(backend, B, K, P, C):
    s = Step(backend, B, K, P, C, seed=B)
    s.run(backend)
    first = s.results(backend)
    s.check(first)
    for _ in range(5):
        s.run(backend)
    assert same(s.results(backend), first)


def test_captured_steps_that_share_their_scratch(backend):
    steps = [Step(backend, 3, 4, 70, 40, seed=1), Step(backend, 64, 3, 1100, 50, seed=2)]
    graphs = []
    for s in steps:
        s.run(backend)
    for s in steps:
        backend.graph_begin()
        s.run(backend)
        graphs.append(backend.graph_end())
    for seed in (5, 6):
        for s in steps:
            s.state(backend, seed)
        for g in graphs + graphs[::-1] + graphs:
            backend.graph_launch(g)
        steps[0].run(backend)
        backend.graph_launch(graphs[0])
        for s in steps:
            s.check(s.results(backend))
    for g in graphs:
        backend.graph_destroy(g)


def test_two_contexts_at_once(backend):
    """A context per thread on one device: neither sees the other's scratch."""
    sizes = [(5, 4, 200, 40), (64, 3, 1100, 50)]
    alone = []
    for i, n in enumerate(sizes):
        s = Step(backend, *n, seed=i)
        s.run(backend)
        alone.append(s.results(backend))
    wrong, errors = [], []

    def work(i):
        try:
            b = CudaB200Backend(0)
            s = Step(b, *sizes[i], seed=i)
            for _ in range(10):
                for _ in range(5):
                    s.run(b)
                if not same(s.results(b), alone[i]):
                    wrong.append(i)
            b.close()
        except Exception as e:  # (a thread's exception would be lost)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1, 0)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and not wrong

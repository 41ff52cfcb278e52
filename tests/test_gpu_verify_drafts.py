"""Verification of drafted tokens (csrc/verify.cu) against its definition in 64 bits.  Tokens are whole numbers: they have to be equal.  The random numbers are drawn so that none lies
within 2^-29 of a border (in units of the whole), more than the 2^-30 that its sums may be off by."""

import numpy as np
import pytest

from yule_b200 import CudaB200Backend, YuleGpuError

pytestmark = pytest.mark.gpu
NONE = 0xFFFFFFFF


def soft(row, temperature):
    """Probabilities of a row of logits, or None where no token can be."""
    x = np.asarray(row, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    x = np.minimum(x, np.finfo(np.float32).max)
    if x.max() == -np.inf:
        return None
    e = np.exp((x - x.max()) / np.float64(np.float32(temperature)))
    return e / e.sum()


def reference(c):
    tokens, accepted, close = np.full((c.B, c.K + 1), NONE, np.uint32), np.zeros(c.B, np.uint32), 1.0
    for b in range(c.B):
        k = c.K if c.lens is None else min(int(c.lens[b]), c.K)
        a = 0
        q = None
        while a < k:
            x, p = int(c.drafts[b, a]), soft(c.target[b, a], c.temperature)
            q = None
            if c.greedy:
                row = np.where(np.isnan(c.target[b, a]), -np.inf, np.minimum(c.target[b, a], np.finfo(np.float32).max))
                fits = p is not None and x < c.V and x == c.V - 1 - int(row[::-1].argmax())
            else:
                q = np.zeros(c.V)
                if c.draft is None:
                    if x < c.V:
                        q[x] = 1.0
                else:
                    d = soft(c.draft[b, a], c.temperature)
                    q = q if d is None else d
                fits = x < c.V and p is not None and float(c.random[b, a]) * q[x] < p[x]
                if x < c.V and p is not None:
                    close = min(close, abs(float(c.random[b, a]) * q[x] - p[x]) / max(p[x], 1e-300))
            if not fits:
                break
            a += 1
        accepted[b] = a
        tokens[b, :a] = c.drafts[b, :a]
        p = soft(c.target[b, a], c.temperature)
        if p is None:
            continue
        if c.greedy:
            row = np.where(np.isnan(c.target[b, a]), -np.inf, np.minimum(c.target[b, a], np.finfo(np.float32).max))
            tokens[b, a] = c.V - 1 - int(row[::-1].argmax())
            continue
        w = np.maximum(p - q, 0) if a < k else p
        run = np.cumsum(w)
        if run[-1] > 0:
            goal = float(c.random[b, c.K]) * run[-1]
            over = np.nonzero((run > goal) & (w > 0))[0]
            tokens[b, a] = over[0] if len(over) else np.nonzero(w > 0)[0][-1]
            close = min(close, np.abs(run[w > 0] - goal).min() / run[-1])
    return tokens, accepted, close


class Call:
    def __init__(self, B=4, K=3, V=500, temperature=0.8, by="model", lens=None, greedy=False, seed=0, near=0.6, spread=2.0, pad=0):
        r = np.random.default_rng(seed)
        self.B, self.K, self.V, self.temperature, self.greedy, self.pad = B, K, V, temperature, greedy, pad
        self.target = (r.standard_normal((B, K + 1, V)) * spread).astype(np.float32)
        self.draft = (self.target[:, :K] + near * r.standard_normal((B, K, V))).astype(np.float32) if by == "model" else None
        like = self.draft if by == "model" else self.target[:, :K] + 0.3 * r.standard_normal((B, K, V))
        self.drafts = (like / temperature + (r.gumbel(size=(B, K, V)) if by == "model" else 0)).argmax(-1).astype(np.uint32)
        self.lens = None if lens is None else np.asarray(lens, np.uint32)
        self.random = r.random((B, K + 1)).astype(np.float32)
        self.random[self.random >= 1] = 0.5

    def upload(self, b):
        def wide(a):
            return np.concatenate([a.reshape(-1, self.V), np.full((a.shape[0] * a.shape[1], self.pad), np.inf, np.float32)], 1)

        self.h = dict(target=b.upload(wide(self.target)), draft=b.upload(wide(self.draft)) if self.draft is not None else None, drafts=b.upload(self.drafts),
                      lens=b.upload(self.lens) if self.lens is not None else None, random=b.upload(self.random), tokens=b.upload(np.full(self.B * (self.K + 1) + 8, 5, np.uint32)),
                      accepted=b.upload(np.full(self.B + 8, 5, np.uint32)))
        return self

    def run(self, b):
        h = self.h
        b.verify_drafts(h["target"], h["draft"], h["drafts"], h["lens"], h["random"], h["tokens"], h["accepted"], self.V, self.B, self.K, temperature=self.temperature,
                        greedy=self.greedy, target_stride=self.V + self.pad, draft_stride=self.V + self.pad)

    def got(self, b):
        n = self.B * (self.K + 1)
        t, a = b.download(self.h["tokens"], n + 8, np.uint32), b.download(self.h["accepted"], self.B + 8, np.uint32)
        assert (t[n:] == 5).all() and (a[self.B:] == 5).all()
        return t[:n].reshape(self.B, -1), a[:self.B]

    def check(self, b):
        tokens, accepted, close = reference(self)
        assert close > 2.0 ** -29, "a random number on a border says nothing"
        got = self.got(b)
        assert (got[1] == accepted).all() and (got[0] == tokens).all()
        return accepted

    def free(self, b):
        for h in self.h.values():
            if h:
                b.free(h)


def go(b, **kw):
    c = Call(**kw)
    again = np.random.default_rng(kw.get("seed", 0) + 77)
    while reference(c)[2] <= 2.0 ** -29:  # a random number on a border says nothing: others
        c.random = again.random(c.random.shape).astype(np.float32) * np.float32(0.999)
    c.upload(b)
    c.run(b)
    accepted = c.check(b)
    c.free(b)
    return accepted


WAYS = pytest.mark.parametrize("way", [dict(by="model"), dict(by="lookup"), dict(by="lookup", greedy=True)], ids=["model", "lookup", "greedy"])


@WAYS
@pytest.mark.parametrize("V", [1, 2, 31, 255, 256, 1000, 1024, 1025, 4095, 4096, 4097, 8192, 8193, 32000, 50257, 128256])
def test_vocabularies(backend, way, V):
    go(backend, V=V, seed=V, B=3 if V > 10000 else 6, **way)
    go(backend, V=V, seed=V + 1, B=20, K=2, **way)  # (fewer CTAs a sequence)


@WAYS
def test_all_numbers_of_accepted_drafts_come_up(backend, way):
    seen = np.concatenate([go(backend, B=32, K=3, V=300, seed=s, near=0.5, **way) for s in range(4)])
    assert set(seen.tolist()) == {0, 1, 2, 3}


@WAYS
@pytest.mark.parametrize("K", [1, 2, 7, 31, 32, 33, 70, 256])
def test_numbers_of_drafts(backend, way, K):
    """Drafts that nearly always stand, so that runs are long."""
    go(backend, B=3, K=K, V=40, near=0.01, seed=K, spread=3.0, **way)


@WAYS
def test_lengths_of_the_drafts(backend, way):
    go(backend, B=7, K=4, V=200, lens=[0, 1, 2, 3, 4, 5, NONE], near=0.05, **way)


@WAYS
@pytest.mark.parametrize("pad", [1, 3, 8])
def test_strides(backend, way, pad):
    go(backend, pad=pad, V=1001, **way)


@pytest.mark.parametrize("temperature", [1e-6, 0.05, 0.5, 1.0, 3.0, 100.0, 1e6])
def test_temperatures(backend, temperature):
    go(backend, temperature=temperature, B=8, V=300)
    go(backend, temperature=temperature, B=8, V=300, by="lookup")


@WAYS
def test_logits_of_any_size(backend, way):
    for spread in (1e-30, 1e-3, 50.0, 1e4, 1e30):
        go(backend, spread=spread, B=6, V=300, near=0.0 if spread > 1e5 else 0.3 * spread, **way)


@WAYS
def test_tokens_that_cannot_be(backend, way):
    """NaN and −infinity are tokens without probability, rows of them have none at all; +infinity is the largest number."""
    c = Call(B=8, K=3, V=300, **way)
    c.target[0, :, ::2] = -np.inf
    c.target[1, :, 5:] = np.nan
    c.target[2] = -np.inf
    c.target[3, 1] = np.nan
    c.target[4, 0, 7], c.target[4, 0, 9] = np.inf, np.inf
    c.target[5, 3, :] = -np.finfo(np.float32).max
    if c.draft is not None:
        c.draft[6, 0] = -np.inf
        c.draft[7, 0, c.drafts[7, 0]] = -np.inf
    c.upload(backend).run(backend)
    c.check(backend)


@WAYS
def test_drafts_outside_the_vocabulary(backend, way):
    c = Call(B=4, K=3, V=300, near=0.01, **way)
    c.drafts[0, 0], c.drafts[1, 1], c.drafts[2, 2] = 300, NONE, 1 << 31
    c.upload(backend).run(backend)
    c.check(backend)


def test_equal_distributions_accept_everything(backend):
    c = Call(B=16, K=3, V=500, near=0.0)
    c.upload(backend).run(backend)
    assert (c.check(backend) == 3).all()


@pytest.mark.parametrize("V", [300, 50257])
@pytest.mark.parametrize("step", [1e-2, 1e-4, 1e-6])
def test_models_that_are_as_good_as_the_same(backend, V, step):
    """Distributions that hardly differ, rejected all the same: all of w is where p and q are near.  (Half of the tokens a step more likely than drafted, half less.)"""
    c = Call(B=6, K=2, V=V, temperature=1.0, spread=1.0)
    r = np.random.default_rng(3)
    c.target[:, :2] = np.round(c.target[:, :2] * 2 ** 10) / 2 ** 10
    c.draft = (c.target[:, :2] + np.where(r.random((6, 2, V)) < 0.5, np.float32(step), np.float32(-step))).astype(np.float32)
    for b in range(6):
        c.drafts[b] = [np.nonzero(c.draft[b, t] > c.target[b, t])[0][0] for t in range(2)]
    c.random[:, :2] = np.nextafter(np.float32(1), np.float32(0))
    c.upload(backend).run(backend)
    c.check(backend)


@pytest.mark.parametrize("V", [40, 300, 40000])
@pytest.mark.parametrize("log_w", [-30, -37, -46, -120, -600])
def test_what_p_has_more_of_is_next_to_nothing(backend, V, log_w):
    """Both distributions are one token up to e^log_w, and the draft is neither's.  p has less of that token, by what it has more of the others in all, so w is p − q at the others,
    of the size of e^log_w, where the whole of p is 1 or a few steps of 2^-52 from it."""
    B = 24
    c = Call(B=B, K=1, V=V, temperature=1.0)
    r = np.random.default_rng(V - log_w)
    others = 1 + r.permutation(V - 2)[:9]  # not the first token, nor the last, which is the draft
    c.target[:], c.draft[:], c.drafts[:] = -np.inf, -np.inf, V - 1
    c.target[:, :, 0], c.draft[:, :, 0] = 3.0, 3.0
    c.target[:, :, others] = 3 + log_w + r.random((B, 2, 9))
    c.draft[:, :, others] = np.nextafter(c.target[:, :1, others], np.float32(0)) - r.random((B, 1, 9)).astype(np.float32)
    p, q = (np.exp(a[:, 0].astype(np.float64) - 3) for a in (c.target, c.draft))
    # the wholes are 1 + sp and 1 + sq: their ratio from the difference of sp and sq
    sp, sq = p[:, 1:].sum(-1, keepdims=True), q[:, 1:].sum(-1, keepdims=True)
    w = np.maximum(p - q * ((sp - sq) / (1 + sq) + 1), 0)
    w[:, 0] = 0
    run = np.cumsum(w, -1)
    for _ in range(100):
        goal = c.random[:, 1].astype(np.float64)[:, None] * run[:, -1:]
        near = (np.abs(run[:, others] - goal) / run[:, -1:]).min(-1) < 2.0 ** -10
        if not near.any():
            break
        c.random[near, 1] = r.random(near.sum())
    assert not near.any()
    c.upload(backend).run(backend)
    tokens, accepted = c.got(backend)
    assert (accepted == 0).all() and (tokens[:, 0] == ((run > goal) & (w > 0)).argmax(-1)).all()


def test_a_draft_that_the_same_distribution_does_not_have(backend):
    """p = q: nothing is left of p − q, and the token is drawn from p."""
    for V in (300, 40000):
        c = Call(B=24, K=2, V=V, near=0.0)
        c.drafts[:8, 0] = NONE
        c.target[8:16, 0, 7] = c.draft[8:16, 0, 7] = -np.inf
        c.drafts[8:16, 0] = 7
        c.target[16:, 0, 5:] = c.draft[16:, 0, 5:] = -np.inf
        c.drafts[16:, 0] = 9
        c.upload(backend).run(backend)
        tokens, accepted = c.got(backend)
        assert (accepted == 0).all()
        for b in range(24):
            run = np.cumsum(soft(c.target[b, 0], c.temperature))
            goal = float(c.random[b, 2]) * run[-1]
            assert np.abs(run - goal).min() > 2.0 ** -29
            assert tokens[b].tolist() == [np.nonzero(run > goal)[0][0], NONE, NONE]


def test_random_numbers_at_the_ends(backend):
    for u in (0.0, np.nextafter(np.float32(1), np.float32(0))):
        c = Call(B=8, K=3, V=300)
        c.random[:] = u
        c.upload(backend).run(backend)
        tokens, accepted, _ = reference(c)
        got = c.got(backend)
        assert (got[0] == tokens).all() and (got[1] == accepted).all()
    # what is no random number gives a token of the vocabulary all the same
    for u in (1.0, 2.0, -1.0, np.nan, np.inf):
        c = Call(B=8, K=3, V=300)
        c.random[:] = u
        c.upload(backend).run(backend)
        tokens, accepted = c.got(backend)
        for b in range(8):
            assert accepted[b] <= 3 and tokens[b, accepted[b]] < 300 and (tokens[b, accepted[b] + 1:] == NONE).all()


@pytest.mark.parametrize("bits", [100, 125, 130, 135, 137, 160, 700])
def test_drafts_that_are_next_to_impossible(backend, bits):
    """p of a draft is 2^-bits or some bits less, and its random number times q 0.1 % of that above or below it: where probabilities have few bits in fp32, or none."""
    B, V = 256, 300
    c = Call(B=B, K=1, V=V, temperature=1.0, spread=1.0, near=0.3)
    r = np.random.default_rng(bits)
    x = r.integers(0, V, B)
    c.drafts[:, 0] = x
    b = np.arange(B)
    c.target[b, 0, x] = -bits * np.log(2) + r.random(B)
    c.draft[b, 0, x] = c.target[b, 0, x] + 0.5
    p, q = (np.array([soft(row, 1.0)[i] for row, i in zip(a[:, 0], x)]) for a in (c.target, c.draft))
    above = r.random(B) < 0.5
    c.random[:, 0] = np.where(above, 1.001, 0.999) * p / q
    assert (c.random[:, 0] > 0).all() and (c.random[:, 0] < 1).all()
    c.upload(backend).run(backend)
    assert (c.check(backend) == ~above).all()


def test_greedy_ties_go_to_the_highest_index(backend):
    c = Call(B=2, K=2, V=9000, by="lookup", greedy=True)
    c.target[:] = 0
    c.target[:, :, [3, 4000, 8500]] = 2.0
    c.drafts[0], c.drafts[1] = [8500, 8500], [8500, 4000]
    c.upload(backend).run(backend)
    tokens, accepted = c.got(backend)
    assert accepted.tolist() == [2, 1] and tokens.tolist() == [[8500, 8500, 8500], [8500, 8500, NONE]]


def test_tokens_are_distributed_as_the_target(backend):
    """Many sequences of one distribution: the first token's frequencies are the target's, within five standard deviations, although the drafts' are others."""
    B, V = 20000, 6
    c = Call(B=B, K=1, V=V, temperature=1.0)
    p, q = np.array([.3, .05, .2, .25, .1, .1]), np.array([.1, .3, .3, .1, .15, .05])
    r = np.random.default_rng(1)
    c.target[:] = np.log(p)
    c.draft[:] = np.log(q)
    c.drafts[:, 0] = r.choice(V, B, p=q)
    c.random = r.random((B, 2)).astype(np.float32)
    c.upload(backend).run(backend)
    tokens, _ = c.got(backend)
    share = np.bincount(tokens[:, 0], minlength=V) / B
    assert (np.abs(share - p) < 5 * np.sqrt(p * (1 - p) / B)).all()


def test_captured_and_replayed_with_other_inputs(backend):
    c = Call(B=5, K=3, V=3000, lens=[3, 3, 3, 3, 3]).upload(backend)
    c.run(backend)
    backend.graph_begin()
    c.run(backend)
    g = backend.graph_end()
    for seed in (5, 6):
        d = Call(B=5, K=3, V=3000, lens=[0, 1, 2, 3, 3], seed=seed)
        for name in ("target", "draft", "drafts", "lens", "random"):
            setattr(c, name, getattr(d, name))
            backend.copy_to_device(getattr(d, name), c.h[name])
        backend.graph_launch(g)
        c.check(backend)
    backend.graph_destroy(g)


def test_handles_that_are_not_looked_at(backend):
    """Greedy: draft logits and random numbers may be anything, an output among them."""
    c = Call(by="lookup", greedy=True).upload(backend)
    c.h["draft"], c.h["random"] = c.h["tokens"], c.h["accepted"]
    c.run(backend)
    c.check(backend)


def test_refusals(backend):
    c = Call(lens=[1, 2, 3, 3]).upload(backend)
    h = c.h
    good = [h["target"], h["draft"], h["drafts"], h["lens"], h["random"], h["tokens"], h["accepted"], 500, 4, 3]
    small = backend.allocate(4)

    def refused(code, at, value, **more):
        args = list(good)
        args[at] = value
        with pytest.raises(YuleGpuError) as e:
            backend.verify_drafts(*args, **more)
        assert e.value.code == code

    for at in range(7):
        refused(3, at, small)
    for at in range(5):
        refused(1, at, h["tokens"])
        refused(1, at, h["accepted"])
    refused(1, 5, h["accepted"])
    refused(2, 4, None)
    refused(1, 7, 0)
    refused(3, 7, 501)
    refused(1, 9, 0)
    refused(1, 9, 3, temperature=0.0)
    c.run(backend)
    c.check(backend)


def test_first_call_in_a_capture():
    """The call needs no scratch."""
    b = CudaB200Backend(0)
    c = Call().upload(b)
    b.graph_begin()
    c.run(b)
    g = b.graph_end()
    b.graph_launch(g)
    c.check(b)
    b.close()

"""Performance cases of the operators for a batch of requests that is served together.

Three operators are covered, as a server's step meets them: attention of a batch whose sequences share a long prefix
(``prefix_attention``), low-rank adapters of many requests beside a shared projection (``adapter_matmul_batched``), and
verification of drafted tokens (``verify_drafts``).  Head layouts, widths and vocabularies are those of the 1.1B, 8B and
70B architectures the package is tested with, and a few odd ones.

``run`` computes a case in plain torch operations, or with ``own`` set through the package.  A case is a dict: ``kind``
names the operator, the other keys its sizes.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

# query heads, KV heads, head_dim
HEADS = {"1b": (32, 4, 64), "8b": (32, 8, 128), "70b": (64, 8, 128), "odd": (20, 5, 96)}
# rows and columns of projections (the 1.1B, 8B and 70B shapes, and an odd one)
LINEARS = {"1b-q": (2048, 2048), "1b-down": (2048, 5632), "8b-q": (4096, 4096), "8b-up": (14336, 4096),
           "8b-down": (4096, 14336), "70b-q": (8192, 8192), "odd": (1000, 2560)}
NOTHING = 0xFFFFFFFF


# ── the cases ──────────────────────────────────────────────────────────────────────────────────


def listed() -> list[dict]:
    return [
        # Two short chats behind a short system prompt: the smallest call, all latency.
        {"name": "attention-1b-2", "kind": "attention", "heads": "1b", "seqs": 2, "query": 1, "prefix": 100, "tail": 20},
        # A server's batch: thirty-two requests behind one set of instructions.
        {"name": "attention-8b-32", "kind": "attention", "heads": "8b", "seqs": 32, "query": 1, "prefix": 2048, "tail": 300},
        # The same with four drafted tokens a request, odd lengths.
        {"name": "attention-8b-drafts", "kind": "attention", "heads": "8b", "seqs": 8, "query": 5, "prefix": 1777, "tail": 211},
        # Many requests about one long document, 70B head layout.
        {"name": "attention-70b-64", "kind": "attention", "heads": "70b", "seqs": 64, "query": 1, "prefix": 8192, "tail": 500},
        # One token of one request with a small adapter: the smallest call.
        {"name": "adapter-1b-1", "kind": "adapter", "linear": "1b-q", "rows": 1, "adapters": 4, "rank": 8, "type": "F16"},
        # A decode step of thirty-two requests with an adapter each.
        {"name": "adapter-8b-32", "kind": "adapter", "linear": "8b-q", "rows": 32, "adapters": 32, "rank": 16, "type": "F16"},
        # Prompts of six requests in one pass, large ranks, the widest projection.
        {"name": "adapter-8b-prompts", "kind": "adapter", "linear": "8b-up", "rows": 1501, "adapters": 6, "rank": 64, "type": "F16"},
        # Adapters kept in 32 bits, long rows, a few requests of an adapter each.
        {"name": "adapter-8b-f32", "kind": "adapter", "linear": "8b-down", "rows": 9, "adapters": 5, "rank": 32, "type": "F32"},
        # One request, four drafts of a small model with the 1.1B model's vocabulary.
        {"name": "verify-1b-1", "kind": "verify", "vocab": 32000, "seqs": 1, "drafts": 4, "temperature": 1.0, "by": "model"},
        # A server's batch with four drafts each, large vocabulary.
        {"name": "verify-8b-32", "kind": "verify", "vocab": 128256, "seqs": 32, "drafts": 4, "temperature": 0.7, "by": "model"},
        # Drafts looked up in the prompt (no probabilities of their own), not the same number for every request.
        {"name": "verify-8b-lookup", "kind": "verify", "vocab": 128256, "seqs": 13, "drafts": 7, "temperature": 0.8, "by": "lookup"},
        # Greedy decoding with drafts.
        {"name": "verify-1b-greedy", "kind": "verify", "vocab": 32000, "seqs": 24, "drafts": 3, "temperature": 1.0, "by": "greedy"},
    ]


def _log(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["attention", "adapter", "verify"])
    if kind == "attention":
        case = {"kind": kind, "heads": rng.choice(["1b", "8b", "8b", "70b", "odd"]), "seqs": _log(rng, 1, 64), "query": rng.choice([1, 1, 1, 2, 3, 5, 8]),
                "prefix": _log(rng, 16, 8192), "tail": _log(rng, 9, 1000)}
        while work(case)["flops"] > 1.7e10 or work(case)["bytes"] > 2e8:
            case["prefix"] = case["prefix"] * 2 // 3
            case["seqs"] = max(1, case["seqs"] * 3 // 4)
        return case
    if kind == "adapter":
        case = {"kind": kind, "linear": rng.choice(sorted(LINEARS)), "rows": rng.choice([1, 2, 3, 5, 8, 17, 32, _log(rng, 33, 1500)]), "adapters": _log(rng, 1, 48),
                "rank": rng.choice([4, 8, 8, 12, 16, 16, 32, 50, 64]), "type": rng.choice(["F16", "F16", "F32"])}
        while work(case)["bytes"] > 2e8:
            case["adapters"] = case["adapters"] * 3 // 4
        return case
    return {"kind": kind, "vocab": rng.choice([32000, 128256, 50257, _log(rng, 1000, 128000)]), "seqs": _log(rng, 1, 32), "drafts": rng.randint(1, 4),
            "temperature": rng.choice([1.0, 0.6, 0.8, 1.3]), "by": rng.choice(["model", "model", "lookup", "greedy"])}


# ── inputs ─────────────────────────────────────────────────────────────────────────────────────

_backend = None
_spare: dict = {}


class _View:
    """A buffer of the package as an array that torch can look at."""

    def __init__(self, address: int, count: int, kind: str):
        self.__cuda_array_interface__ = {"data": (address, False), "shape": (count,), "typestr": kind, "version": 3}


class _Buffers:
    """The buffers of one state.  A program has its buffers once: those of a state that is gone serve the next one."""

    def __init__(self):
        global _backend
        if _backend is None:
            from yule_b200 import CudaB200Backend
            _backend = CudaB200Backend(0)
        self.held = []

    def of(self, tensor: torch.Tensor):
        """(handle, view) of a buffer with the tensor's values."""
        n, dt = tensor.numel(), tensor.dtype
        size, kind = tensor.element_size(), {torch.float32: "<f4", torch.float16: "<f2", torch.int32: "<i4"}[dt]
        free = _spare.setdefault(n * size, [])
        h = free.pop() if free else _backend.allocate(n * size)
        self.held.append((n * size, h))
        _backend.synchronize()  # (a new buffer is filled with zeros on the package's stream)
        view = torch.as_tensor(_View(_backend.buffer_address(h), n, kind), device="cuda").view(tensor.shape)
        view.copy_(tensor)
        return h, view

    def __del__(self):
        for size, h in self.held:
            _spare[size].append(h)


def _lengths(case: dict) -> np.ndarray:
    """Lengths of the sequences' own caches: from a few tokens to all of `tail`."""
    lo = min(case["tail"], case["query"] + 1)
    return np.linspace(lo, case["tail"], case["seqs"]).astype(np.int32) if case["seqs"] > 1 else np.array([case["tail"]], np.int32)


def _ranks(case: dict) -> np.ndarray:
    """Every third adapter has half of the largest rank."""
    return np.array([case["rank"] if a % 3 else max(1, case["rank"] // 2) for a in range(case["adapters"])], np.int32)


def _of_rows(case: dict) -> np.ndarray:
    """The adapter of each row: a run of rows per request; in a batch of several requests the last one has none."""
    requests = min(case["rows"], case["adapters"] if case["rows"] > 64 else max(case["adapters"], case["rows"]))
    request = np.arange(case["rows"]) * requests // case["rows"]
    ids = (request * 7 + 1) % case["adapters"]
    return np.where((request == requests - 1) & (requests > 2), -1, ids).astype(np.int32)


def _draft_lens(case: dict) -> np.ndarray:
    n = np.full(case["seqs"], case["drafts"], np.int32)
    if case["by"] == "lookup":
        n = (np.arange(case["seqs"]) * 3 + 1) % (case["drafts"] + 1)
    return n.astype(np.int32)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def numbers(a):
        return torch.from_numpy(np.ascontiguousarray(a)).cuda()

    if case["kind"] == "attention":
        heads, kv, hd = HEADS[case["heads"]]
        b, p, cap = case["seqs"], case["prefix"], case["tail"] + 4
        # keys have a common part, as a trained model's do
        common = normal(kv, hd)
        lens = numbers(np.random.RandomState(seed & 0x7FFFFFFF).permutation(_lengths(case)))
        t = {"q": normal(b, case["query"], heads, hd) * 1.3, "prefix_k": normal(p, kv, hd) + common, "prefix_v": normal(p, kv, hd),
             "tail_k": normal(b, cap, kv, hd) + common, "tail_v": normal(b, cap, kv, hd), "tail_lens": lens}
        t["out"] = torch.zeros_like(t["q"])
    elif case["kind"] == "adapter":
        rows, cols = LINEARS[case["linear"]]
        a, r = case["adapters"], case["rank"]
        kind = torch.float16 if case["type"] == "F16" else torch.float32
        t = {"down": (normal(a, r, cols) / math.sqrt(cols)).to(kind), "up": (normal(a, rows, r) * 0.1).to(kind), "ranks": numbers(_ranks(case)),
             "scales": 0.5 + torch.rand(a, generator=g, device="cuda"), "row_adapter": numbers(_of_rows(case)), "x": normal(case["rows"], cols),
             "y": normal(case["rows"], rows)}
        # (a program may pass one buffer for both: kept apart here, so that every pass adds to the same result of the projection)
        t["out"] = torch.zeros_like(t["y"])
    else:
        b, k, v = case["seqs"], case["drafts"], case["vocab"]
        # a model's distribution has few likely tokens; a draft model's is near the target's
        target = normal(b, k + 1, v) * 2.5
        draft = target[:, :k] + normal(b, k, v) * 0.5
        if case["by"] == "model":
            noise = -torch.log(-torch.log(torch.rand(b, k, v, generator=g, device="cuda", dtype=torch.float64).clamp_(1e-300, 1 - 1e-16)))
            drafts = (draft.double() / case["temperature"] + noise).argmax(-1)
            del noise
        else:
            drafts = (target[:, :k] + normal(b, k, v) * 0.3).argmax(-1)
        t = {"target": target, "drafts": drafts.int(), "draft_lens": numbers(_draft_lens(case)), "random": torch.rand(b, k + 1, generator=g, device="cuda"),
             "out_tokens": torch.zeros(b, k + 1, dtype=torch.int32, device="cuda"), "out_accepted": torch.zeros(b, dtype=torch.int32, device="cuda")}
        if case["by"] == "model":
            t["draft"] = draft
    s = {"case": dict(case), "t": t}
    if own:  # the same values in the package's buffers
        s["buffers"] = _Buffers()
        made = {name: s["buffers"].of(x) for name, x in t.items()}
        s["h"], s["t"] = {name: m[0] for name, m in made.items()}, {name: m[1] for name, m in made.items()}
        torch.cuda.synchronize()  # (they were copied on torch's stream, behind which the package's is not ordered)
    return s


# ── a pass ─────────────────────────────────────────────────────────────────────────────────────


def _plain_attention(case: dict, t: dict) -> torch.Tensor:
    heads, kv, hd = HEADS[case["heads"]]
    b, nq, p = case["seqs"], case["query"], case["prefix"]
    q = t["q"].view(b * nq, kv, heads // kv, hd)
    cap = t["tail_k"].shape[1]
    of_prefix = torch.matmul(q.permute(1, 0, 2, 3).reshape(kv, -1, hd), t["prefix_k"].permute(1, 2, 0))  # [kv][rows][P]
    of_prefix = of_prefix.view(kv, b, nq, heads // kv, p)
    of_tail = torch.matmul(q.view(b, nq, kv, heads // kv, hd).permute(2, 0, 1, 3, 4).reshape(kv, b, -1, hd), t["tail_k"].permute(2, 0, 3, 1)).view(kv, b, nq, heads // kv, cap)
    seen = t["tail_lens"].view(b, 1) - torch.arange(nq - 1, -1, -1, device="cuda")  # [b][nq]
    hidden = torch.arange(cap, device="cuda") >= seen[..., None]
    of_tail = of_tail.masked_fill(hidden.view(1, b, nq, 1, cap), -math.inf)
    s = torch.cat([of_prefix, of_tail], -1) / math.sqrt(hd)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e[..., :p].reshape(kv, -1, p), t["prefix_v"].permute(1, 0, 2)).view(kv, b, nq, heads // kv, hd)
    o = o + torch.matmul(e[..., p:].reshape(kv, b, -1, cap), t["tail_v"].permute(2, 0, 1, 3)).view(kv, b, nq, heads // kv, hd)
    return (o / total).permute(1, 2, 0, 3, 4).reshape(b, nq, heads, hd)


def _plain_adapter(case: dict, t: dict) -> torch.Tensor:
    a, r = case["adapters"], case["rank"]
    v = t["x"] @ t["down"].float().view(a * r, -1).T  # every row with every adapter
    mine = t["row_adapter"].view(-1, 1) == torch.arange(a, device="cuda")
    there = torch.arange(r, device="cuda") < t["ranks"].view(a, 1)
    v = torch.where(mine[..., None] & there, v.view(-1, a, r) * t["scales"].view(a, 1), 0.0)
    return t["y"] + v.view(-1, a * r) @ t["up"].float().permute(0, 2, 1).reshape(a * r, -1)


def _plain_verify(case: dict, t: dict) -> tuple[torch.Tensor, torch.Tensor]:
    b, k, v = case["seqs"], case["drafts"], case["vocab"]
    lens, drafts = t["draft_lens"].long(), t["drafts"].long()
    at = torch.arange(k, device="cuda")
    target = t["target"]
    if case["by"] == "greedy":
        best = v - 1 - target.flip(-1).argmax(-1)  # ties: the highest index
        fits = (best[:, :k] == drafts) & (at < lens[:, None])
        accepted = fits.long().cumprod(-1).sum(-1)
        pick = best.gather(1, accepted[:, None])[:, 0]
    else:
        p = target.double() / case["temperature"]
        p = torch.exp(p - p.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        if case["by"] == "model":
            q = t["draft"].double() / case["temperature"]
            q = torch.exp(q - q.amax(-1, keepdim=True))
            q = q / q.sum(-1, keepdim=True)
        else:
            q = torch.zeros(b, k, v, dtype=torch.float64, device="cuda").scatter_(2, drafts[..., None], 1.0)
        u = t["random"].double()
        fits = (u[:, :k] * q.gather(2, drafts[..., None])[..., 0] < p[:, :k].gather(2, drafts[..., None])[..., 0]) & (at < lens[:, None])
        accepted = fits.long().cumprod(-1).sum(-1)
        w = p[torch.arange(b, device="cuda"), accepted]
        less = q[torch.arange(b, device="cuda"), accepted.clamp(max=k - 1)]
        w = torch.where((accepted < lens)[:, None], (w - less).clamp(min=0), w)
        c = w.cumsum(-1)
        pick = (c > u[:, k:] * c[:, -1:]).long().argmax(-1)
    places = torch.arange(k + 1, device="cuda")
    tokens = torch.cat([drafts, torch.zeros_like(drafts[:, :1])], 1)
    tokens = torch.where(places < accepted[:, None], tokens, torch.where(places == accepted[:, None], pick[:, None], -1))
    return tokens.int(), accepted.int()


def run(state: dict):
    """One pass.  With ``own`` it is under way on the package's stream: ``_backend.synchronize()``, or torch's of the device, before torch reads the outputs."""
    case, t = state["case"], state["t"]
    kind = case["kind"]
    if not own:
        return {"attention": _plain_attention, "adapter": _plain_adapter, "verify": _plain_verify}[kind](case, t)
    from yule_b200 import DType
    h = state["h"]
    if kind == "attention":
        heads, kv, hd = HEADS[case["heads"]]
        _backend.prefix_attention(h["q"], h["prefix_k"], h["prefix_v"], h["tail_k"], h["tail_v"], h["tail_lens"], h["out"], hd, heads, kv, case["prefix"], case["seqs"],
                                  t["tail_k"].shape[1], n_query=case["query"])
        return t["out"]
    if kind == "adapter":
        rows, cols = LINEARS[case["linear"]]
        # beside the shared projection, whose result is y
        _backend.adapter_matmul_batched(h["down"], h["up"], h["ranks"], h["scales"], h["row_adapter"], h["x"], h["y"], h["out"], rows, cols,
                                        DType.F16 if case["type"] == "F16" else DType.F32, case["adapters"], case["rank"], case["rows"])
        return t["out"]
    _backend.verify_drafts(h["target"], h.get("draft"), h["drafts"], h["draft_lens"], h["random"], h["out_tokens"], h["out_accepted"], case["vocab"], case["seqs"],
                           case["drafts"], temperature=case["temperature"], greedy=case["by"] == "greedy")
    return t["out_tokens"], t["out_accepted"]


# ── what a pass cannot do without ──────────────────────────────────────────────────────────────


def work(case: dict) -> dict:
    if case["kind"] == "attention":
        heads, kv, hd = HEADS[case["heads"]]
        lens, nq = _lengths(case).astype(np.int64), case["query"]
        seen = sum(int(np.maximum(0, lens - i).sum()) for i in range(nq)) + case["prefix"] * case["seqs"] * nq
        keys = case["prefix"] + int(lens.sum())
        return {"bytes": 8 * keys * kv * hd + 8 * case["seqs"] * nq * heads * hd + 4 * case["seqs"], "flops": 4 * hd * heads * seen}
    if case["kind"] == "adapter":
        rows, cols = LINEARS[case["linear"]]
        ids, ranks = _of_rows(case), _ranks(case)
        used = sorted({int(i) for i in ids if i >= 0})
        weights = sum(int(ranks[i]) for i in used) * (rows + cols) * (2 if case["type"] == "F16" else 4)
        adapted = int((ids >= 0).sum())
        return {"bytes": weights + 4 * adapted * cols + 8 * case["rows"] * rows + 4 * case["rows"], "flops": 2 * sum(int(ranks[i]) for i in ids if i >= 0) * (rows + cols)}
    lens = _draft_lens(case)
    rows = int((lens + 1).sum()) + (int(lens.sum()) if case["by"] == "model" else 0)
    # of a logit: largest, difference, exponential, sum
    return {"bytes": 4 * rows * case["vocab"] + 16 * case["seqs"] * case["drafts"], "flops": 4 * rows * case["vocab"]}


# ── the definitions in 64 bits ─────────────────────────────────────────────────────────────────


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    t = {name: x.double() if x.is_floating_point() else x.long() for name, x in s["t"].items()}
    if case["kind"] == "attention":
        heads, kv, hd = HEADS[case["heads"]]
        group, nq, out = heads // kv, case["query"], torch.zeros_like(t["q"])
        for b in range(case["seqs"]):
            for i in range(nq):
                n = max(0, int(t["tail_lens"][b]) - (nq - 1 - i))
                k = torch.cat([t["prefix_k"], t["tail_k"][b, :n]])
                v = torch.cat([t["prefix_v"], t["tail_v"][b, :n]])
                q = t["q"][b, i].view(kv, group, hd)
                p = torch.softmax(torch.einsum("ghd,jgd->ghj", q, k) * hd ** -0.5, -1)
                out[b, i] = torch.einsum("ghj,jgd->ghd", p, v).reshape(heads, hd)
        return out
    if case["kind"] == "adapter":
        out = t["y"].clone()
        ids, ranks = t["row_adapter"].tolist(), t["ranks"].tolist()
        for a in sorted(set(ids) - {-1}):
            rows = torch.tensor([i for i, x in enumerate(ids) if x == a], device="cuda")
            delta = torch.matmul(t["up"][a, :, :ranks[a]], torch.matmul(t["down"][a, :ranks[a]], t["x"][rows].T))
            out[rows] += t["scales"][a] * delta.T
        return out
    return None  # whole numbers only

"""The hand-offs of the shared prefix on tcgen05 (csrc/prefix_attention_tc.cu) under random interleavings, on the CPU: one buffer of raw K and V and of K operands, two of V operands, of
scores and of probabilities by tile parity, waits that know a phase's parity only, MMAs that run in the order of their issue some time after it, and the words through which workers meet."""

import random

import pytest

from interleavings import Barrier, interleave

WORK, SUM = 8, 4


class Meeting:
    """bar.sync of so many warps."""

    def __init__(self, warps):
        self.warps, self.here, self.over = warps, 0, 0

    def meet(self):
        mine = self.over
        self.here += 1
        if self.here == self.warps:
            self.here, self.over = 0, self.over + 1
        return lambda: self.over > mine


def simulate(seed, n, s_wait=True, pv_wait=True, alpha_wait=True, raw_wait=True, inverses=4):
    rng = random.Random(seed)
    pair = lambda c: [Barrier(c), Barrier(c)]  # noqa: E731
    v_full, s_full, s_empty, p_full, pv_done, a_empty = pair(WORK), pair(1), pair(WORK), pair(WORK), pair(1), pair(SUM)
    k_full, o_full, o_empty, l_full = Barrier(WORK), Barrier(2), Barrier(SUM), Barrier(WORK)
    meet_k, meet_v, meet_rows = Meeting(WORK), Meeting(WORK), [Meeting(2) for _ in range(4)]
    raw = {x: {"full": Barrier(1), "empty": Barrier(WORK), "is": -1, "read": [-1] * WORK} for x in "kv"}
    K, V, P = [None] * WORK, [[None] * WORK for _ in range(2)], [[None] * WORK for _ in range(2)]
    S, O, alpha, inverse = [None, None], None, [[None] * SUM for _ in range(2)], [None] * 4
    k_used, v_used, p_used, s_read, o_read, alpha_read, inverse_read = -1, {-1, -2}, {-1, -2}, [[-2 + b] * WORK for b in range(2)], [-1] * SUM, [[-2 + b] * SUM for b in range(2)], [-1] * SUM
    most = {"k": [[None] * WORK for _ in range(2)], "v": [[None] * WORK for _ in range(2)]}
    most_read = {"k": [-1] * WORK, "v": [-1] * WORK}
    rows, rows_read = [[[None] * 2 for _ in range(2)] for _ in range(4)], [[-1] * 2 for _ in range(4)]
    queue = []

    def worker(w):
        quarter, half = w & 3, w >> 2

        def largest(which, meeting, j):
            at = j & 1
            assert min(most_read[which]) >= j - 2, "a word overwritten before it was read"
            most[which][at][w] = j
            yield meeting.meet()
            assert most[which][at] == [j] * WORK, "a largest element of another tile"
            yield lambda: True
            assert most[which][at] == [j] * WORK, "a largest element of another tile"
            most_read[which][w] = j

        def read(x, j):
            yield lambda: raw[x]["full"].over(j & 1)
            assert raw[x]["is"] == j, "another tile's fp32 values"
            yield lambda: True
            assert raw[x]["is"] == j, "another tile's fp32 values"
            raw[x]["read"][w] = j
            raw[x]["empty"].arrive()

        def read_k(j):
            yield from read("k", j)
            yield from largest("k", meet_k, j)

        def store_k(j):
            assert k_used >= j - 1, "K overwritten before its scores"
            K[w] = j
            yield lambda: True
            k_full.arrive()

        def convert_v(j):
            yield from read("v", j)
            yield from largest("v", meet_v, j)
            if pv_wait:
                yield lambda: pv_done[j & 1].over(j // 2 & 1 ^ 1)
            assert j - 2 in v_used, "V overwritten before it was used"
            V[j & 1][w] = j
            if w == 0:
                assert min(inverse_read) >= j - inverses, "an inverse scale overwritten before it was read"
                inverse[j % inverses] = j
            yield lambda: True
            v_full[j & 1].arrive()

        yield from read_k(0)
        yield from store_k(0)
        yield from convert_v(0)
        for j in range(n):
            b, ph = j & 1, j >> 1 & 1
            if j + 1 < n:
                yield from read_k(j + 1)
            if s_wait:
                yield lambda: s_full[b].over(ph)
            if j + 1 < n:
                yield from store_k(j + 1)
            assert S[b] == j, "scores of another tile"
            yield lambda: True
            assert S[b] == j
            s_read[b][w] = j
            s_empty[b].arrive()
            other = rows_read[quarter][half ^ 1]
            assert other >= j - 2, "a row's word overwritten before it was read"
            rows[quarter][b][half] = j
            yield meet_rows[quarter].meet()
            assert rows[quarter][b][half ^ 1] == j, "another tile's largest score"
            rows_read[quarter][half] = j
            if alpha_wait:
                yield lambda: a_empty[b].over(ph ^ 1)
            if half == 0:
                assert alpha_read[b][quarter] >= j - 2, "alpha overwritten before it was read"
                alpha[b][quarter] = j
            yield lambda: True
            assert j - 2 in p_used, "probabilities overwritten before they were used"
            P[b][w] = j
            p_full[b].arrive()
            if j + 1 < n:
                yield from convert_v(j + 1)
        l_full.arrive()

    def loader():
        def copy(x, j):
            def go():
                assert raw[x]["read"] == [j - 1] * WORK, "fp32 values overwritten before they were read"
                raw[x]["is"] = j
            return go

        for j in range(n):
            for x in "kv":
                if raw_wait:
                    yield lambda: raw[x]["empty"].over(j & 1 ^ 1)
                copies[x].extend([copy(x, j), raw[x]["full"].arrive])
                yield lambda: True

    copies = {"k": [], "v": []}

    def issue():
        def scores(j):
            def go():
                nonlocal k_used
                b = j & 1
                assert K == [j] * WORK, "scores of another tile's K"
                assert s_read[b] == [j - 2] * WORK, "scores overwritten before they were read"
                S[b], k_used = j, j
            return go

        def output(j):
            def go():
                nonlocal O
                assert V[j & 1] == [j] * WORK and P[j & 1] == [j] * WORK, "output of other operands"
                assert o_read == [j - 1] * SUM, "output overwritten before it was read"
                O = j
                v_used.add(j)
                p_used.add(j)
            return go

        for j in range(-1, n):
            if j + 1 < n:
                i = j + 1
                yield lambda: s_empty[i & 1].over(i >> 1 & 1 ^ 1)
                yield lambda: k_full.over(i & 1)
                queue.extend([scores(i), s_full[i & 1].arrive])
            if j >= 0:
                b, ph = j & 1, j >> 1 & 1
                yield lambda: v_full[b].over(ph)
                yield lambda: o_empty.over(j & 1 ^ 1)
                yield lambda: p_full[b].over(ph)
                queue.extend([output(j), o_full.arrive, pv_done[b].arrive])
                o_full.arrive()

    def sums(w):
        for j in range(n):
            yield lambda: o_full.over(j & 1)
            assert O == j and alpha[j & 1][w] == j and inverse[j % inverses] == j, "output, alpha or scale of another tile"
            inverse_read[w] = j
            alpha_read[j & 1][w] = j
            a_empty[j & 1].arrive()
            yield lambda: True
            assert O == j
            o_read[w] = j
            o_empty.arrive()
        yield lambda: l_full.over(0)

    interleave(rng, [issue(), loader()] + [worker(w) for w in range(WORK)] + [sums(w) for w in range(SUM)], [queue, *copies.values()])


@pytest.mark.parametrize("n", [1, 2, 3, 4, 9, 14])
def test_hand_offs_hold(n):
    for seed in range(60):
        simulate(seed, n)


@pytest.mark.parametrize("missing", [dict(s_wait=False), dict(pv_wait=False), dict(alpha_wait=False), dict(raw_wait=False), dict(inverses=1)])
def test_the_model_catches_what_is_missing(missing):
    with pytest.raises(AssertionError):
        for seed in range(400):
            simulate(seed, 9, **missing)

"""The hand-offs of the shared prefix on tcgen05 (csrc/prefix_attention_tc.cu) under random interleavings, on the CPU: three buffers of K, two of V, of scores and of
probabilities by tile parity, waits that know a phase's parity only, MMAs and copies that run in the order of their issue
(scores and outputs each in theirs) some time after it, and the words through which the halves of a row meet."""

import random

import pytest

from interleavings import Barrier, interleave

SOFT, SUM, PARTS = 8, 4, 2


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


def simulate(seed, n, k_wait=True, v_wait=True, alpha_wait=True, s_wait=True, o_wait=True):
    rng = random.Random(seed)
    pair = lambda c: [Barrier(c), Barrier(c)]  # noqa: E731
    k_full, k_empty = [Barrier(1) for _ in range(3)], [Barrier(1) for _ in range(3)]
    v_full, v_empty, s_full, s_empty, p_full, a_empty = pair(1), pair(1), pair(1), pair(SOFT), pair(SOFT), pair(SUM)
    o_full, o_empty, l_full = pair(2), pair(SUM), Barrier(SOFT)
    meet_rows = [Meeting(2) for _ in range(4)]
    K, V, S, P, O = [None] * 3, [None] * 2, [None] * 2, [[None] * SOFT for _ in range(2)], [None] * PARTS
    alpha = [[None] * SUM for _ in range(2)]
    k_used, v_used, p_used, s_read, o_read, alpha_read = {-1, -2, -3}, {-1, -2}, {-1, -2}, [[-2 + b] * SOFT for b in range(2)], [[-1] * SUM for _ in range(PARTS)], [[-2 + b] * SUM for b in range(2)]
    rows, rows_read = [[[None] * 2 for _ in range(2)] for _ in range(4)], [[-1] * 2 for _ in range(4)]
    queue, outputs, copies, value_copies = [], [], [], []

    def copy(to, used, j):
        def go():
            assert j - len(to) in used, "an operand overwritten before it was used"
            to[j % len(to)] = j
        return go

    def keys():
        for j in range(n):
            if j >= 2 and k_wait:
                yield lambda: k_empty[j % 3].over(j // 3 & 1 ^ 1)
            copies.extend([copy(K, k_used, j), k_full[j % 3].arrive])
            yield lambda: True

    def values():
        for j in range(n):
            b, ph = j & 1, j >> 1 & 1
            if v_wait:
                yield lambda: v_empty[b].over(ph ^ 1)
            value_copies.extend([copy(V, v_used, j), v_full[b].arrive])
            yield lambda: True

    def softmax(w):
        quarter, half = w & 3, w >> 2
        for j in range(n):
            b, ph = j & 1, j >> 1 & 1
            if alpha_wait:
                yield lambda: a_empty[b].over(ph ^ 1)
            yield lambda: s_full[b].over(ph)
            assert S[b] == j, "scores of another tile"
            yield lambda: True
            assert S[b] == j, "scores of another tile"
            s_read[b][w] = j
            s_empty[b].arrive()
            assert rows_read[quarter][half ^ 1] >= j - 2, "a row's word overwritten before it was read"
            rows[quarter][b][half] = j
            yield meet_rows[quarter].meet()
            assert rows[quarter][b][half ^ 1] == j, "another tile's largest score"
            rows_read[quarter][half] = j
            if half == 0:
                assert alpha_read[b][quarter] >= j - 2, "alpha overwritten before it was read"
                alpha[b][quarter] = j
            assert j - 2 in p_used, "probabilities overwritten before they were used"
            P[b][w] = j
            yield lambda: True
            p_full[b].arrive()
        l_full.arrive()

    def issue_scores():
        def scores(j):
            def go():
                b = j & 1
                assert K[j % 3] == j, "scores of another tile's K"
                assert s_read[b] == [j - 2] * SOFT, "scores overwritten before they were read"
                S[b] = j
                k_used.add(j)
            return go

        for j in range(n):
            if s_wait:
                yield lambda: s_empty[j & 1].over(j >> 1 & 1 ^ 1)
            yield lambda: k_full[j % 3].over(j // 3 & 1)
            queue.extend([scores(j), k_empty[j % 3].arrive, s_full[j & 1].arrive])

    def issue_output():
        def output(j, part):
            def go():
                assert V[j & 1] == j and P[j & 1] == [j] * SOFT, "output of other operands"
                assert o_read[part] == [j - 1] * SUM, "output overwritten before it was read"
                O[part] = j
                if part + 1 == PARTS:
                    v_used.add(j)
                    p_used.add(j)
            return go

        for j in range(n):
            b, ph = j & 1, j >> 1 & 1
            yield lambda: v_full[b].over(ph)
            yield lambda: p_full[b].over(ph)
            for part in range(PARTS):
                if o_wait:
                    yield lambda: o_empty[part].over(j & 1 ^ 1)
                outputs.append(output(j, part))
                if part + 1 == PARTS:
                    outputs.append(v_empty[b].arrive)
                outputs.append(o_full[part].arrive)
                o_full[part].arrive()

    def sums(w):
        for j in range(n):
            for part in range(PARTS):
                yield lambda: o_full[part].over(j & 1)
                assert O[part] == j and alpha[j & 1][w] == j, "output or alpha of another tile"
                if part + 1 == PARTS:
                    alpha_read[j & 1][w] = j
                    a_empty[j & 1].arrive()
                yield lambda: True
                assert O[part] == j
                o_read[part][w] = j
                o_empty[part].arrive()
        yield lambda: l_full.over(0)
        assert k_used >= set(range(n)) and v_used >= set(range(n)) and not queue and not outputs and not copies and not value_copies, "the operands' memory taken while they are in use"

    interleave(rng, [issue_scores(), issue_output(), keys(), values()] + [softmax(w) for w in range(SOFT)] + [sums(w) for w in range(SUM)], [queue, outputs, copies, value_copies])


@pytest.mark.parametrize("n", [1, 2, 3, 4, 9, 14])
def test_hand_offs_hold(n):
    for seed in range(60):
        simulate(seed, n)


@pytest.mark.parametrize("missing", ["k_wait", "v_wait", "alpha_wait", "s_wait", "o_wait"])
def test_the_model_catches_what_is_missing(missing):
    with pytest.raises(AssertionError):
        for seed in range(400):
            simulate(seed, 9, **{missing: False})

"""A model of the loss kernels' barrier protocol (loss_main_kernel), run under random schedules.

Roles, barriers, their arrival counts and phase bookkeeping are the kernel's; work is replaced by
checks of what each role must find: scores of the right tile in a buffer, probabilities of both
halves before the second product, offsets of the right tile in the ring, an accumulator that is
drained before it is started again. A wait models try_wait.parity: it passes when the phase of that
parity is over, whichever phase that is; the model then asserts that it was the phase meant, so a
wait that runs a phase early or late is caught as well as a deadlock.
"""
import random

import pytest


class Bar:
    def __init__(self, count):
        self.count, self.left, self.phase = count, count, 0

    def arrive(self, n=1):
        for _ in range(n):
            self.left -= 1
            if self.left == 0:
                self.left, self.phase = self.count, self.phase + 1


class Wait:
    """Waits for phase `index` (0-based) of `bar` by its parity."""

    def __init__(self, bar, index):
        self.bar, self.index = bar, index

    def ready(self):
        if self.index < 0:  # a fresh barrier's "previous" phase
            return True
        passed = (self.bar.phase & 1) != (self.index & 1)
        if passed:
            assert self.bar.phase == self.index + 1, f"phase {self.index} meant, {self.bar.phase} over"
        return passed


def simulate(units, f32, seed, wrong=None):
    """units: list of (tiles, add_every, bounded); returns the adds done per unit."""
    rng = random.Random(seed)
    stages, bufs = (3, 2) if f32 else (4, 3)
    full = [Bar(1) for _ in range(stages)]
    empty = [Bar(1 + 4) for _ in range(stages)]      # the commit; one arrival per modelled softmax role
    a_full = [Bar(4 if f32 else 1) for _ in range(2)]
    a_empty = [Bar(1) for _ in range(2)]
    s_full, s_free = [Bar(1) for _ in range(bufs)], [Bar(1) for _ in range(bufs)]
    p_full = [[Bar(1), Bar(1)] for _ in range(bufs)]
    o_full, o_empty = Bar(1), Bar(2)
    ring_bar = [Bar(1) for _ in range(4)]
    ms_full, ms_empty = Bar(4), Bar(1)
    top = [Bar(2), Bar(2)]
    # the pair that does not take a tile does not arrive on its stage: two of four roles do
    for b in empty:
        b.count = b.left = 1 + 2
    score, probs, ring = [None] * bufs, [[None, None] for _ in range(bufs)], [None] * 4
    acc, adds = {"tiles": [], "open": False}, []
    queues = {"s": [], "o": []}                       # products in flight, in order within an issuer

    def producer():
        cc = 0
        for uc, (n, _, _) in enumerate(units):
            if not f32:
                w = uc & 1
                yield Wait(a_empty[w], (uc >> 1) - 1)
                a_full[w].arrive()
            for _ in range(n):
                s = cc % stages
                yield Wait(empty[s], cc // stages - 1)
                full[s].arrive()
                cc += 1

    def score_issuer():
        cc = 0
        for uc, (n, _, _) in enumerate(units):
            w = 0 if f32 else uc & 1
            yield Wait(a_full[w], uc if f32 else uc >> 1)
            for _ in range(n):
                s, b = cc % stages, cc % bufs
                yield Wait(full[s], cc // stages)
                yield Wait(s_free[b], cc // bufs - 1)

                def done(b=b, cc=cc):
                    score[b], probs[b] = cc, [None, None]
                    s_full[b].arrive()
                queues["s"].append(done)
                cc += 1
            queues["s"].append(a_empty[w].arrive)

    def product_issuer():
        cc, taken = 0, 0
        for n, every, _ in units:
            held = 0
            for i in range(n):
                s, b = cc % stages, cc % bufs
                for half in range(2):
                    yield Wait(p_full[b][half], cc // bufs)
                yield Wait(o_empty, taken - 1)
                assert probs[b] == [cc, cc]
                held += 1
                last = held == every or i + 1 == n

                def done(b=b, s=s, cc=cc, first=held == 1, last=last):
                    assert probs[b] == [cc, cc] and acc["open"] != first
                    acc["tiles"] = [cc] if first else acc["tiles"] + [cc]
                    acc["open"] = True
                    if last:
                        o_full.arrive()
                    s_free[b].arrive()
                    empty[s].arrive()
                queues["o"].append(done)
                if last:
                    held, taken = 0, taken + 1
                cc += 1

    def softmax(g, half):
        cc = rc = tc = 0
        for uc, (n, every, bounded) in enumerate(units):
            i0 = (g ^ cc) & 1
            if f32:
                yield Wait(a_empty[0], uc - 1)
                a_full[0].arrive()
            ringed = every == 1
            for i in range(i0, n, 2):
                t = cc + i
                b = t % bufs
                yield Wait(s_full[b], t // bufs)
                assert score[b] == t and probs[b][half] is None
                if not bounded:
                    top[g].arrive()
                    yield Wait(top[g], tc if wrong != "tile count" else t // 2)
                    tc += 1
                if ringed and half == 0:
                    ring[(rc + i) & 3] = t
                yield None
                probs[b][half] = t
                p_full[b][half].arrive()
                empty[t % stages].arrive()
                if ringed and half == 0:
                    ring_bar[(rc + i) & 3].arrive()
            cc += n
            rc += n if ringed else 0
            yield Wait(ms_empty, uc - 1)
            ms_full.arrive()

    def adder(g):
        fc = rc = cc = 0
        for uc, (n, every, _) in enumerate(units):
            for c in range(0, n, every):
                if every == 1:
                    yield Wait(ring_bar[rc & 3], rc >> 2)
                    assert ring[rc & 3] == cc + c
                    rc += 1
                yield Wait(o_full, fc)
                assert acc["tiles"] == list(range(cc + c, cc + min(c + every, n)))
                yield None
                if g == 0:
                    adds.append(list(acc["tiles"]))
                drained[fc] = drained.get(fc, 0) + 1
                if drained[fc] == 2:
                    acc["open"] = False
                o_empty.arrive()
                fc += 1
            cc += n
            if g == 0:
                yield Wait(ms_full, uc)
                ms_empty.arrive()

    drained = {}
    roles = [producer(), score_issuer(), product_issuer(), adder(0), adder(1)]
    roles += [softmax(g, half) for g in range(2) for half in range(2)]
    blocked = {i: None for i in range(len(roles))}
    while blocked or queues["s"] or queues["o"]:
        moves = [i for i, w in blocked.items() if w is None or w.ready()]
        moves += [q for q in queues if queues[q]]
        assert moves, f"deadlock: {[type(w).__name__ for w in blocked.values()]}"
        m = rng.choice(moves)
        if isinstance(m, str):
            queues[m].pop(0)()
            continue
        try:
            blocked[m] = next(roles[m])
        except StopIteration:
            del blocked[m]
    return adds


def unit_lists(rng):
    return [(rng.choice([1, 1, 2, 3, 4, 5, 7, 9, 37]), rng.choice([1, 1, 32, 4]), rng.random() < 0.5)
            for _ in range(rng.randint(1, 7))]


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("seed", range(40))
def test_no_deadlock_and_every_tile_added_once(f32, seed):
    rng = random.Random(seed)
    units = unit_lists(rng)
    if f32:
        units = [(n, 1, False) for n, _, _ in units]  # f32 adds every tile and follows the maximum
    else:
        # offsets are handed on, and maxima exchanged, where a unit's rows are not all bounded; a warp
        # whose own rows are bounded exchanges nothing even then
        units = [(n, e, b or e != 1) for n, e, b in units]
    adds = simulate(units, f32, seed)
    assert [t for a in adds for t in a] == list(range(sum(n for n, _, _ in units)))


def test_the_model_sees_a_phase_counted_by_the_wrong_thing():
    """An exchange of maxima counted by tiles instead of by exchanges fails once a unit had none."""
    units = [(3, 32, True), (4, 1, False), (5, 32, True), (6, 1, False)]
    with pytest.raises(AssertionError):
        for seed in range(20):
            simulate(units, False, seed, wrong="tile count")

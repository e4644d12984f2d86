"""A discrete model of the mbarrier protocol of the chunk kernel over an 8-bit cache
(csrc/kv8_prefill.cu), checked for deadlocks over random schedules on the CPU, with the phase
semantics of the hardware (tests/test_prefill_barrier_model.py).

Roles, as in the kernel: converters that fill KS = 2 key buffers and one or two value buffers in
turn; for each of two query tiles an issuer (S(j), then PV(j) behind the softmax's P(j), the next
S either behind that PV or, with P beside S, ahead of it) and a softmax of two halves that exchange
their maxima. Tile 1's issuer starts a softmax behind tile 0's. Products complete in the order they
were issued; a commit arrives when everything before it is complete.

If that start is a wait for the barrier on which tile 0's softmax hands over every P, tile 1's
queries may come so late that the barrier is two phases ahead and looks as if none were complete:
then tile 0 waits for the key buffer that tile 1 has not read, and tile 1 for a tile 0 that waits.
A barrier of its own, completed once, cannot be missed."""
import os
import random
import re

import pytest

from tests.conftest import ROOT
from tests.test_prefill_barrier_model import Bar

KS = 2  # key buffers


def run(n_tiles, beside, vs, late, seed, own_start, steps=60000):
    """Whether every role ends. late: steps before tile 1's queries are there."""
    rnd = random.Random(seed)
    q_full, s_full, s_free = ([Bar(n) for _ in range(2)] for n in (2, 2, 2))
    p_full, pv_done = ([Bar(n) for _ in range(2)] for n in (2, 1))
    k_full, k_empty = ([Bar(n) for _ in range(KS)] for n in (1, 2))
    v_full, v_empty = ([Bar(n) for _ in range(vs)] for n in (1, 2))
    started = Bar(1)
    pipe = []
    met = [[0, 0], [0, 0]]  # exchanges that each half of a query tile has come to

    def wait(bar, parity):
        while not bar.done(parity & 1):
            yield

    def pause(most):
        for _ in range(rnd.randint(0, most)):
            yield

    def converters():
        for j in range(n_tiles):
            if j >= KS:
                yield from wait(k_empty[j % KS], j // KS - 1)
            yield from pause(3)
            k_full[j % KS].arrive()
            if j >= vs:
                yield from wait(v_empty[j % vs], j // vs - 1)
            yield from pause(3)
            v_full[j % vs].arrive()

    def issuer(t):
        def scores(j):
            yield from wait(k_full[j % KS], j // KS)
            if j:
                yield from wait(s_free[t] if beside else pv_done[t], j - 1)
            pipe.append([rnd.randint(1, 10), [s_full[t], k_empty[j % KS]]])
            s_full[t].arrive()

        yield from wait(q_full[t], 0)
        if t == 1:
            yield from wait(started if own_start else p_full[0], 0)
        if beside:
            yield from scores(0)
        for j in range(n_tiles):
            if not beside:
                yield from scores(j)
            elif j + 1 < n_tiles:
                yield from scores(j + 1)
            yield from wait(p_full[t], j)
            if t == 0 and j == 0:
                started.arrive()
            yield from wait(v_full[j % vs], j // vs)
            pipe.append([rnd.randint(1, 10), [pv_done[t], v_empty[j % vs]]])

    def softmax(t, half):
        if t == 1:
            for _ in range(late):
                yield
        q_full[t].arrive()
        for j in range(n_tiles):
            yield from wait(s_full[t], j)
            yield from pause(10)
            met[t][half] += 1
            while met[t][half ^ 1] < met[t][half]:
                yield
            if beside and j:
                yield from wait(pv_done[t], j - 1)
            yield from pause(10)
            if beside:
                s_free[t].arrive()
            p_full[t].arrive()
        yield from wait(pv_done[t], n_tiles - 1)

    alive = {"converters": converters()}
    for t in range(2):
        alive[f"issuer{t}"] = issuer(t)
        for half in range(2):
            alive[f"softmax{t}.{half}"] = softmax(t, half)
    for _ in range(steps):
        if not alive:
            return True
        if pipe:
            pipe[0][0] -= 1
            if pipe[0][0] <= 0:
                for b in pipe.pop(0)[1]:
                    b.arrive()
        for k in list(alive):
            if rnd.random() < 0.3:
                continue
            try:
                next(alive[k])
            except StopIteration:
                del alive[k]
    return False


FORMS = [(False, 1), (False, 2), (True, 2)]  # P beside S or over it, value buffers


@pytest.mark.parametrize("beside,vs", FORMS)
def test_a_start_of_its_own_never_deadlocks(beside, vs):
    for seed in range(120):
        rnd = random.Random(seed)
        n_tiles, late = rnd.choice([1, 2, 3, 8]), rnd.choice([0, 5, 40, 200, 2000])
        assert run(n_tiles, beside, vs, late, seed, True), (n_tiles, late, seed)


@pytest.mark.parametrize("beside,vs", FORMS)
@pytest.mark.parametrize("n_tiles", [2, 3, 8])
def test_a_start_on_the_barrier_of_every_tile_can_be_missed(beside, vs, n_tiles):
    assert not all(run(n_tiles, beside, vs, 2000, seed, False, 20000) for seed in range(10))


def test_the_kernel_waits_once_only_on_barriers_that_complete_once():
    """In the source: a barrier that some wait names with a constant parity is one whose every wait does, so it
    is not also the barrier of a loop, whose phases go on behind the waiter's back."""
    with open(os.path.join(ROOT, "zwhisper_b200", "csrc", "kv8_prefill.cu")) as f:
        code = f.read()
    once, many = set(), set()
    for call in re.findall(r"mbar_wait(?:_warp|_drain)?\((.*?)\)", code):
        names = re.findall(r"&sm\.(\w+)", call)
        assert names, call
        parity = re.sub(r".*\]|.*&sm\.\w+", "", call.split("err")[0]).strip(" ,")
        (once if parity == "0" else many).update(names)
    assert {"q_full", "drained"} <= once and {"p_full", "k_full", "pv_done"} <= many
    assert not once & many, once & many

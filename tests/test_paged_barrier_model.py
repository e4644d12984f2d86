"""A discrete model of the mbarrier protocol of the chunk kernel over a cache in pages
(csrc/paged_chunk.cu), checked over random schedules on the CPU for deadlocks, for barriers that complete twice
behind a waiter's back and for buffers that are written while they are read, with the phase semantics of the
hardware (tests/test_prefill_barrier_model.py).

Roles, as in the kernel: a loader that fills key and value buffers in turn; the warp that goes over values;
for each of two slots an issuer and a softmax of two halves. `two`: both slots take every key tile, else
every other one each. `early`: the next S is issued once this one has been read, else behind the PV. `turns`: the
slots' exponentials follow each other.
Products complete in the order each issuer gave them; a commit arrives when everything before it is complete."""
import os
import random
import re

import pytest

from tests.conftest import ROOT
from tests.test_prefill_barrier_model import Bar

# early, key buffers, value buffers with two slots of rows (with one both have two), exponentials in turns
FORMS = {"d64": (True, 2, 2, True), "d128": (True, 1, 2, True), "d64 f32": (False, 2, 2, False), "d128 f32": (False, 2, 1, True)}


class Broken(Exception):
    pass


def run(form, two, n_tiles, seed, steps=200000):
    """Whether every role ends."""
    early, ks, vs, turns = FORMS[form]
    if not two:
        ks = vs = 2
    rnd = random.Random(seed)
    slots = 2 if two else 1
    k_full, v_full, v_ready = ([Bar(1) for _ in range(2)] for _ in range(3))
    k_empty, v_empty = ([Bar(slots) for _ in range(2)] for _ in range(2))
    s_full, s_free, p_full, pv_done = ([Bar(n) for _ in range(2)] for n in (2, 2, 2, 1))
    started, turn = Bar(1), [Bar(2), Bar(2)]
    pipes = [[], []]
    buffers = {}  # what lies in a buffer, and how many still read it
    met = [[0, 0], [0, 0]]

    def write(name, what):
        if buffers.get(name, (None, 0))[1]:
            raise Broken(f"{name} is written while it is read")
        buffers[name] = (what, 0)

    def read(name, what, more):
        have, readers = buffers.get(name, (None, 0))
        if have != what:
            raise Broken(f"{name} holds {have}, not {what}")
        buffers[name] = (have, readers + more)

    def wait(bar, parity):
        while not bar.done(parity & 1):
            yield

    def pause(most):
        for _ in range(rnd.randint(0, most)):
            yield

    def loader():
        for j in range(n_tiles):
            if j >= ks:
                yield from wait(k_empty[j % ks], j // ks - 1)
            write(f"k{j % ks}", j)
            yield from pause(6)
            k_full[j % ks].arrive()
            if j >= vs:
                yield from wait(v_empty[j % vs], j // vs - 1)
            write(f"v{j % vs}", j)
            yield from pause(6)
            v_full[j % vs].arrive()

    def sweeper():
        for j in range(n_tiles):
            yield from wait(v_full[j % vs], j // vs)
            read(f"v{j % vs}", j, 0)
            yield from pause(8)
            v_ready[j % vs].arrive()

    def tile(t, it):
        return it if two else 2 * it + t

    def count(t):
        return n_tiles if two else (n_tiles - t + 1) // 2

    def issuer(t):
        mine = count(t)

        def give(reads, bars):
            for name, what in reads:
                read(name, what, 1)
            pipes[t].append([rnd.randint(1, 10), reads, bars])

        def keys(it):
            j = tile(t, it)
            yield from wait(k_full[j % ks], j // ks)

        def scores(it):
            j = tile(t, it)
            if it:
                yield from wait(s_free[t] if early else pv_done[t], it - 1)
            write(f"s{t}", it)
            give([(f"k{j % ks}", j)], [s_full[t], k_empty[j % ks]])
            s_full[t].arrive()

        if mine == 0:
            return
        yield from keys(0)
        yield from scores(0)
        for it in range(mine):
            j, more = tile(t, it), it + 1 < mine
            if more and two:
                yield from keys(it + 1)
                if early:
                    yield from scores(it + 1)
            yield from wait(v_full[j % vs], j // vs)
            yield from wait(v_ready[j % vs], j // vs)
            yield from wait(p_full[t], it)
            give([(f"v{j % vs}", j), (f"p{t}", (it, 2))], [pv_done[t], v_empty[j % vs]])
            if t == 0 and it == 0:
                started.arrive()
            if more and not two:
                yield from keys(it + 1)
            if more and not (early and two):
                yield from scores(it + 1)

    def softmax(t, half):
        for it in range(count(t)):
            if not turns and t == 1 and it == 0:
                yield from wait(started, 0)
            yield from wait(s_full[t], it)
            read(f"s{t}", it, 1)
            yield from pause(10)
            met[t][half] += 1
            while met[t][half ^ 1] < met[t][half]:
                yield
            if early:
                read(f"s{t}", it, -1)
                s_free[t].arrive()
                if it:
                    yield from wait(pv_done[t], it - 1)
            if turns and (t == 1 or it):
                yield from wait(turn[t], it - 1 if t == 0 else it)
            yield from pause(10)
            if turns:
                turn[t ^ 1].arrive()
            if not early:
                read(f"s{t}", it, -1)
            have = buffers.get(f"p{t}", (None, 0))
            if have[1]:
                raise Broken("P is written while it is read")
            buffers[f"p{t}"] = ((it, have[0][1] + 1 if have[0] and have[0][0] == it else 1), 0)
            p_full[t].arrive()
        if count(t):
            yield from wait(pv_done[t], count(t) - 1)

    alive = {"loader": loader(), "sweeper": sweeper()}
    for t in range(2):
        alive[f"issuer{t}"] = issuer(t)
        for half in range(2):
            alive[f"softmax{t}.{half}"] = softmax(t, half)
    slow = {k: rnd.choice([0.1, 0.3, 0.9]) for k in alive}
    for _ in range(steps):
        if not alive:
            return True
        for pipe in pipes:
            if pipe:
                pipe[0][0] -= 1
                if pipe[0][0] <= 0:
                    _, reads, bars = pipe.pop(0)
                    for name, what in reads:
                        read(name, what, -1)
                    for b in bars:
                        b.arrive()
        for k in list(alive):
            if rnd.random() < slow[k]:
                continue
            try:
                next(alive[k])
            except StopIteration:
                del alive[k]
    return False


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("two", [True, False])
def test_no_deadlock_and_no_buffer_written_while_read(form, two):
    for seed in range(150):
        n_tiles = random.Random(seed).choice([0, 1, 2, 3, 4, 5, 9])
        assert run(form, two, n_tiles, seed), (n_tiles, seed)


def test_the_model_would_find_a_buffer_too_few():
    """Values that one slot still reads, overwritten: a loader that waits for one slot's products only."""
    global FORMS
    kept = dict(FORMS)
    try:
        FORMS["d64"] = (True, 2, 3, True)  # a third buffer of barriers that there are two of
        with pytest.raises((Broken, IndexError)):
            for seed in range(20):
                run("d64", True, 9, seed)
    finally:
        FORMS.update(kept)


def test_the_kernel_waits_once_only_on_barriers_that_complete_once():
    """In the source: a barrier that some wait names with a constant parity is one whose every wait does."""
    with open(os.path.join(ROOT, "zwhisper_b200", "csrc", "paged_chunk.cu")) as f:
        code = f.read()
    once, many = set(), set()
    for call in re.findall(r"mbar_wait(?:_warp|_drain)?\((.*?)\)", code):
        names = re.findall(r"&sm\.(\w+)", call)
        assert names, call
        parity = re.sub(r".*\]|.*&sm\.\w+", "", call.split("err")[0]).strip(" ,")
        (once if parity == "0" else many).update(names)
    assert {"q_full", "drained", "started"} <= once and {"p_full", "k_full", "pv_done"} <= many
    assert not once & many, once & many

"""The barrier model of the chunk kernel over a cache in pages (tests/test_paged_barrier_model.py) tells faults that are
planted in it: a buffer given back by one of the two slots that read it, a pass over the values that nobody waits for, a score
tile taken for free before it has been read. Each has to end in the buffer it spoils, not in any other error."""
import pytest

from tests import test_paged_barrier_model as M

# the order in which the model makes its barriers: k_full, v_full, v_ready, k_empty, v_empty, s_full, s_free, p_full, pv_done
# (two each), started, turn (two)
NAMES = ["k_full", "v_full", "v_ready", "k_empty", "v_empty", "s_full", "s_free", "p_full", "pv_done"]
COUNTS = {"k_full": 1, "v_full": 1, "v_ready": 1, "k_empty": 2, "v_empty": 2, "s_full": 2, "s_free": 2, "p_full": 2, "pv_done": 1}


def planted(monkeypatch, name, count):
    """Barriers `name` of the next runs of two slots complete at `count` arrivals."""
    made = []

    def bar(n):
        which = NAMES[len(made) // 2] if len(made) < 2 * len(NAMES) else None
        assert which is None or n == COUNTS[which], (which, n)
        made.append(n)
        return M_BAR(count if which == name else n)

    M_BAR = M.Bar
    monkeypatch.setattr(M, "Bar", bar)
    return made


# not told, as another wait covers it: scores that are taken back behind the values' product (not early), and keys where values
# have one buffer (tile j + 2's come behind tile j + 1's values, which wait for both slots' products of tile j)
CASES = [(form, name, buffer) for form, (early, _, vs, _) in M.FORMS.items()
         for name, buffer in (("k_empty", "k"), ("v_empty", "v"), ("s_free", "s"), ("p_full", "p"))
         if not (name == "s_free" and not early) and not (name == "k_empty" and vs == 1)]


@pytest.mark.parametrize("form,name,buffer", CASES)
def test_a_barrier_that_completes_too_soon_is_found(monkeypatch, form, name, buffer):
    made, found = planted(monkeypatch, name, 1), []
    for seed in range(60):
        del made[:]
        try:
            M.run(form, True, 9, seed, steps=20000)
        except M.Broken as e:
            found.append(str(e))
    assert found and all(e.startswith((buffer, buffer.upper())) for e in found), found[:3]


def test_the_barriers_are_named_in_the_models_order(monkeypatch):
    made = planted(monkeypatch, "k_full", 1)
    for form in M.FORMS:
        del made[:]
        assert M.run(form, True, 4, 0)
        assert len(made) == 2 * len(NAMES) + 3

"""Model check of the paged decode kernel's load ring (csrc/paged_attention.cu).

One warp issues loads in order into ``S`` stages; loads land in any order; ``W`` warps wait for
their tiles by barrier parity, which cannot tell a phase from the one before the last. With the
stage count a multiple of the warp count every stage belongs to one warp and all schedules are
safe; otherwise a warp can pass a barrier two phases early.
"""

import random

import pytest


def _run(stages, warps, tiles, seed):
    """'ok', 'early' (a warp read a stage before its tile landed) or 'stuck'."""
    rng = random.Random(seed)
    full, empty = [0] * stages, [0] * stages      # completed phases
    issued, flying = 0, []
    todo = [[j for j in range(tiles) if j % warps == w] for w in range(warps)]
    while True:
        moves = []
        if issued < tiles and empty[issued % stages] >= issued // stages:
            moves.append(("issue", None))
        moves += [("land", j) for j in flying]
        moves += [("use", w) for w in range(warps)
                  if todo[w] and full[todo[w][0] % stages] % 2 != (todo[w][0] // stages) % 2]
        if not moves:
            return "stuck" if any(todo) else "ok"
        what, x = rng.choice(moves)
        if what == "issue":
            flying.append(issued)
            issued += 1
        elif what == "land":
            flying.remove(x)
            full[x % stages] += 1
        else:
            j = todo[x].pop(0)
            if full[j % stages] != j // stages + 1:
                return "early"
            empty[j % stages] += 1


@pytest.mark.parametrize("stages", [8, 12, 16])
def test_stage_count_multiple_of_warps_is_safe(stages):
    assert all(_run(stages, 4, 70, seed) == "ok" for seed in range(100))


@pytest.mark.parametrize("stages", [7, 11])
def test_other_stage_counts_read_early(stages):
    assert any(_run(stages, 4, 70, seed) == "early" for seed in range(100))

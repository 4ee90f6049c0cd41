"""How the loaders of the tcgen05 prompt kernel over a 4-bit cache share its ring, as a model on the CPU: workers fill units in turn, one or two of
them an item, an item a stage, and the products take the items in order.  A barrier tells a phase from its neighbours only (one bit), so the
model looks through every order of events for a stage that is overwritten, a wait that passes too early, and a wait that never ends."""

import pytest

STAGES = 4


def outcomes(items, workers, units_per_item, waits_for):
    """All ends that some order of events has: "done", "stuck", "early".  A worker's next unit is filled in two events, the waits and the
    arrival.  ``waits_for(i)``: the items for whose stages a worker polls before a unit of item i, one poll after the other."""
    # state: per worker (its unit, polls passed, or -1 while it fills), the units that have arrived of items not yet consumed, and the number
    # of items that were
    start = (tuple((worker, 0) for worker in range(workers)), frozenset(), 0)
    seen, todo, ends = {start}, [start], set()
    while todo:
        state, arrived, consumed = todo.pop()
        moves = []
        whole = {consumed * units_per_item + u for u in range(units_per_item)}
        if whole <= arrived:
            moves.append((state, arrived - whole, consumed + 1))
        for worker, (unit, passed) in enumerate(state):
            item = unit // units_per_item
            if item >= items:
                continue
            if passed < 0:          # the rows are written, the arrival is made
                moves.append((state[:worker] + ((unit + workers, 0),) + state[worker + 1:], arrived | {unit}, consumed))
                continue
            polled = waits_for(item)[passed]
            done = len(range(polled % STAGES, consumed, STAGES))             # phases that the stage's barrier has behind it
            if done % 2 != (polled // STAGES) % 2:
                continue
            if passed + 1 < len(waits_for(item)):
                now = (unit, passed + 1)
            else:
                if item >= STAGES and consumed <= item - STAGES:
                    ends.add("early")
                    continue
                now = (unit, -1)
            moves.append((state[:worker] + (now,) + state[worker + 1:], arrived, consumed))
        if not moves:
            ends.add("done" if consumed == items else "stuck")
        for move in moves:
            if move not in seen:
                seen.add(move)
                todo.append(move)
    return ends


@pytest.mark.parametrize("items", [1, 2, 5, 8, 13])
@pytest.mark.parametrize("workers,units_per_item", [(6, 2), (3, 1)])
def test_a_worker_that_waits_for_its_own_stage_is_never_early_and_never_stuck(items, workers, units_per_item):
    assert outcomes(items, workers, units_per_item, lambda i: [i]) == {"done"}


def test_a_worker_that_waits_for_the_stages_of_others_can_be_stuck():
    assert "stuck" in outcomes(13, 3, 1, lambda i: list(range(max(i - 2, 0), i + 1)))

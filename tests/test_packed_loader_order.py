"""How the loaders of the tcgen05 prompt kernel over a 4-bit cache share its ring, as a model on the CPU: teams fill items in turn, a stage
each, and the products take the items in order.  A barrier tells a phase from its neighbours only (one bit), so the model looks through
every order of events for a stage that is overwritten, a wait that passes too early, and a wait that never ends."""

import pytest

TEAMS, STAGES = 3, 4


def outcomes(items, waits_for):
    """All ends that some order of events has: "done", "stuck", "early".  A team's next item is filled in two events, the waits and the
    arrival.  ``waits_for(i)``: the items for whose stages the team polls before item i, one poll after the other."""
    # state: per team (its item, polls passed, or -1 while it fills), the items that have arrived, the number that were consumed
    start = (tuple((team, 0) for team in range(TEAMS)), frozenset(), 0)
    seen, todo, ends = {start}, [start], set()
    while todo:
        teams, arrived, consumed = todo.pop()
        moves = []
        if consumed in arrived:
            moves.append((teams, arrived, consumed + 1))
        for team, (item, passed) in enumerate(teams):
            if item >= items:
                continue
            if passed < 0:          # the rows are written, the arrival is made
                moves.append((teams[:team] + ((item + TEAMS, 0),) + teams[team + 1:], arrived | {item}, consumed))
                continue
            polled = waits_for(item)[passed]
            done = sum(1 for i in range(polled % STAGES, consumed, STAGES))             # phases that the stage's barrier has behind it
            if done % 2 != (polled // STAGES) % 2:
                continue
            if passed + 1 < len(waits_for(item)):
                now = (item, passed + 1)
            else:
                if item >= STAGES and consumed <= item - STAGES:
                    ends.add("early")
                    continue
                now = (item, -1)
            moves.append((teams[:team] + (now,) + teams[team + 1:], arrived, consumed))
        if not moves:
            ends.add("done" if consumed == items else "stuck")
        for state in moves:
            if state not in seen:
                seen.add(state)
                todo.append(state)
    return ends


@pytest.mark.parametrize("items", [1, 2, 5, 8, 13, 18])
def test_a_team_that_waits_for_its_own_stage_is_never_early_and_never_stuck(items):
    assert outcomes(items, lambda i: [i]) == {"done"}


def test_a_team_that_waits_for_the_stages_of_others_can_be_stuck():
    assert "stuck" in outcomes(13, lambda i: list(range(max(i - TEAMS + 1, 0), i + 1)))

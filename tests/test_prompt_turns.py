"""The hand-over of turns at the exponentials, every interleaving of it (no GPU).

Two warps, one of each query tile, take turns through two mbarriers: a warp waits for its own, does its share, and
lane 0 arrives on the other's before the warp meets again at its tensor-memory store.  An mbarrier shows only the parity
of its phases, so a lane that looks late must never find its phase two steps behind.  The model below walks through every
order in which the lanes can run; whether the lanes of a warp leave the wait together is read from the kernel's source.
"""

from __future__ import annotations

from pathlib import Path
import re

SOURCE = Path(__file__).resolve().parents[1] / "fragpack_b200" / "csrc" / "prompt_attn.cu"
LANES, ROUNDS = 2, 3
WAIT, MEET, PASS_ON, STORE = range(4)  # steps of a round: wait, leave together, lane 0 passes the turn on, store (all lanes)


def _stuck_states(synced: bool) -> int:
    """How many reachable states have unfinished lanes and none that can go on."""
    steps = [WAIT, MEET, PASS_ON, STORE] if synced else [WAIT, PASS_ON, STORE]
    size, end = len(steps), len(steps) * ROUNDS

    def can_go(state, warp, lane):
        at, phases = state
        pc = at[warp * LANES + lane]
        if pc == end:
            return False
        step, turn = steps[pc % size], pc // size
        if step == WAIT:  # true once the phase of this parity is complete
            return (phases[warp] & 1) != (turn + warp + 1) & 1
        if step in (MEET, STORE):
            return all(other >= pc for other in at[warp * LANES : (warp + 1) * LANES])
        return True

    start = ((0,) * (2 * LANES), (0, 0))
    seen, todo, stuck = {start}, [start], 0
    while todo:
        state = todo.pop()
        moved = False
        for warp in (0, 1):
            for lane in range(LANES):
                if not can_go(state, warp, lane):
                    continue
                moved = True
                at, phases = list(state[0]), list(state[1])
                if steps[at[warp * LANES + lane] % size] == PASS_ON and lane == 0:
                    phases[warp ^ 1] += 1
                at[warp * LANES + lane] += 1
                after = (tuple(at), tuple(phases))
                if after not in seen:
                    seen.add(after)
                    todo.append(after)
        stuck += not moved and any(pc < end for pc in state[0])
    return stuck


def test_lanes_that_leave_the_wait_one_by_one_could_miss_a_phase() -> None:
    assert _stuck_states(synced=False) > 0


def test_a_turn_is_taken_by_the_whole_warp() -> None:
    text = SOURCE.read_text()
    start = text.index("const auto take_turn = [&] {")
    taking = text[start : text.index("};", start)]
    synced = re.search(r"sm\.turn\[mine\].*__syncwarp\(\);", taking, re.DOTALL) is not None
    assert _stuck_states(synced) == 0


def test_a_wait_that_ends_a_loop_ends_it_for_the_whole_warp() -> None:
    """A lane that saw the wait give up must not leave a loop that the others go on with: the warp meets in it."""
    text = SOURCE.read_text()
    load = text.index("void prompt_load(")  # one lane's waits
    code = text[text.index("void prompt_items(") : load] + text[text.index("void issue_scores(") :]
    deciding = [line.strip() for line in code.splitlines() if re.search(r"(!|=\s*|return\s+|&&\s*)await\(", line)]
    assert not deciding

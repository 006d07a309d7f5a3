"""The ring of code units in the two-tile attention over the INT8 cache, as a
model: one thread copies the units of K and V in turn (K, K, V, V per key tile),
two teams use them, and copies may land in any order.

An mbarrier's parity wait tells the current phase from the one before it and no
more. A team that waits for its use of a slot may therefore only wait on a
barrier whose earlier phases it has seen complete. With one barrier per slot it
need not have: the other team's copy into that slot may still be on its way."""
import random
import re
from pathlib import Path

import pytest

SOURCE = (Path(__file__).resolve().parents[1] / "qwen-image-2.1-accel_b200" / "csrc" / "cached_attn_tiles.cu").read_text()


class Barrier:
    """Completed phases of a barrier of one arrival and its bytes."""

    def __init__(self):
        self.phase, self.pending = 0, None        # pending: the unit of the current phase, once announced

    def announce(self, unit):
        assert self.pending is None, "a second arrival in one phase"
        self.pending = unit

    def land(self):
        self.phase, self.pending = self.phase + 1, None

    def passes(self, parity):                     # the phase before the current one has that parity
        return (self.phase - 1) % 2 == parity


def run(units, tiles, per_team, rng):
    """One random schedule; the units that a team used before they had landed."""
    full = [[Barrier() for _ in range(units)] for _ in range(2 if per_team else 1)]
    empty = [0] * units                           # uses of a slot that are done
    issued, flying, landed, early = 0, [], set(), []
    order = [[u for u in range(4 * tiles) if (u >> 1) & 1 == z] for z in range(2)]
    done, phases = [0, 0], [0, 0]
    barrier_of = lambda u: full[(u >> 1) & 1 if per_team else 0][u % units]       # noqa: E731

    def parity(z, u):
        return (phases[z] >> (u % units)) & 1 if per_team else (u // units) & 1

    while done != [2 * tiles, 2 * tiles]:
        moves = []
        if issued < 4 * tiles and empty[issued % units] == issued // units:
            moves.append("issue")
        moves += [("land", u) for u in flying]
        for z in range(2):
            if done[z] < 2 * tiles and barrier_of(order[z][done[z]]).passes(parity(z, order[z][done[z]])):
                moves.append(("use", z))
        assert moves, "nothing can move"
        move = rng.choice(moves)
        if move == "issue":
            barrier_of(issued).announce(issued)
            flying.append(issued)
            issued += 1
        elif move[0] == "land":
            flying.remove(move[1])
            landed.add(move[1])
            barrier_of(move[1]).land()
        else:
            z = move[1]
            u = order[z][done[z]]
            if u not in landed:
                return [u]
            phases[z] ^= 1 << (u % units)
            empty[u % units] += 1
            done[z] += 1
    return early


@pytest.mark.parametrize("units", [3, 7])
def test_a_team_waits_for_its_own_copy(units):
    rng = random.Random(units)
    for _ in range(400):
        assert not run(units, rng.randint(1, 12), True, rng)
    assert any(run(units, 8, False, rng) for _ in range(400))       # one barrier per slot: used too early


def test_the_kernel_has_a_barrier_per_slot_and_team():
    full = re.findall(r"uint64_t\* (stage_full\w*) = bars \+ (\d+);", SOURCE)
    most = 7                                      # units of a CTA with one query tile
    assert len(full) == 2 and abs(int(full[0][1]) - int(full[1][1])) >= most

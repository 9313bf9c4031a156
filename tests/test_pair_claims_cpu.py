"""The pair kernel's claims (scan_dfa.h pair_static_group / pair_ticket_group, the kernel's own functions) under every residency.

The model: at most `slots` of the grid's workgroups run at once, the next one starts when one ends; a workgroup scans its groups in order,
waits — before it publishes a group's count — for the counts in front of the group before it, and draws the group after next while it scans.
With every group a ticket the launch ends whatever fits on the device.  With the static start it ends if the whole grid is resident, which is
why a launch that met the spin limit is repeated on tickets."""
import random

import pytest

import emu

NONE = 0xFFFFFFFF


def _launch(ngroups, nwg, slots, static_start, seed):
    """(groups in the order in which they were counted, ended) of one launch; the order of the steps is random."""
    L, rng = emu.lib(), random.Random(seed)
    counted, order, ticket = set(), [], 0
    waiting_to_start, running, handed = list(range(nwg)), {}, []

    def draw():
        nonlocal ticket
        g = L.emu_pair_ticket_group(ticket, nwg, ngroups, int(static_start))
        ticket += 1
        if g != NONE:
            handed.append(g)
        return g

    def start():
        while waiting_to_start and len(running) < slots:
            b = waiting_to_start.pop(0)
            if static_start:
                q = [L.emu_pair_static_group(b, k, nwg, ngroups) for k in (0, 1)]
                handed.extend(g for g in q if g != NONE)
            else:
                q = [draw(), draw()]
            running[b] = {"q": q, "prev": None}

    start()
    while running:
        ready = [b for b, w in running.items() if w["prev"] is None or all(g in counted for g in range(w["prev"]))]
        if not ready:
            return order, handed, False                              # every running workgroup waits: the spin limit ends the launch
        b = rng.choice(ready)
        w = running[b]
        g = w["q"].pop(0)
        if g == NONE:
            del running[b]
            start()
            continue
        assert w["prev"] is None or g > w["prev"]                    # a workgroup's groups ascend
        counted.add(g)
        order.append(g)
        w["prev"] = g
        w["q"].append(draw())
    return order, handed, True


GRIDS = [(1, 1), (2, 2), (5, 2), (9, 4), (16, 8), (33, 8), (100, 8)]


@pytest.mark.parametrize("ngroups,nwg", GRIDS)
def test_on_tickets_every_launch_ends_whatever_is_resident(ngroups, nwg):
    for slots in range(1, nwg + 1):
        for seed in range(12):
            order, handed, ended = _launch(ngroups, nwg, slots, False, seed)
            assert ended and sorted(order) == list(range(ngroups))
            assert handed == list(range(ngroups))                    # handed out in order, each once


@pytest.mark.parametrize("ngroups,nwg", GRIDS)
def test_with_the_static_start_a_resident_grid_ends(ngroups, nwg):
    for seed in range(30):
        order, handed, ended = _launch(ngroups, nwg, nwg, True, seed)
        assert ended and sorted(order) == list(range(ngroups)) and sorted(handed) == list(range(ngroups))


def test_with_the_static_start_a_grid_that_is_not_resident_can_wait_for_ever():
    assert not _launch(33, 8, 7, True, 0)[2]                         # workgroup 7 never starts: group 7 is counted by nobody


@pytest.mark.parametrize("nwg,ngroups", [(1, 1), (256, 256), (256, 100_000), (256, 0xFFFFFFFE)])
def test_the_functions_at_their_borders(nwg, ngroups):
    L = emu.lib()
    assert L.emu_pair_static_group(nwg - 1, 0, nwg, ngroups) == (nwg - 1 if nwg - 1 < ngroups else NONE)
    assert L.emu_pair_static_group(nwg - 1, 1, nwg, ngroups) == (2 * nwg - 1 if 2 * nwg - 1 < ngroups else NONE)
    for static in (0, 1):
        first = 2 * nwg if static else 0
        assert L.emu_pair_ticket_group(0, nwg, ngroups, static) == (first if first < ngroups else NONE)
        if ngroups > first:
            assert L.emu_pair_ticket_group(ngroups - 1 - first, nwg, ngroups, static) == ngroups - 1
            assert L.emu_pair_ticket_group(ngroups - first, nwg, ngroups, static) == NONE
        assert L.emu_pair_ticket_group(NONE, nwg, ngroups, static) == NONE    # (also where first + ticket passes 2^32)

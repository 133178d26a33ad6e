"""The barrier protocol of the block-sparse attention kernel, as a model that runs on the CPU.

The load warp, the two MMA warps and the softmax warps of a CTA are generators that yield what they
wait for; copies and MMAs in flight land later. A schedule picks at random who goes next, and now
and then a copy lands as late as it can. A slot read before its rows have landed, a barrier that gets one
arrival too many and a wait that never ends are errors.
"""

from __future__ import annotations

import random
from pathlib import Path

import pytest

KERNEL = Path(__file__).parents[1] / "h3_flash_b200" / "csrc" / "sparse_attention.cu"


class Barrier:
    def __init__(self, count):
        self.count = self.pending = count
        self.phase = 0

    def arrive(self):
        self.pending -= 1
        assert self.pending >= 0, "one arrival too many"
        if self.pending == 0:
            self.pending, self.phase = self.count, self.phase + 1

    def done(self, parity):  # what a wait on a parity sees: the phase before counts as done
        return self.phase & 1 != parity


def _barriers(count, *shape):
    return [_barriers(count, *shape[1:]) for _ in range(shape[0])] if shape else Barrier(count)


def run(items, slots, shared, passes, seed, late):
    """``items``: units of both tiles. ``passes``: a tile without units passes its item's shared slots one
    by one; otherwise it steps over them and the other tile releases them for both."""

    rng = random.Random(seed)
    q_full, q_empty = _barriers(1, 2), _barriers(1, 2)
    s_bar, p_bar, pv_bar = _barriers(1, 2, 2), _barriers(4, 2, 2), _barriers(1, 2, 2)
    full, empty = _barriers(1, slots), _barriers(2 if shared else 1, slots)
    i_full, i_empty = _barriers(1, 2), _barriers(10, 2)
    info, content, tags = [None, None], [None] * slots, [-1] * slots
    copies, issued, pv_done = [], [[], []], [0, 0]

    def load():
        pos, phase = 0, [0, 0]
        for n, units in enumerate(items):
            yield lambda: i_empty[n & 1].done(((n >> 1) & 1) ^ 1)
            info[n & 1] = units
            i_full[n & 1].arrive()

            def push(tile, unit):
                nonlocal pos
                slot = pos % slots
                yield lambda: empty[slot].done(((pos // slots) & 1) ^ 1)
                content[slot], tags[slot] = None, pos

                def land(slot=slot, what=(n, tile, unit)):
                    content[slot] = what
                    full[slot].arrive()

                copies.append((rng.random() < late, land))
                pos += 1

            for t in range(2):
                if units[t] == 0:
                    continue
                yield lambda: q_empty[t].done(phase[t] ^ 1)
                phase[t] ^= 1
                copies.append((False, q_full[t].arrive))
                if t == 0 or not shared:
                    yield from push(t, -1)
            for u in range(max(units)):
                for t in range(2):
                    if u < units[t] and (t == 0 or not shared):
                        yield from push(t, u)

    def mma(t):
        base = n_s = n_pv = phase = 0
        reader = 0 if shared else t
        for n in range(len(items)):
            yield lambda: i_full[n & 1].done((n >> 1) & 1)
            both = info[n & 1]
            i_empty[n & 1].arrive()
            units, other = both[t], both[1 - t]
            lead = int(t == 1 and not shared and both[0] > 0)
            firsts = 1 if shared else (both[0] > 0) + (both[1] > 0)
            at = base + firsts + lead

            def slot_there(where):
                if not shared:
                    yield lambda: tags[where % slots] == where
                yield lambda: full[where % slots].done((where // slots) & 1)

            def issue_s():
                nonlocal n_s
                issued[t].append(s_bar[t][n_s & 1].arrive)
                n_s += 1

            def release(where):
                for _ in range(2 if shared and other == 0 and not passes else 1):
                    issued[t].append(empty[where % slots].arrive)

            if units > 0:
                yield lambda: q_full[t].done(phase)
                yield from slot_there(base + lead)
                phase ^= 1
                assert content[(base + lead) % slots] == (n, reader, -1), "slot read too early"
                for _ in range(min(2, units)):
                    issue_s()
                release(base + lead)
                if units <= 2:
                    issued[t].append(q_empty[t].arrive)
            for u in range(units):
                yield lambda: p_bar[t][n_pv & 1].done((n_pv >> 1) & 1)
                yield from slot_there(at)
                assert content[at % slots] == (n, reader, u), "slot read too early"

                def pv(buffer=n_pv & 1):
                    pv_done[t] += 1
                    pv_bar[t][buffer].arrive()

                issued[t].append(pv)
                if u + 2 < units:
                    issue_s()
                release(at)
                if u + 3 == units:
                    issued[t].append(q_empty[t].arrive)
                n_pv += 1
                at += 1 if shared else 1 + ((u < other) if t == 0 else (u + 1 < other))
            taken = 0 if both == (0, 0) else firsts + (max(both) if shared else sum(both))
            if shared and passes and units == 0:
                for i in range(base, base + taken):
                    yield from slot_there(i)
                    assert content[i % slots][0] == n, "slot passed too early"
                    empty[i % slots].arrive()
            base += taken

    def softmax(t, idle):
        n = 0
        for i in range(len(items)):
            yield lambda: i_full[i & 1].done((i >> 1) & 1)
            units = info[i & 1][t]
            i_empty[i & 1].arrive()
            for u in range(units):
                yield lambda: s_bar[t][n & 1].done((n >> 1) & 1)
                if not idle and u > 0 and rng.random() < 0.3:
                    yield lambda: pv_bar[t][(n - 1) & 1].done(((n - 1) >> 1) & 1)
                    assert pv_done[t] >= n, "O rescaled under an MMA"
                p_bar[t][n & 1].arrive()
                n += 1
            if units:
                yield lambda: pv_bar[t][(n - 1) & 1].done(((n - 1) >> 1) & 1)
                assert pv_done[t] == n, "O read under an MMA"

    roles = [load(), mma(0), mma(1)] + [softmax(t, w > 0 and seed % 2) for t in range(2) for w in range(4)]
    waits = {role: None for role in roles}
    while waits or copies or issued[0] or issued[1]:
        acts = [("role", r) for r, wait in waits.items() if wait is None or wait()]
        acts += [("mma", t) for t in range(2) if issued[t]]
        acts += [("copy", c) for c in copies if not c[0]]
        acts = acts or [("copy", c) for c in copies]
        assert acts, "a wait that never ends"
        kind, what = rng.choice(acts)
        if kind == "copy":
            copies.remove(what)
            what[1]()
        elif kind == "mma":
            issued[what].pop(0)()
        else:
            try:
                waits[what] = next(what)
            except StopIteration:
                del waits[what]


def _schedules(shared, count):
    rng = random.Random(1)
    for seed in range(count):
        items = []
        for _ in range(rng.randint(2, 8)):
            a = rng.choice([0, 1, 2, 3, rng.randint(0, 20), rng.randint(4, 12)])
            items.append((a, rng.choice([a, 0]) if shared else rng.choice([0, 1, 2, 3, a, rng.randint(0, 20)])))
        yield items, rng.choice([5, 10]), shared, seed, rng.choice([0.0, 0.05, 0.2])


@pytest.mark.parametrize("shared", [False, True])
def test_every_slot_is_read_after_it_landed(shared):
    for items, slots, _, seed, late in _schedules(shared, 800):
        run(items, slots, shared, True, seed, late)


def test_a_tile_must_not_step_over_shared_slots():
    """Parity alone does not name a slot to a tile that skipped an item: it reads rows that have not landed."""

    wrong = 0
    for items, slots, _, seed, late in _schedules(True, 800):
        try:
            run(items, slots, True, False, seed, late)
        except AssertionError:
            wrong += 1
    assert wrong > 0


def test_the_kernel_passes_shared_slots_one_by_one():
    source = KERNEL.read_text()
    body = source[source.index("auto release"):]
    assert body.index("SHARED && units == 0 && i < slots") < body.index("mbar_arrive(bar_empty(slot))") < body.index("if (units > 0)")
    assert "other == 0" not in body

"""How the roles of the portions' attention over a cache in 8 bits wait for one another (``e4m3_attention_tcgen05.cu``), walked through on the host.

A barrier counts phases, and a wait names the parity of one: it lets a role through when the phase before the one in progress has that
parity, be it the phase that was meant or the one two phases earlier.  So a role may only wait where nothing but these two answers is
possible: the phase meant is over, or the one before it is.  The model runs the roles in any order that the barriers allow, and looks whether the
softmax of a tile finds beside a stage what the converters left there for its block."""

import os
import random
import re

import pytest

import mini_llm_b200

SOURCE = os.path.join(os.path.dirname(mini_llm_b200.__file__), "csrc", "e4m3_attention_tcgen05.cu")


class Barriers(dict):
    """Completed phases of each barrier, and arrivals of the one in progress."""

    def __missing__(self, key):
        self[key] = [0, 0]
        return self[key]

    def arrive(self, key, needed=1):
        phases = self[key]
        phases[1] += 1
        if phases[1] == needed:
            phases[0], phases[1] = phases[0] + 1, 0

    def lets_through(self, key, parity):
        return (self[key][0] - 1) & 1 == parity


class Ring:
    def __init__(self, stages):
        self.stages, self.stage, self.parity = stages, 0, 0

    def next(self):
        self.stage += 1
        if self.stage == self.stages:
            self.stage, self.parity = 0, self.parity ^ 1


def converter(b, side, units, stages):
    ring, block = Ring(stages), 0
    for unit in units:
        for _ in range(max(unit)):
            yield ("k_empty", ring.stage), ring.parity ^ 1
            b.arrive(("k_full", ring.stage))
            yield ("v_empty", ring.stage), ring.parity ^ 1
            side[ring.stage] = block
            b.arrive(("v_full", ring.stage))
            ring.next()
            block += 1


def products(b, units, stages, apart):
    ring, seen, seen_units = Ring(stages), [0, 0], [0, 0]

    def after():
        other = Ring(stages)
        other.stage, other.parity = ring.stage, ring.parity
        other.next()
        return other

    for n in units:
        most = max(n)
        yield ("k_full", ring.stage), ring.parity
        for tile in (0, 1):
            if n[tile]:
                yield ("q_full", tile), seen_units[tile] & 1
                b.arrive(("s_ready", tile))
        b.arrive(("k_empty", ring.stage))
        for j in range(most):
            behind = after()
            yield ("v_full", ring.stage), ring.parity
            if j + 1 < most:
                yield ("k_full", behind.stage), behind.parity
            for tile in (0, 1):
                if j >= n[tile]:
                    continue
                parity = (seen[tile] + j) & 1
                if apart and j + 1 < n[tile]:
                    yield ("s_read", tile), parity
                    b.arrive(("s_ready", tile))
                if j == 0:
                    yield ("o_free", tile), (seen_units[tile] & 1) ^ 1
                yield ("p_ready", tile), parity
                b.arrive(("o_added", tile))
                if not apart and j + 1 < n[tile]:
                    b.arrive(("s_ready", tile))
            b.arrive(("v_empty", ring.stage))
            if j + 1 < most:
                b.arrive(("k_empty", behind.stage))
            ring.next()
        for tile in (0, 1):
            seen[tile] += n[tile]
            seen_units[tile] += n[tile] > 0


def softmax(b, side, units, stages, apart, tile, order):
    ring, seen, block = Ring(stages), 0, 0
    for n in units:
        if n[tile]:
            b.arrive(("q_full", tile))
        for j in range(n[tile]):
            for name in order:
                yield (name, ring.stage if name == "v_full" else tile), ring.parity if name == "v_full" else seen & 1
            assert side[ring.stage] == block + j, f"tile {tile}: block {block + j} met what is beside block {side[ring.stage]}"
            stage = ring.stage
            ring.next()
            if j > 0:
                yield ("o_added", tile), (seen - 1) & 1
            if apart:
                b.arrive(("s_read", tile))
            yield None                                                      # (its weights; what is beside the stage is read until then)
            assert side[stage] == block + j
            b.arrive(("p_ready", tile))
            seen += 1
        if n[tile]:
            yield ("o_added", tile), (seen - 1) & 1
            b.arrive(("o_free", tile))
        for _ in range(max(n) - n[tile]):
            ring.next()
        block += max(n)


def walk(units, stages, apart, order, rng):
    b, side = Barriers(), [None] * stages
    roles = [converter(b, side, units, stages), products(b, units, stages, apart)] + [softmax(b, side, units, stages, apart, t, order) for t in (0, 1)]
    # (one role is slower than the others in most runs)
    weights = [rng.choice((1.0, 1.0, 0.02)) for _ in roles]
    waits = [next(role, "done") for role in roles]
    while any(w != "done" for w in waits):
        able = [i for i, w in enumerate(waits) if w is None or (w != "done" and b.lets_through(*w))]
        assert able, f"all roles wait: {waits}"
        i = rng.choices(able, [weights[i] for i in able])[0]
        waits[i] = next(roles[i], "done")


def all_walks(order, runs):
    rng = random.Random(5)
    for run in range(runs):
        # units of one tile, of two, and of two of which one walks fewer blocks
        units = [rng.choice([(n, 0), (n, 0), (n, n), (n, n + 1), (n, n), (0, n)]) for n in (rng.randint(1, 5) for _ in range(rng.randint(2, 8)))]
        stages, apart = rng.choice([(4, True), (2, False)])
        walk(units, stages, apart, order, rng)


def test_softmax_finds_what_stands_beside_its_block():
    """In the order in which the kernel waits."""
    with open(SOURCE) as f:
        order = re.findall(r"ok = wait_or_fail\(sh, &sh\.(\w+)\[\w+\], [^)]*\) && wait_or_fail\(sh, &sh\.(\w+)\[\w+\],", f.read())
    assert len(order) == 1 and set(order[0]) == {"v_full", "s_ready"}
    all_walks(order[0], 3000)


def test_the_model_sees_a_phase_taken_for_another():
    """The other order lets a tile that has skipped a short unit's blocks take an older phase of its next block's barrier for the one it means."""
    with pytest.raises(AssertionError, match="met what is beside"):
        all_walks(("v_full", "s_ready"), 3000)

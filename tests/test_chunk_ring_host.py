"""CPU: the order that the chunk attention's ring of key tiles keeps.

A model of the roles that touch the ring in a piece whose key tiles two groups share (each takes every
second one): loads are issued in order as stages fall free and land in any order, the value
conversion takes the tiles in order, a group waits for its tiles by parity, as the kernel does. Whatever
the interleaving, a wait that passes has to mean that this tile's keys are there, and every role
has to come to its end. The number of stages and of barriers is read from the kernel's source."""

import random
import re
from pathlib import Path

import pytest

SRC = Path(__file__).resolve().parent.parent / "superl8_serve_b200" / "csrc" / "chunk_attn.cu"


def _ring():
    src = SRC.read_text()
    stages = int(re.search(r"constexpr int kStages = (\d+);", src).group(1))
    full = re.search(r"constexpr int kFull = (\d*) ?\*? ?kStages;", src)
    return stages, stages * int(full.group(1) or 1) if full else stages


class Wrong(Exception):
    pass


def _run(tiles, stages, barriers, rng):
    """One interleaving; raises Wrong if a wait passed for keys that had not landed."""
    phase = [0] * barriers  # completed phases of the barriers of landed keys
    landed, vlanded, issued = set(), set(), []
    scored, soft, conv, product = set(), set(), set(), set()

    def empty(t):  # a stage's reads are over: scores, softmax (scales) and conversion
        return t < 0 or (t in scored and t in soft and t in conv)

    def loader():
        for t in range(tiles):
            yield lambda t=t: empty(t - stages)
            issued.append(t)

    def land(seen, count):
        for _ in range(tiles):
            yield lambda: any(t not in seen for t in issued)
            t = rng.choice([t for t in issued if t not in seen])
            seen.add(t)
            if count:
                phase[t % barriers] += 1

    def convert():
        for t in range(tiles):
            yield lambda t=t: t in vlanded and (t < 2 or t - 2 in product)
            conv.add(t)

    def softmax(g):
        for t in range(g, tiles, 2):
            yield lambda t=t: t in scored
            soft.add(t)

    def group(g):
        def keys(t):  # the parity wait
            return phase[t % barriers] & 1 != (t // barriers) & 1

        def scores(t):
            if t not in landed:
                raise Wrong(t)
            scored.add(t)

        own = range(g, tiles, 2)
        if own:
            yield lambda: keys(g)
            scores(g)
        for t in own:
            yield lambda t=t: t in conv
            if t + 2 < tiles:
                yield lambda t=t: keys(t + 2)
            yield lambda t=t: t in soft
            product.add(t)
            if t + 2 < tiles:
                scores(t + 2)

    roles = [loader(), land(landed, True), land(vlanded, False), convert(), softmax(0), softmax(1),
             group(0), group(1)]
    speed = [rng.choice((0.02, 0.3, 1.0)) for _ in roles]  # some roles far behind others
    ready = {}
    for i, r in enumerate(roles):
        ready[i] = next(r, None)
    while any(c is not None for c in ready.values()):
        can = [i for i, c in ready.items() if c is not None and c()]
        if not can:
            raise Wrong("no role can go on")
        i = rng.choices(can, [speed[i] for i in can])[0]
        ready[i] = next(roles[i], None)


@pytest.mark.parametrize("tiles", [1, 2, 3, 4, 7, 16])
def test_keys_are_there_when_a_wait_passes(tiles):
    stages, barriers = _ring()
    assert barriers % stages == 0
    for seed in range(1500):
        _run(tiles, stages, barriers, random.Random(seed))


def test_one_barrier_per_stage_would_not_do():
    """The model is able to show the fault: a group then passes the wait for a tile whose stage
    the other group's keys have not reached yet."""
    with pytest.raises(Wrong):
        for seed in range(1500):
            _run(16, 3, 3, random.Random(seed))

"""How the products of the feed-forward ops share their work, on the host: every K block of every tile runs once, whoever finishes a
tile waits only for units that leave their share first, and no unit leaves more than one."""
import ctypes as C
import random

import pytest

SEGMENTS = 4096


def _walk(lib, tiles, kblocks, units):
    used = C.c_int()
    assert lib.fp4ar_layer_plan(tiles, kblocks, units, 0, C.byref(used), None, 0) == 0
    buf = (C.c_int * (5 * SEGMENTS))()
    out = []
    for u in range(used.value):
        n = lib.fp4ar_layer_plan(tiles, kblocks, units, u, C.byref(used), buf, SEGMENTS)
        assert 0 <= n <= SEGMENTS
        out.append([tuple(buf[5 * i:5 * i + 5]) for i in range(n)])
    return out


def _cases():
    rng = random.Random(5)
    listed = [(1, 1, 74), (1, 96, 74), (16, 96, 74), (34, 32, 74), (55, 96, 74), (73, 200, 74), (74, 10, 74), (75, 1, 74), (75, 96, 74), (148, 3, 74),
              (1024, 96, 74), (3, 1000, 2), (5, 7, 1)]
    return listed + [(rng.randint(1, 400), rng.randint(1, 260), rng.choice([74, 66, 60, 1, 2, 7])) for _ in range(150)]


@pytest.mark.parametrize("tiles,kblocks,units", _cases())
def test_every_block_runs_once(cuda_lib, tiles, kblocks, units):
    plan = _walk(cuda_lib, tiles, kblocks, units)
    assert len(plan) <= units
    runs = {}
    for u, segs in enumerate(plan):
        kinds = [s[3] for s in segs]
        assert kinds.count(1) <= 1 and 1 not in kinds[1:]                # one partial, and it comes first
        for tile, lo, count, kind, others in segs:
            assert 0 <= tile < tiles and count >= 1 and 0 <= lo and lo + count <= kblocks
            assert (kind == 0) == (count == kblocks)
            runs.setdefault(tile, []).append((u, lo, count, kind, others))
    assert len(runs) == tiles
    for parts in runs.values():
        blocks = sorted(b for _, lo, n, _, _ in parts for b in range(lo, lo + n))
        assert blocks == list(range(kblocks))
        if len(parts) > 1:
            first = [p for p in parts if p[3] == 2]
            assert len(first) == 1
            u, lo, n, _, others = first[0]
            assert lo + n == kblocks                                     # the last K blocks: what follows the K loop belongs to it
            assert sorted(p[0] for p in parts if p[3] == 1) == list(range(u + 1, u + 1 + others))
    load = [sum(s[2] for s in segs) for segs in plan]
    if tiles >= units:
        assert max(load) - min(load) <= kblocks

"""How the attention over a paged cache deals out its tiles, and the hand-overs of a warp's ring of steps, walked on the CPU: every tile once,
every piece of a cut unit where the launch that adds pieces up looks for it, every wait with a copy on its way, no slot filled that is
still to be read."""
import os
import random
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lact_b200", "csrc")


def _constant(name):
    for f in ("paged_attention.cuh", "lact_b200.cu"):
        m = re.search(r"constexpr int %s = (\d+);" % name, open(os.path.join(CSRC, f)).read())
        if m:
            return int(m.group(1))
    raise AssertionError(name)


WARPS, LEAST, WHOLE, CLUSTERED, STAGES, LONG, MOST = (_constant("kPaged" + n) for n in
                                                      ("Warps", "Least", "Whole", "Clustered", "Stages", "Long", "JoinMost"))
SMS = 148


def _span(length, window, room, step):
    length = max(length, 0)
    last = min(length, room)
    first = min(max(length - window, 0) if window else 0, last)
    base = first // step * step
    return first, last, base, max(-(-(last - base) // (step * WARPS)), 1)


def _plan(c):
    """As paged_step_plan: (runs, CTAs of a cluster, slots, slots of long runs, query blocks)."""
    step = {256: 16, 128: 32, 64: 64}[c["row_bytes"]]
    nq = 2 if c["share"] > 8 else 1
    blocks = -(-c["share"] // (8 * nq))
    units = len(c["lengths"]) * c["heads"] * blocks
    room = c["cols"] * c["page"]
    tokens = min(c["window"] + step - 1, room) if 0 < c["window"] < room else room
    tiles = -(-tokens // (step * WARPS))
    per_sm = 3 if nq == 1 else 2
    ctas = SMS * per_sm
    cluster, runs = 1, 0
    while cluster < 8 and cluster < tiles and 2 * cluster * units <= ctas:
        cluster *= 2
    if tiles > (CLUSTERED * cluster if cluster > 1 else WHOLE):
        cluster, runs = 1, min(ctas, -(-units * tiles // LEAST), MOST)
    e4 = c["row_bytes"] == c["d"]
    stage = 2 * step * (c["row_bytes"] + e4)
    sums = min(c["share"], 8 * nq) * (c["d"] + 4) * 4
    at_end = (WARPS + (cluster > 1)) * sums
    stages = min(STAGES, (227 * 1024 // per_sm - 3 * 1024 - at_end) // (WARPS * stage))
    assert stages >= 1 and WARPS * stages * stage + at_end + 1024 <= 227 * 1024 // per_sm - 2048
    return runs, cluster, stages, min(stages, max(1, 8192 // stage)), blocks, step


def _case(rng):
    d, bits = rng.choice((64, 128)), rng.choice((8, 16))
    top = int(2 ** rng.uniform(0, 14))
    n = rng.choice((1, 2, 3, 7, 40, 130))
    page = rng.choice((16, 32, 64, 256))
    lengths = [rng.choice((0, -4, 1, top, rng.randint(1, top), rng.randint(1, top))) for _ in range(n)]
    return dict(d=d, row_bytes=d * bits // 8, lengths=lengths, heads=rng.choice((1, 2, 5, 12)), share=rng.choice((1, 4, 8, 9, 20)), page=page,
                cols=max(1, -(-max(lengths + [1]) // page) - rng.choice((0, 0, 0, 1))), window=rng.choice((0, 0, 1, 30, 500, 4000)),
                bad=rng.random() < 0.3)


def _runs(c):
    """Every CTA's tiles, in order: lists of (sequence, unit, first tile, end); and the cuts it writes down."""
    runs, cluster, _, _, blocks, step = _plan(c)
    spans = [_span(n, c["window"], c["cols"] * c["page"], step) for n in c["lengths"]]
    units = c["heads"] * blocks
    out = []
    if runs == 0:
        for s, (_, _, _, tiles) in enumerate(spans):
            each = -(-tiles // cluster)
            for u in range(units):
                out += [([(s, u, min(r * each, tiles), min(r * each, tiles) + min(each, tiles - min(r * each, tiles)))], None) for r in range(cluster)]
        return out, spans, units
    total = sum(t for *_, t in spans) * units
    per = max(-(-total // runs), LEAST)
    order = [(s, u) for s in range(len(spans)) for u in range(units)]
    starts, at = {}, 0
    for s, u in order:
        starts[s, u] = at
        at += spans[s][3]
    begins = sorted((b, k) for k, b in starts.items())
    k = 0
    for cta in range(runs):
        run0 = cta * per
        if run0 >= total:
            out.append(([], 0))
            continue
        left = min(per, total - run0)
        while k + 1 < len(begins) and begins[k + 1][0] <= run0:
            k += 1
        (s, u), t = begins[k][1], run0 - begins[k][0]
        mine, cut, done = [], 0, 0
        while left > 0:
            t1 = min(spans[s][3], t + left)
            mine.append((s, u, t, t1))
            if t == 0 and t1 < spans[s][3]:
                cut = (run0 + done + spans[s][3] - 1) // per - cta + 1
            done += t1 - t
            left -= t1 - t
            t, u = 0, u + 1
            if u == units:
                s, u = s + 1, 0
        out.append((mine, cut))
    return out, spans, units


@pytest.mark.parametrize("seed", range(60))
def test_every_tile_once_and_every_piece_found(seed):
    c = _case(random.Random(seed))
    ctas, spans, units = _runs(c)
    assert len(ctas) <= 1 << 20
    seen, pieces = {}, {}
    for cta, (mine, _) in enumerate(ctas):
        for s, u, t0, t1 in mine:
            for t in range(t0, t1):
                assert (s, u, t) not in seen
                seen[s, u, t] = cta
            if ctas[cta][1] is not None and not (t0 == 0 and t1 == spans[s][3]):
                slot = (cta, 1 if t0 == 0 else 0)
                assert slot not in pieces               # (a run leaves at most one of each)
                pieces[slot] = (s, u)
    assert len(seen) == units * sum(t for *_, t in spans)
    found = set()
    for cta, (mine, cut) in enumerate(ctas):
        if not cut:
            continue
        unit = pieces[cta, 1]
        slots = [(cta + i, 1 if i == 0 else 0) for i in range(cut)]
        assert all(pieces.get(x) == unit for x in slots) and 2 <= cut <= MOST and not found & set(slots)
        found |= set(slots)
    assert found == set(pieces)
    # positions and pages of every step lie within the window and the table
    step = _plan(c)[5]
    for first, last, base, tiles in spans:
        covered = set()
        for t in range(tiles):
            for w in range(WARPS):
                p = base + (t * WARPS + w) * step
                if p < last:
                    assert p // c["page"] < c["cols"] and p % c["page"] % 16 == 0 and (c["page"] < step or p % c["page"] + step <= c["page"])
                    covered |= set(range(p, min(p + step, last)))
        assert set(range(first, last)) <= covered


@pytest.mark.parametrize("seed", range(60))
def test_the_ring_of_a_warp(seed):
    """One warp of a CTA: `issue` and the use of steps as in the kernel, with pages that are not there; copies arrive whenever they like."""
    rng = random.Random(1000 + seed)
    c = _case(rng)
    ctas, spans, units = _runs(c)
    _, _, stages, long_stages, _, step = _plan(c)
    for mine, _ in rng.sample(ctas, min(6, len(ctas))):
        tiles = [(s, u, t) for s, u, t0, t1 in mine for t in range(t0, t1)]
        warp, n = rng.randrange(WARPS), len(tiles)
        ring = long_stages if n > LONG else stages
        real = [spans[s][2] + (t * WARPS + warp) * step < spans[s][1] and not (c["bad"] and rng.random() < 0.2) for s, u, t in tiles]
        slots, completed, phase = [None] * ring, [0] * ring, [0] * ring    # what a slot holds; phases its barrier has completed; next wait's parity
        made = used = 0

        def issue():
            nonlocal made
            if made == n:
                return
            slot = made % ring
            assert slots[slot] is None                                     # read and done with
            slots[slot] = (made, real[made])
            made += 1
        for _ in range(ring):
            issue()
        while used < n:
            slot = used % ring
            held, there = slots[slot]
            assert held == used
            if there:
                completed[slot] += 1                                       # (its copies arrive: one phase for one filling)
                assert (completed[slot] - 1) % 2 == phase[slot]            # the wait is for this phase and not for one that is over
                phase[slot] ^= 1
            slots[slot] = None
            used += 1
            issue()
        assert made == n and all(x is None for x in slots)

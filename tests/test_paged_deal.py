"""The attention over a paged cache, walked on the CPU: how its tiles are dealt out (with the source's own functions for the plan and the
spans, compiled here), and every step of a warp's ring with the state that the kernel keeps of it.  What the walk restates of the kernel is
compared with the source's text, so that a changed formula is seen here."""
import ctypes as C
import os
import random
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "lact_b200", "csrc")
KERNEL = open(os.path.join(CSRC, "paged_attention.cuh")).read()
HOST = open(os.path.join(CSRC, "lact_b200.cu")).read()
SMS = 148


def _cut(source, begin, end="\n}\n"):
    """The source from `begin` to the first `end` behind it."""
    at = source.index(begin)
    return source[at:source.index(end, at) + len(end)]


@pytest.fixture(scope="module")
def own(tmp_path_factory):
    """paged_step_plan and paged_span of the source as a library."""
    constants = "\n".join(re.findall(r"^(?:__host__ __device__ )?constexpr int kPaged\w+(?: = |\().*$", KERNEL + HOST, flags=re.M))
    code = f'''
#include <algorithm>
#include <atomic>
#include "{ROOT}/include/lact_b200.h"
#define __device__
#define __host__
#define __forceinline__ inline
using std::max; using std::min;
static int sm_count() {{ return {SMS}; }}
static int64_t ceil_div(int64_t a, int64_t b) {{ return (a + b - 1) / b; }}
struct PagedCut {{ int64_t o; int32_t rows, count; }};
struct PagedStepArgs {{ struct {{ int32_t cols, shift; const int32_t* lengths; }} c; int32_t window; }};
{constants}
{_cut(HOST, "struct PagedStepPlan {", chr(10) + "};" + chr(10))}
{_cut(HOST, "int paged_step_plan(")}
{_cut(KERNEL, "struct PagedSpan {", chr(10) + "};" + chr(10))}
{_cut(KERNEL, "template <int STEP, int TILE>")}
extern "C" int plan(const lact_paged_cache* c, int64_t heads, int64_t window, int64_t* out) {{
  PagedStepPlan p;
  const int rc = paged_step_plan(c, heads, window, &p);
  const int64_t x[] = {{p.nq, p.blocks, p.runs, p.cluster, p.stages, p.long_stages, (int64_t)p.bytes, (int64_t)p.smem}};
  for (int i = 0; i < 8; ++i) out[i] = x[i];
  return rc;
}}
extern "C" void span(int step, int cols, int shift, int length, int window, int* out) {{
  PagedStepArgs a;
  a.c.cols = cols; a.c.shift = shift; a.c.lengths = &length; a.window = window;
  const PagedSpan s = step == 16 ? paged_span<16, 16 * kPagedWarps>(a, 0) : step == 32 ? paged_span<32, 32 * kPagedWarps>(a, 0) : paged_span<64, 64 * kPagedWarps>(a, 0);
  out[0] = s.first; out[1] = s.last; out[2] = s.base; out[3] = s.tiles; out[4] = s.over;
}}
extern "C" int constant(int i) {{
  const int x[] = {{kPagedWarps, kPagedLeast, kPagedLong, kPagedStages, kPagedJoinMost, kPagedSub(64), kPagedSub(128), kPagedSub(256)}};
  return x[i];
}}
'''
    at = tmp_path_factory.mktemp("deal")
    (at / "own.cpp").write_text(code)
    subprocess.run(["g++", "-O1", "-std=c++17", "-w", "-shared", "-fPIC", "-o", str(at / "own.so"), str(at / "own.cpp")], check=True)
    return _Own(C.CDLL(str(at / "own.so")))


class _Cache(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("k", "v", "k_exponent", "v_exponent")] + [
        (n, C.c_int64) for n in ("pages", "kv_heads", "page_size", "head_dim", "k_page_stride", "v_page_stride", "ke_page_stride", "ve_page_stride")] + [
        ("page_table", C.c_void_p), ("table_cols", C.c_int64), ("table_stride", C.c_int64), ("lengths", C.c_void_p), ("sequences", C.c_int64)]


class _Own:
    def __init__(self, lib):
        self.lib = lib
        self.warps, self.least, self.long, self.slots, self.join_most, *self.sub = (lib.constant(i) for i in range(8))

    def step(self, c):
        return 16 * dict(zip((64, 128, 256), self.sub))[c["row_bytes"]]

    def plan(self, c):
        k = _Cache(k=4096, v=4096, pages=100, kv_heads=c["heads"], page_size=c["page"], head_dim=c["d"], table_cols=c["cols"], sequences=len(c["lengths"]))
        if c["row_bytes"] == c["d"]:
            k.k_exponent = k.v_exponent = 4096
        out = (C.c_int64 * 8)()
        assert self.lib.plan(C.byref(k), C.c_int64(c["heads"] * c["share"]), C.c_int64(c["window"]), out) == 0
        return dict(zip(("nq", "blocks", "runs", "cluster", "stages", "long_stages", "bytes", "smem"), out))

    def span(self, c, length):
        out = (C.c_int * 5)()
        self.lib.span(self.step(c), c["cols"], c["page"].bit_length() - 1, length, c["window"], out)
        return dict(zip(("first", "last", "base", "tiles", "over"), out))


# What the walk restates of the kernel, line by line
RESTATED = [
    # the deal
    "const int tiles = paged_span<STEP, TILE>(a, make.seq).tiles, each = (tiles + a.cluster - 1) / a.cluster;",
    "make.t = min(rank * each, tiles);", "make.left = min(each, tiles - make.t);",
    "all *= units;", "per = max((all + a.runs - 1) / a.runs, static_cast<int64_t>(a.least));", "run0 = blockIdx.x * per;", "if (run0 >= all) return;",
    "make.left = static_cast<int>(min(per, all - run0));", "plan[1] = static_cast<int>((run0 - at) / n);", "plan[2] = static_cast<int>((run0 - at) % n);",
    "w.t1 = min(span.tiles, w.t + w.left);", "w.left -= w.t1 - from; w.t = 0; if (++w.unit == units) { w.unit = 0; ++w.seq; }",
    "const bool whole = use.t1 == use.tiles && t0 == 0", "if (a.cluster == 1 && whole) {", "begin = run0 + done;",
    "(static_cast<int64_t>(blockIdx.x) * 2 + (t0 == 0 ? 1 : 0)) * sum_rows * ROW;",
    "if (threadIdx.x == 0 && t0 == 0) a.cuts[blockIdx.x] = {at, rows, static_cast<int32_t>((begin + tiles - 1) / per - blockIdx.x) + 1};",
    "auto piece = [&](int i) { return base + static_cast<int64_t>(2 * i + (i == 0 ? 1 : 0)) * sum_rows * ROW; };",
    # positions and pages
    "return w.base + (w.t * W + warp) * STEP;",
    "const int parts = max(STEP >> a.c.shift, 1), part_rows = min(STEP, 1 << a.c.shift), part_bytes = (STAGE + EB) / parts;",
    "const int p = position(w), at = p >> a.c.shift; pg[0] = p < w.last ? w.table[at] : -1;",
    "for (int i = 1; i < SUB; ++i) pg[i] = i < parts && p + i * part_rows < w.last ? w.table[at + i] : -1;",
    # the ring
    "const int stages = make.left > kPagedLong ? a.long_stages : a.stages;", "uint32_t has = 0, gone = 0, phase = 0;",
    "auto issue = [&]() { if (make.left <= 0) return; const int p = position(make), row = (make.head << a.c.shift) + (p & ((1 << a.c.shift) - 1));",
    "const bool real = p + at < make.last; if (real && static_cast<uint32_t>(pg) >= static_cast<uint32_t>(a.c.pages)) {",
    "const bool real = there(page[0], 0); has = real ? has | 1u << make_slot : has & ~(1u << make_slot); if (real) { mbar_expect_tx_if(leader, bar, STAGE + EB); "
    "copy(page[0], 0, STEP, leader); }",
    "if (i < parts && there(page[i], i * part_rows)) on |= 1u << i; has = on != 0 ? has | 1u << make_slot : has & ~(1u << make_slot);",
    "if ((on >> (u * 16 >> a.c.shift) & 1) == 0) lost |= 1u << u; gone = (gone & ~(((1u << SUB) - 1) << make_slot * SUB)) | lost << make_slot * SUB;",
    "mbar_expect_tx_if(leader, bar, __popc(on) * part_bytes);", "if (on >> i & 1) copy(page[i], i * part_rows, part_rows, leader);",
    "if (++make_slot == stages) make_slot = 0; if (++make.t == make.t1) { leave(make, make_from); make_from = 0; if (make.left > 0) enter(make); } "
    "if (make.left > 0) pages_of(make, page);",
    "for (int i = 0; i < stages; ++i) issue();",
    "const int slot = use_slot, p = position(use); if (++use_slot == stages) use_slot = 0; if ((has >> slot & 1) && !failed) { "
    "if (!mbar_wait_warp(&full[warp * kPagedStages + slot], phase >> slot & 1, &gave_up)) {",
    "make.left = 0; for (int s = 0; s < stages; ++s) if (has >> s & 1) mbar_wait(&full[warp * kPagedStages + s], phase >> s & 1); } phase ^= 1u << slot; }",
    "if (!(has >> slot & 1) || failed) { issue(); continue; }",
    "const uint32_t lost = gone >> slot * SUB & ((1u << SUB) - 1); if (p < use.first || p + STEP > use.last || lost != 0) {",
]


def _plain(text):
    return re.sub(r"\s+", " ", re.sub(r"//[^\n]*|#pragma unroll", "", text))


def test_the_walk_restates_the_source():
    source = _plain(KERNEL)
    for line in RESTATED:
        assert _plain(line) in source, line


def _case(rng):
    d, bits = rng.choice((64, 128)), rng.choice((8, 16))
    top = int(2 ** rng.uniform(0, 14))
    n = rng.choice((1, 2, 3, 7, 40, 130))
    page = rng.choice((16, 16, 32, 64, 256))
    lengths = [rng.choice((0, -4, 1, top, rng.randint(1, top), rng.randint(1, top))) for _ in range(n)]
    return dict(d=d, row_bytes=d * bits // 8, lengths=lengths, heads=rng.choice((1, 2, 5, 12)), share=rng.choice((1, 4, 8, 9, 20)), page=page,
                cols=max(1, -(-max(lengths + [1]) // page) - rng.choice((0, 0, 0, 1)) + rng.choice((0, 0, 3, 500))), window=rng.choice((0, 0, 1, 17, 30, 500, 4000)),
                bad=rng.choice((0.0, 0.0, 0.1, 0.6)))


def _deal(own, c):
    """Every CTA's units in order, (sequence, unit, first tile, end), and the count that it writes down of a cut unit."""
    p = own.plan(c)
    spans = [own.span(c, n) for n in c["lengths"]]
    units = c["heads"] * p["blocks"]
    out = []
    if p["runs"] == 0:
        for s, x in enumerate(spans):
            each = -(-x["tiles"] // p["cluster"])
            for u in range(units):
                for rank in range(p["cluster"]):
                    t = min(rank * each, x["tiles"])
                    out.append(([(s, u, t, t + min(each, x["tiles"] - t))], None))
        return p, spans, units, out
    total = sum(x["tiles"] for x in spans) * units
    per = max(-(-total // p["runs"]), own.least)
    for cta in range(p["runs"]):
        run0, mine, cut, done = cta * per, [], 0, 0
        if run0 < total:
            left, at = min(per, total - run0), 0
            for s, x in enumerate(spans):
                if run0 < at + x["tiles"] * units:
                    u, t = divmod(run0 - at, x["tiles"])
                    break
                at += x["tiles"] * units
            while left > 0:
                tiles = spans[s]["tiles"]
                t1 = min(tiles, t + left)
                mine.append((s, u, t, t1))
                if t == 0 and t1 < tiles:
                    cut = (run0 + done + tiles - 1) // per - cta + 1
                done, left, t, u = done + t1 - t, left - (t1 - t), 0, u + 1
                if u == units:
                    s, u = s + 1, 0
        out.append((mine, cut))
    return p, spans, units, out


@pytest.mark.parametrize("seed", range(80))
def test_every_tile_once_and_every_piece_found(own, seed):
    c = _case(random.Random(seed))
    p, spans, units, ctas = _deal(own, c)
    seen, pieces = set(), {}
    for cta, (mine, _) in enumerate(ctas):
        for s, u, t0, t1 in mine:
            for t in range(t0, t1):
                assert (s, u, t) not in seen
                seen.add((s, u, t))
            if p["runs"] and not (t0 == 0 and t1 == spans[s]["tiles"]):
                assert (cta, t0 == 0) not in pieces                     # (a run leaves at most one of each)
                pieces[cta, t0 == 0] = (s, u)
    assert len(seen) == units * sum(x["tiles"] for x in spans)
    found = set()
    for cta, (_, cut) in enumerate(ctas):
        if cut:
            slots = [(cta + i, i == 0) for i in range(cut)]
            assert all(pieces.get(x) == pieces[cta, True] for x in slots) and 2 <= cut <= own.join_most and not found & set(slots)
            found |= set(slots)
    assert found == set(pieces)
    # what is on a SM at a time fits; pieces have their room
    rows, per_sm = min(c["share"], 8 * p["nq"]), 3 if p["nq"] == 1 else 2
    assert 1 <= p["long_stages"] <= p["stages"] <= own.slots and p["smem"] <= 227 * 1024 // per_sm - 2048
    assert p["bytes"] >= p["runs"] * (16 + 2 * rows * (c["d"] + 4) * 4)


@pytest.mark.parametrize("seed", range(80))
def test_steps_hold_the_window_and_no_page_in_front_of_it(own, seed):
    c = _case(random.Random(500 + seed))
    step = own.step(c)
    part = min(step, c["page"])
    for n in c["lengths"]:
        x = own.span(c, n)
        room = c["cols"] * c["page"]
        assert x["last"] == min(max(n, 0), room) and x["over"] == (n > room) and x["tiles"] >= 1
        assert x["first"] == min(max(n - c["window"], 0) if c["window"] else 0, x["last"])
        held = set()
        for t in range(x["tiles"]):
            for w in range(own.warps):
                p = x["base"] + (t * own.warps + w) * step
                for at in range(p, min(p + step, x["last"]), part):
                    assert at // c["page"] < c["cols"] and at % part == 0 and at // c["page"] == (at + part - 1) // c["page"]   # (one page, within the table)
                    assert at + part > x["first"]                       # a part in front of the window is in no step
                    held |= set(range(at, min(at + part, x["last"])))
        assert set(range(x["first"], x["last"])) <= held


class _Ring:
    """One warp: what the kernel keeps (has, gone, phase, the two slots), and beside it what its slots and barriers really hold."""

    def __init__(self, own, c, tiles, spans, stages, long_stages, warp, rng, stuck=None, mistake=None):
        self.own, self.c, self.spans, self.warp, self.rng, self.stuck, self.mistake = own, c, spans, warp, rng, stuck, mistake
        self.step, self.page = own.step(c), c["page"]
        self.sub = self.step // 16
        self.parts, self.part_rows = max(self.step // self.page, 1), min(self.step, self.page)
        self.stage = 2 * self.step * (c["row_bytes"] + (c["row_bytes"] == c["d"]))
        self.tiles = tiles
        self.stages = long_stages if len(tiles) > own.long else stages
        self.has = self.gone = self.phase = 0
        self.make_slot = self.use_slot = self.made = 0
        self.left = len(tiles)
        self.held = [None] * self.stages          # what a slot's memory is of: (tile, parts that were copied), and whether it is still to be read
        self.expected, self.arrived, self.completed = [0] * self.stages, [0] * self.stages, [0] * self.stages
        self.flying = []                          # (slot, bytes) on their way
        self.tables = {s: [rng.random() >= c["bad"] for _ in range(c["cols"])] for s in {s for s, _, _ in tiles}}

    def position(self, i):
        s, _, t = self.tiles[i]
        return self.spans[s]["base"] + (t * self.own.warps + self.warp) * self.step

    def real(self, i):
        """Parts of a step that are there."""
        s, p, last = self.tiles[i][0], self.position(i), self.spans[self.tiles[i][0]]["last"]
        return [p + j * self.part_rows < last and self.tables[s][(p + j * self.part_rows) // self.page] for j in range(self.parts)]

    def land(self, some=False):
        """Copies arrive in any order; a barrier's phase is over when all that it expects is there."""
        self.rng.shuffle(self.flying)
        for _ in range(self.rng.randint(1, len(self.flying)) if some else len(self.flying)):
            slot, n = self.flying.pop()
            if (slot, self.completed[slot]) == self.stuck:
                self.kept = (slot, n)
                continue
            self.arrived[slot] += n
            assert self.arrived[slot] <= self.expected[slot]
            if self.arrived[slot] == self.expected[slot]:
                self.completed[slot] += 1
                self.arrived[slot] = self.expected[slot] = 0

    def issue(self):
        if self.left <= 0:
            return
        i, slot = self.made, self.make_slot
        assert self.held[slot] is None and self.expected[slot] == 0 and not any(s == slot for s, _ in self.flying)   # read and done with, nothing on its way
        on = self.real(i)
        there = any(on)
        self.has = self.has | 1 << slot if there or self.mistake == "has" else self.has & ~(1 << slot)
        if self.parts > 1:
            lost = sum(1 << u for u in range(self.sub) if not on[u * 16 // self.page])
            if self.mistake != "gone":
                self.gone = self.gone & ~(((1 << self.sub) - 1) << slot * self.sub) | lost << slot * self.sub
        if there:
            n = self.stage // self.parts
            self.expected[slot] = sum(on) * n if self.mistake != "bytes" else self.stage
            self.flying += [(slot, n) for x in on if x]
        self.held[slot] = (i, on)
        self.make_slot = 0 if self.make_slot + 1 == self.stages else self.make_slot + 1
        self.made += 1
        self.left -= 1

    def wait(self, slot):
        """Until the barrier has completed the phase of this parity; False: it never does."""
        if self.mistake != "phase":
            assert self.expected[slot] > 0 or self.completed[slot] % 2 != self.phase >> slot & 1
        while self.completed[slot] % 2 == self.phase >> slot & 1:
            if not self.flying:
                return False
            self.land(some=True)
        return True

    def run(self):
        failed = False
        for _ in range(self.stages):
            self.issue()
        for i in range(len(self.tiles)):
            slot, p = self.use_slot, self.position(i)
            self.use_slot = 0 if self.use_slot + 1 == self.stages else self.use_slot + 1
            if self.has >> slot & 1 and not failed:
                if not self.wait(slot):
                    failed = True
                    self.left = 0
                    for s in range(self.stages):
                        if self.has >> s & 1:
                            while self.completed[s] % 2 == self.phase >> s & 1 and self.flying:   # (as long again, and then on)
                                self.land(some=True)
                self.phase ^= 1 << slot
                if self.mistake == "phase":
                    self.phase ^= 1 << slot
            if not self.has >> slot & 1 or failed:
                if not failed:
                    assert not any(self.held[slot][1])                  # a step that is passed over had nothing to be read
                    self.held[slot] = None
                self.issue()
                continue
            # the slot's contents are those of this step, all there; what of it counts is what was copied and lies in the window
            tile, on = self.held[slot]
            assert tile == i and self.completed[slot] % 2 == self.phase >> slot & 1 and not any(s == slot for s, _ in self.flying)
            x = self.spans[self.tiles[i][0]]
            lost = self.gone >> slot * self.sub & ((1 << self.sub) - 1)
            masked = p < x["first"] or p + self.step > x["last"] or lost != 0
            for r in range(0, self.step):
                counts = not masked or (not lost >> r // 16 & 1 and x["first"] <= p + r < x["last"])
                assert counts == (x["first"] <= p + r < x["last"] and on[r // self.part_rows])
            self.held[slot] = None
            self.issue()
        if not failed:
            assert self.made == len(self.tiles) and not self.flying and all(h is None for h in self.held) and not any(self.expected)
        return failed


def _rings(own, seed, mistake=None, stuck=False, wide=False):
    rng = random.Random(2000 + seed)
    c = _case(rng)
    if wide:
        c.update(d=64, row_bytes=64, page=16, bad=0.5)
        c["cols"] = max(1, -(-max(c["lengths"] + [300]) // 16))
        c["lengths"][0] = 300
    p, spans, _, ctas = _deal(own, c)
    used = [mine for mine, _ in ctas if mine and any(t1 > t0 for _, _, t0, t1 in mine)]
    for mine in rng.sample(used, min(6, len(used))):
        tiles = [(s, u, t) for s, u, t0, t1 in mine for t in range(t0, t1)]
        at = (rng.randrange(p["stages"]), rng.randrange(2)) if stuck else None
        yield _Ring(own, c, tiles, spans, p["stages"], p["long_stages"], rng.randrange(own.warps), rng, at, mistake)


@pytest.mark.parametrize("seed", range(80))
def test_the_ring_of_a_warp(own, seed):
    """Copies arrive whenever they like: every wait is for what is on its way to its slot, no slot is filled that is still to be read, and
    the tokens that count are those of the window whose pages are there."""
    for ring in _rings(own, seed):
        assert not ring.run()


@pytest.mark.parametrize("seed", range(80))
def test_a_wait_that_runs_out_leaves_nothing_on_its_way(own, seed):
    """One copy never arrives: the warp goes on through its tiles without copies, after all the others have landed."""
    for ring in _rings(own, seed, stuck=True):
        if ring.run():
            assert not ring.flying


@pytest.mark.parametrize("mistake", ["has", "gone", "bytes", "phase"])
def test_the_walk_sees_a_mistake(own, mistake):
    """One planted in the walk's own state: a bit that is not taken back, missing parts not noted, bytes of parts that were not copied, a parity not turned."""
    seen = 0
    for seed in range(20):
        for ring in _rings(own, seed, mistake, wide=True):
            try:
                seen += ring.run()
            except AssertionError:
                seen += 1
    assert seen > 0

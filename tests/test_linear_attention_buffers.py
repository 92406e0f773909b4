"""What the warps of linear_chunks_kernel put where, walked through on the CPU in any order the hardware may run them: every place in shared
and in tensor memory is followed by its address, what is in it is read by all that need it before it is written over, nobody reads what
is not there yet, no barrier completes a phase that a waiting warp has not looked at, and all come to their end.  The rows' and the
state's warps are two agents each, so that warps of a role run ahead of one another.

Every wait of the kernel is left out in turn: the walk has to fail without it, or the wait is listed with the reason why others hold the
same.  The sequence of waits, arrivals, commits, loads and products is compared with the source, so that a change there is one here."""
import os
import random
import re

import pytest

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lact_b200", "csrc", "linear_chunks.cuh")


class Fault(AssertionError):
    pass


def _must(ok, *what):
    if not ok:
        raise Fault(what)


class _Barrier:
    def __init__(self, count=1):
        self.count, self.arrived, self.phases = count, 0, 0

    def arrive(self):
        self.arrived += 1
        if self.arrived == self.count:
            self.arrived, self.phases = 0, self.phases + 1

    def passes(self, index):
        """The wait of the code: by parity of the phase `index`."""
        return (self.phases & 1) != (index & 1)


class _Smem:
    """LinearSmem<A, B>."""

    def __init__(self, A, B):
        self.ring5, self.twice = A == 128 and B == 128, A == 64
        self.stages = 2 if A == 128 or B == 128 else 3
        self.piece_stages = 3 if B == 128 or A == 128 else 4
        self.XY, self.Z = 128 * A * 2, 128 * B * 2
        self.tiles = 5 * self.XY if self.ring5 else self.stages * (2 * self.XY + self.Z)
        self.S = self.tiles
        self.Low = self.S + self.XY
        self.end = self.Low + (4 if self.twice else 1) * self.XY
        _must(self.end + 320 <= 232448)

    def x(self, t):
        return 3 * t % 5 * self.XY if self.ring5 else t % self.stages * (2 * self.XY + self.Z)

    def y(self, t):
        return (3 * t + 1) % 5 * self.XY if self.ring5 else self.x(t) + self.XY

    def z(self, t):
        return (3 * t + 2) % 5 * self.XY if self.ring5 else self.x(t) + 2 * self.XY

    def piece_y(self, t):
        return 2 * t % 5 * self.XY if self.ring5 else t % self.piece_stages * (self.XY + self.Z)

    def piece_z(self, t):
        return (2 * t + 1) % 5 * self.XY if self.ring5 else self.piece_y(t) + self.XY

    def low(self, t, spare):
        return self.Low + (t & 1) * self.XY if self.twice else self.S if spare and t & 1 else self.Low

    def lowest(self, t):
        return self.Low + (2 + (t & 1)) * self.XY if self.twice else self.S


class _Content:
    """What lies in [begin, end): `need`: who has yet to read it; `made`: which agents have made their part (None: all at once)."""

    def __init__(self, label, begin, end, need, made=None):
        self.label, self.begin, self.end, self.need, self.made = label, begin, end, set(need), made
        self.cleared = set()


TMEM = 1 << 24    # columns of tensor memory, behind the addresses of shared memory
AGENTS = (0, 1)


class _Kernel:
    """One CTA of `tiles` tiles; `without`: the wait that is left out."""

    def __init__(self, rng, tiles, A, B, piece, three, without=None):
        self.rng, self.T, self.piece, self.three, self.without = rng, tiles, piece, three, without
        self.m = _Smem(A, B)
        self.NS = self.m.piece_stages if piece else self.m.stages
        bars = lambda n=1, c=1: [_Barrier(c) for _ in range(n)]
        self.xy_full, self.z_full, self.stage_empty = bars(4), bars(4), bars(4)
        self.g_full, self.o_full = bars()[0], bars()[0]
        self.p_full, self.s_ready, self.o_empty = (bars(1, 2)[0] for _ in range(3))
        self.x_done, self.d_full = bars(2), bars(2)
        self.y_ready, self.rest_ready, self.d_read = bars(2, 2), bars(2, 2), bars(2, 2)
        self.there, self.queue, self.loads = [], [], []
        self.broken = [rng.random() < 0.3 for _ in range(tiles)]
        self.seen = set()

    # ---- places
    def over(self, begin, end):
        return [c for c in self.there if c.begin < end and begin < c.end]

    def busy(self, begin, end, what):
        """No load or issued product touches the place."""
        for touched in [q[1] for q in self.queue] + [p[1] for p in self.loads]:
            for b, e in touched:
                _must(not (b < end and begin < e), what, "while a load or a product is at it")

    def replace(self, label, begin, end, need, made=None, issued=()):
        """A new content: all readers of what was there are done (`issued`: or in the queue ahead of the product that writes)."""
        for c in self.over(begin, end):
            _must(not (c.need - set(issued)), label, "over", c.label, "which is still needed by", c.need)
        self.there = [c for c in self.there if not (c.begin < end and begin < c.end)]
        c = _Content(label, begin, end, need, made)
        self.there.append(c)
        return c

    def find(self, label, begin, end):
        for c in self.there:
            if c.label == label and c.begin == begin and c.end == end:
                return c
        raise Fault(label, "is not there; there is", [c.label for c in self.over(begin, end)])

    def part(self, label, begin, end, need, agent):
        """An agent's part of a content that several make."""
        self.busy(begin, end, label)
        for c in self.over(begin, end):
            if c.label == label:
                c.made.add(agent)
                return
        self.replace(label, begin, end, need, {agent})

    def load(self, label, begin, size, need, bar, count):
        """A bulk copy: the place is its own from now until it lands."""
        self.busy(begin, begin + size, label)
        for c in self.over(begin, begin + size):
            _must(not c.need, label, "over", c.label, "which is still needed by", c.need)
        self.there = [c for c in self.there if not (c.begin < begin + size and begin < c.end)]

        def lands():
            self.replace(label, begin, begin + size, need)
            count[0] -= 1
            if count[0] == 0:
                bar.arrive()
        self.loads.append((lands, [(begin, begin + size)]))

    def product(self, who, reads, writes, commits):
        """Products in the order of their issue.  reads: (label, begin, end, parts that have to be made, what else has to hold); writes:
        (label, begin, end, need) or None; the check of what is written over is made at the issue, where the code has to be sure."""
        if writes:
            label, b, e, need = writes
            ahead = {q[2] for q in self.queue}
            for c in self.over(b, e):
                _must(c.label == label or not (c.need - ahead - {who}), who, "over", c.label, "which is still needed by", c.need)
            for _, place in self.loads:
                _must(not any(x < e and b < y for x, y in place))

        def runs():
            for label_, b_, e_, holds in reads:
                c = self.find(label_, b_, e_)
                _must(holds(c), who, "reads", label_, "too early or too late")
                c.need.discard(who)
            if writes and not any(c.label == label and c.begin == b for c in self.there):
                self.replace(label, b, e, need)
            for bar in commits:
                bar.arrive()
        # what it reads has to be there at the issue, too (but for products ahead of it in the queue that make it)
        for label_, b_, e_, holds in reads:
            if label_[0] not in ("P",):
                c = self.find(label_, b_, e_)
                _must(holds(c), who, "is issued on", label_, "too early or too late")
        places = [(b_, e_) for _, b_, e_, _ in reads] + ([(b, e)] if writes else [])
        self.queue.append((runs, places, who))

    # ---- the walk
    def wait(self, name, bar, index):
        """One wait of the code.  (The agent goes on some time after it has passed.)"""
        self.seen.add(name)
        if name == self.without:
            return
        yield bar, index
        yield None, 0

    def run(self):
        agents = {"load": self.loader(), "mma": self.mma()}
        for a in AGENTS:
            agents[f"rows {a}"], agents[f"state {a}"] = self.rows(a), self.state(a)
        speed = {n: self.rng.choice((1.0, 0.2, 0.02)) for n in [*agents, "queue", "loads"]}
        at = {n: next(g, None) for n, g in agents.items()}
        for _ in range(3000 * (self.T + 2)):
            live = [n for n in at if at[n] is not None]
            if not live:
                while self.queue:
                    self.queue.pop(0)[0]()
                return
            moves = [n for n in live if at[n][0] is None or at[n][0].passes(at[n][1])]
            moves += (["queue"] if self.queue else []) + (["loads"] if self.loads else [])
            for n in live:
                bar, index = at[n]
                _must(bar is None or bar.phases <= index + 1, n, "has missed a phase")
            _must(moves, "nobody can go on")
            n = self.rng.choices(moves, [speed[x] for x in moves])[0]
            if n == "queue":
                self.queue.pop(0)[0]()
            elif n == "loads":
                self.loads.pop(self.rng.randrange(len(self.loads)))[0]()
            else:
                at[n] = next(agents[n], None)
        raise Fault("no end")

    # ---- the roles, wait by wait as in the source
    def loader(self):
        m, NS = self.m, self.NS
        for t in range(self.T):
            if t >= NS:
                yield from self.wait("load stage_empty", self.stage_empty[t % NS], t // NS - 1)
            count = [1 if self.piece else 2]
            if self.piece:
                self.load(("Y", t), m.piece_y(t), m.XY, {"rows 0", "rows 1", ("D", t)}, self.xy_full[t % NS], count)
            else:
                self.load(("X", t), m.x(t), m.XY, {("G", t), ("OX", t)}, self.xy_full[t % NS], count)
                self.load(("Y", t), m.y(t), m.XY, {("G", t), "rows 0", "rows 1", ("D", t)}, self.xy_full[t % NS], count)
            yield None, 0
            if m.ring5 and self.piece and t >= 2:
                yield from self.wait("load stage_empty of the ring", self.stage_empty[(t - 2) % NS], (t - 2) // NS)
            if m.ring5 and not self.piece and t >= 1:
                yield from self.wait("load x_done of the ring", self.x_done[(t - 1) & 1], (t - 1) >> 1)
            self.load(("Z", t), m.piece_z(t) if self.piece else m.z(t), m.Z, {("D", t)} if self.piece else {("O", t), ("D", t)},
                      self.z_full[t % NS], [1])
            yield None, 0

    def y_of(self, t):
        return self.m.piece_y(t) if self.piece else self.m.y(t)

    def z_of(self, t):
        return self.m.piece_z(t) if self.piece else self.m.z(t)

    def clean(self, t):
        return lambda c: not self.broken[t] or c.cleared == set(AGENTS)

    def issue_g(self, t):
        m = self.m
        self.product(("G", t), [(("X", t), m.x(t), m.x(t) + m.XY, lambda c: True), (("Y", t), m.y(t), m.y(t) + m.XY, lambda c: not c.made)],
                     (("P", t), TMEM + 128, TMEM + 256, {"rows 0", "rows 1", ("O", t)}), [self.g_full])

    def mma(self):
        m, NS, all_made = self.m, self.NS, lambda c: c.made == set(AGENTS)
        if not self.piece:
            yield from self.wait("mma xy_full of the first", self.xy_full[0], 0)
            self.issue_g(0)
        for t in range(self.T):
            later = False
            z = (("Z", t), self.z_of(t), self.z_of(t) + m.Z, self.clean(t))
            if not self.piece:
                yield from self.wait("mma s_ready", self.s_ready, t)
                if t >= 1:
                    yield from self.wait("mma o_empty", self.o_empty, t - 1)
                self.product(("OX", t), [(("X", t), m.x(t), m.x(t) + m.XY, lambda c: True), (("S", t), m.S, m.S + m.XY, all_made)],
                             (("Ox", t), TMEM + 384, TMEM + 512, {"rows 0", "rows 1"}), [self.x_done[t & 1]])
                yield from self.wait("mma p_full", self.p_full, t)
                yield from self.wait("mma z_full", self.z_full[t % NS], t // NS)
                self.product(("O", t), [(("P", t), TMEM + 128, TMEM + 256, all_made), z],
                             (("Oz", t), TMEM + 256, TMEM + 384, {"rows 0", "rows 1"}), [self.o_full])
                later = t + 1 < self.T
                if later and not self.y_ready[t & 1].passes(t >> 1) and self.xy_full[(t + 1) % NS].passes((t + 1) // NS):
                    self.issue_g(t + 1)
                    later = False
                yield None, 0
            yield from self.wait("mma y_ready", self.y_ready[t & 1], t >> 1)
            if self.piece:
                yield from self.wait("mma z_full", self.z_full[t % NS], t // NS)
                if t >= 2:
                    yield from self.wait("mma d_read", self.d_read[t & 1], (t >> 1) - 1)
            d = TMEM + (128 * (t & 1) if self.piece else 0)
            low = m.low(t, self.piece and not self.three)
            write = (("D", t), d, d + 128, {"state 0", "state 1"})
            done = [self.d_full[t & 1], self.stage_empty[t % NS]]
            reads = [(("Y", t), self.y_of(t), self.y_of(t) + m.XY, all_made), z, (("low", t), low, low + m.XY, all_made)]
            if self.three:
                for label, b, e, holds in reads:
                    _must(holds(self.find(label, b, e)), "D is issued on", label)
                _must(not any(c.need - {q[2] for q in self.queue} for c in self.over(d, d + 128) if c.label != ("D", t)), "D over what is read")
                yield from self.wait("mma rest_ready", self.rest_ready[t & 1], t >> 1)
                b = m.lowest(t)
                reads = reads + [(("lowest", t), b, b + m.XY, all_made)]
            self.product(("D", t), reads, write, done)
            if later:
                yield from self.wait("mma xy_full", self.xy_full[(t + 1) % NS], (t + 1) // NS)
                self.issue_g(t + 1)
            yield None, 0

    def decay(self, t, a, low):
        """An agent's rows of Y: read, scaled in place, and the second piece stored."""
        m, b = self.m, self.y_of(t)
        c = self.find(("Y", t), b, b + m.XY)
        self.busy(b, b + m.XY, ("decay", t))
        _must(("G", t) not in c.need, "Y is scaled before G has read it")
        c.made = (c.made or set()) | {a}
        c.need.discard(f"rows {a}")
        self.part(("low", t), low, low + m.XY, {("D", t)}, a)

    def clear(self, t, a):
        b = self.z_of(t)
        c = self.find(("Z", t), b, b + self.m.Z)
        self.busy(b, b + self.m.Z, ("clear", t))
        c.cleared.add(a)

    def rows(self, a):
        m, NS = self.m, self.NS
        for t in range(self.T):
            if self.piece:
                used = t - 1 if self.three and not m.twice else t - 2
                yield from self.wait("rows xy_full", self.xy_full[t % NS], t // NS)
                if used >= 0:
                    yield from self.wait("rows d_full", self.d_full[used & 1], used >> 1)
                self.decay(t, a, m.low(t, not self.three))
                yield None, 0
                if self.three:
                    self.part(("lowest", t), m.lowest(t), m.lowest(t) + m.XY, {("D", t)}, a)
                if self.broken[t]:
                    yield from self.wait("rows z_full", self.z_full[t % NS], t // NS)
                    self.clear(t, a)
                yield None, 0
                self.y_ready[t & 1].arrive()
                yield None, 0
                if self.three:
                    self.rest_ready[t & 1].arrive()
                continue
            yield from self.wait("rows g_full", self.g_full, t)
            c = self.find(("P", t), TMEM + 128, TMEM + 256)
            c.made = (c.made or set()) | {a}
            c.need.discard(f"rows {a}")
            yield None, 0
            if self.broken[t]:
                yield from self.wait("rows z_full", self.z_full[t % NS], t // NS)
                self.clear(t, a)
            yield None, 0
            self.p_full.arrive()
            yield None, 0
            used = t - (2 if m.twice else 1)
            yield from self.wait("rows xy_full", self.xy_full[t % NS], t // NS)
            if used >= 0:
                yield from self.wait("rows d_full", self.d_full[used & 1], used >> 1)
            self.decay(t, a, m.low(t, False))
            yield None, 0
            self.y_ready[t & 1].arrive()
            yield None, 0
            if self.three:
                if not m.twice:
                    yield from self.wait("rows x_done", self.x_done[t & 1], t >> 1)
                self.part(("lowest", t), m.lowest(t), m.lowest(t) + m.XY, {("D", t)}, a)
                yield None, 0
                self.rest_ready[t & 1].arrive()
            yield from self.wait("rows o_full", self.o_full, t)
            for label, b in ((("Oz", t), TMEM + 256), (("Ox", t), TMEM + 384)):
                self.find(label, b, b + 128).need.discard(f"rows {a}")
            yield None, 0
            self.o_empty.arrive()

    def take(self, t, a, d):
        self.find(("D", t), d, d + 128).need.discard(f"state {a}")

    def state(self, a):
        m = self.m
        if self.piece:
            for t in range(self.T):
                yield from self.wait("state d_full", self.d_full[t & 1], t >> 1)
                self.take(t, a, TMEM + 128 * (t & 1))
                yield None, 0
                self.d_read[t & 1].arrive()
            return
        for t in range(self.T + 1):
            if t >= 1:
                yield from self.wait("state d_full", self.d_full[(t - 1) & 1], (t - 1) >> 1)
                self.take(t - 1, a, TMEM)
                yield None, 0
            if t < self.T:
                self.part(("S", t), m.S, m.S + m.XY, {("OX", t)}, a)
                yield None, 0
                self.s_ready.arrive()


SIZES = [(128, 128), (128, 64), (64, 128), (64, 64)]
COUNTS = (1, 2, 3, 4, 5, 7, 9)


def _walk(seed, A, B, piece, three, without=None):
    rng = random.Random(seed)
    k = _Kernel(rng, rng.choice(COUNTS), A, B, piece, three, without)
    k.run()
    return k.seen


@pytest.mark.parametrize("three", [False, True])
@pytest.mark.parametrize("piece", [False, True])
@pytest.mark.parametrize("A,B", SIZES)
def test_nothing_is_read_early_or_written_over(A, B, piece, three):
    for seed in range(150):
        _walk(seed, A, B, piece, three)


# Waits that order nothing which another does not order already, and where that is so.
MAIN = {(A, B, False, three) for A, B in SIZES for three in (False, True)}
SHARES = {(A, B, True, three) for A, B in SIZES for three in (False, True)}
REDUNDANT = {
    # G has read the tile, so it is there; the warps wait themselves for what the copy has written to be visible to them
    "rows xy_full": MAIN,
    # two sets of pieces: the last tile's output stands behind its X S, that behind the state's copy, that behind D of the tile before
    "rows d_full": {k for k in MAIN if k[0] == 64},
    # the ring of five, the shares: the wait for the place of the Z before it was for a later tile
    "load stage_empty": {k for k in SHARES if k[:2] == (128, 128)},
    # the shares: both pieces' arrivals come behind both stores
    "mma rest_ready": {k for k in SHARES if k[3]},
}


@pytest.mark.parametrize("three", [False, True])
@pytest.mark.parametrize("piece", [False, True])
@pytest.mark.parametrize("A,B", SIZES)
def test_every_wait_is_needed(A, B, piece, three):
    names = set()
    for seed in range(20):
        names |= _walk(seed, A, B, piece, three)
    for name in sorted(names):
        failed = False
        for seed in range(300):
            try:
                _walk(seed, A, B, piece, three, name)
            except Fault:
                failed = True
                break
        assert failed != ((A, B, piece, three) in REDUNDANT.get(name, ())), (name, failed)


CALLS = ("mbar_init", "mbar_wait_warp", "mbar_test", "mbar_arrive", "mbar_expect_tx_if", "tma_load_4d_if", "umma_bf16_if", "umma_bf16_ta_if",
         "umma_commit_if", "issue_g", "add", "decay", "put_rest", "linear_clear_rows<B>", "take", "tmem_ld32", "tmem_ld16", "tmem_st16")


def _calls(text):
    """The kernel's calls that the walk follows, in the order of the source, without blanks."""
    text = re.sub(r"//[^\n]*", "", text)
    out = []
    for found in re.finditer(r"(?<![\w<])(" + "|".join(re.escape(c) for c in CALLS) + r")\(", text):
        at, depth = found.end(), 1
        while depth:
            depth += {"(": 1, ")": -1}.get(text[at], 0)
            at += 1
        out.append(re.sub(r"\s+", "", found.group(0) + text[found.end():at]).replace(",abort_flag", "").replace("(leader,", "("))
    return out


PLACES = """
  static __device__ __forceinline__ uint32_t x(int t) { return kRing5 ? 3 * t % 5 * kXY : t % kStages * (2 * kXY + kZ); }
  static __device__ __forceinline__ uint32_t y(int t) { return kRing5 ? (3 * t + 1) % 5 * kXY : x(t) + kXY; }
  static __device__ __forceinline__ uint32_t z(int t) { return kRing5 ? (3 * t + 2) % 5 * kXY : x(t) + 2 * kXY; }
  static __device__ __forceinline__ uint32_t piece_y(int t) { return kRing5 ? 2 * t % 5 * kXY : t % kPieceStages * (kXY + kZ); }
  static __device__ __forceinline__ uint32_t piece_z(int t) { return kRing5 ? (2 * t + 1) % 5 * kXY : piece_y(t) + kXY; }
    return kTwice ? kLow + (t & 1) * kXY : spare && (t & 1) ? kS : kLow;
  static __device__ __forceinline__ uint32_t lowest(int t) { return kTwice ? kLow + (2 + (t & 1)) * kXY : kS; }
  static constexpr uint32_t kTiles = kRing5 ? 5 * kXY : kStages * (2 * kXY + kZ);
  static constexpr uint32_t kLow = kS + kXY;
  static constexpr int kStages = A == 128 || B == 128 ? 2 : 3;
  static constexpr int kPieceStages = B == 128 || A == 128 ? 3 : 4;
  constexpr int NS = PIECE ? SM::kPieceStages : SM::kStages;
  used = three && !SM::kTwice ? t - 1 : t - 2;
  used = t - (SM::kTwice ? 2 : 1);
  if (!SM::kTwice && !mbar_wait_warp(&x_done[par]
  if (SM::kRing5 && (PIECE ? t >= 2 && !mbar_wait_warp(&stage_empty[(t - 2) % NS]
  if (t >= NS && !mbar_wait_warp(&stage_empty[st]
  if (PIECE && (!mbar_wait_warp(&z_full[t % NS], (t / NS) & 1, abort_flag) ||
  (t >= 2 && !mbar_wait_warp(&d_read[t & 1], ((t >> 1) - 1) & 1, abort_flag))
  kTmemCols = 512, kG = 128, kO = 256, kOx = 384;
  kLinearRowThreads = 512, kLinearRowWarps = 16;
"""


SEQUENCE = """
mbar_init(&xy_full[s],1)
mbar_init(&z_full[s],1)
mbar_init(&stage_empty[s],1)
mbar_init(g_full,1)
mbar_init(p_full,kLinearRowWarps)
mbar_init(s_ready,8)
mbar_init(o_full,1)
mbar_init(o_empty,kLinearRowWarps)
mbar_init(&x_done[s],1)
mbar_init(&y_ready[s],kLinearRowWarps)
mbar_init(&rest_ready[s],kLinearRowWarps)
mbar_init(&d_full[s],1)
mbar_init(&d_read[s],8)
mbar_wait_warp(&stage_empty[st],(t/NS-1)&1)
mbar_expect_tx_if(&xy_full[st],PIECE?SM::kXY:2*SM::kXY)
tma_load_4d_if(base+SM::x(t)+j*kBox,&args.x,&xy_full[st],64*j,row,it.head/a.x_share,it.s.entry)
tma_load_4d_if(y_of(t)+j*kBox,&args.y,&xy_full[st],64*j,row,it.head/a.y_share,it.s.entry)
mbar_wait_warp(&stage_empty[(t-2)%NS],((t-2)/NS)&1)
mbar_wait_warp(&x_done[(t-1)&1],((t-1)>>1)&1)
mbar_expect_tx_if(&z_full[st],SM::kZ)
tma_load_4d_if(z_of(t)+j*kBox,&args.z,&z_full[st],64*j,row,it.head/a.z_share,it.s.entry)
umma_bf16_if(tmem+kG,desc.at((x+kk*kBox+k4*32)>>4),desc.at((y+kk*kBox+k4*32)>>4),idesc_g,(kk|k4)!=0)
umma_commit_if(g_full)
mbar_wait_warp(&xy_full[0],0)
issue_g(0)
mbar_wait_warp(s_ready,par)
mbar_wait_warp(o_empty,par^1)
umma_bf16_if(tmem+kOx,desc.at((x+kk*kBox+k4*32)>>4),desc.at((base+SM::kS+kk*kSBox+k4*32)>>4),idesc_ox,(kk|k4)!=0)
umma_commit_if(&x_done[par])
mbar_wait_warp(p_full,par)
mbar_wait_warp(&z_full[t%NS],(t/NS)&1)
umma_bf16_ta_if(tmem+kO,tmem+kG+(k>>1)*32+(k&1)*8,desc.at((z+k*2048)>>4),idesc_o,k!=0)
umma_commit_if(o_full)
mbar_test(&y_ready[par],(t>>1)&1)
mbar_test(&xy_full[(t+1)%NS],((t+1)/NS)&1)
issue_g(t+1)
mbar_wait_warp(&y_ready[par],(t>>1)&1)
mbar_wait_warp(&z_full[t%NS],(t/NS)&1)
mbar_wait_warp(&d_read[t&1],((t>>1)-1)&1)
umma_bf16_if(d,desc.at((z+k*2048)>>4),desc.at((piece+k*2048)>>4),idesc_d,!fresh||k!=0)
add(y,true)
add(base+SM::low(t,PIECE&&!three),false)
mbar_wait_warp(&rest_ready[par],(t>>1)&1)
add(base+SM::lowest(t),false)
umma_commit_if(&d_full[par])
umma_commit_if(&stage_empty[t%NS])
mbar_wait_warp(&xy_full[(t+1)%NS],((t+1)/NS)&1)
issue_g(t+1)
mbar_wait_warp(&xy_full[st],(t/NS)&1)
mbar_wait_warp(&d_full[used&1],(used>>1)&1)
decay(y_of(t),base+SM::low(t,!three),three,tid,f,j<nv)
put_rest(base+SM::lowest(t),tid)
mbar_wait_warp(&z_full[st],(t/NS)&1)
linear_clear_rows<B>(z_of(t),nv,tid)
mbar_arrive(&y_ready[t&1])
mbar_arrive(&rest_ready[t&1])
mbar_wait_warp(g_full,par)
tmem_ld32(tmem+lane_off+kG+c0,bits)
tmem_st16(tmem+lane_off+kG+c0,w)
mbar_wait_warp(&z_full[t%NS],(t/NS)&1)
linear_clear_rows<B>(z_of(t),nv,tid)
mbar_arrive(p_full)
mbar_wait_warp(&xy_full[t%NS],(t/NS)&1)
mbar_wait_warp(&d_full[used&1],(used>>1)&1)
decay(y_of(t),base+SM::low(t,false),three,tid,f,j<nv)
mbar_arrive(&y_ready[par])
mbar_wait_warp(&x_done[par],(t>>1)&1)
put_rest(base+SM::lowest(t),tid)
mbar_arrive(&rest_ready[par])
mbar_wait_warp(o_full,par)
tmem_ld16(tmem+lane_off+kO+cb*(B/4)+c,bi)
tmem_ld16(tmem+lane_off+kOx+cb*(B/4)+c,bx)
mbar_arrive(o_empty)
tmem_ld16(tmem+lane_off+d+c0+c,v)
mbar_wait_warp(&d_full[t&1],(t>>1)&1)
take((t&1)*kG,1.f,exp2f(g2*static_cast<float>(behind)))
mbar_arrive(&d_read[t&1])
mbar_wait_warp(&d_full[par^1],((t-1)>>1)&1)
take(0,decay,1.f)
mbar_arrive(s_ready)
"""


def test_the_walk_follows_the_source():
    text = open(SRC).read()
    for line in filter(None, (x.strip() for x in PLACES.splitlines())):
        assert line in text, line
    body = text[text.index("linear_chunks_kernel(const __grid_constant__"):text.index("linear_carry_kernel(const float*")]
    assert _calls(body) == [x.strip() for x in SEQUENCE.strip().splitlines()]

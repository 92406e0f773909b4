"""The hand-overs between the warps of linear_chunks_kernel, walked through on the CPU in any order the hardware may run them: a wait by
parity holds for one phase of a barrier, so that no barrier may complete a second phase before the waiting warp has looked at the
first; what a buffer holds may not be replaced before its last reader; and all have to come to their end.

The agents below follow the kernel's roles wait by wait (each wait names the barrier and the tile it is for); the products of the
tensor core complete in the order of their issue, some time after it."""
import os
import random
import re

import pytest

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lact_b200", "csrc", "linear_chunks.cuh")


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


class _Kernel:
    """One CTA: `tiles` tiles; `ring5` and `twice` as in LinearSmem, `three` pieces of Y, `piece` the pass over the shares."""

    def __init__(self, rng, tiles, piece, ring5, twice, three, stages):
        self.rng, self.T, self.piece, self.ring5, self.twice, self.three, self.NS = rng, tiles, piece, ring5, twice, three, stages
        B = lambda n=1, c=1: [_Barrier(c) for _ in range(n)]
        self.xy_full, self.z_full, self.stage_empty = B(4), B(4), B(4)
        self.g_full, self.p_full, self.s_ready, self.o_full, self.o_empty = (b for b in B(5))
        self.x_done, self.y_ready, self.rest_ready, self.d_full, self.d_read = B(2), B(2), B(2), B(2), B(2)
        self.queue, self.loads = [], []        # issued products and their commits, in order; loads in flight, in any order
        self.low = {}                          # place of a second piece -> (tile, whether D has read it)
        self.mma_at = self.rows_at = 0

    def run(self):
        agents = {"load": self.load(), "mma": self.mma(), "rows": self.rows(), "state": self.state()}
        at = {n: next(g, None) for n, g in agents.items()}
        for _ in range(400 * (self.T + 2)):
            live = [n for n in at if at[n] is not None]
            if not live:
                return True
            moves = [n for n in live if at[n][0].passes(at[n][1])] + (["queue"] if self.queue else []) + (["loads"] if self.loads else [])
            for n in live:   # a phase that the waiting warp has not looked at may not be followed by another
                bar, index = at[n]
                assert bar.phases <= index + 1, (n, index, bar.phases)
            if not moves:
                return False
            n = self.rng.choice(moves)
            if n == "queue":
                self.queue.pop(0)()
            elif n == "loads":
                self.loads.pop(self.rng.randrange(len(self.loads)))()
            else:
                at[n] = next(agents[n], None)
        return False

    def load(self):
        NS = self.NS
        for t in range(self.T):
            if t >= NS:
                yield self.stage_empty[t % NS], t // NS - 1
            self.loads.append(self.xy_full[t % NS].arrive)
            if self.ring5:
                if self.piece and t >= 2:
                    yield self.stage_empty[(t - 2) % NS], (t - 2) // NS
                if not self.piece and t >= 1:
                    yield self.x_done[(t - 1) & 1], (t - 1) >> 1
            self.loads.append(self.z_full[t % NS].arrive)

    def place(self, t):
        return t & 1 if self.twice or (self.piece and not self.three) else 0

    def mma(self):
        NS = self.NS
        if not self.piece:
            yield self.xy_full[0], 0
            self.queue.append(self.g_full.arrive)
        for t in range(self.T):
            later = False
            if not self.piece:
                yield self.s_ready, t
                if t >= 1:
                    yield self.o_empty, t - 1
                self.queue.append(self.x_done[t & 1].arrive)
                yield self.p_full, t
                yield self.z_full[t % NS], t // NS
                self.queue.append(self.o_full.arrive)
                later = t + 1 < self.T
                if later and not self.y_ready[t & 1].passes(t >> 1) and self.xy_full[(t + 1) % NS].passes((t + 1) // NS):
                    self.queue.append(self.g_full.arrive)
                    later = False
            yield self.y_ready[t & 1], t >> 1
            if self.piece:
                yield self.z_full[t % NS], t // NS
                if t >= 2:
                    yield self.d_read[t & 1], (t >> 1) - 1
            if self.three:
                yield self.rest_ready[t & 1], t >> 1

            def d_done(t=t):
                assert self.low[self.place(t)] == t
                self.low[self.place(t)] = None      # read
                self.d_full[t & 1].arrive()
                self.stage_empty[t % NS].arrive()
            self.queue.append(d_done)
            if later:
                yield self.xy_full[(t + 1) % NS], (t + 1) // NS
                self.queue.append(self.g_full.arrive)

    def pieces(self, t):
        assert self.low.get(self.place(t)) is None, "the pieces of a tile that D has not read yet"
        self.low[self.place(t)] = t

    def rows(self):
        NS = self.NS
        for t in range(self.T):
            if self.piece:
                used = t - 1 if self.three and not self.twice else t - 2
                yield self.xy_full[t % NS], t // NS
                if used >= 0:
                    yield self.d_full[used & 1], used >> 1
                self.pieces(t)
                if self.rng.random() < 0.3:      # (a tile that ends within it)
                    yield self.z_full[t % NS], t // NS
                self.y_ready[t & 1].arrive()
                if self.three:
                    self.rest_ready[t & 1].arrive()
                continue
            yield self.g_full, t
            if self.rng.random() < 0.3:
                yield self.z_full[t % NS], t // NS
            self.p_full.arrive()
            used = t - (2 if self.twice else 1)
            yield self.xy_full[t % NS], t // NS
            if used >= 0:
                yield self.d_full[used & 1], used >> 1
            self.pieces(t)
            self.y_ready[t & 1].arrive()
            if self.three:
                if not self.twice:
                    yield self.x_done[t & 1], t >> 1
                self.rest_ready[t & 1].arrive()
            yield self.o_full, t
            self.o_empty.arrive()

    def state(self):
        if self.piece:
            for t in range(self.T):
                yield self.d_full[t & 1], t >> 1
                self.d_read[t & 1].arrive()
            return
        for t in range(self.T + 1):
            if t >= 1:
                yield self.d_full[(t - 1) & 1], (t - 1) >> 1
            if t < self.T:
                self.s_ready.arrive()


@pytest.mark.parametrize("three", [False, True])
@pytest.mark.parametrize("piece", [False, True])
@pytest.mark.parametrize("ring5,twice,main,shares", [(True, False, 2, 3), (False, False, 2, 3), (False, True, 2, 3), (False, True, 3, 4)])
def test_every_order_comes_to_its_end(ring5, twice, main, shares, piece, three):
    for seed in range(300):
        rng = random.Random(seed)
        k = _Kernel(rng, rng.choice((1, 2, 3, 4, 5, 9, 14)), piece, ring5, twice, three, shares if piece else main)
        assert k.run(), (seed, k.T)


def test_the_model_has_the_stages_of_the_kernel():
    text = open(SRC).read()
    assert "kStages = A == 128 || B == 128 ? 2 : 3;" in text and "kPieceStages = B == 128 || A == 128 ? 3 : 4;" in text
    assert "used = t - (SM::kTwice ? 2 : 1);" in text and "used = three && !SM::kTwice ? t - 1 : t - 2;" in text
    waits = re.findall(r"mbar_wait_warp\(&?(\w+)", text)
    assert set(waits) == {"stage_empty", "x_done", "xy_full", "s_ready", "o_empty", "p_full", "z_full", "y_ready", "d_read", "rest_ready",
                          "g_full", "d_full", "o_full"}
    assert not re.search(r"\bmbar_wait\(", text)     # a whole warp waits, and meets again for the aligned instructions behind

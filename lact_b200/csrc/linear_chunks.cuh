// Linear attention with a decay per head (linear_steps.cuh has the formulas), tiles of 128 tokens on the tensor cores:
//   G = X Y^T,  P_ij = G_ij lambda^(i-j) (j <= i),  out = scale (P Z + diag(lambda^(i+1)) X S),
//   S <- lambda^n S + D,  D = (diag(lambda^(n-1-j)) Y)^T Z                             (backwards in time: the mirror image).
// A CTA takes a run of tiles of consecutive (sequence, head)s and reads every tile once:
//   warp 0       loads the tiles of X, Y, Z through a ring of stages;
//   warp 1       issues the products: X S, P Z, D and the next tile's G (before D if D has to wait);
//   warps 4-19   ("rows") G -> P (to tensor memory, the first operand of P Z from there), Y -> diag(lambda^(n-1-j)) Y in bf16 pieces,
//                the first in place, then both parts of the output -> memory;
//   warps 20-27  ("state") keep S in registers: S <- lambda^n S + D, its copy in bf16 to shared memory for X S.
// A tile is 131 KB at 128 features and arrives in 5700 clocks; the chain from one D to the next through these passes has to be shorter,
// and what a warp does one instruction after the other takes 7 clocks each: hence many warps with little work, four threads a row.
// Roundings: P and the copy of S to bf16, as operands of products whose sum is rounded to bf16 in the end.  S itself is added up in
// fp32 (D alone is summed by the tensor core, which truncates: over a long sequence that would show): the decayed rows of Y are two
// bf16 pieces (16 bits of the product; what is lost, 2^-17, is far below the copy's rounding), three (24 bits) where the last state
// is an output.
// Measured (2 x 32768 tokens, 12 heads of 128, 42 tiles a CTA): 141 us forwards, 805 MB at 5.7 TB/s, 3.4 us a tile where its 131 KB take 3.0;
// with three pieces 4.0 (48 products of 68 clocks).  What is left is the chain from D through the state's copy, X S and P Z to the next G.
// Long sequences of few heads: `per` tiles a CTA may begin within a sequence.  linear_chunks_kernel<.., PIECE, ..> first leaves every CTA's
// share of the state of the sequence that goes on behind it, linear_carry_kernel adds the shares up in order.  The shares are taken
// from the last tile to the first, and only as far as fp32 has room for their decay.  (So the tiles that a CTA begins with afterwards have
// been read last; what that leaves in L2 has not been measured by itself.)
#pragma once
#include "linear_steps.cuh"
#include "umma_gemm.cuh"

namespace lact {

constexpr int kLinearThreads = 896;   // a warpgroup for loads and products, four for the rows, two for the state
constexpr int kLinearRowThreads = 512, kLinearRowWarps = 16;
// registers per thread of each; together what the launch has.  (The little L1 beside 227 KB of shared memory misses: with a tile's
// bookkeeping on the stack it alone waited 1700 clocks.  Two of 128 features spill 10 bytes a thread, their shares' pass 68; the others none.)
constexpr int kLinearIssueRegs = 40, kLinearRowRegs = 56, kLinearStateRegs = 120, kLinearLaunchRegs = 72;
static_assert(kLinearIssueRegs + 4 * kLinearRowRegs + 2 * kLinearStateRegs <= 7 * kLinearLaunchRegs, "the shares of the registers");

struct LinearPiece {
  int32_t goes_on;    // the CTA's last sequence goes on in the next CTA
  int32_t inherits;   // ... and began before this one
  int32_t state;      // its state's index (sequence * heads + head)
  float mult;         // what the state before these tokens is multiplied with
};

struct LinearChunkArgs {
  LinearArgs a;
  CUtensorMap x, y, z;   // 4-D maps (feature, token, head, entry), box {64, 128, 1, 1}
  uint32_t per;          // tiles a CTA takes; packed sequences: 0, as many as make the CTAs even
  float* slots;          // [CTA] states: what the next CTA's sequence begins with ([A][B]; those of another pass may be read as [B][A]: slots_t)
  LinearPiece* pieces;   // [CTA]
  int32_t slots_t;
  int32_t* status;
};

template <int A, int B>
struct LinearSmem {
  static constexpr bool kRing5 = A == 128 && B == 128;   // no room for two whole stages beside the rest: five tiles of 32 KB in a ring
  static constexpr bool kTwice = A == 64;                // room for two sets of the second and third pieces of Y
  static constexpr int kStages = A == 128 || B == 128 ? 2 : 3;
  static constexpr int kPieceStages = B == 128 || A == 128 ? 3 : 4;   // of Y and Z alone (the ring of five holds two and a half)
  static constexpr uint32_t kXY = 128 * A * 2, kZ = 128 * B * 2;
  static constexpr uint32_t kTiles = kRing5 ? 5 * kXY : kStages * (2 * kXY + kZ);
  static constexpr uint32_t kS = kTiles;            // copy of S; one set of pieces: the third of Y
  static constexpr uint32_t kLow = kS + kXY;        // second piece of Y (two sets: two of them, two of the third)
  static constexpr uint32_t kBars = kLow + (kTwice ? 4 : 1) * kXY;
  static constexpr uint32_t kBytes = kBars + 320;
  static_assert(kRing5 || kPieceStages * (kXY + kZ) <= kTiles + (kTwice ? kXY : 0), "the stages of the shares fit");
  // where X, Y, Z of the CTA's tile t lie
  static __device__ __forceinline__ uint32_t x(int t) { return kRing5 ? 3 * t % 5 * kXY : t % kStages * (2 * kXY + kZ); }
  static __device__ __forceinline__ uint32_t y(int t) { return kRing5 ? (3 * t + 1) % 5 * kXY : x(t) + kXY; }
  static __device__ __forceinline__ uint32_t z(int t) { return kRing5 ? (3 * t + 2) % 5 * kXY : x(t) + 2 * kXY; }
  static __device__ __forceinline__ uint32_t piece_y(int t) { return kRing5 ? 2 * t % 5 * kXY : t % kPieceStages * (kXY + kZ); }
  static __device__ __forceinline__ uint32_t piece_z(int t) { return kRing5 ? (2 * t + 1) % 5 * kXY : piece_y(t) + kXY; }
  // the second and third pieces of Y; `spare`: the place of the copy of S is free for every other second one
  static __device__ __forceinline__ uint32_t low(int t, bool spare) {
    return kTwice ? kLow + (t & 1) * kXY : spare && (t & 1) ? kS : kLow;
  }
  static __device__ __forceinline__ uint32_t lowest(int t) { return kTwice ? kLow + (2 + (t & 1)) * kXY : kS; }
};

// The tiles of a launch in order: sequence, head, tile (backwards in time: from the last).
struct LinearTiles {
  int n, head, c, tiles;   // sequence, head, tile of the sequence in the order of the walk, its number of tiles
  LinearSpan s;
  static __device__ __forceinline__ int tiles_of(int len) { return (len + 127) >> 7; }
  // all tiles; every lane of a warp takes part
  static __device__ __forceinline__ uint32_t total(const LinearArgs& a) {   // (the host has seen to it that 31 bits are enough)
    if (a.cu == nullptr) return static_cast<uint32_t>(a.sequences) * a.heads * tiles_of(a.L);
    uint32_t sum = 0;
    for (int n = threadIdx.x & 31; n < a.sequences; n += 32) sum += tiles_of(linear_span(a, n).len);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    return sum * a.heads;
  }
  // tile number f (< total); every lane of a warp takes part
  __device__ __forceinline__ void seek(const LinearArgs& a, uint32_t f) {
    if (a.cu == nullptr) {
      tiles = tiles_of(a.L);
      const uint32_t chain = f / static_cast<uint32_t>(tiles);
      c = f - chain * tiles;
      n = chain / static_cast<uint32_t>(a.heads);
      head = chain - n * a.heads;
      s = linear_span(a, n);
      return;
    }
    const int lane = threadIdx.x & 31;
    for (int n0 = 0;; n0 += 32) {
      const int mine = n0 + lane < a.sequences ? tiles_of(linear_span(a, n0 + lane).len) : 0;
      uint32_t upto = mine;   // tiles of one head
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
        if (lane >= o) upto += v;
      }
      const uint32_t past = __ballot_sync(0xFFFFFFFFu, upto * a.heads > f);
      if (past != 0) {
        const int w = __ffs(past) - 1;
        n = n0 + w;
        tiles = __shfl_sync(0xFFFFFFFFu, mine, w);
        f -= (__shfl_sync(0xFFFFFFFFu, upto, w) - tiles) * a.heads;
        break;
      }
      f -= __shfl_sync(0xFFFFFFFFu, upto, 31) * a.heads;
      if (n0 + 32 >= a.sequences) {   // (f is not below the total: cannot be)
        n = a.sequences - 1;
        tiles = 1;
        f = 0;
        break;
      }
    }
    head = f / static_cast<uint32_t>(tiles);
    c = f - head * tiles;
    s = linear_span(a, n);
  }
  __device__ __forceinline__ void next(const LinearArgs& a) {
    if (++c < tiles) return;
    c = 0;
    if (++head < a.heads) return;
    head = 0;
    do {
      if (++n >= a.sequences) return;
      s = linear_span(a, n);
    } while (s.len == 0);
    tiles = tiles_of(s.len);
  }
  __device__ __forceinline__ int place(bool reverse) const { return (reverse ? tiles - 1 - c : c) * 128; }  // first token
  __device__ __forceinline__ int valid(int place) const { return min(128, s.len - place); }
  // backwards in time the state before the first token (the gradient of the last state) is not decayed by it
  __device__ __forceinline__ int first_decay(bool reverse) const { return reverse && c == 0 ? 0 : 1; }
};

struct LinearStart {
  LinearTiles it;
  int count, mid;
};

__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// Rows of a tile of Y times their decay until the tile's end, as bf16 pieces: the first in place, the second to `low`, a third (with
// `three`) into `rest`, which put_rest stores.  Thread j of 512 works on row j % 128; rows past the sequence become
// zeros.  (All loads before the first store: one after the other, they took twice as long.)
template <int A>
struct LinearRows {
  static constexpr int kUnits = A / 32;   // 16-byte units a thread
  static __device__ __forceinline__ uint32_t place(int tid, int k) {
    const int j = tid & 127, unit = (tid >> 7) * kUnits + k;
    return (unit >> 3) * (128 * 128) + j * 128 + (((unit & 7) ^ (j & 7)) << 4);
  }
  static __device__ __forceinline__ void put(uint32_t to, const uint32_t* v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
  }
  uint32_t rest[kUnits][4];
  __device__ __forceinline__ void decay(uint32_t y, uint32_t low, bool three, int tid, float f, bool real) {
    const F32x2 ff = f32x2(f, f), minus = f32x2(-1.f, -1.f);
    auto pair = [](uint32_t b) { return f32x2(__uint_as_float(b << 16), __uint_as_float(b & 0xFFFF0000u)); };
    auto round = [](F32x2 p) {
      float p0, p1;
      f32x2_split(p, p0, p1);
      return pack_bf16x2(p0, p1);
    };
#pragma unroll
    for (int k = 0; k < kUnits; ++k)
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(rest[k][0]), "=r"(rest[k][1]), "=r"(rest[k][2]), "=r"(rest[k][3]) : "r"(y + place(tid, k)));
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      uint32_t w[4], l[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        F32x2 p = f32x2_mul(pair(real ? rest[k][e] : 0u), ff);
        w[e] = round(p);
        p = f32x2_fma(pair(w[e]), minus, p);
        l[e] = round(p);
        if (three) rest[k][e] = round(f32x2_fma(pair(l[e]), minus, p));
      }
      put(y + place(tid, k), w);
      put(low + place(tid, k), l);
    }
  }
  __device__ __forceinline__ void put_rest(uint32_t lowest, int tid) const {
#pragma unroll
    for (int k = 0; k < kUnits; ++k) put(lowest + place(tid, k), rest[k]);
  }
};
// Rows `from` to 127 of a tile of Z become zeros.
template <int B>
__device__ __forceinline__ void linear_clear_rows(uint32_t z, int from, int tid) {
  for (int i = tid; i < (128 - from) * (B / 8); i += kLinearRowThreads) {
    const int row = from + i / (B / 8), u = i % (B / 8);
    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(z + (u >> 3) * (128 * 128) + row * 128 + (u & 7) * 16), "r"(0) : "memory");
  }
}

// A warpgroup's own number of registers: `dec` may not name more than the launch has, `inc` not less.
template <int N>
__device__ __forceinline__ void linear_registers() {
  if constexpr (N > kLinearLaunchRegs) registers_grow<N>();
  else registers_shrink<N>();
}

// THREE: pieces of Y; BACK: backwards in time (the shares' pass takes both).  Parameters of the template: as run-time choices in the rows'
// loop the one cost 12 %, the other 5 % (170 and 153 us of calls that take 151 and 145).
template <int A, int B, bool PIECE, bool THREE, bool BACK>
__global__ void __launch_bounds__(kLinearThreads, 1) linear_chunks_kernel(const __grid_constant__ LinearChunkArgs args) {
  static_assert((A == 64 || A == 128) && (B == 64 || B == 128), "64 or 128 features");
  using SM = LinearSmem<A, B>;
  constexpr int NS = PIECE ? SM::kPieceStages : SM::kStages;   // tiles on their way or in use, at most
  constexpr uint32_t kBox = 128 * 128;       // [128 rows][64 features] box of a tile
  constexpr uint32_t kSBox = B * 128;        // [B rows][64 columns] box of the copy of S
  constexpr uint32_t kTmemCols = 512, kG = 128, kO = 256, kOx = 384;   // D at 0, G and P (PIECE: a second D), P Z, X S
  extern __shared__ __align__(1024) uint8_t linear_smem[];
  const uint32_t base = smem_u32(linear_smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(linear_smem + SM::kBars);
  uint64_t* xy_full = bars;             // [stages, at most 4]
  uint64_t* z_full = bars + 4;          // [..]
  uint64_t* stage_empty = bars + 8;     // [..] Y and Z (and, the ring of five aside, X) have been used
  uint64_t* g_full = bars + 12;         // G is in tensor memory
  uint64_t* p_full = bars + 13;         // an arrival per row warp: P is there (and Z is clean)
  uint64_t* s_ready = bars + 14;        // an arrival per state warp: D has been read, the copy of S is there
  uint64_t* o_full = bars + 16;         // both parts of the output are there
  uint64_t* o_empty = bars + 17;        // an arrival per row warp: they have been read
  // Two of each of these, for every other tile: one role may be a tile ahead of another that waits (the rows of the products, with two
  // sets of pieces; X S of the loads, in the ring of five), and a wait by parity on one barrier would then miss a phase.
  uint64_t* x_done = bars + 18;         // [2] X and the copy of S have been used
  uint64_t* y_ready = bars + 20;        // [2] an arrival per warp that makes them: the first two pieces of Y are there
  uint64_t* rest_ready = bars + 22;     // [2] likewise the third
  uint64_t* d_full = bars + 24;         // [2] D is there
  uint64_t* d_read = bars + 26;         // [2] PIECE: an arrival per state warp
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 28);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  LinearStart* start = reinterpret_cast<LinearStart*>(tmem_slot + 2);
  const LinearArgs& a = args.a;
  const bool reverse = PIECE ? a.reverse != 0 : BACK;

  const int warp = uniform_warp_index(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < 4; ++s) { mbar_init(&xy_full[s], 1); mbar_init(&z_full[s], 1); mbar_init(&stage_empty[s], 1); }
    mbar_init(g_full, 1);
    mbar_init(p_full, kLinearRowWarps);
    mbar_init(s_ready, 8);
    mbar_init(o_full, 1);
    mbar_init(o_empty, kLinearRowWarps);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&x_done[s], 1);
      mbar_init(&y_ready[s], kLinearRowWarps);
      mbar_init(&rest_ready[s], kLinearRowWarps);
      mbar_init(&d_full[s], 1);
      mbar_init(&d_read[s], 8);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  griddep_launch_dependents();
  griddep_wait();

  // This CTA's tiles: worked out by one warp (by every warp, its values lay on the stack for the rest of the kernel)
  if (warp == 2) {
    const uint32_t total = LinearTiles::total(a);
    const uint32_t per = args.per > 0 ? args.per : (total + gridDim.x - 1) / gridDim.x;
    const uint32_t first = blockIdx.x * per, end = min(first + per, total);
    LinearStart w{};
    w.count = end > first ? static_cast<int>(end - first) : 0;
    if (w.count > 0) {
      w.it.seek(a, PIECE ? end - 1 : first);
      w.mid = w.it.c > 0;
      if (PIECE) {   // the tiles of the last one's sequence, from the last to the first
        const bool goes_on = w.it.c + 1 < w.it.tiles;
        const int back = min(w.it.c, w.count - 1);
        LinearTiles at = w.it;
        at.c -= back;
        // tokens of these tiles: all whole, but for the first of a walk backwards
        const int tokens = (back + 1) * 128 - (reverse && at.c == 0 ? 128 - at.valid(at.place(reverse)) : 0);
        if (lane == 0)
          args.pieces[blockIdx.x] = {goes_on, at.c > 0, w.it.n * a.heads + w.it.head,
                                     exp2f(decay_log2(a, w.it.head) * static_cast<float>(tokens - 1 + at.first_decay(reverse)))};
        w.count = goes_on ? back + 1 : 0;
        // tiles whose decay is below the smallest fp32 would be added as zeros
        const float g2 = decay_log2(a, w.it.head);
        if (g2 * 128.f * static_cast<float>(w.count) < -160.f) w.count = min(w.count, static_cast<int>(160.f / (-128.f * g2)) + 2);
      }
    } else if (PIECE && lane == 0) {
      args.pieces[blockIdx.x] = {0, 0, 0, 0.f};
    }
    if (lane == 0) *start = w;
  }
  __syncthreads();
  const int count = start->count;
  const bool mid = start->mid != 0;    // the first tile goes on with a sequence that the CTA before this one has begun
  LinearTiles it = start->it;
  auto advance = [&]() {
    if (PIECE) --it.c;
    else it.next(a);
  };
  // (swizzled tiles need the alignment asked for above)
  bool failed = uniform(static_cast<uint32_t>(*reinterpret_cast<volatile int32_t*>(args.status))) != kStatusOk || (base & 1023u) != 0;
  constexpr bool three = THREE;
  auto y_of = [&](int t) { return base + (PIECE ? SM::piece_y(t) : SM::y(t)); };
  auto z_of = [&](int t) { return base + (PIECE ? SM::piece_z(t) : SM::z(t)); };

  if (warp < 4) {
    linear_registers<kLinearIssueRegs>();
    if (warp == 0) {
      const uint32_t leader = elect_leader();
      for (int t = 0; t < count && !failed; ++t, advance()) {
        const int st = t % NS, row = it.s.first + it.place(reverse);
        if (t >= NS && !mbar_wait_warp(&stage_empty[st], (t / NS - 1) & 1, abort_flag)) { failed = true; break; }
        mbar_expect_tx_if(leader, &xy_full[st], PIECE ? SM::kXY : 2 * SM::kXY);
        for (int j = 0; j < A / 64; ++j) {
          if (!PIECE) tma_load_4d_if(leader, base + SM::x(t) + j * kBox, &args.x, &xy_full[st], 64 * j, row, it.head / a.x_share, it.s.entry);
          tma_load_4d_if(leader, y_of(t) + j * kBox, &args.y, &xy_full[st], 64 * j, row, it.head / a.y_share, it.s.entry);
        }
        // (ring of five: Z comes to where X of the tile before was; for the shares, where Y of the tile two before was)
        if (SM::kRing5 && (PIECE ? t >= 2 && !mbar_wait_warp(&stage_empty[(t - 2) % NS], ((t - 2) / NS) & 1, abort_flag)
                                 : t >= 1 && !mbar_wait_warp(&x_done[(t - 1) & 1], ((t - 1) >> 1) & 1, abort_flag))) { failed = true; break; }
        mbar_expect_tx_if(leader, &z_full[st], SM::kZ);
        for (int j = 0; j < B / 64; ++j)
          tma_load_4d_if(leader, z_of(t) + j * kBox, &args.z, &z_full[st], 64 * j, row, it.head / a.z_share, it.s.entry);
      }
    } else if (warp == 1) {
      const uint32_t leader = elect_leader();
      const uint32_t idesc_g = make_idesc_bf16(128, 128, 0, 0);   // X Y^T, both K-major
      const uint32_t idesc_ox = make_idesc_bf16(128, B, 0, 0);    // X S: the copy of S is [B][A], K-major
      const uint32_t idesc_o = make_idesc_bf16(128, B, 0, 1);     // P Z: P in tensor memory, Z MN-major
      const uint32_t idesc_d = make_idesc_bf16(128, A, 1, 1);     // Z^T Y, both MN-major (64 features: the upper lanes take what follows Z)
      const SmemDescBase desc(kBox);
      auto issue_g = [&](int t) {
        const uint32_t x = base + SM::x(t), y = y_of(t);
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < A / 64; ++kk)
#pragma unroll
          for (int k4 = 0; k4 < 4; ++k4)
            umma_bf16_if(leader, tmem + kG, desc.at((x + kk * kBox + k4 * 32) >> 4), desc.at((y + kk * kBox + k4 * 32) >> 4), idesc_g,
                         (kk | k4) != 0);
        umma_commit_if(leader, g_full);
      };
      if (!PIECE && count > 0 && !failed) {
        if (mbar_wait_warp(&xy_full[0], 0, abort_flag)) issue_g(0);
        else failed = true;
      }
      for (int t = 0; t < count && !failed; ++t) {
        const uint32_t par = t & 1, x = base + SM::x(t), y = y_of(t), z = z_of(t);
        bool g_next = false;
        if (!PIECE) {
          if (!mbar_wait_warp(s_ready, par, abort_flag) || (t >= 1 && !mbar_wait_warp(o_empty, par ^ 1, abort_flag))) { failed = true; break; }
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < A / 64; ++kk)
#pragma unroll
            for (int k4 = 0; k4 < 4; ++k4)
              umma_bf16_if(leader, tmem + kOx, desc.at((x + kk * kBox + k4 * 32) >> 4),
                           desc.at((base + SM::kS + kk * kSBox + k4 * 32) >> 4), idesc_ox, (kk | k4) != 0);
          umma_commit_if(leader, &x_done[par]);
          if (!mbar_wait_warp(p_full, par, abort_flag) || !mbar_wait_warp(&z_full[t % NS], (t / NS) & 1, abort_flag)) { failed = true; break; }
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < 8; ++k)
            umma_bf16_ta_if(leader, tmem + kO, tmem + kG + (k >> 1) * 32 + (k & 1) * 8, desc.at((z + k * 2048) >> 4), idesc_o, k != 0);
          umma_commit_if(leader, o_full);
          g_next = t + 1 < count;
          // D before the next G, if its operands are there: what the next tile waits for comes behind D
          if (g_next && !__all_sync(0xFFFFFFFFu, mbar_test(&y_ready[par], (t >> 1) & 1)) &&
              __all_sync(0xFFFFFFFFu, mbar_test(&xy_full[(t + 1) % NS], ((t + 1) / NS) & 1))) {
            issue_g(t + 1);
            g_next = false;
          }
        }
        if (!mbar_wait_warp(&y_ready[par], (t >> 1) & 1, abort_flag)) { failed = true; break; }
        if (PIECE && (!mbar_wait_warp(&z_full[t % NS], (t / NS) & 1, abort_flag) ||
                      (t >= 2 && !mbar_wait_warp(&d_read[t & 1], ((t >> 1) - 1) & 1, abort_flag)))) { failed = true; break; }
        tc_fence_after();
        const uint32_t d = tmem + (PIECE ? par * kG : 0);
        auto add = [&](uint32_t piece, bool fresh) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            umma_bf16_if(leader, d, desc.at((z + k * 2048) >> 4), desc.at((piece + k * 2048) >> 4), idesc_d, !fresh || k != 0);
        };
        add(y, true);
        add(base + SM::low(t, PIECE && !three), false);
        if (three) {
          if (!mbar_wait_warp(&rest_ready[par], (t >> 1) & 1, abort_flag)) { failed = true; break; }
          tc_fence_after();
          add(base + SM::lowest(t), false);
        }
        umma_commit_if(leader, &d_full[par]);
        umma_commit_if(leader, &stage_empty[t % NS]);
        if (g_next) {
          if (!mbar_wait_warp(&xy_full[(t + 1) % NS], ((t + 1) / NS) & 1, abort_flag)) { failed = true; break; }
          issue_g(t + 1);
        }
      }
    }
  } else if (warp < 4 + kLinearRowWarps) {
    linear_registers<kLinearRowRegs>();
    // ---------------- rows: four threads per row of the tile (tensor-memory lane), 32 columns of G and a quarter of the output each
    const int quarter = warp & 3, cb = (warp - 4) >> 2, r = quarter * 32 + lane, tid = threadIdx.x - 128;
    int head = -1;
    float g2 = 0.f;
    if constexpr (PIECE) {   // the pieces of Y; the tiles' own end is where their decays count from
      for (int t = 0; t < count && !failed; ++t, advance()) {
        const int st = t % NS, nv = it.valid(it.place(reverse)), used = three && !SM::kTwice ? t - 1 : t - 2;   // (the tile whose places these are)
        if (it.head != head) {
          head = it.head;
          g2 = decay_log2(a, head);
        }
        const int j = tid & 127;
        const float f = exp2f(g2 * static_cast<float>(reverse ? j : max(nv - 1 - j, 0)));
        if (!mbar_wait_warp(&xy_full[st], (t / NS) & 1, abort_flag) ||
            (used >= 0 && !mbar_wait_warp(&d_full[used & 1], (used >> 1) & 1, abort_flag))) { failed = true; break; }
        LinearRows<A> rows;
        rows.decay(y_of(t), base + SM::low(t, !three), three, tid, f, j < nv);
        if (three) rows.put_rest(base + SM::lowest(t), tid);
        if (nv < 128 && a.cu != nullptr) {
          if (!mbar_wait_warp(&z_full[st], (t / NS) & 1, abort_flag)) { failed = true; break; }
          linear_clear_rows<B>(z_of(t), nv, tid);
        }
        fence_async_proxy();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&y_ready[t & 1]);
          if (three) mbar_arrive(&rest_ready[t & 1]);
        }
      }
    } else {
      const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
      linear_zero_rest<B>(a, static_cast<int64_t>(blockIdx.x) * kLinearRowThreads + tid, static_cast<int64_t>(gridDim.x) * kLinearRowThreads);
      if (a.cu != nullptr && a.s_out != nullptr) {   // empty sequences keep their states
        for (int i = blockIdx.x; i < a.sequences * a.heads; i += gridDim.x) {
          if (linear_span(a, i / a.heads).len != 0) continue;
          const int64_t at = static_cast<int64_t>(i) * (A * B / 4);
          for (int e = tid; e < A * B / 4; e += kLinearRowThreads)
            reinterpret_cast<float4*>(a.s_out)[at + e] =
                a.s_in != nullptr ? reinterpret_cast<const float4*>(a.s_in)[at + e] : make_float4(0.f, 0.f, 0.f, 0.f);
        }
      }
      float lambda = 0.f;
      for (int t = 0; t < count && !failed; ++t, advance()) {
        const uint32_t par = t & 1;
        const int place = it.place(reverse), nv = it.valid(place);
        if (it.head != head) {
          head = it.head;
          g2 = decay_log2(a, head);
          lambda = exp2f(g2);
        }
        if (!mbar_wait_warp(g_full, par, abort_flag)) { failed = true; break; }
        tc_fence_after();
        {
          const int c0 = cb * 32;
          uint32_t w[16];
          if (reverse ? cb < quarter : cb > quarter) {
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = 0;
          } else {
            uint32_t bits[32];
            tmem_ld32(tmem + lane_off + kG + c0, bits);
            if (cb != quarter) {
              // from the column nearest to the diagonal on, a factor of lambda each (two columns at a time; no table of them: shared memory is
              // what the products wait for)
              const float f = exp2_ftz(g2 * static_cast<float>(reverse ? c0 - r : r - c0 - 31)), f1 = f * lambda;
              const F32x2 two = f32x2(lambda * lambda, lambda * lambda);
              const int hi = reverse ? nv - 1 - c0 : 31;
              F32x2 d = reverse ? f32x2(f, f1) : f32x2(f1, f);
              tmem_ld_wait();
              auto column = [&](int j) {
                float p0, p1;
                f32x2_split(f32x2_mul(f32x2(__uint_as_float(bits[j]), __uint_as_float(bits[j + 1])), d), p0, p1);
                if (hi < 31) {
                  p0 = j > hi ? 0.f : p0;
                  p1 = j + 1 > hi ? 0.f : p1;
                }
                w[j / 2] = pack_bf16x2(p0, p1);
                d = f32x2_mul(d, two);
              };
              if (reverse) {
#pragma unroll
                for (int j = 0; j < 32; j += 2) column(j);
              } else {
#pragma unroll
                for (int j = 30; j >= 0; j -= 2) column(j);
              }
            } else {
              // column j is |lane - j| tokens away; visible from / up to its own
              const float step = reverse ? g2 : -g2, from = (reverse ? -lane : lane) * g2;
              const int lo = reverse ? lane : 0, hi = reverse ? nv - 1 - c0 : lane;
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 32; j += 2) {
                float p0 = __uint_as_float(bits[j]) * exp2_ftz(fmaf(static_cast<float>(j), step, from));
                float p1 = __uint_as_float(bits[j + 1]) * exp2_ftz(fmaf(static_cast<float>(j + 1), step, from));
                p0 = j < lo || j > hi ? 0.f : p0;
                p1 = j + 1 < lo || j + 1 > hi ? 0.f : p1;
                w[j / 2] = pack_bf16x2(p0, p1);
              }
            }
          }
          __syncwarp();
          tmem_st16(tmem + lane_off + kG + c0, w);
        }
        if (nv < 128 && a.cu != nullptr) {   // rows of the next sequence: no part of any sum
          if (!mbar_wait_warp(&z_full[t % NS], (t / NS) & 1, abort_flag)) { failed = true; break; }
          linear_clear_rows<B>(z_of(t), nv, tid);
          fence_async_proxy();
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full);

        // the pieces of Y, where those of the tile before (two sets: before that one) were, once D has used them.  A third, where there is
        // one set, takes the place of the copy of S once X S has used that.
        {
          const int j = tid & 127, used = t - (SM::kTwice ? 2 : 1);
          const float f = exp2f(g2 * static_cast<float>(reverse ? j : max(nv - 1 - j, 0)));
          if (!mbar_wait_warp(&xy_full[t % NS], (t / NS) & 1, abort_flag) ||
              (used >= 0 && !mbar_wait_warp(&d_full[used & 1], (used >> 1) & 1, abort_flag))) { failed = true; break; }
          LinearRows<A> rows;
          rows.decay(y_of(t), base + SM::low(t, false), three, tid, f, j < nv);
          fence_async_proxy();
          __syncwarp();
          if (lane == 0) mbar_arrive(&y_ready[par]);
          if (three) {
            if (!SM::kTwice && !mbar_wait_warp(&x_done[par], (t >> 1) & 1, abort_flag)) { failed = true; break; }
            rows.put_rest(base + SM::lowest(t), tid);
            fence_async_proxy();
            __syncwarp();
            if (lane == 0) mbar_arrive(&rest_ready[par]);
          }
        }

        const int pos = reverse ? nv - 1 - r : r;
        const float since = a.scale * exp2f(g2 * static_cast<float>(max(pos, 0) + it.first_decay(reverse)));
        const F32x2 ss = f32x2(since, since), sc = f32x2(a.scale, a.scale);
        const int64_t o = ((it.s.entry * static_cast<int64_t>(a.L) + it.s.first + place + r) * a.heads + head) * B + cb * (B / 4);
        if (!mbar_wait_warp(o_full, par, abort_flag)) { failed = true; break; }
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < B / 4; c += 16) {
          uint32_t bi[16], bx[16];
          tmem_ld16(tmem + lane_off + kO + cb * (B / 4) + c, bi);
          tmem_ld16(tmem + lane_off + kOx + cb * (B / 4) + c, bx);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            const F32x2 p = f32x2_fma(f32x2(__uint_as_float(bx[j]), __uint_as_float(bx[j + 1])), ss,
                                      f32x2_mul(f32x2(__uint_as_float(bi[j]), __uint_as_float(bi[j + 1])), sc));
            float p0, p1;
            f32x2_split(p, p0, p1);
            if (a.out_f32) {
              bi[j] = __float_as_uint(p0);
              bi[j + 1] = __float_as_uint(p1);
            } else {
              bi[j / 2] = pack_bf16x2(p0, p1);
            }
          }
          if (r < nv) {
            if (a.out_f32) {
              st_global_32(static_cast<float*>(a.out) + o + c, bi);
              st_global_32(static_cast<float*>(a.out) + o + c + 8, bi + 8);
            } else {
              st_global_32(static_cast<bf16*>(a.out) + o + c, bi);
            }
          }
          __syncwarp();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(o_empty);
      }
    }
  } else {
    linear_registers<kLinearStateRegs>();
    // ---------------- state: lane = column of Z (B of them), two threads per lane, half of S's other side each
    const int quarter = warp & 3, half = (warp - 4 - kLinearRowWarps) >> 2, r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const bool holds = quarter * 32 < B;    // (64 columns: the upper lanes of tensor memory are not part of S)
    constexpr int NC = A / 2;
    const int c0 = half * NC;
    int head = -1;
    float g2 = 0.f;
    float S[NC];
#pragma unroll
    for (int j = 0; j < NC; ++j) S[j] = 0.f;
    // state number `n` of an array: element (row of A: c0 + j, column r), j up to NC
    auto load_state = [&](const float* from, int64_t n, bool transposed, float mul) {
      from += n * (A * B) + (transposed ? r * A + c0 : c0 * B + r);
      if (transposed) {
#pragma unroll
        for (int j = 0; j < NC; ++j) S[j] = from[j] * mul;
      } else {
#pragma unroll
        for (int j = 0; j < NC; ++j) S[j] = from[j * B] * mul;
      }
    };
    auto store_state = [&](float* to, int64_t n, float mul) {
      to += n * (A * B) + c0 * B + r;
#pragma unroll
      for (int j = 0; j < NC; ++j) to[j * B] = S[j] * mul;
    };
    // S <- S * x + D * y
    auto take = [&](uint32_t d, float x, float y) {
      const F32x2 xx = f32x2(x, x), yy = f32x2(y, y);
#pragma unroll
      for (int c = 0; c < NC; c += 16) {
        uint32_t v[16];
        tmem_ld16(tmem + lane_off + d + c0 + c, v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          const F32x2 s = f32x2_fma(f32x2(S[c + j], S[c + j + 1]), xx, f32x2_mul(f32x2(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), yy));
          f32x2_split(s, S[c + j], S[c + j + 1]);
        }
      }
    };
    if constexpr (PIECE) {
      int behind = 0;   // tokens of these tiles behind tile t
      for (int t = 0; t < count && !failed; ++t, advance()) {
        if (it.head != head) {
          head = it.head;
          g2 = decay_log2(a, head);
        }
        if (!mbar_wait_warp(&d_full[t & 1], (t >> 1) & 1, abort_flag)) { failed = true; break; }
        tc_fence_after();
        if (holds) take((t & 1) * kG, 1.f, exp2f(g2 * static_cast<float>(behind)));
        behind += it.valid(it.place(reverse));
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&d_read[t & 1]);
      }
      if (!failed && count > 0 && holds) store_state(args.slots, blockIdx.x, 1.f);
    } else {
      float decay = 1.f;        // of the tile before
      bool last = false;        // it was its sequence's last
      int state = 0;            // whose number
      for (int t = 0;; ++t) {
        const uint32_t par = t & 1;
        if (t >= 1) {
          if (!mbar_wait_warp(&d_full[par ^ 1], ((t - 1) >> 1) & 1, abort_flag)) { failed = true; break; }
          tc_fence_after();
          if (holds) {
            take(0, decay, 1.f);
            if (last && a.s_out != nullptr) store_state(a.s_out, state, a.out_mul * (reverse ? exp2f(g2) : 1.f));
          }
          advance();
        }
        if (t >= count || failed) break;
        const int place = it.place(reverse), nv = it.valid(place);
        if (it.head != head) {
          head = it.head;
          g2 = decay_log2(a, head);
        }
        state = it.n * a.heads + head;
        last = it.c + 1 == it.tiles;
        decay = exp2f(g2 * static_cast<float>(nv - 1 + it.first_decay(reverse)));
        if (holds) {
          if (it.c == 0) {
            if (a.s_in != nullptr) {
              load_state(a.s_in, state, a.s_in_t, a.in_mul);
            } else {
#pragma unroll
              for (int j = 0; j < NC; ++j) S[j] = 0.f;
            }
          } else if (mid && t == 0) {   // what the CTA before this one has left
            load_state(args.slots, blockIdx.x - 1, args.slots_t, 1.f);
          }
          // the copy (K-major, 128-byte swizzle: row r of 128-byte rows of 64 columns)
          const uint32_t row = base + SM::kS + (c0 >> 6) * kSBox + r * 128;
#pragma unroll
          for (int g = 0; g < NC / 8; ++g) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(S[g * 8 + 2 * e], S[g * 8 + 2 * e + 1]);
            const uint32_t unit = ((c0 & 63) >> 3) + g;
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row + ((unit ^ (r & 7)) << 4)), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                         "r"(w[3])
                         : "memory");
          }
        }
        tc_fence_before();
        fence_async_proxy();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_ready);
      }
    }
  }
  if (failed && *reinterpret_cast<volatile int32_t*>(args.status) == kStatusOk) {
    *abort_flag = 1;
    report_timeout(args.status);
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag && threadIdx.x == 0) {
    for (int i = 0; i < 256; ++i) __nanosleep(1000);   // bulk copies still in flight land before shared memory goes
  }
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, kTmemCols);
}

// What every CTA's first sequence begins with: along a sequence, slots[i] <- slots[i] + mult_i * (state before CTA i's part).  A block
// takes 512 elements of the sequence whose first share is CTA blockIdx.y's; shares are fetched eight at a time.
constexpr int kLinearMaxCtas = 256;
__global__ void __launch_bounds__(128) linear_carry_kernel(const float* __restrict__ s_in, float in_mul, float* __restrict__ slots,
                                                           const LinearPiece* __restrict__ pieces, int32_t ctas, int32_t size) {
  __shared__ LinearPiece info[kLinearMaxCtas];
  griddep_launch_dependents();
  griddep_wait();
  const int i0 = blockIdx.y;
  if (!pieces[i0].goes_on || pieces[i0].inherits) return;
  for (int i = i0 + threadIdx.x; i < ctas; i += 128) info[i] = pieces[i];
  __syncthreads();
  const int e = (blockIdx.x * 128 + threadIdx.x) * 4;    // of a state's `size` elements
  float4 carry = make_float4(0.f, 0.f, 0.f, 0.f);
  if (s_in != nullptr) {
    carry = *reinterpret_cast<const float4*>(s_in + static_cast<int64_t>(info[i0].state) * size + e);
    carry.x *= in_mul; carry.y *= in_mul; carry.z *= in_mul; carry.w *= in_mul;
  }
  int last = i0;   // the sequence's last share
  while (last + 1 < ctas && info[last + 1].goes_on && info[last + 1].inherits) ++last;
  float4* const at = reinterpret_cast<float4*>(slots + e);
  const int64_t step = size / 4;
  for (int i = i0; i <= last; i += 8) {
    float4 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = at[min(i + k, last) * step];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (i + k > last) break;
      const float m = info[i + k].mult;
      carry = make_float4(fmaf(m, carry.x, v[k].x), fmaf(m, carry.y, v[k].y), fmaf(m, carry.z, v[k].z), fmaf(m, carry.w, v[k].w));
      at[(i + k) * step] = carry;
    }
  }
}

}  // namespace lact

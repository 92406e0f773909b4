// Linear attention with a decay per head (linear_steps.cuh has the formulas), tiles of 128 tokens on the tensor cores:
//   G = X Y^T,  P_ij = G_ij lambda^(i-j) (j <= i),  out = scale (P Z + diag(lambda^(i+1)) X S),
//   S <- lambda^n S + (diag(lambda^(n-1-j)) Y)^T Z                                     (backwards in time: the mirror image).
// A CTA takes a run of tiles of consecutive (sequence, head)s, keeps S in tensor memory over them and reads every tile once:
//   warp 0       loads the tiles of X, Y, Z through a ring of stages;
//   warp 1       issues the products: G(t + 1) as soon as P(t) has been used and the tile is there;
//   warps 2-9    ("rows") G -> P (to tensor memory, the first operand of P Z from there), later both parts of the output -> memory;
//   warps 10-17  ("state") S -> bf16 in shared memory for X S, S * lambda^n back to tensor memory, then Y -> Y lambda^(n-1-j) in bf16
//                pieces, in place and into the tile's X and the copy of S, which X S has used by then.
// Roundings: P and the copy of S to bf16, as operands of products whose sum is rounded to bf16 in the end.  S itself stays in fp32:
// decayed rows of Y are two bf16 pieces (16 bits of the product; what is lost, 2^-17, is far below the copy's rounding), three
// (24 bits) where the last state is an output.
// Long sequences of few heads: `per` tiles a CTA may begin within a sequence.  linear_chunks_kernel<..., PIECE> first leaves every CTA's
// share of the state of the sequence that goes on behind it, linear_carry_kernel adds the shares up in order.
#pragma once
#include "linear_steps.cuh"
#include "umma_gemm.cuh"

namespace lact {

struct LinearPiece {
  int32_t goes_on;    // the CTA's last sequence goes on in the next CTA
  int32_t inherits;   // ... and began before this one
  int32_t state;      // its state's index (sequence * heads + head)
  float mult;         // what the state before these tokens is multiplied with
};

struct LinearChunkArgs {
  LinearArgs a;
  CUtensorMap x, y, z;   // 4-D maps (feature, token, head, entry), box {64, 128, 1, 1}
  int64_t per;           // tiles a CTA takes; packed sequences: 0, as many as make the CTAs even
  float* slots;          // [CTA] states: what the next CTA's sequence begins with ([A][B], or [B][A] if slots_t)
  LinearPiece* pieces;   // [CTA]
  int32_t slots_t;
  int32_t* status;
};

template <int A, int B>
struct LinearSmem {
  static constexpr int kStages = A == 128 ? 2 : B == 128 ? 3 : 4;
  static constexpr uint32_t kXY = 128 * A * 2, kZ = 128 * B * 2, kStage = 2 * kXY + kZ;   // X, Y, Z of one tile
  static constexpr uint32_t kS = kStages * kStage;                                         // copy of S, third piece of Y
  static constexpr uint32_t kBars = kS + kXY;
  static constexpr uint32_t kBytes = kBars + 256;
};

// The tiles of a launch in order: sequence, head, tile (backwards in time: from the last).
struct LinearTiles {
  int n, head, c, tiles;   // sequence, head, tile of the sequence in the order of the walk, its number of tiles
  LinearSpan s;
  static __device__ __forceinline__ int tiles_of(int len) { return (len + 127) >> 7; }
  // all tiles; every lane of a warp takes part
  static __device__ __forceinline__ int64_t total(const LinearArgs& a) {
    if (a.cu == nullptr) return static_cast<int64_t>(a.sequences) * a.heads * tiles_of(a.L);
    int64_t sum = 0;
    for (int n = threadIdx.x & 31; n < a.sequences; n += 32) sum += tiles_of(linear_span(a, n).len);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    return sum * a.heads;
  }
  // tile number f (< total); every lane of a warp takes part
  __device__ __forceinline__ void seek(const LinearArgs& a, int64_t f) {
    if (a.cu == nullptr) {
      tiles = tiles_of(a.L);
      c = static_cast<int>(f % tiles);
      f /= tiles;
      head = static_cast<int>(f % a.heads);
      n = static_cast<int>(f / a.heads);
      s = linear_span(a, n);
      return;
    }
    const int lane = threadIdx.x & 31;
    for (int n0 = 0;; n0 += 32) {
      const int mine = n0 + lane < a.sequences ? tiles_of(linear_span(a, n0 + lane).len) : 0;
      int upto = mine;   // tiles of one head (fewer than 2^24 + 2^24 in all)
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
        if (lane >= o) upto += v;
      }
      const uint32_t past = __ballot_sync(0xFFFFFFFFu, static_cast<int64_t>(upto) * a.heads > f);
      if (past != 0) {
        const int w = __ffs(past) - 1;
        n = n0 + w;
        tiles = __shfl_sync(0xFFFFFFFFu, mine, w);
        f -= static_cast<int64_t>(__shfl_sync(0xFFFFFFFFu, upto, w) - tiles) * a.heads;
        break;
      }
      f -= static_cast<int64_t>(__shfl_sync(0xFFFFFFFFu, upto, 31)) * a.heads;
      if (n0 + 32 >= a.sequences) {   // (f is not below the total: cannot be)
        n = a.sequences - 1;
        tiles = 1;
        f = 0;
        break;
      }
    }
    head = static_cast<int>(f / tiles);
    c = static_cast<int>(f % tiles);
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
  __device__ __forceinline__ int place(const LinearArgs& a) const { return (a.reverse ? tiles - 1 - c : c) * 128; }  // first token
  __device__ __forceinline__ int valid(int place) const { return min(128, s.len - place); }
  // backwards in time the state before the first token (the gradient of the last state) is not decayed by it
  __device__ __forceinline__ int first_decay(const LinearArgs& a) const { return a.reverse && c == 0 ? 0 : 1; }
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

constexpr int kLinearRowWarps = 8, kLinearStateWarps = 8;
constexpr int kLinearThreads = 64 + 32 * (kLinearRowWarps + kLinearStateWarps);

template <int A, int B, bool PIECE>
__global__ void __launch_bounds__(kLinearThreads, 1) linear_chunks_kernel(const __grid_constant__ LinearChunkArgs args) {
  static_assert((A == 64 || A == 128) && (B == 64 || B == 128), "64 or 128 features");
  using SM = LinearSmem<A, B>;
  constexpr int NS = SM::kStages;
  constexpr uint32_t kBox = 128 * 128;       // [128 rows][64 features] box of a tile
  constexpr uint32_t kSBox = B * 128;        // [B rows][64 columns] box of the copy of S
  constexpr uint32_t kTmemCols = 512, kG = 128, kO = 256, kOx = 384;   // S at 0, G and P, P Z, X S
  extern __shared__ __align__(1024) uint8_t linear_smem[];
  const uint32_t base = smem_u32(linear_smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(linear_smem + SM::kBars);
  uint64_t* xy_full = bars;             // [NS]
  uint64_t* z_full = bars + 4;          // [NS]
  uint64_t* stage_empty = bars + 8;     // [NS]
  uint64_t* g_full = bars + 12;         // G is in tensor memory
  uint64_t* p_full = bars + 13;         // an arrival per row warp: P is there (and Z is clean)
  uint64_t* s_ready = bars + 14;        // an arrival per state warp: the copy of S is there, S is decayed
  uint64_t* x_done = bars + 15;         // X and the copy of S have been used
  uint64_t* o_full = bars + 16;         // both parts of the output are there
  uint64_t* o_empty = bars + 17;        // an arrival per row warp: they have been read
  uint64_t* y_ready = bars + 18;        // an arrival per state warp: the pieces of Y are there
  uint64_t* s_full = bars + 19;         // S has taken the tile in
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 20);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  const LinearArgs& a = args.a;

  const int warp = uniform_warp_index(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) { mbar_init(&xy_full[s], 1); mbar_init(&z_full[s], 1); mbar_init(&stage_empty[s], 1); }
    mbar_init(g_full, 1);
    mbar_init(p_full, kLinearRowWarps);
    mbar_init(s_ready, kLinearStateWarps);
    mbar_init(x_done, 1);
    mbar_init(o_full, 1);
    mbar_init(o_empty, kLinearRowWarps);
    mbar_init(y_ready, kLinearStateWarps);
    mbar_init(s_full, 1);
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

  // this CTA's tiles
  const int64_t total = LinearTiles::total(a);
  const int64_t per = args.per > 0 ? args.per : (total + gridDim.x - 1) / gridDim.x;
  const int64_t first = blockIdx.x * per, end = min(first + per, total);
  int count = end > first ? static_cast<int>(end - first) : 0;
  LinearTiles it;
  bool mid = false;       // the first tile goes on with a sequence that the CTA before this one has begun
  if (count > 0) {
    if (PIECE) {
      it.seek(a, end - 1);
      const bool goes_on = it.c + 1 < it.tiles;
      const int back = min(it.c, count - 1);   // tiles of the last one's sequence before it
      it.c -= back;
      mid = it.c > 0;
      if (threadIdx.x == 0) {
        // tokens of tiles c .. c + back: all whole, but for the first of a walk backwards
        const int tokens = (back + 1) * 128 - (a.reverse && !mid ? 128 - it.valid(it.place(a)) : 0);
        args.pieces[blockIdx.x] = {goes_on, mid, it.n * a.heads + it.head,
                                   exp2f(decay_log2(a, it.head) * static_cast<float>(tokens - 1 + it.first_decay(a)))};
      }
      count = goes_on ? back + 1 : 0;
    } else {
      it.seek(a, first);
      mid = it.c > 0;
    }
  } else if (PIECE && threadIdx.x == 0) {
    args.pieces[blockIdx.x] = {0, 0, 0, 0.f};
  }
  // (swizzled tiles need the alignment asked for above)
  bool failed = uniform(static_cast<uint32_t>(*reinterpret_cast<volatile int32_t*>(args.status))) != kStatusOk || (base & 1023u) != 0;
  const int pieces = !PIECE && a.s_out == nullptr ? 2 : 3;

  if (warp == 0) {
    const uint32_t leader = elect_leader();
    for (int t = 0; t < count && !failed; ++t, it.next(a)) {
      const int st = t % NS, row = it.s.first + it.place(a);
      const uint32_t dst = base + st * SM::kStage;
      if (t >= NS && !mbar_wait_warp(&stage_empty[st], (t / NS - 1) & 1, abort_flag)) { failed = true; break; }
      mbar_expect_tx_if(leader, &xy_full[st], PIECE ? SM::kXY : 2 * SM::kXY);
      for (int j = 0; j < A / 64; ++j) {
        if (!PIECE) tma_load_4d_if(leader, dst + j * kBox, &args.x, &xy_full[st], 64 * j, row, it.head / a.x_share, it.s.entry);
        tma_load_4d_if(leader, dst + SM::kXY + j * kBox, &args.y, &xy_full[st], 64 * j, row, it.head / a.y_share, it.s.entry);
      }
      mbar_expect_tx_if(leader, &z_full[st], SM::kZ);
      for (int j = 0; j < B / 64; ++j)
        tma_load_4d_if(leader, dst + 2 * SM::kXY + j * kBox, &args.z, &z_full[st], 64 * j, row, it.head / a.z_share, it.s.entry);
    }
  } else if (warp == 1) {
    const uint32_t leader = elect_leader();
    const uint32_t idesc_g = make_idesc_bf16(128, 128, 0, 0);   // X Y^T, both K-major
    const uint32_t idesc_ox = make_idesc_bf16(128, B, 0, 0);    // X S: the copy of S is [B][A], K-major
    const uint32_t idesc_o = make_idesc_bf16(128, B, 0, 1);     // P Z: P in tensor memory, Z MN-major
    const uint32_t idesc_s = make_idesc_bf16(128, A, 1, 1);     // Z^T Y, both MN-major (64 features: the upper lanes take what follows Z)
    const SmemDescBase desc(kBox);
    auto stage = [&](int64_t t) { return base + static_cast<uint32_t>(t % NS) * SM::kStage; };
    auto phase = [&](int64_t t) { return (t / NS) & 1; };
    auto issue_g = [&](int64_t t) {
      const uint32_t x = stage(t), y = x + SM::kXY;
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
      const uint32_t par = t & 1, x = stage(t), y = x + SM::kXY, z = y + SM::kXY, s = base + SM::kS;
      bool g_next = true;
      if (!PIECE) {
        if (!mbar_wait_warp(s_ready, par, abort_flag) || (t >= 1 && !mbar_wait_warp(o_empty, par ^ 1, abort_flag))) { failed = true; break; }
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < A / 64; ++kk)
#pragma unroll
          for (int k4 = 0; k4 < 4; ++k4)
            umma_bf16_if(leader, tmem + kOx, desc.at((x + kk * kBox + k4 * 32) >> 4), desc.at((s + kk * kSBox + k4 * 32) >> 4), idesc_ox,
                         (kk | k4) != 0);
        umma_commit_if(leader, x_done);
        if (!mbar_wait_warp(p_full, par, abort_flag) || !mbar_wait_warp(&z_full[t % NS], phase(t), abort_flag)) { failed = true; break; }
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < 8; ++k)
          umma_bf16_ta_if(leader, tmem + kO, tmem + kG + (k >> 1) * 32 + (k & 1) * 8, desc.at((z + k * 2048) >> 4), idesc_o, k != 0);
        umma_commit_if(leader, o_full);
        g_next = t + 1 < count;
        if (g_next && __all_sync(0xFFFFFFFFu, mbar_test(&xy_full[(t + 1) % NS], phase(t + 1)))) {
          issue_g(t + 1);
          g_next = false;
        }
      }
      if (!mbar_wait_warp(y_ready, par, abort_flag) || (PIECE && !mbar_wait_warp(&z_full[t % NS], phase(t), abort_flag))) { failed = true; break; }
      tc_fence_after();
      for (int p = 0; p < pieces; ++p) {
        const uint32_t yp = p == 0 ? y : p == 1 ? x : s;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          umma_bf16_if(leader, tmem, desc.at((z + k * 2048) >> 4), desc.at((yp + k * 2048) >> 4), idesc_s, 1);
      }
      umma_commit_if(leader, s_full);
      umma_commit_if(leader, &stage_empty[t % NS]);
      if (!PIECE && g_next) {
        if (!mbar_wait_warp(&xy_full[(t + 1) % NS], phase(t + 1), abort_flag)) { failed = true; break; }
        issue_g(t + 1);
      }
    }
  } else if (warp < 2 + kLinearRowWarps) {
    // ---------------- rows: two threads per row of the tile (tensor-memory lane), 64 columns of G and half of the output each
    if constexpr (!PIECE) {
      const int quarter = warp & 3, half = (warp - 2) >> 2, r = quarter * 32 + lane;
      const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
      const int tid = threadIdx.x - 64;
      linear_zero_rest<B>(a, static_cast<int64_t>(blockIdx.x) * 256 + tid, static_cast<int64_t>(gridDim.x) * 256);
      if (a.cu != nullptr && a.s_out != nullptr) {   // empty sequences keep their states
        for (int n = blockIdx.x; n < a.sequences; n += gridDim.x) {
          if (linear_span(a, n).len != 0) continue;
          const int64_t size = static_cast<int64_t>(a.heads) * (A * B), at = n * size;
          for (int64_t i = tid; i < size; i += 256) a.s_out[at + i] = a.s_in != nullptr ? a.s_in[at + i] : 0.f;
        }
      }
      int head = -1;
      float g2 = 0.f;
      for (int t = 0; t < count && !failed; ++t, it.next(a)) {
        const uint32_t par = t & 1;
        const int place = it.place(a), nv = it.valid(place);
        if (it.head != head) {
          head = it.head;
          g2 = decay_log2(a, head);
        }
        if (!mbar_wait_warp(g_full, par, abort_flag)) { failed = true; break; }
        tc_fence_after();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int cb = half * 2 + i, c0 = cb * 32;
          uint32_t w[16];
          if (a.reverse ? cb < quarter : cb > quarter) {
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = 0;
          } else {
            uint32_t bits[32];
            tmem_ld32(tmem + lane_off + kG + c0, bits);
            // exponents of columns j: |r - c0 - j| tokens
            const float step = a.reverse ? g2 : -g2, from = (a.reverse ? c0 - r : r - c0) * g2;
            const int lo = a.reverse ? r - c0 : 0, hi = a.reverse ? nv - 1 - c0 : r - c0;   // visible columns
            tmem_ld_wait();
            float p[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) p[j] = __uint_as_float(bits[j]) * exp2_ftz(fmaf(static_cast<float>(j), step, from));
            if (cb == quarter || hi < 31) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (j < lo || j > hi) p[j] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = pack_bf16x2(p[2 * j], p[2 * j + 1]);
          }
          __syncwarp();
          tmem_st16(tmem + lane_off + kG + c0, w);
        }
        if (nv < 128 && a.cu != nullptr) {   // rows of the next sequence: no part of any sum
          const int st = t % NS;
          if (!mbar_wait_warp(&z_full[st], (t / NS) & 1, abort_flag)) { failed = true; break; }
          const uint32_t z = base + st * SM::kStage + 2 * SM::kXY;
          for (int i = tid; i < (128 - nv) * (B / 8); i += 256) {
            const int row = nv + i / (B / 8), u = i % (B / 8);
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(z + (u >> 3) * kBox + row * 128 + (u & 7) * 16), "r"(0) : "memory");
          }
          fence_async_proxy();
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full);

        const int pos = a.reverse ? nv - 1 - r : r;
        const float since = exp2f(g2 * static_cast<float>(max(pos, 0) + it.first_decay(a)));
        if (!mbar_wait_warp(o_full, par, abort_flag)) { failed = true; break; }
        tc_fence_after();
        const int64_t o = ((it.s.entry * static_cast<int64_t>(a.L) + it.s.first + place + r) * a.heads + head) * B + half * (B / 2);
#pragma unroll
        for (int c = 0; c < B / 2; c += 32) {
          uint32_t bi[32], bx[32];
          tmem_ld32(tmem + lane_off + kO + half * (B / 2) + c, bi);
          tmem_ld32(tmem + lane_off + kOx + half * (B / 2) + c, bx);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j)
            bi[j] = __float_as_uint(a.scale * fmaf(since, __uint_as_float(bx[j]), __uint_as_float(bi[j])));
          if (r < nv) {
            if (a.out_f32) {
              float* dst = static_cast<float*>(a.out) + o + c;
#pragma unroll
              for (int j = 0; j < 32; j += 8) st_global_32(dst + j, bi + j);
            } else {
              bf16* dst = static_cast<bf16*>(a.out) + o + c;
              uint32_t w[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) w[j] = pack_bf16x2(__uint_as_float(bi[2 * j]), __uint_as_float(bi[2 * j + 1]));
              st_global_32(dst, w);
              st_global_32(dst + 16, w + 8);
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
    // ---------------- state: lane = column of Z (B of them), two threads per lane, half of S's other side each
    const int quarter = warp & 3, half = (warp - 2 - kLinearRowWarps) >> 2;
    const int r = quarter * 32 + lane, tid = threadIdx.x - 64 - 32 * kLinearRowWarps;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const bool holds = quarter * 32 < B;    // (64 columns: the upper lanes of tensor memory are not part of S)
    constexpr int NC = A / 2;
    const int c0 = half * NC;
    int head = -1;
    float g2 = 0.f;
    // where element (row of A: c0 + j, column r) of state number `n` of an array lies
    auto element = [&](int64_t n, bool transposed, int j) {
      return n * (A * B) + (transposed ? static_cast<int64_t>(r) * A + c0 + j : static_cast<int64_t>(c0 + j) * B + r);
    };
    for (int t = 0; t < count && !failed; ++t, it.next(a)) {
      const uint32_t par = t & 1;
      const int st = t % NS, place = it.place(a), nv = it.valid(place);
      if (it.head != head) {
        head = it.head;
        g2 = decay_log2(a, head);
      }
      const int64_t state = static_cast<int64_t>(it.n) * a.heads + head;
      const float decay = exp2f(g2 * static_cast<float>(nv - 1 + it.first_decay(a)));
      if (t >= 1 && !mbar_wait_warp(s_full, par ^ 1, abort_flag)) { failed = true; break; }
      tc_fence_after();
      if (holds) {
        const float* from = PIECE ? nullptr : it.c == 0 ? a.s_in : mid && t == 0 ? args.slots : nullptr;
        const bool fresh = PIECE ? t == 0 : it.c == 0 || (mid && t == 0);
#pragma unroll
        for (int c = 0; c < NC; c += 32) {
          uint32_t v[32];
          if (!fresh) {
            tmem_ld32(tmem + lane_off + c0 + c, v);
            tmem_ld_wait();
          } else if (from == nullptr) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0;
          } else {
            const bool own = it.c == 0;   // the caller's state, or what the CTA before this one has left
            const float mul = own ? a.in_mul : 1.f;
            const int64_t n = own ? state : blockIdx.x - 1;
            const bool tr = own ? a.s_in_t : args.slots_t;
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(from[element(n, tr, c + j)] * mul);
          }
          if (!PIECE) {
            // (K-major, 128-byte swizzle: row r of 128-byte rows of 64 columns)
            const uint32_t row = base + SM::kS + ((c0 + c) >> 6) * kSBox + r * 128;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(__uint_as_float(v[g * 8 + 2 * e]), __uint_as_float(v[g * 8 + 2 * e + 1]));
              const uint32_t unit = (((c0 + c) & 63) >> 3) + g;
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row + ((unit ^ (r & 7)) << 4)), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                           "r"(w[3])
                           : "memory");
            }
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * decay);
          tmem_st32(tmem + lane_off + c0 + c, v);
        }
        tmem_st_wait();
      }
      if (!PIECE) {
        tc_fence_before();
        fence_async_proxy();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_ready);
      }
      // Y -> pieces: row j of the tile decays until the tile's end (in the order of the walk); two threads a row
      const int j = tid & 127, part = tid >> 7;
      const float f = exp2f(g2 * static_cast<float>(a.reverse ? j : nv - 1 - j));
      if (!mbar_wait_warp(&xy_full[st], (t / NS) & 1, abort_flag) || (!PIECE && !mbar_wait_warp(x_done, par, abort_flag))) {
        failed = true;
        break;
      }
      const uint32_t x = base + st * SM::kStage, y = x + SM::kXY, s = base + SM::kS;
#pragma unroll 4
      for (int i = 0; i < A / 16; ++i) {
        const int unit = part * (A / 16) + i;
        const uint32_t off = (unit >> 3) * kBox + j * 128 + (((unit & 7) ^ (j & 7)) << 4);
        uint4 u;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(y + off));
        float v[8];
        unpack_bf16x8(u, v);
        uint32_t w[3][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float p0 = j < nv ? v[2 * e] * f : 0.f, p1 = j < nv ? v[2 * e + 1] * f : 0.f;
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            w[k][e] = pack_bf16x2(p0, p1);
            p0 -= __uint_as_float(w[k][e] << 16);
            p1 -= __uint_as_float(w[k][e] & 0xFFFF0000u);
          }
        }
#pragma unroll
        for (int k = 0; k < 3; ++k)
          if (k < pieces)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"((k == 0 ? y : k == 1 ? x : s) + off), "r"(w[k][0]), "r"(w[k][1]),
                         "r"(w[k][2]), "r"(w[k][3])
                         : "memory");
      }
      if (PIECE && nv < 128 && a.cu != nullptr) {
        if (!mbar_wait_warp(&z_full[st], (t / NS) & 1, abort_flag)) { failed = true; break; }
        for (int i = tid; i < (128 - nv) * (B / 8); i += 256) {
          const int row = nv + i / (B / 8), u = i % (B / 8);
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(y + SM::kXY + (u >> 3) * kBox + row * 128 + (u & 7) * 16), "r"(0) : "memory");
        }
      }
      tc_fence_before();
      fence_async_proxy();
      __syncwarp();
      if (lane == 0) mbar_arrive(y_ready);
      // the state behind the sequence, or behind this CTA's part of it
      float* const to = PIECE ? (t + 1 == count ? args.slots : nullptr) : it.c + 1 == it.tiles ? a.s_out : nullptr;
      if (to != nullptr) {
        if (!mbar_wait_warp(s_full, par, abort_flag)) { failed = true; break; }
        tc_fence_after();
        if (holds) {
          const float mul = PIECE ? 1.f : a.out_mul * (a.reverse ? exp2f(g2) : 1.f);
          const int64_t n = PIECE ? blockIdx.x : state;
          const bool tr = PIECE ? args.slots_t : a.s_out_t;
#pragma unroll
          for (int c = 0; c < NC; c += 32) {
            uint32_t v[32];
            tmem_ld32(tmem + lane_off + c0 + c, v);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) to[element(n, tr, c + e)] = __uint_as_float(v[e]) * mul;
          }
        }
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

// What every CTA's first sequence begins with: slots[i] <- slots[i] + mult_i * (state before CTA i's part), in order of i.  One element
// of the state per thread; 16 shares are fetched at a time.
constexpr int kLinearMaxCtas = 256;
__global__ void __launch_bounds__(128) linear_carry_kernel(const float* __restrict__ s_in, int32_t s_in_t, float in_mul, float* slots,
                                                           const LinearPiece* __restrict__ pieces, int32_t ctas, int32_t A, int32_t B) {
  __shared__ LinearPiece info[kLinearMaxCtas];
  griddep_launch_dependents();
  griddep_wait();
  for (int i = threadIdx.x; i < ctas; i += 128) info[i] = pieces[i];
  __syncthreads();
  const int e = blockIdx.x * 128 + threadIdx.x, size = A * B;    // element (e / B, e % B)
  const int at = s_in_t ? (e % B) * A + e / B : e;
  float carry = 0.f;
  for (int i0 = 0; i0 + 1 < ctas; i0 += 16) {
    float mine[16], before[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int i = i0 + k;
      const bool on = i + 1 < ctas && info[i].goes_on;
      mine[k] = on ? slots[static_cast<int64_t>(i) * size + e] : 0.f;
      before[k] = on && !info[i].inherits && s_in != nullptr ? s_in[static_cast<int64_t>(info[i].state) * size + at] * in_mul : 0.f;
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int i = i0 + k;
      if (i + 1 >= ctas || !info[i].goes_on) continue;
      carry = fmaf(info[i].mult, info[i].inherits ? carry : before[k], mine[k]);
      slots[static_cast<int64_t>(i) * size + e] = carry;
    }
  }
}

}  // namespace lact

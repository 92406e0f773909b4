// Attention of one new token of every sequence over a paged cache (paged_cache.cuh):
//   o = sum_p w_p v_p / sum_p w_p,   w_p = 2^(x_p - m),  x_p = scale log2(e) q k_p,   p over the last `window` positions of the length.
// Bound by memory: the window's keys and values once; the g query heads of a kv head make 2 g flops of a byte of bf16, 4 g of 8 bits.
// Up to 8 (or 16) of them are the columns of m16n8k16 products with 16 tokens or 16 features as rows.  Those are warp products on
// registers, not tcgen05: fragments come straight from global memory, since the order of a product's inner axis is free (K: a lane's
// 32 bytes of a row are four (8 bits: eight) steps' pieces of that row; V: a lane holds the same features of four tokens, and byte
// permutes pair the tokens), so nothing passes through shared memory, and 16 tokens of 128 take 16 products while 8 KB arrive.
// The maximum m is raised only when a score passes it by 8 (weights up to 2^8 lose nothing), so that a step of 16 tokens needs one vote
// in place of a reduction.  Weights are rounded for the product with V: in two bf16 pieces (2^-17 of each) with bf16 caches, to fp16
// (2^-12) with 8 bits.  There, V is taken as e4m3, exact in fp16, and its powers of two multiply the weights: u_p = 2^(x_p + e_p - M)
// with a maximum M of its own, against which small weights are rounded by 2^-25.  Queries become fp16 after scaling each by a power of
// two, to a largest value of 2^14 (what is below 2^-38 of it is cut).  Sums are in fp32.
//
// Work: a unit is a (sequence, kv head, block of query heads), its tokens tiles of 16 a warp; lengths are known on the device alone.
// All units' tiles, in order, are dealt out in even runs, one for each CTA, whatever the lengths are.  A run that holds all of a unit
// writes its result; of a unit cut among runs each leaves a piece (sums, maxima), and the run that comes last adds the pieces in their
// order.  Where a unit has few tiles at most (`runs` 0), each CTA takes one unit.
#pragma once
#include "paged_cache.cuh"

namespace lact {

struct PagedStepArgs {
  PagedCache c;
  const bf16* q;                   // [sequences][heads][D], features adjacent, other strides in elements
  int64_t q_bs, q_hs;
  bf16* o;                         // contiguous
  int32_t heads, share, blocks;    // query heads; of a kv head; blocks of query heads of a kv head
  int32_t window;                  // 0: all
  float scale;                     // softmax scale * log2(e)
  int32_t runs, least;             // CTAs that share the tiles; tiles of a run at least
  uint32_t* counters;              // [runs], zero before and after
  float* pieces;                   // [runs][2][rows of a block][D + 4]
};

__device__ __forceinline__ void mma_16x8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, bool halves) {
  if (halves)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// An 8 x 8 matrix of 16-bit values turned over among the lanes of a warp
__device__ __forceinline__ uint32_t transposed_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// N words of a row of the cache, read once; zeros where `there` is false
template <int N>
__device__ __forceinline__ void load_cache(uint32_t (&w)[N], const uint8_t* p, bool there) {
  static_assert(N == 2 || N == 4 || N == 8);
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = 0;
  if (!there) return;
  if constexpr (N == 8)
    asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p));
  else if constexpr (N == 4)
    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
  else
    asm volatile("ld.global.nc.L1::no_allocate.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
}

// Tiles of a sequence (one at least: an empty sequence's zeros are a unit's result, too)
struct PagedSpan {
  int first, last;   // positions [first, last)
  int tiles;
};
template <int TILE>
__device__ __forceinline__ PagedSpan paged_span(const PagedStepArgs& a, int seq) {
  PagedSpan s;
  const int64_t room = static_cast<int64_t>(a.c.cols) << a.c.shift;
  const int len = max(a.c.lengths[seq], 0);
  s.last = static_cast<int>(min(static_cast<int64_t>(len), room));
  s.first = a.window > 0 ? max(len - a.window, 0) : 0;
  s.first = min(s.first, s.last);
  s.tiles = max((s.last - (s.first & ~15) + TILE - 1) / TILE, 1);
  return s;
}

constexpr float kLowest = -3.402823466e38f;
__host__ __device__ constexpr int kPagedPieceRow(int D) { return D + 4; }   // sums, then m, l, M

template <int D, bool E4, int NQ, int W, int PER_SM>
__global__ void __launch_bounds__(W * 32, PER_SM) paged_step_kernel(const __grid_constant__ PagedStepArgs a) {
  constexpr int ROWS = 8 * NQ, TILE = 16 * W, ROW = kPagedPieceRow(D), THREADS = W * 32;
  constexpr int BYTES = E4 ? D : 2 * D;                  // of a row
  constexpr int KL = BYTES >= 128 ? 32 : 16;             // bytes of a K row that a lane loads at a time
  constexpr int KN = BYTES / (4 * KL);                   // times
  constexpr int KW = KL / 4;                             // words of one
  constexpr int VW = BYTES / 32;                         // words of a V row that a lane holds
  constexpr int MT = D / 16;                             // products of 16 features
  constexpr int QW = D / 8;                              // words of a lane's queries: two a step of 16 features
  extern __shared__ __align__(16) float paged_smem[];    // [W][ROWS][ROW]
  __shared__ int plan[4];
  __shared__ int64_t warp_sum[W];
  __shared__ uint32_t arrived;
  griddep_launch_dependents();
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int units = a.c.heads * a.blocks;                // of a sequence
  // -------- this CTA's run
  int seq, unit, t0, left;                               // first unit, its first tile of the run, tiles of the run
  int64_t run0 = 0, per = 0;
  if (a.runs == 0) {
    seq = blockIdx.x / units;
    unit = blockIdx.x - seq * units;
    t0 = 0;
    left = paged_span<TILE>(a, seq).tiles;
  } else {
    const int chunk = (a.c.sequences + THREADS - 1) / THREADS, s0 = min(static_cast<int>(threadIdx.x) * chunk, a.c.sequences), s1 = min(s0 + chunk, a.c.sequences);
    int64_t mine = 0;
    for (int s = s0; s < s1; ++s) mine += paged_span<TILE>(a, s).tiles;
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xFFFFFFFFu, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) warp_sum[warp] = upto;
    __syncthreads();
    int64_t all = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w == warp) upto += all;
      all += warp_sum[w];
    }
    all *= units;
    per = max((all + a.runs - 1) / a.runs, static_cast<int64_t>(a.least));
    run0 = blockIdx.x * per;
    if (run0 >= all) return;
    left = static_cast<int>(min(per, all - run0));
    int64_t at = (upto - mine) * units;
    if (run0 >= at && run0 < upto * units) {
      for (int s = s0; s < s1; ++s) {
        const int64_t n = paged_span<TILE>(a, s).tiles;
        if (run0 < at + n * units) {
          plan[0] = s;
          plan[1] = static_cast<int>((run0 - at) / n);
          plan[2] = static_cast<int>((run0 - at) % n);
          break;
        }
        at += n * units;
      }
    }
    __syncthreads();
    seq = plan[0];
    unit = plan[1];
    t0 = plan[2];
  }
  // -------- its units
  for (int64_t done = 0; left > 0; ++unit) {
    if (unit == units) {
      unit = 0;
      ++seq;
    }
    const PagedSpan span = paged_span<TILE>(a, seq);
    const int head = unit / a.blocks, row0 = (unit - head * a.blocks) * ROWS, rows = min(a.share - row0, ROWS);
    const int t1 = min(span.tiles, t0 + left), base = span.first & ~15;
    if (threadIdx.x == 0 && a.c.lengths[seq] > span.last && t1 == span.tiles) report_bad_page();
    // queries: column r of a product is query head row0 + r (+ 8)
    uint32_t q[NQ][QW];
    float qm[NQ][2];                                     // what scores of columns 2 c, 2 c + 1 are multiplied by
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const bool on = n * 8 + r < rows;
      const bf16* from = a.q + seq * a.q_bs + (static_cast<int64_t>(head) * a.share + row0 + n * 8 + r) * a.q_hs;
      if constexpr (!E4) {
#pragma unroll
        for (int i = 0; i < KN; ++i)
#pragma unroll
          for (int e = 0; e < KW; e += 4) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (on) w = *reinterpret_cast<const uint4*>(from + (i * 4 + c) * (KL / 2) + e * 2);
            q[n][i * KW + e] = w.x; q[n][i * KW + e + 1] = w.y; q[n][i * KW + e + 2] = w.z; q[n][i * KW + e + 3] = w.w;
          }
        qm[n][0] = qm[n][1] = a.scale;
      } else {
        uint32_t raw[QW], top = 0;
#pragma unroll
        for (int i = 0; i < KN; ++i)
#pragma unroll
          for (int e = 0; e < 2 * KW; e += 4) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (on) w = *reinterpret_cast<const uint4*>(from + (i * 4 + c) * KL + e * 2);
            uint32_t* const to = raw + i * 2 * KW + e;
            to[0] = w.x; to[1] = w.y; to[2] = w.z; to[3] = w.w;
          }
#pragma unroll
        for (int i = 0; i < QW; ++i) top = __vmaxu2(top, raw[i] & 0x7FFF7FFFu);
        top = max(top & 0xFFFFu, top >> 16);
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
        // the largest becomes 2^14 to 2^15 (not from below 2^-86); of an infinity or a NaN what it is
        const int e = min(max(static_cast<int>(top >> 7), 41), 254);
        const float up = __uint_as_float(static_cast<uint32_t>(127 + 141 - e) << 23), down = a.scale * __uint_as_float(static_cast<uint32_t>(e - 14) << 23);
#pragma unroll
        for (int i = 0; i < QW; ++i) {
          const __half2 h = __floats2half2_rn(__uint_as_float(raw[i] << 16) * up, __uint_as_float(raw[i] & 0xFFFF0000u) * up);
          q[n][i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        qm[n][0] = __shfl_sync(0xFFFFFFFFu, down, c * 8);
        qm[n][1] = __shfl_sync(0xFFFFFFFFu, down, c * 8 + 4);
      }
    }
    // -------- tiles: this warp's 16 tokens of each
    float acc[NQ][MT][4], m[NQ][2], l[NQ][2];
    [[maybe_unused]] float M[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][j][e] = 0.f;
      m[n][0] = m[n][1] = M[n][0] = M[n][1] = kLowest;
      l[n][0] = l[n][1] = 0.f;
    }
    const int32_t* const table = a.c.table + seq * a.c.table_rs;
    const uint8_t* const kh = a.c.k + (static_cast<int64_t>(head) << a.c.shift) * BYTES;
    const uint8_t* const vh = a.c.v + (static_cast<int64_t>(head) << a.c.shift) * BYTES;
    auto position = [&](int t) { return base + (t * W + warp) * 16; };
    // (a step of 16 tokens lies in one page; past the end none is looked up)
    auto page_of = [&](int t) { return t < t1 && position(t) < span.last ? table[position(t) >> a.c.shift] : -2; };
    uint32_t kr[2][KN][KW], vr[4][VW];
    [[maybe_unused]] uint32_t ke[2], ve[2];
    auto load_k = [&](int t, int page) {
      const int p = position(t), row = p & ((1 << a.c.shift) - 1);
      const bool there = page >= 0 && page < a.c.pages;
      if (!there && page != -2 && lane == 0) report_bad_page();
      const uint8_t* const from = kh + page * a.c.k_ps + static_cast<int64_t>(row) * BYTES;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool on = there && p + r + 8 * h >= span.first && p + r + 8 * h < span.last;
#pragma unroll
        for (int i = 0; i < KN; ++i) load_cache<KW>(kr[h][i], from + (r + 8 * h) * BYTES + (i * 4 + c) * KL, on);
        if constexpr (E4) {
          const int64_t at = (static_cast<int64_t>(head) << a.c.shift) + row + r + 8 * h;
          ke[h] = on ? a.c.ke[page * a.c.ke_ps + at] : 127u;
          ve[h] = on ? a.c.ve[page * a.c.ve_ps + at] : 127u;
        }
      }
    };
    auto load_v = [&](int t, int page) {
      const int p = position(t), row = p & ((1 << a.c.shift) - 1);
      const bool there = page >= 0 && page < a.c.pages;
      const uint8_t* const from = vh + page * a.c.v_ps + static_cast<int64_t>(row) * BYTES;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tok = 2 * c + (i & 1) + 8 * (i >> 1);
        load_cache<VW>(vr[i], from + tok * BYTES + r * (VW * 4), there && p + tok >= span.first && p + tok < span.last);
      }
    };
    int page = page_of(t0), next = page_of(t0 + 1);
    load_k(t0, page);
    load_v(t0, page);
    for (int t = t0; t < t1; ++t) {
      float x[NQ][4];
#pragma unroll
      for (int n = 0; n < NQ; ++n) x[n][0] = x[n][1] = x[n][2] = x[n][3] = 0.f;
#pragma unroll
      for (int i = 0; i < KN; ++i)
#pragma unroll
        for (int e = 0; e < KW; e += E4 ? 1 : 2) {
          uint32_t a0, a1, a2, a3;
          if constexpr (E4) {
            a0 = halves_of_e4m3(kr[0][i][e] & 0xFFFFu); a1 = halves_of_e4m3(kr[1][i][e] & 0xFFFFu);
            a2 = halves_of_e4m3(kr[0][i][e] >> 16); a3 = halves_of_e4m3(kr[1][i][e] >> 16);
          } else {
            a0 = kr[0][i][e]; a1 = kr[1][i][e]; a2 = kr[0][i][e + 1]; a3 = kr[1][i][e + 1];
          }
          const int s = E4 ? 2 * (i * KW + e) : i * KW + e;
#pragma unroll
          for (int n = 0; n < NQ; ++n) mma_16x8(x[n], a0, a1, a2, a3, q[n][s], q[n][s + 1], E4);
        }
      [[maybe_unused]] float kx[2], vx[2];
      if constexpr (E4)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          kx[h] = exponent_value(ke[h]);
          vx[h] = ve[h] == 255 ? __uint_as_float(0x7FC00000u) : static_cast<float>(static_cast<int>(ve[h]) - 127);
        }
      const int p = position(t);
      const bool there = page >= 0 && page < a.c.pages;
      const bool on[2] = {there && p + r >= span.first && p + r < span.last, there && p + r + 8 >= span.first && p + r + 8 < span.last};
      page = next;
      if (t + 1 < t1) {
        next = page_of(t + 2);
        load_k(t + 1, page);
      }
      // scores; the maxima, where one passes them by 8
      bool raise = false;
      [[maybe_unused]] float y[NQ][4];
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[n][e] *= qm[n][e & 1];
          if constexpr (E4) x[n][e] *= kx[e >> 1];
          if (!on[e >> 1]) x[n][e] = -INFINITY;
          raise = raise || x[n][e] > m[n][e & 1] + 8.f;
          if constexpr (E4) {
            y[n][e] = x[n][e] + vx[e >> 1];
            raise = raise || y[n][e] > M[n][e & 1] + 8.f;
          }
        }
      if (__any_sync(0xFFFFFFFFu, raise)) {
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            auto top = [&](float old, float u, float v) {
              float z = fmaxf(u, v);
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) z = fmaxf(z, __shfl_xor_sync(0xFFFFFFFFu, z, o));
              return fmaxf(old, z);
            };
            const float now = top(m[n][e], x[n][e], x[n][e + 2]);
            float f = exp2_ftz(m[n][e] - now);
            l[n][e] *= f;
            m[n][e] = now;
            if constexpr (E4) {
              const float big = top(M[n][e], y[n][e], y[n][e + 2]);
              f = exp2_ftz(M[n][e] - big);
              M[n][e] = big;
            }
#pragma unroll
            for (int j = 0; j < MT; ++j) {
              acc[n][j][e] *= f;
              acc[n][j][e + 2] *= f;
            }
          }
      }
      // weights, turned over so that their tokens are the inner axis
      uint32_t hi[NQ][2];
      [[maybe_unused]] uint32_t lo[NQ][2];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = exp2_ftz(x[n][e] - m[n][e & 1]);
          l[n][e & 1] += w[e];
          if constexpr (E4) w[e] = exp2_ftz(y[n][e] - M[n][e & 1]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if constexpr (E4) {
            const __half2 two = __floats2half2_rn(w[2 * h], w[2 * h + 1]);
            hi[n][h] = transposed_8x8(*reinterpret_cast<const uint32_t*>(&two));
          } else {
            const uint32_t two = pack_bf16x2(w[2 * h], w[2 * h + 1]);
            lo[n][h] = transposed_8x8(pack_bf16x2(w[2 * h] - __uint_as_float(two << 16), w[2 * h + 1] - __uint_as_float(two & 0xFFFF0000u)));
            hi[n][h] = transposed_8x8(two);
          }
        }
      }
      if constexpr (E4) {
#pragma unroll
        for (int j = 0; j < MT; j += 2) {
          const uint32_t t01 = __byte_perm(vr[0][j / 2], vr[1][j / 2], 0x5140), u01 = __byte_perm(vr[0][j / 2], vr[1][j / 2], 0x7362);
          const uint32_t t23 = __byte_perm(vr[2][j / 2], vr[3][j / 2], 0x5140), u23 = __byte_perm(vr[2][j / 2], vr[3][j / 2], 0x7362);
          const uint32_t a0 = halves_of_e4m3(t01 & 0xFFFFu), a1 = halves_of_e4m3(t01 >> 16), a2 = halves_of_e4m3(t23 & 0xFFFFu), a3 = halves_of_e4m3(t23 >> 16);
          const uint32_t b0 = halves_of_e4m3(u01 & 0xFFFFu), b1 = halves_of_e4m3(u01 >> 16), b2 = halves_of_e4m3(u23 & 0xFFFFu), b3 = halves_of_e4m3(u23 >> 16);
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            mma_16x8(acc[n][j], a0, a1, a2, a3, hi[n][0], hi[n][1], true);
            mma_16x8(acc[n][j + 1], b0, b1, b2, b3, hi[n][0], hi[n][1], true);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          const uint32_t a0 = __byte_perm(vr[0][j], vr[1][j], 0x5410), a1 = __byte_perm(vr[0][j], vr[1][j], 0x7632);
          const uint32_t a2 = __byte_perm(vr[2][j], vr[3][j], 0x5410), a3 = __byte_perm(vr[2][j], vr[3][j], 0x7632);
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            mma_16x8(acc[n][j], a0, a1, a2, a3, hi[n][0], hi[n][1], false);
            mma_16x8(acc[n][j], a0, a1, a2, a3, lo[n][0], lo[n][1], false);
          }
        }
      }
      if (t + 1 < t1) load_v(t + 1, page);
    }
    // -------- the warps' sums: a lane holds features 16 j.. of r for columns 2 c, 2 c + 1
    float* const mine = paged_smem + warp * ROWS * ROW;
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[n][e] += __shfl_xor_sync(0xFFFFFFFFu, l[n][e], o);
        const int row = n * 8 + 2 * c + e;
        if (row >= rows) continue;
        float* const to = mine + row * ROW;
#pragma unroll
        for (int j = 0; j < MT; j += 2)
          *reinterpret_cast<float4*>(to + r * (D / 8) + 2 * j) = make_float4(acc[n][j][e], acc[n][j][e + 2], acc[n][j + 1][e], acc[n][j + 1][e + 2]);
        if (r == 0) *reinterpret_cast<float4*>(to + D) = make_float4(m[n][e], l[n][e], E4 ? M[n][e] : m[n][e], 0.f);
      }
    __syncthreads();
    const bool whole = t1 == span.tiles && t0 == 0;
    const int64_t begin = run0 + done - t0;               // the unit's first tile among all
    float* const piece = whole ? nullptr : a.pieces + (static_cast<int64_t>(blockIdx.x) * 2 + (t0 == 0 ? 1 : 0)) * ROWS * ROW;
    bf16* const o = a.o + (static_cast<int64_t>(seq) * a.heads + static_cast<int64_t>(head) * a.share + row0) * D;
    for (int i = threadIdx.x; i < rows * D; i += THREADS) {
      const int row = i / D, d = i % D;
      const float* const from = paged_smem + row * ROW;
      float tm = kLowest, tM = kLowest, sum = 0.f, tl = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        tm = fmaxf(tm, from[w * ROWS * ROW + D]);
        tM = fmaxf(tM, from[w * ROWS * ROW + D + 2]);
      }
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float* const f = from + w * ROWS * ROW;
        sum += f[d] * exp2_ftz(f[D + 2] - tM);
        tl += f[D + 1] * exp2_ftz(f[D] - tm);
      }
      if (whole) {
        o[i] = __float2bfloat16_rn(span.last > span.first ? sum * (exp2_ftz(tM - tm) / tl) : 0.f);
      } else {
        piece[row * ROW + d] = sum;
        if (d < 3) piece[row * ROW + D + d] = d == 0 ? tm : d == 1 ? tl : tM;
      }
    }
    if (!whole) {
      // the run that leaves the last of the unit's pieces adds them up
      const int first_run = static_cast<int>(begin / per), last_run = static_cast<int>((begin + span.tiles - 1) / per);
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        const uint32_t before = atomicAdd(a.counters + first_run, 1u);
        arrived = before;
        if (before == static_cast<uint32_t>(last_run - first_run)) a.counters[first_run] = 0;
      }
      __syncthreads();
      if (arrived == static_cast<uint32_t>(last_run - first_run)) {
        __threadfence();
        for (int i = threadIdx.x; i < rows * D; i += THREADS) {
          const int row = i / D, d = i % D;
          auto of = [&](int run) { return a.pieces + (static_cast<int64_t>(run) * 2 + (run == first_run ? 1 : 0)) * ROWS * ROW + row * ROW; };
          float tm = kLowest, tM = kLowest, sum = 0.f, tl = 0.f;
          for (int run = first_run; run <= last_run; ++run) {
            tm = fmaxf(tm, __ldcg(of(run) + D));
            tM = fmaxf(tM, __ldcg(of(run) + D + 2));
          }
          for (int run = first_run; run <= last_run; ++run) {
            const float* const f = of(run);
            sum += __ldcg(f + d) * exp2_ftz(__ldcg(f + D + 2) - tM);
            tl += __ldcg(f + D + 1) * exp2_ftz(__ldcg(f + D) - tm);
          }
          o[i] = __float2bfloat16_rn(sum * (exp2_ftz(tM - tm) / tl));
        }
      }
    }
    __syncthreads();
    done += t1 - t0;
    left -= t1 - t0;
    t0 = 0;
  }
}

}  // namespace lact

// Attention of one new token of every sequence over a paged cache (paged_cache.cuh):
//   o = sum_p w_p v_p / sum_p w_p,   w_p = 2^(x_p - m),  x_p = scale log2(e) q k_p,   p over the last `window` positions of the length.
// Bound by memory: the window's keys and values once; the g query heads of a kv head make 2 g flops of a byte of bf16, 4 g of 8 bits.
// Up to 8 (or 16) of them are the columns of m16n8k16 products with 16 tokens or 16 features as rows.  Those are warp products on
// registers, not tcgen05, whose 128 rows are more tokens than a step has, and whose second product would want V turned over and the
// weights written to tensor memory before it can begin: here a warp goes on by itself, and 16 tokens of 128 features take 24 products
// while their 8 KB arrive (tensor pipe 15 to 17 % busy).  The order of a product's inner axis is free, so that no fragment is turned
// over: of K a lane has 32 bytes of a row, four (8 bits: eight) steps' pieces of it; of V the same features of four tokens, which byte
// permutes pair.
// The maximum m is raised only when a score passes it by 8 (weights up to 2^8 lose nothing), so that a step needs one vote in place of a
// reduction.  Weights are rounded for the product with V: in two bf16 pieces (2^-16 of each) with bf16 caches, to fp16 (2^-11) with 8
// bits.  (A second piece there could bring results from 1.68e-3 off 64 bits to the 1.66e-3 of their own rounding, and takes 198 us in place of
// 192 with 64 sequences of up to 16384 tokens, 58 in place of 52 with 40 heads on one.)  V is then taken as e4m3, exact in fp16, and its
// powers of two multiply the weights: u_p = 2^(x_p + e_p - M) with a maximum M of its own, against which a warp's small weights are rounded
// by 2^-25.  Queries become fp16 after scaling each by a power of two, to a largest value of 2^14 (what is below 2^-38 of it is cut).
// Sums are in fp32.
//
// Loads: every warp keeps a ring of steps of its own in shared memory (16 tokens of rows of 256 bytes, 32 of 128, 64 of 64), filled by tiled copies
// with a swizzle that both kinds of fragment read without conflicts; a step's page number is looked up one step ahead.  A step is in
// registers before its slot is filled again.  96 KB on their way in a SM is what bandwidth gains from (12 warps with one step of 8 KB; two
// steps: step_window 170 in place of 162 us, step_long 103 and 100): longer runs use no more slots than that (with more than 8 query heads a kv
// head, of which 8 warps are on a SM, that is 64 KB: 16 heads 84 % in bf16).
//
// Work: a unit is a (sequence, kv head, block of query heads), its tokens tiles of one step a warp; lengths are known on the device alone.
// All units' tiles, in order, are dealt out in even runs, one for each CTA, whatever the lengths are (more runs than fit at once: two for
// each place step_long 109 in place of 106 us, step_window 173 and 165).  A run that holds all of a unit writes its result; of a unit
// cut among runs each leaves a piece (sums, maxima), and a small launch adds the pieces in a fixed order.  Where units are few and have few
// tiles at most, or have very few (`runs` 0), a unit is a cluster of CTAs that share its tiles evenly and read one another's sums from
// shared memory.
// Measured (of the measured copy rate; from one GPU to another): 4 sequences of up to 131072 tokens, 16 heads on 4 of 128, bf16 94 to 96 us (94 %); 64 of
// up to 16384, 32 on 8 of 128, 8 bits 185 to 193 us (92 to 95 %); 192 of up to 5000, a window of 2048, 12 heads of 64 156 to 160 us (96 to 98 %); one
// of 777, 12 heads 6.4 to 7.2 us.  Less near it: 82 of up to 4000, 12 heads of 64 in 8 bits 59 us (70 %); 64 of up to 8192, 64 heads on 4 of 128
// 105 us (84 %), in 8 bits 70 (64 %); 80 on 4 181 (the cache is read twice: 49 %); 40 on 1 in 8 bits 52 (read three times: 22 %).
#pragma once
#include "paged_cache.cuh"

namespace lact {

constexpr int kPagedStages = 8;   // slots of a warp at most
constexpr int kPagedLong = 8;     // tiles up to which a run uses them all
struct PagedStepArgs {
  PagedCache c;
  const bf16* q;                   // [sequences][heads][D], features adjacent, other strides in elements
  int64_t q_bs, q_hs;
  bf16* o;                         // contiguous
  int32_t heads, share, blocks;    // query heads; of a kv head; blocks of query heads of a kv head
  int32_t window;                  // 0: all
  float scale;                     // softmax scale * log2(e)
  int32_t runs, least;             // CTAs that share the tiles; tiles of a run at least
  int32_t cluster;                 // runs 0: CTAs of a unit (1, 2, 4 or 8)
  struct PagedCut* cuts;           // [runs]
  float* pieces;                   // [runs][2][min(share, rows of a block)][D + 4]: of the unit that a run begins in, of one that begins in it
  int32_t* status;
  int32_t stages, long_stages;     // steps that a warp has on their way or in work; the same in runs of more tiles than kPagedLong
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
// Tiles of a sequence (one at least: an empty sequence's zeros are a unit's result, too).  The first begins with the step that the window begins
// in, or, where a step is several pages, with the page: pages in front of it may have been given back.
struct PagedSpan {
  int first, last;   // positions [first, last)
  int base;          // where the first tile begins
  int tiles;
  bool over;         // the length is past the table's end
};
template <int STEP, int TILE>
__device__ __forceinline__ PagedSpan paged_span(const PagedStepArgs& a, int seq) {
  PagedSpan s;
  const int64_t room = static_cast<int64_t>(a.c.cols) << a.c.shift;
  const int len = max(a.c.lengths[seq], 0);
  s.last = static_cast<int>(min(static_cast<int64_t>(len), room));
  s.over = len > room;
  s.first = a.window > 0 ? max(len - a.window, 0) : 0;
  s.first = min(s.first, s.last);
  s.base = s.first & -min(STEP, 1 << a.c.shift);
  s.tiles = max((s.last - s.base + TILE - 1) / TILE, 1);
  return s;
}

constexpr float kLowest = -3.402823466e38f;
__host__ __device__ constexpr int kPagedPieceRow(int D) { return D + 4; }   // sums, then m, l, M

// An untiled copy (both addresses on 16 bytes, a multiple of 16 bytes)
__device__ __forceinline__ void bulk_load_if(uint32_t leader, uint32_t smem_dst, const void* from, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %4, 0;\n\t"
      "@q cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n\t}" ::"r"(smem_dst),
      "l"(reinterpret_cast<uint64_t>(from)), "r"(bytes), "r"(bar), "r"(leader)
      : "memory");
}
__device__ __forceinline__ uint4 ld_shared_16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ uint2 ld_shared_8(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
  return v;
}

// Where a walk over a run's tiles is.
struct PagedWalk {
  int seq, unit, t, t1, left;      // left: tiles of the run from this unit's first on
  int head, first, last, base, tiles;
  bool over;                       // the length is past the table's end
  const int32_t* table;
};

__device__ __forceinline__ float4 ld_cluster_16(uint32_t at, uint32_t rank) {
  float4 v;
  asm volatile(
      "{\n\t.reg .b32 p;\n\tmapa.shared::cluster.u32 p, %4, %5;\n\tld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [p];\n\t}"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
      : "r"(at), "r"(rank)
      : "memory");
  return v;
}
// The sums of W warps in `sums` ([W][sum_rows][ROW]: D features, then m, l, M), added up for four features of a row at a time:
// put(row, d, sum, float4(m, l, M, 0)).
template <int D, int W, int ROW, class Put>
__device__ __forceinline__ void paged_merge(const float* sums, int sum_rows, int rows, const Put& put) {
  for (int i = threadIdx.x; i < rows * (D / 4); i += W * 32) {
    const int row = i / (D / 4), d = i % (D / 4) * 4;
    float4 s[W], sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float tm = kLowest, tM = kLowest, tl = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      s[w] = *reinterpret_cast<const float4*>(sums + (w * sum_rows + row) * ROW + D);
      tm = fmaxf(tm, s[w].x);
      tM = fmaxf(tM, s[w].z);
    }
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float4 x = *reinterpret_cast<const float4*>(sums + (w * sum_rows + row) * ROW + d);
      const float by = exp2_ftz(s[w].z - tM);
      sum.x += x.x * by; sum.y += x.y * by; sum.z += x.z * by; sum.w += x.w * by;
      tl += s[w].y * exp2_ftz(s[w].x - tm);
    }
    put(row, d, sum, make_float4(tm, tl, tM, 0.f));
  }
}
__device__ __forceinline__ void store_bf16x4(bf16* to, const float4& x, float by) {
  *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(x.x * by, x.y * by), pack_bf16x2(x.z * by, x.w * by));
}

// The sums of a cluster's CTAs, each added up in `mine` ([rows][ROW]), as the unit's result.
template <int D, int W, int ROW>
__device__ __forceinline__ void paged_join_cluster(int ctas, const float* mine, int rows, bool any, bf16* o) {
  cluster_arrive();
  cluster_wait();
  const uint32_t at = smem_u32(mine);
  for (int i = cluster_rank() * W * 32 + threadIdx.x; i < rows * (D / 4); i += ctas * W * 32) {
    const int row = i / (D / 4), d = i % (D / 4) * 4;
    float4 s[8], x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      s[k] = make_float4(kLowest, 0.f, kLowest, 0.f);
      x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k >= ctas) continue;
      s[k] = ld_cluster_16(at + (row * ROW + D) * 4, k);
      x[k] = ld_cluster_16(at + (row * ROW + d) * 4, k);
    }
    float tm = kLowest, tM = kLowest, tl = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      tm = fmaxf(tm, s[k].x);
      tM = fmaxf(tM, s[k].z);
    }
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float by = exp2_ftz(s[k].z - tM);
      sum.x += x[k].x * by; sum.y += x[k].y * by; sum.z += x[k].z * by; sum.w += x[k].w * by;
      tl += s[k].y * exp2_ftz(s[k].x - tm);
    }
    store_bf16x4(o + row * D + d, sum, any ? exp2_ftz(tM - tm) / tl : 0.f);
  }
  cluster_arrive();   // (nobody leaves while its sums are read)
  cluster_wait();
}

// CTAs of a SM, by registers: 12 warps of 168, or 8 of 255.  (One CTA of 12 warps: step_many 203 in place of 192 us, step_window 174 and 169:
// nothing is computed while one adds up its warps' sums.)
constexpr int kPagedWarps = 4;
__host__ __device__ constexpr int kPagedPerSm(int nq) { return nq == 1 ? 3 : 2; }
// 16 tokens of a step times this
__host__ __device__ constexpr int kPagedSub(int row_bytes) { return row_bytes > 128 ? 1 : row_bytes > 64 ? 2 : 4; }

// A unit that begins in a run and does not end there: its result, and how many runs have pieces of it (0: there is none).
struct PagedCut {
  int64_t o;
  int32_t rows, count;
};
// The pieces of the units that were cut, added up: blockIdx.x is the run that one begins in, blockIdx.y 64 times four of its sums; groups
// of 64 threads share the pieces, eight of a group on their way at a time.  A launch of its own, so that nothing is left behind in the
// kernel that has to wait for pieces (which would cost its loop registers: there, by who comes last, step_long took 101 in place of 97 us).
constexpr int kPagedJoinMost = 1024;   // pieces of a unit at most: the runs of a call
template <int D>
__global__ void __launch_bounds__(512) paged_join_kernel(const float* pieces, const PagedCut* cuts, bf16* out, int32_t sum_rows) {
  constexpr int ROW = kPagedPieceRow(D), ROWS = 256 / D, N = 8;   // rows of 64 times four sums
  __shared__ float factor[ROWS][kPagedJoinMost], scale[ROWS];
  __shared__ float4 part[7][64];
  // (the next launch begins when this one ends: begun beside its blocks, which hold shared memory that three CTAs of the next call's kernel
  // need, that finds fewer places: step_window 208 in place of 159 us, generate 62 and 48, call after call)
  griddep_wait();
  const PagedCut u = cuts[blockIdx.x];
  const int row0 = blockIdx.y * ROWS, rows = min(u.rows - row0, ROWS), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (u.count == 0 || rows <= 0) return;
  // (the first piece is its run's second)
  const float* const base = pieces + static_cast<int64_t>(blockIdx.x) * 2 * sum_rows * ROW + row0 * ROW;
  auto piece = [&](int i) { return base + static_cast<int64_t>(2 * i + (i == 0 ? 1 : 0)) * sum_rows * ROW; };
  for (int row = warp; row < rows; row += blockDim.x >> 5) {
    float tm = kLowest, tM = kLowest, tl = 0.f;                   // (a lane's own, until they are put together)
    for (int i0 = lane; i0 < u.count; i0 += 4 * 32) {
      float4 s[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        s[k] = make_float4(kLowest, 0.f, kLowest, 0.f);
        if (i0 + k * 32 < u.count) s[k] = *reinterpret_cast<const float4*>(piece(i0 + k * 32) + row * ROW + D);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float now = fmaxf(tm, s[k].x);
        tl = tl * exp2_ftz(tm - now) + s[k].y * exp2_ftz(s[k].x - now);
        tm = now;
        tM = fmaxf(tM, s[k].z);
        if (i0 + k * 32 < u.count) factor[row][i0 + k * 32] = s[k].z;
      }
    }
    float top = tm;
#pragma unroll
    for (int e = 16; e > 0; e >>= 1) {
      top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, e));
      tM = fmaxf(tM, __shfl_xor_sync(0xFFFFFFFFu, tM, e));
    }
    tl *= exp2_ftz(tm - top);
#pragma unroll
    for (int e = 16; e > 0; e >>= 1) tl += __shfl_xor_sync(0xFFFFFFFFu, tl, e);
    for (int i = lane; i < u.count; i += 32) factor[row][i] = exp2_ftz(factor[row][i] - tM);
    if (lane == 0) scale[row] = exp2_ftz(tM - top) / tl;
  }
  __syncthreads();
  const int groups = blockDim.x / 64, group = threadIdx.x / 64, at = threadIdx.x % 64, row = at / (D / 4), d = at % (D / 4) * 4;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  if (row < rows) {
    for (int i0 = group; i0 < u.count; i0 += N * groups) {
      float4 x[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i0 + k * groups < u.count) x[k] = *reinterpret_cast<const float4*>(piece(i0 + k * groups) + row * ROW + d);
      }
#pragma unroll
      for (int k = 0; k < N; ++k) {
        if (i0 + k * groups >= u.count) continue;
        const float f = factor[row][i0 + k * groups];
        sum.x += x[k].x * f; sum.y += x[k].y * f; sum.z += x[k].z * f; sum.w += x[k].w * f;
      }
    }
  }
  if (group > 0) part[group - 1][at] = sum;
  __syncthreads();
  if (group > 0 || row >= rows) return;
  for (int g = 0; g < groups - 1; ++g) {
    const float4 x = part[g][at];
    sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
  }
  store_bf16x4(out + u.o + (row0 + row) * D + d, sum, scale[row]);
}

template <int D, bool E4, int NQ, int W>
__global__ void __launch_bounds__(W * 32, kPagedPerSm(NQ)) paged_step_kernel(const __grid_constant__ PagedStepArgs a, const __grid_constant__ CUtensorMap k_map,
                                                            const __grid_constant__ CUtensorMap v_map) {
  constexpr int BYTES = E4 ? D : 2 * D;                  // of a row
  constexpr int SUB = kPagedSub(BYTES), STEP = 16 * SUB; // tokens of a step: 8 KB where rows allow
  constexpr int ROWS = 8 * NQ, TILE = STEP * W, ROW = kPagedPieceRow(D), THREADS = W * 32;
  constexpr int BOX = BYTES >= 128 ? 128 : 64;           // bytes of a row in a box of 16 rows; swizzled over as many
  constexpr int BOXES = BYTES / BOX;
  constexpr int KB = STEP * BYTES, EB = E4 ? 2 * STEP : 0, STAGE = 2 * KB;
  constexpr int KW = BOX / 16;                           // words of a box's K row that a lane has
  constexpr int VW = BOX / 32;                           // words of a box's V row that a lane has
  constexpr int MT = D / 16;                             // products of 16 features
  constexpr int QW = D / 8;                              // words of a lane's queries: two a step of 16 features
  extern __shared__ uint8_t smem_raw[];   // [W][stages] of K and V, [W][stages] of exponents, sums [W][rows][ROW]
  __shared__ uint64_t full[W * kPagedStages];
  __shared__ int plan[4];
  __shared__ int64_t warp_sum[W];
  __shared__ uint32_t gave_up;
  const int warp = uniform_warp_index(), lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const uint32_t leader = elect_leader();
  uint8_t* const paged_smem = smem_raw + ((smem_u32(smem_raw) + 1023u & ~1023u) - smem_u32(smem_raw));
  const uint32_t ring = smem_u32(paged_smem) + warp * a.stages * STAGE, exp_ring = smem_u32(paged_smem) + W * a.stages * STAGE + warp * a.stages * EB;
  float* const sums = reinterpret_cast<float*>(paged_smem + W * a.stages * (STAGE + EB));
  if (lane == 0)
    for (int i = 0; i < a.stages; ++i) mbar_init(&full[warp * kPagedStages + i], 1);
  if (threadIdx.x == 0) gave_up = 0;
  fence_mbar_init();
  griddep_launch_dependents();
  griddep_wait();
  const int units = a.c.heads * a.blocks;                // of a sequence
  const int sum_rows = min(a.share, ROWS);
  // -------- this CTA's run
  PagedWalk make;                                        // (the copies run ahead of the products)
  int64_t run0 = 0, per = 0;
  if (a.runs == 0) {
    const int u = blockIdx.x / a.cluster, rank = blockIdx.x - u * a.cluster;
    make.seq = u / units;
    make.unit = u - make.seq * units;
    const int tiles = paged_span<STEP, TILE>(a, make.seq).tiles, each = (tiles + a.cluster - 1) / a.cluster;
    make.t = min(rank * each, tiles);
    make.left = min(each, tiles - make.t);
    __syncthreads();
  } else {
    const int chunk = (a.c.sequences + THREADS - 1) / THREADS, s0 = min(static_cast<int>(threadIdx.x) * chunk, a.c.sequences), s1 = min(s0 + chunk, a.c.sequences);
    int64_t mine = 0;
    for (int s = s0; s < s1; ++s) mine += paged_span<STEP, TILE>(a, s).tiles;
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
    if (threadIdx.x == 0) a.cuts[blockIdx.x].count = 0;   // (until there is one)
    if (run0 >= all) return;
    make.left = static_cast<int>(min(per, all - run0));
    int64_t at = (upto - mine) * units;
    if (run0 >= at && run0 < upto * units) {
      for (int s = s0; s < s1; ++s) {
        const int64_t n = paged_span<STEP, TILE>(a, s).tiles;
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
    make.seq = plan[0];
    make.unit = plan[1];
    make.t = plan[2];
  }
  auto enter = [&](PagedWalk& w) {                       // seq, unit, t and left are set
    const PagedSpan span = paged_span<STEP, TILE>(a, w.seq);
    w.first = span.first; w.last = span.last; w.base = span.base; w.tiles = span.tiles; w.over = span.over;
    w.t1 = min(span.tiles, w.t + w.left);
    w.head = w.unit / a.blocks;
    w.table = a.c.table + w.seq * a.c.table_rs;
  };
  auto leave = [&](PagedWalk& w, int from) {             // to the next unit; `from`: the tile that this one began with
    w.left -= w.t1 - from;
    w.t = 0;
    if (++w.unit == units) {
      w.unit = 0;
      ++w.seq;
    }
  };
  auto position = [&](const PagedWalk& w) { return w.base + (w.t * W + warp) * STEP; };
  // A step lies in one page, or in `parts` of smaller ones; past the end none is looked up.
  const int parts = max(STEP >> a.c.shift, 1), part_rows = min(STEP, 1 << a.c.shift), part_bytes = (STAGE + EB) / parts;
  auto pages_of = [&](const PagedWalk& w, int (&pg)[SUB]) {
    const int p = position(w), at = p >> a.c.shift;
    pg[0] = p < w.last ? w.table[at] : -1;
#pragma unroll
    for (int i = 1; i < SUB; ++i) pg[i] = i < parts && p + i * part_rows < w.last ? w.table[at + i] : -1;
  };
  enter(make);
  const int stages = make.left > kPagedLong ? a.long_stages : a.stages;
  PagedWalk use = make;
  int make_from = make.t, page[SUB], make_slot = 0, use_slot = 0;
  pages_of(make, page);
  uint32_t has = 0, gone = 0, phase = 0;                 // slots that hold something; 16 tokens that are not there, SUB bits a slot; parities of the next waits
  // the copies of this warp's tokens of the next tile
  auto issue = [&]() {
    if (make.left <= 0) return;
    const int p = position(make), row = (make.head << a.c.shift) + (p & ((1 << a.c.shift) - 1));
    const uint32_t bar = smem_u32(&full[warp * kPagedStages + make_slot]), to = ring + make_slot * STAGE, exps = exp_ring + make_slot * EB;
    auto copy = [&](int pg, int at, int rows, uint32_t on) {
#pragma unroll
      for (int i = 0; i < BOXES; ++i) tma_load_3d_if(on, to + i * STEP * BOX + at * BOX, &k_map, bar, i * 64, row, pg);
#pragma unroll
      for (int i = 0; i < BOXES; ++i) tma_load_3d_if(on, to + KB + i * STEP * BOX + at * BOX, &v_map, bar, i * 64, row, pg);
      if constexpr (E4) {
        bulk_load_if(on, exps + at, a.c.ke + pg * a.c.ke_ps + row, rows, bar);
        bulk_load_if(on, exps + STEP + at, a.c.ve + pg * a.c.ve_ps + row, rows, bar);
      }
    };
    auto there = [&](int pg, int at) {
      const bool real = p + at < make.last;
      if (real && static_cast<uint32_t>(pg) >= static_cast<uint32_t>(a.c.pages)) {
        if (lane == 0) report_bad_page();
        return false;
      }
      return real;
    };
    if (SUB == 1 || parts == 1) {
      const bool real = there(page[0], 0);
      has = real ? has | 1u << make_slot : has & ~(1u << make_slot);
      if (real) {
        mbar_expect_tx_if(leader, bar, STAGE + EB);
        copy(page[0], 0, STEP, leader);
      }
    } else {
      // (a part that is not there is left as it was, and counts as outside of the window)
      uint32_t on = 0;
#pragma unroll
      for (int i = 0; i < SUB; ++i)
        if (i < parts && there(page[i], i * part_rows)) on |= 1u << i;
      has = on != 0 ? has | 1u << make_slot : has & ~(1u << make_slot);
      uint32_t lost = 0;
#pragma unroll
      for (int u = 0; u < SUB; ++u)
        if ((on >> (u * 16 >> a.c.shift) & 1) == 0) lost |= 1u << u;
      gone = (gone & ~(((1u << SUB) - 1) << make_slot * SUB)) | lost << make_slot * SUB;
      if (on != 0) {
        mbar_expect_tx_if(leader, bar, __popc(on) * part_bytes);
#pragma unroll
        for (int i = 0; i < SUB; ++i)
          if (on >> i & 1) copy(page[i], i * part_rows, part_rows, leader);
      }
    }
    if (++make_slot == stages) make_slot = 0;
    if (++make.t == make.t1) {
      leave(make, make_from);
      make_from = 0;
      if (make.left > 0) enter(make);
    }
    if (make.left > 0) pages_of(make, page);
  };
  for (int i = 0; i < stages; ++i) issue();
  bool failed = false;
  // queries: column r of a product is query head row0 + r (+ 8); as they are, and as the products take them
  uint32_t q[NQ][QW];
  float qm[NQ][2];                                       // what scores of columns 2 c, 2 c + 1 are multiplied by
  auto first_row = [&](const PagedWalk& w) { return (w.unit - w.head * a.blocks) * ROWS; };
  auto load_q = [&](const PagedWalk& w) {
    const int row0 = first_row(w), rows = min(a.share - row0, ROWS);
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const bf16* from = a.q + w.seq * a.q_bs + (static_cast<int64_t>(w.head) * a.share + row0 + n * 8 + r) * a.q_hs;
#pragma unroll
      for (int e = 0; e < QW; e += 4) {
        uint4 x = make_uint4(0, 0, 0, 0);
        // (8 bits: QW words from c's on; else KW of each box)
        if (n * 8 + r < rows) x = *reinterpret_cast<const uint4*>(from + (E4 ? c * (2 * QW) + e * 2 : e / KW * 64 + c * 16 + e % KW * 2));
        q[n][e] = x.x; q[n][e + 1] = x.y; q[n][e + 2] = x.z; q[n][e + 3] = x.w;
      }
    }
  };
  auto ready_q = [&]() {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      qm[n][0] = qm[n][1] = a.scale;
      if constexpr (E4) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < QW; ++i) top = __vmaxu2(top, q[n][i] & 0x7FFF7FFFu);
        top = max(top & 0xFFFFu, top >> 16);
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
        // the largest becomes 2^14 to 2^15 (not from below 2^-86); of an infinity or a NaN what it is
        const int e = min(max(static_cast<int>(top >> 7), 41), 254);
        const float up = __uint_as_float(static_cast<uint32_t>(127 + 141 - e) << 23), down = a.scale * __uint_as_float(static_cast<uint32_t>(e - 14) << 23);
#pragma unroll
        for (int i = 0; i < QW; ++i) {
          const __half2 h = __floats2half2_rn(__uint_as_float(q[n][i] << 16) * up, __uint_as_float(q[n][i] & 0xFFFF0000u) * up);
          q[n][i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        qm[n][0] = __shfl_sync(0xFFFFFFFFu, down, c * 8);
        qm[n][1] = __shfl_sync(0xFFFFFFFFu, down, c * 8 + 4);
      }
    }
  };
  load_q(use);
  // -------- its units
  for (int64_t done = 0; use.left > 0 || a.cluster > 1;) {   // (of a cluster every CTA has one turn, with tiles or without)
    const int t0 = use.t, row0 = first_row(use), rows = min(a.share - row0, ROWS);
    if (threadIdx.x == 0 && use.over && use.t1 == use.tiles) report_bad_page();
    ready_q();
    // -------- tiles: this warp's step of each
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
    for (; use.t < use.t1; ++use.t) {
      const int slot = use_slot, p = position(use);
      if (++use_slot == stages) use_slot = 0;
      if ((has >> slot & 1) && !failed) {
        if (!mbar_wait_warp(&full[warp * kPagedStages + slot], phase >> slot & 1, &gave_up)) {
          // out of time: nothing more is copied or computed; what is on its way gets as long again to arrive
          failed = true;
          gave_up = 1;
          if (lane == 0) report_timeout(a.status);
          make.left = 0;
          for (int s = 0; s < stages; ++s)
            if (has >> s & 1) mbar_wait(&full[warp * kPagedStages + s], phase >> s & 1);
        }
        phase ^= 1u << slot;
      }
      if (!(has >> slot & 1) || failed) {
        issue();
        continue;
      }
      const uint32_t ks = ring + slot * STAGE, vs = ks + KB;
      float x[SUB][NQ][4];
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        float z[NQ][4];                                  // (two chains of products)
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[u][n][e] = z[n][e] = 0.f;
#pragma unroll
        for (int i = 0; i < BOXES; ++i) {
          uint32_t kr[2][KW];                            // rows r, r + 8: a lane's BOX / 4 bytes
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < KW / 4; ++e) {
              const uint4 w = ld_shared_16(ks + i * STEP * BOX + (16 * u + r + 8 * h) * BOX + ((c * (KW / 4) + e) ^ (BOX == 128 ? r : r >> 1 & 3)) * 16);
              kr[h][4 * e] = w.x; kr[h][4 * e + 1] = w.y; kr[h][4 * e + 2] = w.z; kr[h][4 * e + 3] = w.w;
            }
#pragma unroll
          for (int e = 0; e < KW; e += E4 ? 1 : 2) {
            uint32_t a0, a1, a2, a3;
            if constexpr (E4) {
              halves_of_e4m3(kr[0][e], a0, a2);
              halves_of_e4m3(kr[1][e], a1, a3);
            } else {
              a0 = kr[0][e]; a1 = kr[1][e]; a2 = kr[0][e + 1]; a3 = kr[1][e + 1];
            }
            const int s = E4 ? 2 * e : i * KW + e;
#pragma unroll
            for (int n = 0; n < NQ; ++n) mma_16x8(s / 2 % 2 ? z[n] : x[u][n], a0, a1, a2, a3, q[n][s], q[n][s + 1], E4);
          }
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[u][n][e] = E4 ? x[u][n][e] + z[n][e] : (x[u][n][e] + z[n][e]) * qm[n][e & 1];
      }
      [[maybe_unused]] float y[SUB][NQ][4];
      if constexpr (E4) {
        const uint8_t* const exps = paged_smem + (exp_ring - smem_u32(paged_smem)) + slot * EB;
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            // 2^(byte - 127) and byte - 127, NaN for 255 (infinity times zero).  The query's factor and the key's come together first: large
            // queries on small keys have scores of an ordinary size, the one or the other alone may not be there in fp32.
            const uint32_t kb = exps[16 * u + r + 8 * h], vb = exps[STEP + 16 * u + r + 8 * h];
            const float k2 = __uint_as_float(max(kb << 23, 0x00400000u)), kx = fmaf(k2, 0.f, k2);
            const float vx = fmaf(__uint_as_float(vb << 23), 0.f, __uint_as_float(0x4B000000u | vb) - 8388735.f);
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
              for (int e = 2 * h; e < 2 * h + 2; ++e) {
                x[u][n][e] *= qm[n][e & 1] * kx;
                y[u][n][e] = x[u][n][e] + vx;
              }
          }
      }
      // a lane's features (8 bits: 16; else 8 of each box) of tokens 2 c, 2 c + 1 and those 8 later
      uint32_t vr[SUB][4][BOXES * VW];
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int tok = 2 * c + (i & 1) + 8 * (i >> 1);
#pragma unroll
          for (int b = 0; b < BOXES; ++b) {
            if constexpr (VW == 4) {
              const uint4 w = ld_shared_16(vs + b * STEP * BOX + (16 * u + tok) * BOX + (r ^ (tok & 7)) * 16);
              vr[u][i][b * 4] = w.x; vr[u][i][b * 4 + 1] = w.y; vr[u][i][b * 4 + 2] = w.z; vr[u][i][b * 4 + 3] = w.w;
            } else {
              const uint2 w = ld_shared_8(vs + (16 * u + tok) * BOX + ((r >> 1) ^ (tok >> 1 & 3)) * 16 + (r & 1) * 8);
              vr[u][i][0] = w.x; vr[u][i][1] = w.y;
            }
          }
        }
      // tokens outside of the window: no weight, and no values (what lies there may be NaN)
      const uint32_t lost = gone >> slot * SUB & ((1u << SUB) - 1);
      if (p < use.first || p + STEP > use.last || lost != 0) {
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int at = p + 16 * u + r + 8 * h;
            if ((lost >> u & 1) == 0 && at >= use.first && at < use.last) continue;
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
              for (int e = 2 * h; e < 2 * h + 2; ++e) x[u][n][e] = y[u][n][e] = -INFINITY;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int at = p + 16 * u + 2 * c + (i & 1) + 8 * (i >> 1);
            if ((lost >> u & 1) == 0 && at >= use.first && at < use.last) continue;
#pragma unroll
            for (int e = 0; e < BOXES * VW; ++e) vr[u][i][e] = 0;
          }
        }
      }
      __syncwarp();
      issue();                                           // (all of the slot is in registers)
      // the maxima, where a score passes them by 8
      float top[NQ][2], high[NQ][2];
      bool raise = false;
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[n][e] = fmaxf(x[0][n][e], x[0][n][e + 2]);
          if constexpr (E4) high[n][e] = fmaxf(y[0][n][e], y[0][n][e + 2]);
#pragma unroll
          for (int u = 1; u < SUB; ++u) {
            top[n][e] = fmaxf(top[n][e], fmaxf(x[u][n][e], x[u][n][e + 2]));
            if constexpr (E4) high[n][e] = fmaxf(high[n][e], fmaxf(y[u][n][e], y[u][n][e + 2]));
          }
          raise = raise || top[n][e] > m[n][e] + 8.f;
          if constexpr (E4) raise = raise || high[n][e] > M[n][e] + 8.f;
        }
      if (__any_sync(0xFFFFFFFFu, raise)) {
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            auto over_rows = [&](float old, float z) {
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) z = fmaxf(z, __shfl_xor_sync(0xFFFFFFFFu, z, o));
              return fmaxf(old, z);
            };
            const float now = over_rows(m[n][e], top[n][e]);
            float f = exp2_ftz(m[n][e] - now);
            l[n][e] *= f;
            m[n][e] = now;
            if constexpr (E4) {
              const float big = over_rows(M[n][e], high[n][e]);
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
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        // weights, turned over so that their tokens are the inner axis
        uint32_t hi[NQ][2];
        [[maybe_unused]] uint32_t lo[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            w[e] = exp2_ftz(x[u][n][e] - m[n][e & 1]);
            l[n][e & 1] += w[e];
            if constexpr (E4) w[e] = exp2_ftz(y[u][n][e] - M[n][e & 1]);
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
            uint32_t a0, a1, a2, a3, b0, b1, b2, b3;
            halves_of_e4m3(__byte_perm(vr[u][0][j / 2], vr[u][1][j / 2], 0x5140), a0, a1);
            halves_of_e4m3(__byte_perm(vr[u][2][j / 2], vr[u][3][j / 2], 0x5140), a2, a3);
            halves_of_e4m3(__byte_perm(vr[u][0][j / 2], vr[u][1][j / 2], 0x7362), b0, b1);
            halves_of_e4m3(__byte_perm(vr[u][2][j / 2], vr[u][3][j / 2], 0x7362), b2, b3);
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
              mma_16x8(acc[n][j], a0, a1, a2, a3, hi[n][0], hi[n][1], true);
              mma_16x8(acc[n][j + 1], b0, b1, b2, b3, hi[n][0], hi[n][1], true);
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            const uint32_t a0 = __byte_perm(vr[u][0][j], vr[u][1][j], 0x5410), a1 = __byte_perm(vr[u][0][j], vr[u][1][j], 0x7632);
            const uint32_t a2 = __byte_perm(vr[u][2][j], vr[u][3][j], 0x5410), a3 = __byte_perm(vr[u][2][j], vr[u][3][j], 0x7632);
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
              mma_16x8(acc[n][j], a0, a1, a2, a3, hi[n][0], hi[n][1], false);
              mma_16x8(acc[n][j], a0, a1, a2, a3, lo[n][0], lo[n][1], false);
            }
          }
        }
      }
    }
    // -------- the warps' sums (rows of D features, then m, l, M)
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[n][e] += __shfl_xor_sync(0xFFFFFFFFu, l[n][e], o);
        const int row = n * 8 + 2 * c + e;
        if (row >= rows) continue;
        float* const to = sums + (warp * sum_rows + row) * ROW;
#pragma unroll
        for (int j = 0; j < MT; j += 2) {
          const int d = BOXES == 1 ? r * (D / 8) + 2 * j : j / 4 * 64 + r * 8 + j % 4 * 2;
          *reinterpret_cast<float4*>(to + d) = make_float4(acc[n][j][e], acc[n][j][e + 2], acc[n][j + 1][e], acc[n][j + 1][e + 2]);
        }
        if (r == 0) *reinterpret_cast<float4*>(to + D) = make_float4(m[n][e], l[n][e], E4 ? M[n][e] : m[n][e], 0.f);
      }
    const bool whole = use.t1 == use.tiles && t0 == 0, any = use.last > use.first;
    const int64_t at = (static_cast<int64_t>(use.seq) * a.heads + static_cast<int64_t>(use.head) * a.share + row0) * D, begin = run0 + done;
    const int tiles = use.tiles;
    done += use.t1 - t0;
    leave(use, t0);
    if (use.left > 0) {   // (the next unit's queries are on their way while this one's sums are added up)
      enter(use);
      load_q(use);
    }
    __syncthreads();
    if (a.cluster == 1 && whole) {
      paged_merge<D, W, ROW>(sums, sum_rows, rows, [&](int row, int d, const float4& sum, const float4& s) {
        store_bf16x4(a.o + at + row * D + d, sum, any ? exp2_ftz(s.z - s.x) / s.y : 0.f);
      });
    } else {
      // a piece: to this CTA's part of the cluster's, or to global memory
      float* const piece = a.cluster > 1 ? sums + W * sum_rows * ROW : a.pieces + (static_cast<int64_t>(blockIdx.x) * 2 + (t0 == 0 ? 1 : 0)) * sum_rows * ROW;
      paged_merge<D, W, ROW>(sums, sum_rows, rows, [&](int row, int d, const float4& sum, const float4& s) {
        *reinterpret_cast<float4*>(piece + row * ROW + d) = sum;
        if (d == 0) *reinterpret_cast<float4*>(piece + row * ROW + D) = s;
      });
      if (a.cluster > 1) {
        paged_join_cluster<D, W, ROW>(a.cluster, piece, rows, any, a.o + at);
        return;
      }
      if (threadIdx.x == 0 && t0 == 0) a.cuts[blockIdx.x] = {at, rows, static_cast<int32_t>((begin + tiles - 1) / per - blockIdx.x) + 1};
    }
    __syncthreads();
  }
}

}  // namespace lact

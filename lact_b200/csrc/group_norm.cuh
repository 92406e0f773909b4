// Group norm with an activation, channels last: x [n][s][C], the C channels in G groups of adjacent ones; per sample and group
//   xhat = (x - mean) / sqrt(var + eps)  over its s spots and C / G channels,  z = xhat w_c + b_c,  y = z or z sigmoid(z).
// Backward, with dz = dy (or dy * d silu(z)):  dw_c = sum dz xhat, db_c = sum dz over samples and spots, and per sample and group
//   dx = (dz w - c1 - xhat c2) / sqrt(var + eps),  c1 = mean(dz w),  c2 = mean(dz w xhat).
// Bound by memory: x and y once are what it cannot do without (x, dy, dx backward).  Two ways:
//   one spot a sample (the norm per head of tokens): a row is read into registers, its groups are summed among the threads that hold
//     them, mean first and then squares of what is left; one pass over memory, one launch.
//   many spots: threads keep their channels and walk the spots, so that 16 bytes are read whatever a group's width is; every thread
//     sums against the first value it sees and hands on a mean and the squares around it (no cancellation where the mean is far from
//     zero); a small launch puts chunks and channels of a group together, a last one reads x again - from L2 as far as it goes: it
//     begins where the sums have ended - and writes.
// All sums are in fp32 and in a fixed order.
#pragma once
#include "ptx.cuh"

namespace lact {

using bf16 = __nv_bfloat16;

struct GroupNormArgs {
  const void* x;
  const void* dy;             // backward; strides as x's own
  const float *w, *b;         // [C] or nullptr: ones, zeros
  void* out;                  // y, or dx: contiguous
  float* stats;               // [n][G][2]: mean, 1 / sqrt(var + eps)
  float* part;                // [n][chunks][C][2]; one spot, backward: [blocks][2][C]
  float* chan;                // [n][C][2]
  float* coef;                // backward: [n][G][2]: c1, c2
  float *dw, *db;             // [C]
  int64_t n, x_ns, x_ss, dy_ns, dy_ss;
  int32_t s, C, G, silu;
  int32_t chunks, per_chunk;  // spots of a sample are dealt to `chunks` blocks
  float eps;
};

// V values of type T, as one access
template <class T, int V>
struct Vec;
template <int BYTES>
struct Raw;
template <> struct Raw<16> { using type = uint4; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<4> { using type = uint32_t; };
template <> struct Raw<2> { using type = uint16_t; };
template <class T, int V>
__device__ __forceinline__ void load_values(const T* p, float (&f)[V]) {
  using R = typename Raw<V * sizeof(T)>::type;
  const R r = *reinterpret_cast<const R*>(p);
  const T* t = reinterpret_cast<const T*>(&r);
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = static_cast<float>(t[i]);
}
template <class T, int V>
__device__ __forceinline__ void store_values(T* p, const float (&f)[V]) {
  using R = typename Raw<V * sizeof(T)>::type;
  R r;
  T* t = reinterpret_cast<T*>(&r);
#pragma unroll
  for (int i = 0; i < V; ++i) t[i] = static_cast<T>(f[i]);
  *reinterpret_cast<R*>(p) = r;
}
__device__ __forceinline__ float silu_of(float z) { return z * sigmoidf_fast(z); }
__device__ __forceinline__ float silu_slope(float z) {
  const float g = sigmoidf_fast(z);
  return g * fmaf(z, 1.f - g, 1.f);
}

// ---------------------------------------------------------------- one spot a sample
// LPR threads a row (a power of two), K vectors of V channels each (a group holds whole vectors); 256 / LPR rows a block at a time.
// Sums of a group: among neighbouring lanes where it has 1, 2, .. 32 vectors, through shared memory otherwise.
template <int K>
struct GroupSums {
  float* vec;     // [rows][vectors]
  float* sum;     // [rows][G]
  int gv, G, nv, lpr, rows;
  bool lanes;     // gv a power of two, at most 32 and lpr
  // p[i]: this thread's sum of vector l + i * lpr -> the sum over the vector's group
  __device__ __forceinline__ void operator()(float (&p)[K], int row, int l) const {
    if (lanes) {
#pragma unroll
      for (int i = 0; i < K; ++i)
        for (int o = 1; o < gv; o <<= 1) p[i] += __shfl_xor_sync(0xFFFFFFFFu, p[i], o);
      return;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < K; ++i)
      if (l + i * lpr < nv) vec[row * nv + l + i * lpr] = p[i];
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int it = warp; it < rows * G; it += 8) {
      const float* from = vec + it / G * nv + it % G * gv;
      float t = 0.f;
      for (int j = lane; j < gv; j += 32) t += from[j];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
      if (lane == 0) sum[it] = t;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < K; ++i)
      if (l + i * lpr < nv) p[i] = sum[row * G + (l + i * lpr) / gv];
  }
};

template <class T, int V, int K, bool BACKWARD>
__global__ void __launch_bounds__(256) group_norm_rows_kernel(const __grid_constant__ GroupNormArgs a, int32_t lpr) {
  extern __shared__ float norm_smem[];
  griddep_launch_dependents();
  griddep_wait();
  const int l = threadIdx.x & (lpr - 1), row = threadIdx.x / lpr, rows = 256 / lpr;
  const int nv = a.C / V, gv = nv / a.G;
  const GroupSums<K> sums{norm_smem, norm_smem + rows * nv, gv, a.G, nv, lpr, rows, (gv & (gv - 1)) == 0 && gv <= 32 && gv <= lpr};
  const float inv = 1.f / (gv * V);
  float w[K][V], b[K][V];
#pragma unroll
  for (int i = 0; i < K; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int v = l + i * lpr, c = v * V + e;
      w[i][e] = v < nv && a.w != nullptr ? a.w[c] : 1.f;
      b[i][e] = v < nv && a.b != nullptr ? a.b[c] : 0.f;
    }
  [[maybe_unused]] float dw[BACKWARD ? K : 1][V], db[BACKWARD ? K : 1][V];
  if (BACKWARD) {
#pragma unroll
    for (int i = 0; i < K; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) dw[i][e] = db[i][e] = 0.f;
  }
  for (int64_t n0 = static_cast<int64_t>(blockIdx.x) * rows; n0 < a.n; n0 += static_cast<int64_t>(gridDim.x) * rows) {
    const int64_t n = n0 + row;
    const bool on = n < a.n;    // (all threads take part in the sums)
    float x[K][V], p[K];
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const int v = l + i * lpr;
#pragma unroll
      for (int e = 0; e < V; ++e) x[i][e] = 0.f;
      if (on && v < nv) load_values<T, V>(static_cast<const T*>(a.x) + n * a.x_ns + v * V, x[i]);
    }
    if constexpr (!BACKWARD) {
#pragma unroll
      for (int i = 0; i < K; ++i) {
        p[i] = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) p[i] += x[i][e];
      }
      sums(p, row, l);
#pragma unroll
      for (int i = 0; i < K; ++i) {
        const float mean = p[i] * inv;
        if (on && l + i * lpr < nv && (l + i * lpr) % gv == 0) a.stats[(n * a.G + (l + i * lpr) / gv) * 2] = mean;
        p[i] = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          x[i][e] -= mean;
          p[i] = fmaf(x[i][e], x[i][e], p[i]);
        }
        if (l + i * lpr >= nv) p[i] = 0.f;
      }
      sums(p, row, l);
#pragma unroll
      for (int i = 0; i < K; ++i) {
        const int v = l + i * lpr;
        const float rstd = rsqrtf(fmaf(p[i], inv, a.eps));
        if (!on || v >= nv) continue;
        if (v % gv == 0) a.stats[(n * a.G + v / gv) * 2 + 1] = rstd;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float z = fmaf(x[i][e] * rstd, w[i][e], b[i][e]);
          x[i][e] = a.silu ? silu_of(z) : z;
        }
        store_values<T, V>(static_cast<T*>(a.out) + n * a.C + v * V, x[i]);
      }
    } else {
      float t[K][V], q[K], rstd[K];
#pragma unroll
      for (int i = 0; i < K; ++i) {
        const int v = l + i * lpr;
        p[i] = q[i] = rstd[i] = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) t[i][e] = 0.f;
        if (!on || v >= nv) continue;
        load_values<T, V>(static_cast<const T*>(a.dy) + n * a.dy_ns + v * V, t[i]);
        const float2 st = *reinterpret_cast<const float2*>(a.stats + (n * a.G + v / gv) * 2);
        rstd[i] = st.y;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          x[i][e] = (x[i][e] - st.x) * st.y;
          if (a.silu) t[i][e] *= silu_slope(fmaf(x[i][e], w[i][e], b[i][e]));
          db[i][e] += t[i][e];
          dw[i][e] = fmaf(t[i][e], x[i][e], dw[i][e]);
          t[i][e] *= w[i][e];
          p[i] += t[i][e];
          q[i] = fmaf(t[i][e], x[i][e], q[i]);
        }
      }
      sums(p, row, l);
      sums(q, row, l);
#pragma unroll
      for (int i = 0; i < K; ++i) {
        const int v = l + i * lpr;
        if (!on || v >= nv) continue;
        const float c1 = p[i] * inv, c2 = q[i] * inv;
#pragma unroll
        for (int e = 0; e < V; ++e) x[i][e] = rstd[i] * (t[i][e] - c1 - x[i][e] * c2);
        store_values<T, V>(static_cast<T*>(a.out) + n * a.C + v * V, x[i]);
      }
    }
  }
  if constexpr (BACKWARD) {
    // the block's sums over its rows: [2][C], rows of threads added in their order
    float* const acc = norm_smem;
    for (int turn = 0; turn < rows; ++turn) {
      __syncthreads();
      if (row != turn) continue;
#pragma unroll
      for (int i = 0; i < K; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int v = l + i * lpr, c = v * V + e;
          if (v >= nv) continue;
          acc[c] = turn == 0 ? dw[i][e] : acc[c] + dw[i][e];
          acc[a.C + c] = turn == 0 ? db[i][e] : acc[a.C + c] + db[i][e];
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * a.C; c += 256) a.part[static_cast<int64_t>(blockIdx.x) * 2 * a.C + c] = acc[c];
  }
}

// ---------------------------------------------------------------- many spots
// Threads of a block: up to 256 vectors of V channels, and as many spots at a time as there are threads left.
struct NormSpots {
  int v, row, rows, first, last;   // this thread's vector, its spot among `rows` at a time, the chunk's spots
  bool on;
};
template <int V>
__device__ __forceinline__ NormSpots norm_spots(const GroupNormArgs& a, int chunk, int cblock) {
  const int nv = a.C / V, here = min(nv, 256);
  NormSpots p;
  p.rows = 256 / here;
  p.row = threadIdx.x / here;
  p.v = cblock * 256 + threadIdx.x % here;
  p.on = p.row < p.rows && p.v < nv;
  p.first = chunk * a.per_chunk;
  p.last = min(p.first + a.per_chunk, a.s);
  return p;
}
constexpr int kNormAhead = 4;   // spots fetched before the first is worked on

// Per channel of a chunk -> part[n][chunk][c]: forward the mean and the sum of squares around it, backward the sums of dz and dz xhat.
template <class T, int V, bool BACKWARD>
__global__ void __launch_bounds__(256) group_norm_sums_kernel(const __grid_constant__ GroupNormArgs a) {
  __shared__ float acc[256 * V * 2];
  griddep_launch_dependents();
  griddep_wait();
  const int chunk = blockIdx.x % a.chunks;
  const int64_t n = blockIdx.x / a.chunks;
  const NormSpots p = norm_spots<V>(a, chunk, blockIdx.y);
  const T* const x = static_cast<const T*>(a.x) + n * a.x_ns + p.v * V;
  const T* const dy = BACKWARD ? static_cast<const T*>(a.dy) + n * a.dy_ns + p.v * V : nullptr;
  float s0[V], s1[V], ref[V];   // ref: the first value (forward), the mean (backward)
  [[maybe_unused]] float rs[V], w[V], b[V];
#pragma unroll
  for (int e = 0; e < V; ++e) s0[e] = s1[e] = 0.f;
  const auto spots_of = [&](int row) { return max(0, (p.last - p.first - row + p.rows - 1) / p.rows); };
  if (p.on && spots_of(p.row) > 0) {
    if (!BACKWARD) {
      load_values<T, V>(x + (p.first + p.row) * a.x_ss, ref);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int c = p.v * V + e;
        const float2 st = *reinterpret_cast<const float2*>(a.stats + (n * a.G + c / (a.C / a.G)) * 2);
        ref[e] = st.x;
        rs[e] = st.y;
        w[e] = a.w != nullptr ? a.w[c] : 1.f;
        b[e] = a.b != nullptr ? a.b[c] : 0.f;
      }
    }
    auto take = [&](const float (&f)[V], const float (&g)[V]) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (!BACKWARD) {
          const float d = f[e] - ref[e];
          s0[e] += d;
          s1[e] = fmaf(d, d, s1[e]);
        } else {
          const float h = (f[e] - ref[e]) * rs[e];
          const float dz = a.silu ? g[e] * silu_slope(fmaf(h, w[e], b[e])) : g[e];
          s0[e] += dz;
          s1[e] = fmaf(dz, h, s1[e]);
        }
      }
    };
    int i = p.first + p.row;
    for (; i + (kNormAhead - 1) * p.rows < p.last; i += kNormAhead * p.rows) {
      float f[kNormAhead][V], g[kNormAhead][V];
#pragma unroll
      for (int k = 0; k < kNormAhead; ++k) {
        load_values<T, V>(x + (i + k * p.rows) * a.x_ss, f[k]);
        if (BACKWARD) load_values<T, V>(dy + (i + k * p.rows) * a.dy_ss, g[k]);
      }
#pragma unroll
      for (int k = 0; k < kNormAhead; ++k) take(f[k], g[k]);
    }
    for (; i < p.last; i += p.rows) {
      float f[V], g[V];
      load_values<T, V>(x + i * a.x_ss, f);
      if (BACKWARD) load_values<T, V>(dy + i * a.dy_ss, g);
      take(f, g);
    }
  }
  const int here = min(a.C / V, 256);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    if (!BACKWARD && p.on && spots_of(p.row) > 0) {
      const float d = s0[e] / static_cast<float>(spots_of(p.row));
      s1[e] = fmaf(-d, s0[e], s1[e]);
      s0[e] = ref[e] + d;
    }
    acc[(threadIdx.x * V + e) * 2] = s0[e];
    acc[(threadIdx.x * V + e) * 2 + 1] = s1[e];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < here * V; c += 256) {
    const int at = blockIdx.y * 256 * V + c;
    if (at >= a.C) break;
    float t0 = acc[c * 2], t1 = acc[c * 2 + 1], n0 = static_cast<float>(spots_of(0));
    for (int r = 1; r < p.rows; ++r) {
      const float m = acc[(r * here * V + c) * 2], q = acc[(r * here * V + c) * 2 + 1], n1 = static_cast<float>(spots_of(r));
      if (BACKWARD) {
        t0 += m;
        t1 += q;
      } else if (n1 > 0.f) {   // two means and the squares around each
        const float d = m - t0, f = n1 / (n0 + n1);
        t0 = fmaf(d, f, t0);
        t1 += fmaf(d * d, n0 * f, q);
        n0 += n1;
      }
    }
    *reinterpret_cast<float2*>(a.part + ((n * a.chunks + chunk) * a.C + at) * 2) = make_float2(t0, t1);
  }
}

// Block (group, sample): chunks of a channel, then the group's channels.  Forward: mean and 1 / sqrt(var + eps); backward: the channel's
// sums to `chan`, c1 and c2.
__device__ __forceinline__ float2 block_sum2(float a, float b) {
  __shared__ float2 w[8];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
    b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) w[threadIdx.x >> 5] = make_float2(a, b);
  __syncthreads();
  float2 t = w[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) t = make_float2(t.x + w[i].x, t.y + w[i].y);
  return t;
}
template <bool BACKWARD>
__global__ void __launch_bounds__(256) group_norm_groups_kernel(const __grid_constant__ GroupNormArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  const int g = blockIdx.x % a.G, cg = a.C / a.G, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t n = blockIdx.x / a.G;
  const float spots = static_cast<float>(a.s);
  float2* const chan = reinterpret_cast<float2*>(a.chan) + n * a.C + g * cg;
  float u0 = 0.f, u1 = 0.f;
  for (int j = warp; j < cg; j += 8) {
    const int c = g * cg + j;
    const float2* const part = reinterpret_cast<const float2*>(a.part) + n * a.chunks * a.C + c;
    auto weight = [&](int k) { return static_cast<float>(min(a.per_chunk, a.s - k * a.per_chunk)); };
    float t0 = 0.f, t1 = 0.f;
    for (int k = lane; k < a.chunks; k += 32) {
      const float2 v = part[static_cast<int64_t>(k) * a.C];
      t0 += BACKWARD ? v.x : v.x * weight(k);
      if (BACKWARD) t1 += v.y;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      t0 += __shfl_xor_sync(0xFFFFFFFFu, t0, o);
      if (BACKWARD) t1 += __shfl_xor_sync(0xFFFFFFFFu, t1, o);
    }
    if (!BACKWARD) {   // the channel's mean, and its squares around it
      t0 /= spots;
      for (int k = lane; k < a.chunks; k += 32) {
        const float2 v = part[static_cast<int64_t>(k) * a.C];
        const float d = v.x - t0;
        t1 += fmaf(d * d, weight(k), v.y);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) t1 += __shfl_xor_sync(0xFFFFFFFFu, t1, o);
    }
    if (lane == 0) {
      chan[j] = make_float2(t0, t1);
      const float w = BACKWARD && a.w != nullptr ? a.w[c] : 1.f;
      u0 = fmaf(w, t0, u0);
      if (BACKWARD) u1 = fmaf(w, t1, u1);
    }
  }
  const float2 t = block_sum2(u0, u1);   // (its barriers: `chan` is there, too)
  if (!BACKWARD) {
    const float mean = t.x / static_cast<float>(cg);
    float m2 = 0.f;
    for (int j = threadIdx.x; j < cg; j += 256) {
      const float2 v = chan[j];
      const float d = v.x - mean;
      m2 += fmaf(spots * d, d, v.y);
    }
    const float m2s = block_sum2(m2, 0.f).x, var = (m2s < 0.f ? 0.f : m2s) / (spots * static_cast<float>(cg));
    if (threadIdx.x == 0) *reinterpret_cast<float2*>(a.stats + (n * a.G + g) * 2) = make_float2(mean, rsqrtf(var + a.eps));
  } else if (threadIdx.x == 0) {
    const float m = spots * static_cast<float>(cg);
    *reinterpret_cast<float2*>(a.coef + (n * a.G + g) * 2) = make_float2(t.x / m, t.y / m);
  }
}

// Backward: dw, db = sums of `chan` over the samples: 32 channels a block, 8 samples at a time.
__global__ void __launch_bounds__(256) group_norm_weights_kernel(const __grid_constant__ GroupNormArgs a) {
  __shared__ float2 acc[8][32];
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float2 t = make_float2(0.f, 0.f);
  if (c < a.C)
    for (int64_t n = warp; n < a.n; n += 8) {
      const float2 v = reinterpret_cast<const float2*>(a.chan)[n * a.C + c];
      t = make_float2(t.x + v.x, t.y + v.y);
    }
  acc[warp][lane] = t;
  __syncthreads();
  if (warp == 0 && c < a.C) {
    for (int i = 1; i < 8; ++i) t = make_float2(t.x + acc[i][lane].x, t.y + acc[i][lane].y);
    a.db[c] = t.x;
    a.dw[c] = t.y;
  }
}

// y, or dx.  The blocks go through samples and chunks from the last to the first: what the sums have read last is still in L2.
template <class T, int V, bool BACKWARD>
__global__ void __launch_bounds__(256) group_norm_apply_kernel(const __grid_constant__ GroupNormArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  const int turn = gridDim.x - 1 - blockIdx.x;
  const int64_t n = turn / a.chunks;
  const NormSpots p = norm_spots<V>(a, turn % a.chunks, blockIdx.y);
  if (!p.on) return;
  const T* const x = static_cast<const T*>(a.x) + n * a.x_ns + p.v * V;
  const T* const dy = BACKWARD ? static_cast<const T*>(a.dy) + n * a.dy_ns + p.v * V : nullptr;
  T* const out = static_cast<T*>(a.out) + n * a.s * a.C + p.v * V;
  // forward: z = (x - m) k + b;  backward: xhat = (x - m) k, z = xhat w + b, dx = dz w k - (c1 + xhat c2) k
  float k[V], m[V], b[V];
  [[maybe_unused]] float w[V], c1[V], c2[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int c = p.v * V + e, g = c / (a.C / a.G);
    const float2 st = *reinterpret_cast<const float2*>(a.stats + (n * a.G + g) * 2);
    const float wc = a.w != nullptr ? a.w[c] : 1.f;
    m[e] = st.x;
    b[e] = a.b != nullptr ? a.b[c] : 0.f;
    if (!BACKWARD) {
      k[e] = st.y * wc;
    } else {
      const float2 cc = *reinterpret_cast<const float2*>(a.coef + (n * a.G + g) * 2);
      k[e] = st.y;
      w[e] = wc;
      c1[e] = cc.x * st.y;
      c2[e] = cc.y * st.y;
    }
  }
  auto work = [&](float (&f)[V], const float (&g)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (!BACKWARD) {
        const float z = fmaf(f[e] - m[e], k[e], b[e]);
        f[e] = a.silu ? silu_of(z) : z;
      } else {
        const float h = (f[e] - m[e]) * k[e];
        const float dz = a.silu ? g[e] * silu_slope(fmaf(h, w[e], b[e])) : g[e];
        f[e] = fmaf(dz, w[e] * k[e], -fmaf(h, c2[e], c1[e]));
      }
    }
  };
  int i = p.first + p.row;
  for (; i + (kNormAhead - 1) * p.rows < p.last; i += kNormAhead * p.rows) {
    float f[kNormAhead][V], g[kNormAhead][V];
#pragma unroll
    for (int j = 0; j < kNormAhead; ++j) {
      load_values<T, V>(x + (i + j * p.rows) * a.x_ss, f[j]);
      if (BACKWARD) load_values<T, V>(dy + (i + j * p.rows) * a.dy_ss, g[j]);
    }
#pragma unroll
    for (int j = 0; j < kNormAhead; ++j) {
      work(f[j], g[j]);
      store_values<T, V>(out + static_cast<int64_t>(i + j * p.rows) * a.C, f[j]);
    }
  }
  for (; i < p.last; i += p.rows) {
    float f[V], g[V];
    load_values<T, V>(x + i * a.x_ss, f);
    if (BACKWARD) load_values<T, V>(dy + i * a.dy_ss, g);
    work(f, g);
    store_values<T, V>(out + static_cast<int64_t>(i) * a.C, f);
  }
}

}  // namespace lact

// Group norm with an activation, channels last: x [n][s][C], the C channels in G groups of adjacent ones; per sample and group
//   xhat = (x - mean) / sqrt(var + eps)  over its s spots and C / G channels,  z = xhat w_c + b_c,  y = z or z sigmoid(z).
// Backward, with dz = dy (or dy * d silu(z)):  dw_c = sum dz xhat, db_c = sum dz over samples and spots, and per sample and group
//   dx = (dz w - c1 - xhat c2) / sqrt(var + eps),  c1 = mean(dz w),  c2 = mean(dz w xhat).
// Bound by memory: x and y once are what it cannot do without (x, dy, dx backward).  Two ways:
//   one spot a sample (the norm per head of tokens): a row is read into registers, its groups are summed among the threads that hold
//     them, mean first and then squares of what is left; one pass over memory, one launch.
//   many spots: threads keep their channels and walk the spots, so that 16 bytes are read whatever a group's width is; every thread
//     sums against the first value it sees and hands on a mean and the squares around it (no cancellation where the mean is far from
//     zero); a small launch puts chunks and channels of a group together, a last one reads x again and writes.
// Measured: 65536 tokens of 1536 in 12 groups, bf16, 111 us forward and 167 backward (3.6 TB/s; instruction issue two thirds busy);
// 2 frames of 480 x 832 x 96 38 + 6 + 51 us (sums 4.0, outputs 6.0 TB/s).
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
  float* part;                // [n][C][chunks][2]; one spot, backward: [blocks][2][C]
  float* chan;                // [n][C][2]
  float* coef;                // backward: [n][G][2]: c1, c2
  float *dw, *db;             // [C]
  int64_t n, x_ns, x_ss, dy_ns, dy_ss;
  int32_t s, C, G, silu;
  int32_t chunks, per_chunk;  // spots of a sample are dealt to `chunks` blocks
  float eps;
};

// V values of type T, as one access
template <int BYTES>
struct Raw;
template <> struct Raw<16> { using type = uint4; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<4> { using type = uint32_t; };
template <> struct Raw<2> { using type = uint16_t; };
template <class T, int V>
using RawOf = typename Raw<V * sizeof(T)>::type;
template <class T, int V>
__device__ __forceinline__ RawOf<T, V> load_raw(const T* p) {
  return *reinterpret_cast<const RawOf<T, V>*>(p);
}
// (bf16 in pairs: one instruction a value either way)
template <class T, int V>
__device__ __forceinline__ void values_of(const RawOf<T, V>& r, float (&f)[V]) {
  if constexpr (sizeof(T) == 2 && V >= 2) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      f[i] = __uint_as_float(w[i / 2] << 16);
      f[i + 1] = __uint_as_float(w[i / 2] & 0xFFFF0000u);
    }
  } else {
    const T* t = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = static_cast<float>(t[i]);
  }
}
template <class T, int V>
__device__ __forceinline__ void store_values(T* p, const float (&f)[V]) {
  RawOf<T, V> r;
  if constexpr (sizeof(T) == 2 && V >= 2) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < V; i += 2) w[i / 2] = pack_bf16x2(f[i], f[i + 1]);
  } else {
    T* t = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = static_cast<T>(f[i]);
  }
  *reinterpret_cast<RawOf<T, V>*>(p) = r;
}
// Arithmetic on V values, two at a time (a large call has a budget of 20 instructions an element while its memory arrives)
template <int V>
__device__ __forceinline__ void v_fma(float (&d)[V], const float (&a)[V], const float (&b)[V], const float (&c)[V]) {
  if constexpr (V == 1) d[0] = fmaf(a[0], b[0], c[0]);
  else
#pragma unroll
    for (int i = 0; i < V; i += 2) f32x2_split(f32x2_fma(f32x2(a[i], a[i + 1]), f32x2(b[i], b[i + 1]), f32x2(c[i], c[i + 1])), d[i], d[i + 1]);
}
template <int V>
__device__ __forceinline__ void v_mul(float (&d)[V], const float (&a)[V], const float (&b)[V]) {
  if constexpr (V == 1) d[0] = a[0] * b[0];
  else
#pragma unroll
    for (int i = 0; i < V; i += 2) f32x2_split(f32x2_mul(f32x2(a[i], a[i + 1]), f32x2(b[i], b[i + 1])), d[i], d[i + 1]);
}
template <int V>
__device__ __forceinline__ void v_add(float (&d)[V], const float (&a)[V], const float (&b)[V]) {
  if constexpr (V == 1) d[0] = a[0] + b[0];
  else
#pragma unroll
    for (int i = 0; i < V; i += 2) f32x2_split(f32x2_add(f32x2(a[i], a[i + 1]), f32x2(b[i], b[i + 1])), d[i], d[i + 1]);
}
template <int V>
__device__ __forceinline__ void v_set(float (&d)[V], float x) {
#pragma unroll
  for (int i = 0; i < V; ++i) d[i] = x;
}
template <int V>
__device__ __forceinline__ float v_sum(const float (&a)[V]) {
  if constexpr (V == 1) return a[0];
  else {
    F32x2 t = f32x2(a[0], a[1]);
#pragma unroll
    for (int i = 2; i < V; i += 2) t = f32x2_add(t, f32x2(a[i], a[i + 1]));
    float x, y;
    f32x2_split(t, x, y);
    return x + y;
  }
}
// sum of products
template <int V>
__device__ __forceinline__ float v_dot(const float (&a)[V], const float (&b)[V]) {
  if constexpr (V == 1) return a[0] * b[0];
  else {
    F32x2 t = f32x2_mul(f32x2(a[0], a[1]), f32x2(b[0], b[1]));
#pragma unroll
    for (int i = 2; i < V; i += 2) t = f32x2_fma(f32x2(a[i], a[i + 1]), f32x2(b[i], b[i + 1]), t);
    float x, y;
    f32x2_split(t, x, y);
    return x + y;
  }
}

// sigmoid(z) of V values.  Two special-function results an element (16 a clock and SM) take as long as the memory of a large call
// (77 million elements: 34 us; two frames of 480 x 832 x 96 come and go in 47): two neighbours share one reciprocal, 1 / a = b (1 / ab).
// Below z = -41 the sigmoid stays at 2^-60, so that the product stays finite (silu is off by |z| 2^-60: less than 2^-40 at z = -10^6).
template <int V>
__device__ __forceinline__ void sigmoids(const float (&z)[V], float (&g)[V]) {
  if constexpr (V == 1) {
    g[0] = sigmoidf_fast(z[0]);
  } else {
    const F32x2 k = f32x2(-1.4426950408889634f, -1.4426950408889634f), one = f32x2(1.f, 1.f);
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      float x0, x1, a, b;
      f32x2_split(f32x2_mul(f32x2(z[i], z[i + 1]), k), x0, x1);
      // (of NaN the minimum is 60: the callers multiply by z)
      f32x2_split(f32x2_add(f32x2(exp2_ftz(fminf(x0, 60.f)), exp2_ftz(fminf(x1, 60.f))), one), a, b);
      const float r = rcp_ftz(a * b);
      g[i] = r * b;
      g[i + 1] = r * a;
    }
  }
}
// z -> z sigmoid(z), and its slope
template <int V>
__device__ __forceinline__ void silu_of(float (&z)[V]) {
  float g[V];
  sigmoids(z, g);
  v_mul(z, z, g);
}
template <int V>
__device__ __forceinline__ void silu_slope(float (&z)[V]) {   // g (1 + z (1 - g)) = g + z (g - g g)
  float g[V], h[V], n[V];
  sigmoids(z, g);
#pragma unroll
  for (int i = 0; i < V; ++i) n[i] = -g[i];
  v_fma(h, n, g, g);
  v_fma(z, z, h, g);
}

// ---------------------------------------------------------------- one spot a sample
// A row is a thread per vector of V channels (a group holds whole vectors) and as many rows a block as make 256 threads, or, past 256
// vectors, K of them a thread.  Sums of a group: among neighbouring lanes where it has 1, 2, .. 32 vectors, through shared memory
// otherwise.
struct GroupSums {
  float* vec;     // [rows][vectors]
  float* sum;     // [rows][G]
  int gv, G, nv, rows;
  bool lanes;     // gv a power of two, at most 32
  // p[i]: this thread's sum of vector l + 256 i of its row -> the sum over the vector's group
  template <int K>
  __device__ __forceinline__ void among_lanes(float (&p)[K]) const {
    for (int o = 1; o < gv; o <<= 1)
#pragma unroll
      for (int i = 0; i < K; ++i) p[i] += __shfl_xor_sync(0xFFFFFFFFu, p[i], o);
  }
  template <int K>
  __device__ __forceinline__ void in_memory(float* p, int row, int l, bool here) const {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < K; ++i)
      if (here && l + i * 256 < nv) vec[row * nv + l + i * 256] = p[i];
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int it = warp; it < rows * G; it += blockDim.x >> 5) {
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
      if (here && l + i * 256 < nv) p[i] = sum[row * G + (l + i * 256) / gv];
  }
  // M = K vectors of each of several rows
  template <int K, int M>
  __device__ __forceinline__ void operator()(float (&p)[M], int row, int l, bool here) const {
    if (lanes) among_lanes(p);
    else
#pragma unroll
      for (int r = 0; r < M; r += K) in_memory<K>(p + r, row, l, here);
  }
};

// R rows of a thread at a time, fetched together while those before are worked on side by side.
constexpr int kNormRowsAtOnce = 2;
template <class T, int V, int K, int R, bool BACKWARD>
__global__ void __launch_bounds__(256, 3) group_norm_rows_kernel(const __grid_constant__ GroupNormArgs a, int32_t rows) {
  constexpr int M = K * R;
  extern __shared__ float norm_smem[];
  griddep_launch_dependents();
  griddep_wait();
  const int nv = a.C / V, gv = nv / a.G;
  const int row = K > 1 ? 0 : threadIdx.x / nv, l = K > 1 ? threadIdx.x : threadIdx.x - row * nv;
  const bool here = row < rows;
  const GroupSums sums{norm_smem, norm_smem + rows * nv, gv, a.G, nv, rows, (gv & (gv - 1)) == 0 && gv <= 32};
  const float inv = 1.f / (gv * V);
  float w[K][V], b[K][V];
#pragma unroll
  for (int i = 0; i < K; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int v = l + i * 256, c = v * V + e;
      w[i][e] = here && v < nv && a.w != nullptr ? a.w[c] : 1.f;
      b[i][e] = here && v < nv && a.b != nullptr ? a.b[c] : 0.f;
    }
  [[maybe_unused]] float dw[BACKWARD ? K : 1][V], db[BACKWARD ? K : 1][V];
  if (BACKWARD) {
#pragma unroll
    for (int i = 0; i < K; ++i) {
      v_set(dw[i], 0.f);
      v_set(db[i], 0.f);
    }
  }
  const int64_t step = static_cast<int64_t>(gridDim.x) * rows * R;
  int64_t n0 = static_cast<int64_t>(blockIdx.x) * rows * R;
  // (entry j: vector l + 256 (j % K) of row n0 + row + rows (j / K))
  auto sample = [&](int j) { return n0 + row + static_cast<int64_t>(rows) * (j / K); };
  auto vector = [&](int j) { return l + 256 * (j % K); };
  auto on = [&](int j) { return here && vector(j) < nv && sample(j) < a.n; };
  RawOf<T, V> raw[M];
  [[maybe_unused]] RawOf<T, V> raw_dy[BACKWARD ? M : 1];
  [[maybe_unused]] float2 st[BACKWARD ? M : 1];
  auto fetch = [&]() {   // entries that are not there: zeros all through
#pragma unroll
    for (int j = 0; j < M; ++j) {
      raw[j] = RawOf<T, V>{};
      if constexpr (BACKWARD) {
        raw_dy[j] = RawOf<T, V>{};
        st[j] = make_float2(0.f, 0.f);
      }
      if (!on(j)) continue;
      raw[j] = load_raw<T, V>(static_cast<const T*>(a.x) + sample(j) * a.x_ns + vector(j) * V);
      if constexpr (BACKWARD) {
        raw_dy[j] = load_raw<T, V>(static_cast<const T*>(a.dy) + sample(j) * a.dy_ns + vector(j) * V);
        st[j] = *reinterpret_cast<const float2*>(a.stats + (sample(j) * a.G + vector(j) / gv) * 2);
      }
    }
  };
  fetch();
  for (; n0 < a.n; n0 += step) {
    auto fetch_next = [&]() {   // (on their way while the values of these are worked on)
      n0 += step;
      fetch();
      n0 -= step;
    };
    float x[M][V], p[M];
    if constexpr (!BACKWARD) {
      float mean[M];
#pragma unroll
      for (int j = 0; j < M; ++j) {
        values_of<T, V>(raw[j], x[j]);
        p[j] = v_sum(x[j]);
      }
      fetch_next();
      sums.template operator()<K>(p, row, l, here);
#pragma unroll
      for (int j = 0; j < M; ++j) {
        mean[j] = p[j] * inv;
        float m[V];
        v_set(m, -mean[j]);
        v_add(x[j], x[j], m);
        p[j] = v_dot(x[j], x[j]);
      }
      sums.template operator()<K>(p, row, l, here);
#pragma unroll
      for (int j = 0; j < M; ++j) {
        const float rstd = rsqrtf(fmaf(p[j], inv, a.eps));
        if (!on(j)) continue;
        if (vector(j) % gv == 0) *reinterpret_cast<float2*>(a.stats + (sample(j) * a.G + vector(j) / gv) * 2) = make_float2(mean[j], rstd);
        float k[V];
        v_set(k, rstd);
        v_mul(k, k, w[j % K]);
        v_fma(x[j], x[j], k, b[j % K]);
        if (a.silu) silu_of(x[j]);
        store_values<T, V>(static_cast<T*>(a.out) + sample(j) * a.C + vector(j) * V, x[j]);
      }
    } else {
      float t[M][V], q[M], rstd[M];
#pragma unroll
      for (int j = 0; j < M; ++j) {
        rstd[j] = st[j].y;
        values_of<T, V>(raw[j], x[j]);
        values_of<T, V>(raw_dy[j], t[j]);
        float k[V], z[V];
        v_set(k, -st[j].x);
        v_add(x[j], x[j], k);
        v_set(k, st[j].y);
        v_mul(x[j], x[j], k);
        if (a.silu) {
          v_fma(z, x[j], w[j % K], b[j % K]);
          silu_slope(z);
          v_mul(t[j], t[j], z);
        }
        v_add(db[j % K], db[j % K], t[j]);
        v_fma(dw[j % K], t[j], x[j], dw[j % K]);
        v_mul(t[j], t[j], w[j % K]);
        p[j] = v_sum(t[j]);
        q[j] = v_dot(t[j], x[j]);
      }
      fetch_next();
      sums.template operator()<K>(p, row, l, here);
      sums.template operator()<K>(q, row, l, here);
#pragma unroll
      for (int j = 0; j < M; ++j) {
        if (!on(j)) continue;
        float c1[V], c2[V], k[V];   // (dz w - c1 first: where a group is one value, nothing is left of it)
        v_set(c1, -p[j] * inv);
        v_set(c2, -q[j] * inv);
        v_set(k, rstd[j]);
        v_add(t[j], t[j], c1);
        v_fma(x[j], x[j], c2, t[j]);
        v_mul(x[j], x[j], k);
        store_values<T, V>(static_cast<T*>(a.out) + sample(j) * a.C + vector(j) * V, x[j]);
      }
    }
  }
  if constexpr (BACKWARD) {
    // the block's sums over its rows, [2][C]: a column's rows of threads are added in their order
    float* const part = a.part + static_cast<int64_t>(blockIdx.x) * 2 * a.C;
    if (K > 1) {
#pragma unroll
      for (int i = 0; i < K; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int c = (l + i * 256) * V + e;
          if (l + i * 256 >= nv) continue;
          part[c] = dw[i][e];
          part[a.C + c] = db[i][e];
        }
      return;
    }
    float* const acc = norm_smem;   // [2][rows][C]
    __syncthreads();
    if (here) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        acc[row * a.C + l * V + e] = dw[0][e];
        acc[(rows + row) * a.C + l * V + e] = db[0][e];
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * a.C; c += blockDim.x) {
      const float* from = acc + (c < a.C ? c : rows * a.C + c - a.C);
      float t = 0.f;
      for (int r = 0; r < rows; ++r) t += from[r * a.C];
      part[c] = t;
    }
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
// A thread's spots, N of them fetched together.
constexpr int kNormAhead = 4;
template <class T, int V, bool BOTH, class Work>
__device__ __forceinline__ void norm_walk(const T* x, const T* dy, const GroupNormArgs& a, const NormSpots& p, const Work& work) {
  constexpr int N = kNormAhead;
  int i = p.first + p.row;
  for (; i + (N - 1) * p.rows < p.last; i += N * p.rows) {
    RawOf<T, V> rx[N], rdy[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      rx[k] = load_raw<T, V>(x + (i + k * p.rows) * a.x_ss);
      if (BOTH) rdy[k] = load_raw<T, V>(dy + (i + k * p.rows) * a.dy_ss);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) work(i + k * p.rows, rx[k], BOTH ? rdy[k] : rx[k]);
  }
  for (; i < p.last; i += p.rows) {
    const RawOf<T, V> rx = load_raw<T, V>(x + i * a.x_ss);
    work(i, rx, BOTH ? load_raw<T, V>(dy + i * a.dy_ss) : rx);
  }
}

// Per channel of a chunk -> part[n][c][chunk]: forward the mean and the sum of squares around it, backward the sums of dz and dz xhat.
template <class T, int V, bool BACKWARD>
__global__ void __launch_bounds__(256, BACKWARD ? 2 : 4) group_norm_sums_kernel(const __grid_constant__ GroupNormArgs a) {
  __shared__ float acc[256 * V * 2];
  griddep_launch_dependents();
  griddep_wait();
  const int chunk = blockIdx.x % a.chunks;
  const int64_t n = blockIdx.x / a.chunks;
  const NormSpots p = norm_spots<V>(a, chunk, blockIdx.y);
  const T* const x = static_cast<const T*>(a.x) + n * a.x_ns + p.v * V;
  const T* const dy = BACKWARD ? static_cast<const T*>(a.dy) + n * a.dy_ns + p.v * V : nullptr;
  float s0[V], s1[V], ref[V];   // ref: minus the first value (forward) or the mean (backward)
  [[maybe_unused]] float rs[V], w[V], b[V];
#pragma unroll
  for (int e = 0; e < V; ++e) s0[e] = s1[e] = 0.f;
  const auto spots_of = [&](int row) { return max(0, (p.last - p.first - row + p.rows - 1) / p.rows); };
  if (p.on && spots_of(p.row) > 0) {
    if (!BACKWARD) {
      values_of<T, V>(load_raw<T, V>(x + (p.first + p.row) * a.x_ss), ref);
#pragma unroll
      for (int e = 0; e < V; ++e) ref[e] = -ref[e];
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int c = p.v * V + e;
        const float2 st = *reinterpret_cast<const float2*>(a.stats + (n * a.G + c / (a.C / a.G)) * 2);
        ref[e] = -st.x;
        rs[e] = st.y;
        w[e] = a.w != nullptr ? a.w[c] : 1.f;
        b[e] = a.b != nullptr ? a.b[c] : 0.f;
      }
    }
    auto take = [&](const RawOf<T, V>& rx, const RawOf<T, V>& rdy) {
      float f[V], g[V], z[V];
      values_of<T, V>(rx, f);
      v_add(f, f, ref);
      if (!BACKWARD) {
        v_add(s0, s0, f);
        v_fma(s1, f, f, s1);
      } else {
        values_of<T, V>(rdy, g);
        v_mul(f, f, rs);
        if (a.silu) {
          v_fma(z, f, w, b);
          silu_slope(z);
          v_mul(g, g, z);
        }
        v_add(s0, s0, g);
        v_fma(s1, g, f, s1);
      }
    };
    norm_walk<T, V, BACKWARD>(x, dy, a, p, [&](int, const RawOf<T, V>& rx, const RawOf<T, V>& rdy) { take(rx, rdy); });
  }
  const int here = min(a.C / V, 256);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    if (!BACKWARD && p.on && spots_of(p.row) > 0) {
      const float d = s0[e] / static_cast<float>(spots_of(p.row));
      s1[e] = fmaf(-d, s0[e], s1[e]);
      s0[e] = d - ref[e];
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
    reinterpret_cast<float2*>(a.part)[(n * a.C + at) * a.chunks + chunk] = make_float2(t0, t1);
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
    const float2* const part = reinterpret_cast<const float2*>(a.part) + (n * a.C + c) * a.chunks;
    auto weight = [&](int k) { return static_cast<float>(min(a.per_chunk, a.s - k * a.per_chunk)); };
    float t0 = 0.f, t1 = 0.f;
#pragma unroll 4
    for (int k = lane; k < a.chunks; k += 32) {
      const float2 v = part[k];
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
#pragma unroll 4
      for (int k = lane; k < a.chunks; k += 32) {
        const float2 v = part[k];
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

// Backward: dw, db: 32 channels, from sums of `n` rows, eight at a time.
__device__ __forceinline__ void norm_weights(const GroupNormArgs& a, int c, int64_t n, const float* first, const float* second, int64_t step,
                                             int64_t next) {
  __shared__ float2 acc[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float2 t = make_float2(0.f, 0.f);
  if (c < a.C) {
#pragma unroll 16
    for (int64_t i = warp; i < n; i += 8) {
      t.x += first[c * step + i * next];
      t.y += second[c * step + i * next];
    }
  }
  acc[warp][lane] = t;
  __syncthreads();
  if (warp == 0 && c < a.C) {
    for (int i = 1; i < 8; ++i) t = make_float2(t.x + acc[i][lane].x, t.y + acc[i][lane].y);
    a.dw[c] = t.x;
    a.db[c] = t.y;
  }
}
// ... of the blocks of group_norm_rows_kernel
__global__ void __launch_bounds__(256) group_norm_weights_kernel(const __grid_constant__ GroupNormArgs a, int32_t blocks) {
  griddep_launch_dependents();
  griddep_wait();
  norm_weights(a, blockIdx.x * 32 + (threadIdx.x & 31), blocks, a.part, a.part + a.C, 1, 2ll * a.C);
}

// y, or dx.  The blocks go through samples and chunks from the last to the first.  Forward, where all of them are resident at once (as the
// sums' are), that changes nothing: 46.1 us of a whole call at 51 MB, 54.3 at 67, 99.4 at 153 either way.  Backward there are two waves, and
// the first takes what the sums' second has read: 52.2, 66.6 and 80.9 us at 34, 51 and 67 MB a tensor against 54.3, 68.7 and 83.0 from the
// first to the last; past L2 (133 MB and more) the same.
template <class T, int V, bool BACKWARD>
__global__ void __launch_bounds__(256, BACKWARD ? 2 : 4) group_norm_apply_kernel(const __grid_constant__ GroupNormArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  const int64_t most = a.n * a.chunks;
  if (BACKWARD && blockIdx.x >= most) {   // (sums of dz and of dz xhat per sample and channel)
    const int64_t c = ((blockIdx.x - most) * gridDim.y + blockIdx.y) * 32 + (threadIdx.x & 31);
    norm_weights(a, static_cast<int>(min(c, static_cast<int64_t>(a.C))), a.n, a.chan + 1, a.chan, 2, 2ll * a.C);
    return;
  }
  const int turn = static_cast<int>(most - 1 - blockIdx.x);
  const int64_t n = turn / a.chunks;
  const NormSpots p = norm_spots<V>(a, turn % a.chunks, blockIdx.y);
  if (!p.on) return;
  const T* const x = static_cast<const T*>(a.x) + n * a.x_ns + p.v * V;
  const T* const dy = BACKWARD ? static_cast<const T*>(a.dy) + n * a.dy_ns + p.v * V : nullptr;
  T* const out = static_cast<T*>(a.out) + n * a.s * a.C + p.v * V;
  // forward: z = (x + m) k + b, m minus the mean;  backward: xhat = (x + m) k, z = xhat w + b, dx = (dz w - c1 - xhat c2) k
  float k[V], m[V], b[V];
  [[maybe_unused]] float w[V], c1[V], c2[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int c = p.v * V + e, g = c / (a.C / a.G);
    const float2 st = *reinterpret_cast<const float2*>(a.stats + (n * a.G + g) * 2);
    const float wc = a.w != nullptr ? a.w[c] : 1.f;
    m[e] = -st.x;
    b[e] = a.b != nullptr ? a.b[c] : 0.f;
    if (!BACKWARD) {
      k[e] = st.y * wc;
    } else {
      const float2 cc = *reinterpret_cast<const float2*>(a.coef + (n * a.G + g) * 2);
      k[e] = st.y;
      w[e] = wc;
      c1[e] = -cc.x;
      c2[e] = -cc.y;
    }
  }
  norm_walk<T, V, BACKWARD>(x, dy, a, p, [&](int i, const RawOf<T, V>& rx, const RawOf<T, V>& rdy) {
    float f[V], g[V], z[V];
    values_of<T, V>(rx, f);
    v_add(f, f, m);
    if (!BACKWARD) {
      v_fma(f, f, k, b);
      if (a.silu) silu_of(f);
    } else {
      values_of<T, V>(rdy, g);
      v_mul(f, f, k);
      if (a.silu) {
        v_fma(z, f, w, b);
        silu_slope(z);
        v_mul(g, g, z);
      }
      v_mul(g, g, w);
      v_add(g, g, c1);
      v_fma(f, f, c2, g);
      v_mul(f, f, k);
    }
    store_values<T, V>(out + static_cast<int64_t>(i) * a.C, f);
  });
}

}  // namespace lact

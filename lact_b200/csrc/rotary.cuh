// Rotary positions with several axes.  A token has one position per axis (text: one; images: two; video: time, height, width), the P
// rotated pairs of a head are dealt to the axes in sections, and pair j of axis a turns by  t = position[a] * frequency[j]:
//   (x, y) -> (x cos t - y sin t,  y cos t + x sin t);   the gradient turns by -t (`sign`).
// Pairs are (j, j + P) or neighbours (2j, 2j + 1); elements from 2 P on are copied.
// Bound by memory: every element is read and written once.  A block takes several tokens, works out their cosines and sines once into
// shared memory, and each thread keeps those of its V pairs in registers while it goes through its share of the token's heads (queries
// first, then keys).  Angles are taken in turns, in fp64 (a position of 2^31 leaves 2^-21 of a turn), and reduced to half a turn
// before they become fp32.
#pragma once
#include "group_norm.cuh"

namespace lact {

constexpr int kRotaryAxes = 8;
struct RotaryArgs {
  const void* x[2];             // queries, keys: [batch][tokens][heads][d], features adjacent, other strides in elements
  void* y[2];                   // contiguous
  int64_t bs[2], ts[2], hs[2];
  int32_t heads[2];
  const void* pos;              // int32 or int64, [batch or shared][tokens][axes]
  int64_t pos_bs, pos_ts, pos_as;
  int32_t pos_wide, axes;
  int32_t ends[kRotaryAxes];    // pair j is of the first axis whose end is above j
  const double* freq;           // [P], radians per position
  int64_t tokens;               // batch * L
  int32_t L, d, P;
  float sign;
  int32_t share, per_block;     // thread groups that share a token's heads; tokens of a block
};

// cos and sin of `turn` (-1/2 to 1/2 of a full turn).  For bf16 results the hardware's own approximations do (absolute error 2^-20.9
// in this range, a bf16 result is rounded by 2^-9); fp32 results take the accurate functions.
template <class T>
__device__ __forceinline__ float2 rotary_angle(float turn) {
  float s, c;
  if constexpr (sizeof(T) == 2) {
    const float t = turn * 6.283185307179586f;
    s = __sinf(t);
    c = __cosf(t);
  } else {
    sincospif(2.f * turn, &s, &c);
  }
  return make_float2(c, s);
}

// (the products and sums are named, so that a result's last bit does not depend on the width of the accesses)
__device__ __forceinline__ void turned_pair(float x, float y, float c, float s, float& u, float& v) {
  u = fmaf(x, c, -__fmul_rn(y, s));
  v = fmaf(y, c, __fmul_rn(x, s));
}

constexpr int kRotaryThreads = 256;
constexpr int kRotaryHeadsAtOnce = 3;   // of a thread, fetched together
template <class T, int V, bool HALVES>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  extern __shared__ float2 rotary_smem[];   // [per_block][P]
  griddep_launch_dependents();
  griddep_wait();
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.per_block;
  const int here = static_cast<int>(min(static_cast<int64_t>(a.per_block), a.tokens - t0));
  for (int i = threadIdx.x; i < here * a.P; i += kRotaryThreads) {
    const int j = i % a.P;
    const int64_t t = t0 + i / a.P, b = t / a.L, l = t - b * a.L;
    int axis = 0;
    while (axis < a.axes - 1 && j >= a.ends[axis]) ++axis;
    const int64_t at = b * a.pos_bs + l * a.pos_ts + axis * a.pos_as;
    const double p = a.pos_wide ? static_cast<double>(static_cast<const int64_t*>(a.pos)[at]) : static_cast<double>(static_cast<const int32_t*>(a.pos)[at]);
    const double turns = p * (a.freq[j] * 0.15915494309189535);
    float2 cs = rotary_angle<T>(static_cast<float>(turns - rint(turns)));
    cs.y *= a.sign;
    rotary_smem[i] = cs;
  }
  __syncthreads();
  const int nc = a.d / (2 * V), c = threadIdx.x % nc, slot = threadIdx.x / nc;   // this thread's 2 V features
  const int tok = slot / a.share, part = slot - tok * a.share;
  if (tok >= here) return;
  const int64_t t = t0 + tok, b = t / a.L, l = t - b * a.L;
  const bool turned = c * V < a.P;   // (the others are copied)
  float co[V], si[V];
  if (turned) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float2 cs = rotary_smem[tok * a.P + c * V + e];
      co[e] = cs.x;
      si[e] = cs.y;
    }
  }
  const int first = turned && HALVES ? c * V : 2 * c * V, second = turned && HALVES ? a.P + c * V : 2 * c * V + V;
  const int all = a.heads[0] + a.heads[1];
  using Raw = RawOf<T, V>;
  constexpr int N = kRotaryHeadsAtOnce;
  for (int h0 = part; h0 < all; h0 += N * a.share) {
    Raw ra[N], rb[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int h = h0 + k * a.share;
      if (h >= all) continue;
      const int w = h >= a.heads[0];
      const T* x = static_cast<const T*>(a.x[w]) + b * a.bs[w] + l * a.ts[w] + (w ? h - a.heads[0] : h) * a.hs[w];
      ra[k] = load_raw<T, V>(x + first);
      rb[k] = load_raw<T, V>(x + second);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int h = h0 + k * a.share;
      if (h >= all) continue;
      const int w = h >= a.heads[0];
      T* y = static_cast<T*>(a.y[w]) + (t * a.heads[w] + (w ? h - a.heads[0] : h)) * a.d;
      if (!turned) {
        *reinterpret_cast<Raw*>(y + first) = ra[k];
        *reinterpret_cast<Raw*>(y + second) = rb[k];
        continue;
      }
      float p[V], q[V], u[V], z[V];
      values_of<T, V>(ra[k], p);
      values_of<T, V>(rb[k], q);
      if constexpr (HALVES) {
#pragma unroll
        for (int e = 0; e < V; ++e) turned_pair(p[e], q[e], co[e], si[e], u[e], z[e]);
      } else {   // 2 V neighbours: V values in p, V in q
        float f[2 * V], g[2 * V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          f[e] = p[e];
          f[V + e] = q[e];
        }
#pragma unroll
        for (int e = 0; e < V; ++e) turned_pair(f[2 * e], f[2 * e + 1], co[e], si[e], g[2 * e], g[2 * e + 1]);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          u[e] = g[e];
          z[e] = g[V + e];
        }
      }
      store_values<T, V>(y + first, u);
      store_values<T, V>(y + second, z);
    }
  }
}

}  // namespace lact

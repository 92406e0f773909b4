// Rotary positions with several axes.  A token has one position per axis (text: one; images: two; video: time, height, width), the P
// rotated pairs of a head are dealt to the axes in sections, and pair j of axis a turns by  t = position[a] * frequency[j]:
//   (x, y) -> (x cos t - y sin t,  y cos t + x sin t);   the gradient turns by -t (`sign`).
// Pairs are (j, j + P) or neighbours (2j, 2j + 1); elements from 2 P on are copied.
// Bound by memory: every element is read and written once.  A block takes several tokens, works out their cosines and sines once into
// shared memory, and each thread keeps those of its V pairs in registers for its share of the token's heads (queries
// first, then keys).  Angles are whole numbers of 2^-64 turns, in which products with a position drop full turns by themselves: what a
// position of 2^31 is off by is 2^-24 of a turn at a frequency of 1 (2^-56 each from the frequency's product in fp64 and its constant).
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
template <class T, int V, bool HALVES, bool AHEAD, int N, int PER_SM>   // N heads of a thread are fetched together; AHEAD: all it has, ahead of the angles
__global__ void __launch_bounds__(kRotaryThreads, PER_SM) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  extern __shared__ float rotary_smem[];   // cosines [per_block][P], sines
  griddep_launch_dependents();
  griddep_wait();
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.per_block, b0 = t0 / a.L;
  const int l0 = static_cast<int>(t0 - b0 * a.L), here = static_cast<int>(min(static_cast<int64_t>(a.per_block), a.tokens - t0));
  auto token = [&](int i, int64_t& b, int& l) {   // batch entry and token of the block's i-th
    b = b0;
    l = l0 + i;
    if (l >= a.L) {
      b += l / a.L;
      l %= a.L;
    }
  };
  const int nc = a.d / (2 * V), c = threadIdx.x % nc, slot = threadIdx.x / nc;
  const int tok = slot / a.share, part = slot - tok * a.share;
  const int64_t t = t0 + tok;
  const int all = tok < here ? a.heads[0] + a.heads[1] : 0;   // (behind the last token: none)
  int64_t b;
  int l;
  token(tok, b, l);
  // This thread's two accesses of V features: of halves, those of V pairs (or two that are copied); of neighbours one in each half of
  // the head, V / 2 pairs each (accesses next to one another would leave every other one to a second instruction: 185 against 160 us
  // for 32760 tokens of 24 heads of 128, forward and backward); single features are a pair's two.
  constexpr bool APART = !HALVES && V > 1;
  const bool turned[2] = {APART ? c * V < 2 * a.P : c * V < a.P, APART ? (c + nc) * V < 2 * a.P : c * V < a.P};
  const int first = APART || (HALVES && turned[0]) ? c * V : 2 * c * V, second = APART ? (c + nc) * V : HALVES && turned[0] ? a.P + c * V : 2 * c * V + V;
  using Raw = RawOf<T, V>;
  Raw ra[N], rb[N];
  auto fetch = [&](int h0) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int h = h0 + k * a.share;
      if (h >= all) continue;
      const int w = h >= a.heads[0];
      const T* x = static_cast<const T*>(a.x[w]) + b * a.bs[w] + l * a.ts[w] + (w ? h - a.heads[0] : h) * a.hs[w];
      ra[k] = load_raw<T, V>(x + first);
      rb[k] = load_raw<T, V>(x + second);
    }
  };
  if constexpr (AHEAD) fetch(part);
  {
    // a thread has one pair, of every so many tokens
    const int j = threadIdx.x % a.P, rows = kRotaryThreads / a.P;
    int axis = 0;
    while (axis < a.axes - 1 && j >= a.ends[axis]) ++axis;
    const double f = a.freq[j] * 0.15915494309189535;   // turns per position
    const uint64_t step = __double2ull_rn((f - floor(f)) * 18446744073709551616.0);
    const float spoiled = static_cast<float>(f * 0.0);   // (NaN if that is not finite)
    for (int i = threadIdx.x / a.P; i < here && threadIdx.x < rows * a.P; i += rows) {
      int64_t b;
      int l;
      token(i, b, l);
      const int64_t at = b * a.pos_bs + l * a.pos_ts + axis * a.pos_as;
      const int64_t p = a.pos_wide ? static_cast<const int64_t*>(a.pos)[at] : static_cast<const int32_t*>(a.pos)[at];
      const int32_t turn = static_cast<int32_t>((static_cast<uint64_t>(p) * step) >> 32);   // of 2^32
      const float2 cs = rotary_angle<T>(static_cast<float>(turn) * 2.3283064365386963e-10f + spoiled);
      rotary_smem[i * a.P + j] = cs.x;
      rotary_smem[(a.per_block + i) * a.P + j] = cs.y * a.sign;
    }
  }
  __syncthreads();
  if (all == 0) return;
  float co[V], si[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const bool late = APART && e >= V / 2;
    co[e] = si[e] = 0.f;
    if (!turned[late]) continue;
    const int at = tok * a.P + (APART ? (late ? second : first) / 2 + e % (V / 2) : c * V + e);
    co[e] = rotary_smem[at];
    si[e] = rotary_smem[a.per_block * a.P + at];
  }
  for (int h0 = part; h0 < all; h0 += N * a.share) {
    if constexpr (!AHEAD) fetch(h0);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int h = h0 + k * a.share;
      if (h >= all) continue;
      const int w = h >= a.heads[0];
      T* y = static_cast<T*>(a.y[w]) + (t * a.heads[w] + (w ? h - a.heads[0] : h)) * a.d;
      // (in place, two values at a time: registers bound how many threads are there)
      Raw &x0 = ra[k], &x1 = rb[k];
      if constexpr (sizeof(T) == 2 && V >= 2) {
        uint32_t *w0 = reinterpret_cast<uint32_t*>(&x0), *w1 = reinterpret_cast<uint32_t*>(&x1);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          const float a0 = __uint_as_float(w0[i] << 16), a1 = __uint_as_float(w0[i] & 0xFFFF0000u);
          const float b0 = __uint_as_float(w1[i] << 16), b1 = __uint_as_float(w1[i] & 0xFFFF0000u);
          float u0, u1, z0, z1;
          if constexpr (HALVES) {
            turned_pair(a0, b0, co[2 * i], si[2 * i], u0, z0);
            turned_pair(a1, b1, co[2 * i + 1], si[2 * i + 1], u1, z1);
          } else {
            turned_pair(a0, a1, co[i], si[i], u0, u1);
            turned_pair(b0, b1, co[V / 2 + i], si[V / 2 + i], z0, z1);
          }
          if (turned[0]) w0[i] = pack_bf16x2(u0, u1);
          if (turned[1]) w1[i] = pack_bf16x2(z0, z1);
        }
      } else {
        T *f0 = reinterpret_cast<T*>(&x0), *f1 = reinterpret_cast<T*>(&x1);
        constexpr int PAIRS = APART ? V / 2 : V;
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
          float u0, u1, z0, z1;
          if constexpr (APART) {
            turned_pair(static_cast<float>(f0[2 * i]), static_cast<float>(f0[2 * i + 1]), co[i], si[i], u0, u1);
            turned_pair(static_cast<float>(f1[2 * i]), static_cast<float>(f1[2 * i + 1]), co[V / 2 + i], si[V / 2 + i], z0, z1);
            if (turned[0]) { f0[2 * i] = static_cast<T>(u0); f0[2 * i + 1] = static_cast<T>(u1); }
            if (turned[1]) { f1[2 * i] = static_cast<T>(z0); f1[2 * i + 1] = static_cast<T>(z1); }
          } else {
            turned_pair(static_cast<float>(f0[i]), static_cast<float>(f1[i]), co[i], si[i], u0, z0);
            if (turned[0]) { f0[i] = static_cast<T>(u0); f1[i] = static_cast<T>(z0); }
          }
        }
      }
      *reinterpret_cast<Raw*>(y + first) = x0;
      *reinterpret_cast<Raw*>(y + second) = x1;
    }
  }
}

}  // namespace lact

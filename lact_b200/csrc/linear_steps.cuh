// Linear attention with a decay per head, token by token.  Per sequence and head, with a state S of A x B (fp32):
//   S_t = lambda S_(t-1) + y_t z_t^T,   out_t = scale x_t^T S_t,                        lambda = exp(log_decay[head]) .
// With (x, y, z) = (q, k, v) that is the forward.  All three gradients are the same operator on other operands:
//   dq_t = scale S_t do_t                                    (x, y, z) = (do, v, k), the state transposed;
//   dv_t = R_t^T k_t,  dk_t = R_t v_t,  R_t = lambda R_(t+1) + scale q_t do_t^T, from the last token to the first, where R starts
//          from the gradient of the last state (not decayed before its first token):  (k, q, do), and (v, do, q) transposed;
//   the first state's gradient is lambda R_0.  (R is kept divided by the scale: `in_mul`, `out_mul`.)
// This kernel keeps S in registers and reads every token once, the state once: what a call of one token needs.
#pragma once
#include "ptx.cuh"

namespace lact {

using bf16 = __nv_bfloat16;

struct LinearArgs {
  const bf16 *x, *y, *z;               // [entry][token][head / share][A or B], heads adjacent, token / entry strides in elements
  int64_t x_ts, x_bs, y_ts, y_bs, z_ts, z_bs;
  int32_t x_share, y_share, z_share;   // heads of the state that one head of the operand serves
  void* out;                           // [entry][token][heads][B], contiguous
  int32_t out_f32;                     // fp32 instead of bf16 (gradients that are still to be added over shared heads)
  const float* log_decay;              // [heads]
  const int32_t* cu;                   // packed sequences: [sequences + 1] bounds within the one entry; or nullptr: an entry is one
  int32_t sequences, L, heads;         // L: tokens of an entry
  const float* s_in;                   // [sequences][heads] states, or nullptr: zeros
  float* s_out;                        // or nullptr
  int32_t s_in_t;                      // stored [B][A] instead of [A][B]
  float scale, in_mul, out_mul;        // of the outputs; of a state that is read / written
  int32_t reverse;
};

// lambda as a power of two: 2^(n * decay_log2) after n tokens.  A decay of exp(-inf) = 0 stays 0 from the first token on (2^-200
// is below the smallest fp32) and makes no 0 x inf at n = 0.
__device__ __forceinline__ float decay_log2(const LinearArgs& a, int head) {
  const float g = a.log_decay[head] * 1.4426950408889634f;
  return g < -200.f ? -200.f : g;
}

struct LinearSpan {
  int entry, first, len;   // batch entry, first token, tokens
};
// (bounds that do not rise or pass the end are cut to what is there: nothing is read or written outside)
__device__ __forceinline__ LinearSpan linear_span(const LinearArgs& a, int n) {
  if (a.cu == nullptr) return {n, 0, a.L};
  const int t0 = min(max(a.cu[n], 0), a.L), t1 = min(max(a.cu[n + 1], t0), a.L);
  return {0, t0, t1 - t0};
}

// Tokens before the first and behind the last packed sequence have outputs of zero.
template <int B>
__device__ __forceinline__ void linear_zero_rest(const LinearArgs& a, int64_t worker, int64_t workers) {
  if (a.cu == nullptr) return;
  const int head = min(max(a.cu[0], 0), a.L), tail = min(max(a.cu[a.sequences], head), a.L);
  const int64_t row = static_cast<int64_t>(a.heads) * B * (a.out_f32 ? 4 : 2) / 16;   // 16-byte units
  const int64_t lead = head * row, all = lead + (a.L - tail) * row;
  uint4* const o = static_cast<uint4*>(a.out);
  for (int64_t i = worker; i < all; i += workers) o[i < lead ? i : i - lead + tail * row] = make_uint4(0, 0, 0, 0);
}

__device__ __forceinline__ void unpack_bf16x8(const uint4& u, float* f) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

// One CTA per (sequence, head, 32 columns of the state); 8 threads hold a row's columns, 4 each, 32 rows at a time.
// Bound by the state's bytes (8 A B a head and token of generation): 32 columns a CTA keep 148 SMs busy from about 40 heads on and
// have 16 KB in flight per CTA.  (8 tokens of 12 heads of 128: 4.7 us; linear_plan has the rule between this and the tiles.)
constexpr int kStepTokens = 8;   // tokens staged at a time
template <int A, int B>
__global__ void __launch_bounds__(256) linear_steps_kernel(const __grid_constant__ LinearArgs a) {
  constexpr int R = A / 32;
  __shared__ __align__(16) float sx[kStepTokens][A], sy[kStepTokens][A], sz[kStepTokens][32], part[kStepTokens][8][32];
  griddep_launch_dependents();
  griddep_wait();
  const int tid = threadIdx.x, cl = tid & 7, rg = tid >> 3, warp = tid >> 5, lane = tid & 31;
  const int unit = blockIdx.x / (B / 32), n = unit / a.heads, head = unit % a.heads, c0 = blockIdx.x % (B / 32) * 32;
  float S[R][4];
  const int64_t at = (static_cast<int64_t>(n) * a.heads + head) * (A * B);
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = rg + 32 * i;
    if (a.s_in == nullptr) {
#pragma unroll
      for (int e = 0; e < 4; ++e) S[i][e] = 0.f;
    } else if (!a.s_in_t) {
      const float4 v = *reinterpret_cast<const float4*>(a.s_in + at + row * B + c0 + cl * 4);
      S[i][0] = v.x * a.in_mul; S[i][1] = v.y * a.in_mul; S[i][2] = v.z * a.in_mul; S[i][3] = v.w * a.in_mul;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) S[i][e] = a.s_in[at + (c0 + cl * 4 + e) * A + row] * a.in_mul;
    }
  }
  const float lambda = exp2f(decay_log2(a, head));
  const bf16* const x = a.x + n * a.x_bs + (head / a.x_share) * A;
  const bf16* const y = a.y + n * a.y_bs + (head / a.y_share) * A;
  const bf16* const z = a.z + n * a.z_bs + (head / a.z_share) * B + c0;
  for (int p0 = 0; p0 < a.L; p0 += kStepTokens) {
    const int count = min(kStepTokens, a.L - p0);
    auto token = [&](int tt) { return static_cast<int64_t>(a.reverse ? a.L - 1 - p0 - tt : p0 + tt); };
    for (int u = tid; u < count * (A / 8); u += 256) {
      const int tt = u / (A / 8), c = u % (A / 8) * 8;
      unpack_bf16x8(*reinterpret_cast<const uint4*>(x + token(tt) * a.x_ts + c), &sx[tt][c]);
      unpack_bf16x8(*reinterpret_cast<const uint4*>(y + token(tt) * a.y_ts + c), &sy[tt][c]);
    }
    if (tid < count * 4) unpack_bf16x8(*reinterpret_cast<const uint4*>(z + token(tid >> 2) * a.z_ts + (tid & 3) * 8), &sz[tid >> 2][(tid & 3) * 8]);
    __syncthreads();
    for (int tt = 0; tt < count; ++tt) {
      const float dec = a.reverse && p0 + tt == 0 ? 1.f : lambda;
      const float4 zv = *reinterpret_cast<const float4*>(&sz[tt][cl * 4]);
      const float zc[4] = {zv.x, zv.y, zv.z, zv.w};
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float yv = sy[tt][rg + 32 * i], xv = sx[tt][rg + 32 * i];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          S[i][e] = fmaf(S[i][e], dec, yv * zc[e]);
          acc[e] = fmaf(xv, S[i][e], acc[e]);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        acc[e] += __shfl_xor_sync(0xFFFFFFFFu, acc[e], 8);
        acc[e] += __shfl_xor_sync(0xFFFFFFFFu, acc[e], 16);
      }
      if (lane < 8) *reinterpret_cast<float4*>(&part[tt][warp][cl * 4]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
    }
    __syncthreads();
    const int tt = tid >> 5, c = tid & 31;
    if (tt < count) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) sum += part[tt][w][c];
      const int64_t o = ((n * static_cast<int64_t>(a.L) + token(tt)) * a.heads + head) * B + c0 + c;
      if (a.out_f32) static_cast<float*>(a.out)[o] = sum * a.scale;
      else static_cast<bf16*>(a.out)[o] = __float2bfloat16_rn(sum * a.scale);
    }
    __syncthreads();
  }
  if (a.s_out == nullptr) return;
  const float mul = a.out_mul * (a.reverse ? lambda : 1.f);
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = rg + 32 * i;
    *reinterpret_cast<float4*>(a.s_out + at + row * B + c0 + cl * 4) = make_float4(S[i][0] * mul, S[i][1] * mul, S[i][2] * mul, S[i][3] * mul);
  }
}

// One token of every sequence, forward, states as they are stored: the same split without the staging and the loops, so that more CTAs
// are resident (192 sequences of 12 heads of 128 x 128, 304 MB: 46.4 us, 6.5 TB/s; 66 with the kernel above).
template <int A, int B>
__global__ void __launch_bounds__(256, 6) linear_token_kernel(const __grid_constant__ LinearArgs a) {
  constexpr int R = A / 32;
  __shared__ __align__(16) float part[8][32];
  griddep_launch_dependents();
  griddep_wait();
  const int tid = threadIdx.x, cl = tid & 7, rg = tid >> 3, warp = tid >> 5, lane = tid & 31;
  const int unit = blockIdx.x / (B / 32), n = unit / a.heads, head = unit % a.heads, c0 = blockIdx.x % (B / 32) * 32;
  const int64_t at = static_cast<int64_t>(unit) * (A * B) + rg * B + c0 + cl * 4;
  float4 S[R];
#pragma unroll
  for (int i = 0; i < R; ++i) S[i] = *reinterpret_cast<const float4*>(a.s_in + at + i * 32 * B);
  const bf16* const x = a.x + n * a.x_bs + (head / a.x_share) * A + rg;
  const bf16* const y = a.y + n * a.y_bs + (head / a.y_share) * A + rg;
  const uint2 zr = *reinterpret_cast<const uint2*>(a.z + n * a.z_bs + (head / a.z_share) * B + c0 + cl * 4);
  float xv[R], yv[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    xv[i] = __bfloat162float(x[i * 32]);
    yv[i] = __bfloat162float(y[i * 32]);
  }
  const float lambda = exp2f(decay_log2(a, head));
  const float4 z = make_float4(__uint_as_float(zr.x << 16), __uint_as_float(zr.x & 0xFFFF0000u), __uint_as_float(zr.y << 16),
                               __uint_as_float(zr.y & 0xFFFF0000u));
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < R; ++i) {
    S[i] = make_float4(fmaf(S[i].x, lambda, yv[i] * z.x), fmaf(S[i].y, lambda, yv[i] * z.y), fmaf(S[i].z, lambda, yv[i] * z.z),
                       fmaf(S[i].w, lambda, yv[i] * z.w));
    *reinterpret_cast<float4*>(a.s_out + at + i * 32 * B) = S[i];
    acc[0] = fmaf(xv[i], S[i].x, acc[0]);
    acc[1] = fmaf(xv[i], S[i].y, acc[1]);
    acc[2] = fmaf(xv[i], S[i].z, acc[2]);
    acc[3] = fmaf(xv[i], S[i].w, acc[3]);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    acc[e] += __shfl_xor_sync(0xFFFFFFFFu, acc[e], 8);
    acc[e] += __shfl_xor_sync(0xFFFFFFFFu, acc[e], 16);
  }
  if (lane < 8) *reinterpret_cast<float4*>(&part[warp][cl * 4]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
  __syncthreads();
  if (tid < 32) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) sum += part[w][tid];
    static_cast<bf16*>(a.out)[static_cast<int64_t>(unit) * B + c0 + tid] = __float2bfloat16_rn(sum * a.scale);
  }
}

// Gradients of shared heads: out[t][g] = sum over the `share` heads of group g, added in their order in fp32 and rounded once.
__global__ void __launch_bounds__(256) linear_sum_heads_kernel(const float* __restrict__ in, bf16* __restrict__ out, int64_t rows4,
                                                               int32_t share, int32_t d4) {
  griddep_launch_dependents();
  griddep_wait();
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < rows4; i += gridDim.x * 256ll) {
    const int64_t row = i / d4;
    const float4* src = reinterpret_cast<const float4*>(in) + row * share * d4 + i % d4;
    float4 s = src[0];
    for (int e = 1; e < share; ++e) {
      const float4 v = src[static_cast<int64_t>(e) * d4];
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    *reinterpret_cast<uint2*>(out + i * 4) = make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
  }
}

}  // namespace lact

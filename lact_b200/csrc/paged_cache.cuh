// A paged cache of keys and values: pages [page][kv head][row][d] of bf16, or of e4m3 with one byte a row of a head for a power of two.
// Sequence i has lengths[i] tokens; token p lies in page table[i][p / page_size], row p % page_size.  The calls below deal with the
// last n_i tokens of every sequence (the rows of a batch entry, or of a packed sequence): row j has position lengths[i] - n_i + j, and
// none where that is negative (rows that pad a batch in front).
//
// 8 bits: x = e4m3 * 2^(byte - 127), the smallest power of two with max |x| over the row at most 448 times it (between 2^-126
// and 2^119: values above 1.75 x 2^127 would come back as infinities, and are cut to that).
// Powers of two make scaling exact, so that e4m3 alone rounds (2^-4 of a value at most, 2^-10 of the power for the smallest); a scale
// of max / 448 would gain at most one bit of the range below 2^-15 of the row's largest value, and round twice.  Byte 255 is NaN: a
// row with a NaN or an infinity is NaN throughout.
#pragma once
#include <cuda_fp8.h>

#include "group_norm.cuh"

namespace lact {

struct PagedCache {
  uint8_t *k, *v;                  // pages
  uint8_t *ke, *ve;                // exponents [page][kv head][row], or nullptr: bf16
  int64_t k_ps, v_ps;              // bytes from page to page
  int64_t ke_ps, ve_ps;
  int32_t pages, heads, shift;     // page_size = 1 << shift
  const int32_t* table;            // [sequences][cols]
  int64_t table_rs;
  int32_t cols;
  const int32_t* lengths;
  int32_t sequences;
};

// A page number or a length that the cache does not have is left out, and told to the host (which raises on its next call): in the second
// byte of its word, so that a wait that ran out (the first byte), which spoils more than the rows left out here, stays to be read.  (A
// compare-and-swap of the whole word would do it too, at 7 us each, one after the other: 2.4 s for 80000 rows without a page in place of 80 us.)
__device__ __forceinline__ void report_bad_page() {
  if (g_host_status != nullptr) {
    reinterpret_cast<volatile uint8_t*>(g_host_status)[1] = kStatusBadPage;
    __threadfence_system();
  }
}

// 2^(byte - 127)
__device__ __forceinline__ float exponent_value(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7FC00000u : byte << 23);
}
// The byte of a row whose largest |bf16| has these 15 bits
__device__ __forceinline__ uint32_t exponent_byte(uint32_t top) {
  const int e = static_cast<int>(top >> 7);
  if (e == 255) return 255;
  return static_cast<uint32_t>(min(max(e - 8 + ((top & 0x7F) > 0x60 ? 1 : 0), 1), 246));
}
// Four e4m3 values as halves, exactly: the lower two and the upper two of a word
__device__ __forceinline__ void halves_of_e4m3(uint32_t four, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(four));
}
// Two values in e4m3 (low byte: the first)
__device__ __forceinline__ uint32_t e4m3_of(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

struct PagedRows {
  PagedCache c;
  const bf16 *xk, *xv;             // written: [entry][token][head][D], features adjacent, other strides in elements
  int64_t k_bs, k_ts, k_hs, v_bs, v_ts, v_hs;
  bf16* out;                       // read: [2][entries][tokens][heads][D], on 32 bytes
  const int32_t* cu;               // packed: [sequences + 1] bounds within the one entry
  int64_t tokens;                  // of all entries
  int32_t L, share;                // of an entry; thread groups that share a token's heads
};

// Where row `t` of the batch lies: its page (-1: nowhere) and row.
__device__ __forceinline__ int2 paged_place(const PagedRows& a, int64_t t) {
  int64_t seq, pos;
  if (a.cu == nullptr) {
    seq = t / a.L;
    pos = static_cast<int64_t>(a.c.lengths[seq]) - a.L + (t - seq * a.L);
  } else {
    int lo = 0, hi = a.c.sequences;   // the last sequence that begins at or before t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.cu[mid] <= t) lo = mid;
      else hi = mid;
    }
    seq = lo;
    if (a.cu[seq] > t || t >= a.cu[seq + 1]) return make_int2(-1, 0);   // outside of the sequences
    pos = static_cast<int64_t>(a.c.lengths[seq]) - (a.cu[seq + 1] - t);
  }
  if (pos < 0) return make_int2(-1, 0);
  if (pos >> a.c.shift >= a.c.cols) {
    report_bad_page();
    return make_int2(-1, 0);
  }
  const int page = a.c.table[seq * a.c.table_rs + (pos >> a.c.shift)];
  if (page < 0 || page >= a.c.pages) {
    report_bad_page();
    return make_int2(-1, 0);
  }
  return make_int2(page, static_cast<int>(pos & ((1 << a.c.shift) - 1)));
}

// Both directions are bound by memory.  A row of a head is held by D / 8 threads, 8 values each, or with 8 bits by D / 16 (16 bytes of the
// cache a thread); such a group takes one token, finds its place, and goes through its share of the heads, keys and values of N at a time on
// their way together (writing, they are fetched before the place is known).  28080 tokens of 12 heads of 128: bf16 written in 54.5 us, read in
// 55.7 (6.3 and 6.2 TB/s), 8 bits in 44.2 and 44.4 (5.9 and 5.8).
constexpr int kPagedThreads = 256;
__host__ __device__ constexpr int kPagedLanes(int D, bool e4) { return D / (e4 ? 16 : 8); }
template <int D, bool E4, bool WRITE, int N, int PER_SM>
__global__ void __launch_bounds__(kPagedThreads, PER_SM) paged_rows_kernel(const __grid_constant__ PagedRows a) {
  constexpr int LANES = kPagedLanes(D, E4), GROUPS = kPagedThreads / LANES, VEC = D / LANES, P = VEC / 8;   // P: 16 bytes of activations
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES, tok = group / a.share, part = group - tok * a.share;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (GROUPS / a.share) + tok;
  // (every thread of a warp takes part in every turn: tokens past the end have no place, and no heads)
  const int heads = t < a.tokens ? a.c.heads : 0;
  const int64_t b = t / a.L, l = t - b * a.L;
  int2 at = make_int2(-1, 0);
  for (int h0 = part; h0 - part < a.c.heads; h0 += N * a.share) {
    uint4 raw[2][N][P];
    [[maybe_unused]] uint32_t byte[2][N];
    if constexpr (WRITE) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int h = h0 + i * a.share;
#pragma unroll
        for (int p = 0; p < P; ++p) {
          raw[0][i][p] = raw[1][i][p] = make_uint4(0, 0, 0, 0);
          if (h >= heads) continue;
          raw[0][i][p] = *reinterpret_cast<const uint4*>(a.xk + b * a.k_bs + l * a.k_ts + h * a.k_hs + lane * VEC + p * 8);
          raw[1][i][p] = *reinterpret_cast<const uint4*>(a.xv + b * a.v_bs + l * a.v_ts + h * a.v_hs + lane * VEC + p * 8);
        }
      }
    }
    if (h0 == part && heads > 0) at = paged_place(a, t);
    const bool there = at.x >= 0;
    auto row_of = [&](int h) { return (static_cast<int64_t>(h) << a.c.shift) + at.y; };
    auto place = [&](int v, int h) { return (v ? a.c.v + at.x * a.c.v_ps : a.c.k + at.x * a.c.k_ps) + (row_of(h) * LANES + lane) * 16; };
    auto exponent = [&](int v, int h) { return (v ? a.c.ve + at.x * a.c.ve_ps : a.c.ke + at.x * a.c.ke_ps) + row_of(h); };
    if constexpr (!WRITE) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int h = h0 + i * a.share;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          raw[v][i][0] = make_uint4(0, 0, 0, 0);
          byte[v][i] = 127;
          if (h >= heads || !there) continue;
          raw[v][i][0] = *reinterpret_cast<const uint4*>(place(v, h));
          if constexpr (E4) byte[v][i] = *exponent(v, h);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int h = h0 + i * a.share;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        uint4(&x)[P] = raw[v][i];
        if constexpr (WRITE) {
          if constexpr (E4) {
            uint32_t w[8], top = 0;
#pragma unroll
            for (int p = 0; p < P; ++p) {
              w[4 * p] = x[p].x; w[4 * p + 1] = x[p].y; w[4 * p + 2] = x[p].z; w[4 * p + 3] = x[p].w;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) top = __vmaxu2(top, w[e] & 0x7FFF7FFFu);
            top = max(top & 0xFFFFu, top >> 16);
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            if (h >= heads || !there) continue;
            const uint32_t e8 = exponent_byte(top);
            const float by = __uint_as_float((254u - min(e8, 253u)) << 23);   // 2^(127 - byte)
            uint32_t q[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t lo = w[2 * e], hi = w[2 * e + 1];
              q[e] = e8 == 255 ? 0x7F7F7F7Fu
                               : e4m3_of(__uint_as_float(lo << 16) * by, __uint_as_float(lo & 0xFFFF0000u) * by) |
                                     e4m3_of(__uint_as_float(hi << 16) * by, __uint_as_float(hi & 0xFFFF0000u) * by) << 16;
            }
            *reinterpret_cast<uint4*>(place(v, h)) = make_uint4(q[0], q[1], q[2], q[3]);
            if (lane == 0) *exponent(v, h) = static_cast<uint8_t>(e8);
          } else {
            if (h >= heads || !there) continue;
            *reinterpret_cast<uint4*>(place(v, h)) = x[0];
          }
        } else {
          if (h >= heads) continue;
          if constexpr (E4) {
            const float by = exponent_value(byte[v][i]);
            const uint32_t w[4] = {x[0].x, x[0].y, x[0].z, x[0].w};
            uint32_t o[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t two[2];
              halves_of_e4m3(w[e], two[0], two[1]);
#pragma unroll
              for (int s = 0; s < 2; ++s) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&two[s]));
                o[2 * e + s] = pack_bf16x2(f.x * by, f.y * by);
              }
            }
            st_global_32(a.out + ((v ? a.tokens : 0) + t) * a.c.heads * D + h * D + lane * VEC, o);
          } else {
            *reinterpret_cast<uint4*>(a.out + ((v ? a.tokens : 0) + t) * a.c.heads * D + h * D + lane * VEC) = x[0];
          }
        }
      }
    }
  }
}

}  // namespace lact

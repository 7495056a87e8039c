// Arguments and helpers shared by the attention kernels over the 8-bit paged cache.
#pragma once

#include "paged_kv.cuh"

namespace nmb {
namespace paged {

// Probabilities in f16. A row's running maximum M of t = score + log2 of the value scale moves when
// a tile exceeds it by 2^6 (most tiles then skip rescaling the accumulator; prompts of up to 2048
// tokens over as many, 32 / 8 heads of 128: 239.6 us with 2^4, 235.2 with 2^8), and probabilities are
// stored as 2^(t - M + 9): at most 2^15, with all 11 bits down to 2^-23 of 2^M and a quantum of
// 2^-24 (error 2^-25) below that.
constexpr float kLazy = 6.f;
constexpr float kShift = 9.f;

// That error of a key's probability matters only where the whole result is small: where M comes
// from a key whose own value is next to nothing, because its page's scale was raised by another
// key or because it just takes the weight. A row whose largest numerator is at least this times its
// keys is within 2^-11 of it (keys * largest code * 2^-25); the others are computed again by
// exact_row. A key with a code of 8 at the maximum is enough for 149,000 keys.
template <bool INT8>
constexpr float kResolved = (INT8 ? 127.f : 448.f) / 16384.f;

struct Params {
  const __nv_bfloat16* q;
  int64_t q_row, q_head;
  __nv_bfloat16* o;                 // [T, Hq, D]
  float* lse;                       // [T, Hq] or null
  const uint8_t *k_codes, *v_codes; // [pages, Hkv, ps, D]
  const float *k_scale, *v_scale;   // [pages, Hkv]
  const int *tables, *q_starts, *kv_lens;
  int64_t table_stride;
  int width, num_pages, ps, page_shift;
  int B, T, Hq, Hkv, G;
  int max_rows;                     // more query rows: the prefill kernel's requests, else decode's
  float scale_log2;
  float* part;                      // [grid][2][rows][D] numerators of shared units
  float2* part_ml;                  // [grid][2][rows] (M, denominator)
  int* counters;                    // tiles finished of each shared unit; zero between calls
  int* status;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// One row of a request over its first `keys` positions by one warp, with fp32 probabilities and
// without the value scales in the maximum: the plain formula. For the few rows that the f16
// probabilities cannot resolve (see kResolved), so simple rather than fast: a lane per key for the
// scores, a lane per D / 32 columns for the sum. (All rows of 128 requests of up to 4096 tokens, 32 / 8
// heads of 128: 3.3 ms, where the kernel takes 0.12.) With `look`, leaves a row alone, and returns
// false, if all the values it sees are zero: its 0 is right already (a cache of zeros: 0.7 ms).
// Pages' value scales may differ by up to 2^100 (beyond, the kernels' fp32 denominators lose keys
// that still count).
template <int D, bool INT8>
__device__ __forceinline__ bool exact_row(const Params& p, int b, int h, const __nv_bfloat16* q,
                                          int keys, bool look, __nv_bfloat16* out, float* lse) {
  constexpr int kCols = D / 32;
  const int lane = threadIdx.x & 31;
  const int* table = p.tables + b * p.table_stride;
  // row of a key's codes, in units of D; -1 on a missing page
  auto row_of = [&](int key) -> int64_t {
    const int page = __ldg(table + (key >> p.page_shift));
    if (page < 0 || page >= p.num_pages) return -1;
    return ((static_cast<int64_t>(page) * p.Hkv + h) << p.page_shift) + (key & (p.ps - 1));
  };
  bool any = !look;
#pragma unroll 1
  for (int k0 = 0; k0 < keys && !any; k0 += 32) {
    const int64_t row = k0 + lane < keys ? row_of(k0 + lane) : -1;
    uint32_t bits = 0;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      const uint4 x = row >= 0 ? __ldg(reinterpret_cast<const uint4*>(p.v_codes + row * D) + c)
                               : make_uint4(0, 0, 0, 0);
      bits |= x.x | x.y | x.z | x.w;
    }
    any = __any_sync(0xffffffffu, (bits & (INT8 ? 0xffffffffu : 0x7f7f7f7fu)) != 0);
  }
  if (!any) return false;

  float qv[kCols], x[kCols] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < kCols; ++i) qv[i] = __bfloat162float(q[lane * kCols + i]);
#pragma unroll 1
  for (int k0 = 0; k0 < keys; k0 += 32) {
    const int64_t row = k0 + lane < keys ? row_of(k0 + lane) : -1;
    const float ks = row >= 0 ? __ldg(p.k_scale + (row >> p.page_shift)) : 0.f;
    const float vs = row >= 0 ? __ldg(p.v_scale + (row >> p.page_shift)) : 0.f;
    float s = 0.f;
#pragma unroll 1
    for (int c0 = 0; c0 < D; c0 += 64) {       // 64 codes in flight
      uint4 x4[4];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        x4[c] = row >= 0 ? __ldg(reinterpret_cast<const uint4*>(p.k_codes + row * D + c0) + c)
                         : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        const uint32_t w4[4] = {x4[c / 4].x, x4[c / 4].y, x4[c / 4].z, x4[c / 4].w};
        uint32_t f[2];
        kv::decode4<INT8>(w4[c % 4], f[0], f[1]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 k2 = kv::f16x2_to_float2(f[e >> 1]);
          const float qd = __shfl_sync(0xffffffffu, qv[e % kCols], (c0 + c * 4 + e) / kCols);
          s = fmaf(qd, (e & 1 ? k2.y : k2.x) * ks, s);
        }
      }
    }
    s = row >= 0 ? s * p.scale_log2 : -INFINITY;
    const float top = fmaxf(m, warp_max(s)), ref = top == -INFINITY ? 0.f : top;
    const float w = ex2(s - ref), down = ex2(m - ref);
    m = top;
    l = fmaf(l, down, warp_sum(w));
#pragma unroll
    for (int i = 0; i < kCols; ++i) x[i] *= down;
#pragma unroll 1
    for (int k = 0; k < min(32, keys - k0); k += 8) {
      uint32_t raw[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {            // a missing page or none: weight 0, codes 0
        const int64_t at = __shfl_sync(0xffffffffu, row, k + i);
        const uint8_t* codes = p.v_codes + at * D + lane * kCols;
        raw[i] = at < 0 ? 0u
                        : kCols == 4 ? __ldg(reinterpret_cast<const uint32_t*>(codes))
                                     : __ldg(reinterpret_cast<const uint16_t*>(codes));
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float wk = __shfl_sync(0xffffffffu, w, k + i), sk = __shfl_sync(0xffffffffu, vs, k + i);
        uint32_t f[2];
        kv::decode4<INT8>(raw[i], f[0], f[1]);
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          const float2 v2 = kv::f16x2_to_float2(f[c >> 1]);
          x[c] = fmaf(wk, (c & 1 ? v2.y : v2.x) * sk, x[c]);
        }
      }
    }
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;   // a row that sees nothing: 0
  __syncwarp();                       // what this warp wrote there before
#pragma unroll
  for (int i = 0; i < kCols; i += 2)
    *reinterpret_cast<uint32_t*>(out + lane * kCols + i) = pack_bf16x2(x[i] * inv, x[i + 1] * inv);
  if (lse != nullptr && lane == 0) *lse = m + log2f(l);
  return true;
}

}  // namespace paged
}  // namespace nmb

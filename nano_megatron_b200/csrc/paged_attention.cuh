// Arguments and helpers shared by the attention kernels over the 8-bit paged cache.
#pragma once

#include "paged_kv.cuh"

namespace nmb {
namespace paged {

// The running max only moves when a tile exceeds it by 2^8: most tiles then skip rescaling the
// accumulator, and P <= 256 keeps its 11 bits in f16.
constexpr float kLazy = 8.f;

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


}  // namespace paged
}  // namespace nmb

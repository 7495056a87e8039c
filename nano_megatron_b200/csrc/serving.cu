// Batched-serving kernels besides attention: the step plan (block tables, slot map), writing
// new keys / values into the 8-bit paged cache, reading it back, and the rules on logits.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "paged_kv.cuh"

namespace nmb {
namespace serving {

// --------------------------------------------------------------------------- step plan
// Every block scans the B request lengths for itself (a few KB out of L2) and then fills its
// own 256 token rows and 256 touched-page entries, so one launch needs no block to wait for
// another. Bound by latency: two dependent loads, three block scans, one binary search (3.3 us for 8
// requests, 4.8 for 700 with 17,000 new tokens).
constexpr int kPlanThreads = 256;
constexpr int kPlanMaxRequests = 4096;

struct PlanParams {
  const int *context, *fresh, *free_pages, *free_count;
  int* tables;
  int64_t table_stride;
  int B, width, T, U, page_shift, num_free;
  int *q_starts, *kv_lens, *positions, *slots, *free_out, *missing;
  int4* touched;
};

// Exclusive scan of one value per thread over the block; `total` for all.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* warp_sums, int64_t& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x / 32;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sums[w] = x;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kPlanThreads / 32; ++i) {
    if (i < w) before += warp_sums[i];
    total += warp_sums[i];
  }
  __syncthreads();
  return before + x - v;
}

// Last index r with start[r] <= v (start is ascending, start[0] = 0).
__device__ __forceinline__ int owner_of(const int* start, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= v) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanParams p) {
  extern __shared__ int sh[];
  __shared__ int64_t warp_sums[kPlanThreads / 32];
  int* s_row = sh;                  // [B + 1] first token row of each request
  int* s_touch = s_row + p.B + 1;   // [B + 1] first touched-page entry
  int* s_fresh = s_touch + p.B + 1; // [B + 1] first new page
  const int ps = 1 << p.page_shift;
  const int per = (p.B + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(p.B, static_cast<int>(threadIdx.x) * per), b1 = min(p.B, b0 + per);
  const int have = min(max(*p.free_count, 0), p.num_free);
  auto context_of = [&](int b) { return min(max(p.context[b], 0), 1 << 30); };

  // Lengths are clamped so that sums of wrong ones stay in range: 64 bits before the cut at T.
  int64_t sum = 0, total;
  for (int b = b0; b < b1; ++b) sum += min(max(p.fresh[b], 0), p.T);
  int64_t at = block_scan(sum, warp_sums, total);
  int touch = 0, fresh = 0, beyond = 0;
  for (int b = b0; b < b1; ++b) {
    // rows past the T that the outputs hold are dropped
    const int row = static_cast<int>(min(at, static_cast<int64_t>(p.T))), n = min(max(p.fresh[b], 0), p.T - row);
    at += min(max(p.fresh[b], 0), p.T);
    const int ctx = context_of(b);
    s_row[b] = row;
    s_touch[b] = n > 0 ? ((ctx + n - 1) >> p.page_shift) - (ctx >> p.page_shift) + 1 : 0;
    // new pages that the table has columns for; the others stay in the free list
    const int old = (ctx + ps - 1) >> p.page_shift, after = (ctx + n + ps - 1) >> p.page_shift;
    s_fresh[b] = max(min(after, p.width) - old, 0);
    touch += s_touch[b];
    fresh += s_fresh[b];
    beyond += after - old - s_fresh[b];
  }
  int64_t touch_total, fresh_total;
  int touch_at = static_cast<int>(block_scan(touch, warp_sums, touch_total));
  // two sums in one scan, each below 2^31: new pages in the low half, those beyond the tables above
  int fresh_at = static_cast<int>(
      block_scan(fresh + (static_cast<int64_t>(beyond) << 32), warp_sums, fresh_total));
  for (int b = b0; b < b1; ++b) {
    const int t = s_touch[b], f = s_fresh[b];
    s_touch[b] = touch_at;
    s_fresh[b] = fresh_at;
    touch_at += t;
    fresh_at += f;
  }
  if (threadIdx.x == 0) {
    s_row[p.B] = static_cast<int>(min(total, static_cast<int64_t>(p.T)));
    s_touch[p.B] = static_cast<int>(touch_total);
    s_fresh[p.B] = static_cast<int>(fresh_total);
  }
  __syncthreads();

  // Physical page of logical page `lp` of request b: from the table where the context has it,
  // else the next of the free list (-1 when the list or the table's width does not reach).
  auto page_of = [&](int b, int lp, int ctx) {
    const int old = (ctx + ps - 1) >> p.page_shift;
    if (lp >= p.width) return -1;
    if (lp < old) return p.tables[b * p.table_stride + lp];
    const int take = have - 1 - (s_fresh[b] + lp - old);
    return take >= 0 ? p.free_pages[take] : -1;
  };

  const int i = blockIdx.x * kPlanThreads + threadIdx.x;
  if (i < p.T) {
    int pos = 0, slot = -1;
    if (i < s_row[p.B]) {
      const int b = owner_of(s_row, p.B, i);
      const int ctx = context_of(b);
      pos = ctx + i - s_row[b];
      const int page = page_of(b, pos >> p.page_shift, ctx);
      if (page >= 0) slot = (page << p.page_shift) + (pos & (ps - 1));
    }
    p.positions[i] = pos;
    p.slots[i] = slot;
  }
  if (i < p.U) {
    int4 e = make_int4(-1, 0, 0, 0);
    if (i < touch_total) {
      const int b = owner_of(s_touch, p.B, i);
      const int ctx = context_of(b), n = s_row[b + 1] - s_row[b];
      const int lp = (ctx >> p.page_shift) + i - s_touch[b];
      const int first = max(lp << p.page_shift, ctx), last = min((lp + 1) << p.page_shift, ctx + n);
      const int page = page_of(b, lp, ctx);
      e = make_int4(page, s_row[b] + first - ctx, first - (lp << p.page_shift), last - first);
      if (lp >= (ctx + ps - 1) >> p.page_shift && lp < p.width)
        p.tables[b * p.table_stride + lp] = page;
    }
    p.touched[i] = e;
  }
  if (blockIdx.x == 0) {
    for (int b = b0; b < b1; ++b) {
      p.q_starts[b] = s_row[b];
      p.kv_lens[b] = context_of(b) + s_row[b + 1] - s_row[b];
    }
    if (threadIdx.x == 0) {
      p.q_starts[p.B] = s_row[p.B];
      const int need = s_fresh[p.B];
      *p.free_out = max(have - need, 0);
      *p.missing = max(need - have, 0) + static_cast<int>(fresh_total >> 32);
    }
  }
}

// ------------------------------------------------------------------------- cache write
// One unit is (touched page, kv head, K or V). Its new rows are read once into registers (at most
// 16 loads of 16 bytes a lane), their largest finite magnitude gives the page's scale, and the
// codes leave as 8-byte stores; codes that were on the page before are rescaled only when the
// scale grows. Bound by reading the rows and writing the codes. A unit takes one warp up to 4096
// values, so small pages need no barrier and no block of their own, two or four beyond. Written and
// read back, 120,000 tokens of 8 heads of 128 take 270 us, 5.4 TB/s or 83 % of the copy rate (a block
// per unit and scalar index arithmetic: 551 us).
constexpr int kAppendThreads = 128;

struct AppendParams {
  const __nv_bfloat16 *k, *v;
  int64_t k_row, k_head, v_row, v_head;
  uint8_t *k_codes, *v_codes;
  float *k_scale, *v_scale;
  const int4* touched;
  int entries, rows, num_pages, H, vec;
};

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  f[0] = bf16_lo(v.x); f[1] = bf16_hi(v.x); f[2] = bf16_lo(v.y); f[3] = bf16_hi(v.y);
  f[4] = bf16_lo(v.z); f[5] = bf16_hi(v.z); f[6] = bf16_lo(v.w); f[7] = bf16_hi(v.w);
}

__device__ __forceinline__ uint4 load8(const __nv_bfloat16* p, bool vec) {
  if (vec) return __ldg(reinterpret_cast<const uint4*>(p));
  const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = q[2 * e] | (static_cast<uint32_t>(q[2 * e + 1]) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <bool INT8, int D, int PS>
__global__ void __launch_bounds__(kAppendThreads, 4) append_kernel(const AppendParams p) {
  constexpr int kCols = D / 8;                                    // 8-value chunks of a row
  constexpr int kWarps = PS * D <= 4096 ? 1 : PS * D / 4096;      // of a unit
  constexpr int kStep = kWarps * 32 / kCols;                      // rows of one pass
  constexpr int kPer = PS / kStep;
  __shared__ float s_max[kAppendThreads / 32];
  const int warp = threadIdx.x / 32;
  const int unit = blockIdx.x * (kAppendThreads / 32 / kWarps) + warp / kWarps;
  const bool value = unit & 1;
  const int entry = (unit >> 1) / p.H, h = (unit >> 1) - entry * p.H;
  int4 t = make_int4(-1, 0, 0, 0);
  if (entry < p.entries) t = __ldg(p.touched + entry);
  const bool live = t.x >= 0 && t.x < p.num_pages && t.w > 0 && t.z >= 0 && t.z + t.w <= PS &&
                    t.y >= 0 && t.y <= p.rows - t.w;
  if (!live) t.w = t.z = 0;
  const int64_t row_stride = value ? p.v_row : p.k_row;
  const __nv_bfloat16* x = (value ? p.v : p.k) + t.y * row_stride + h * (value ? p.v_head : p.k_head);
  const int64_t at = live ? static_cast<int64_t>(t.x) * p.H + h : 0;
  uint8_t* codes = (value ? p.v_codes : p.k_codes) + at * (PS * D);
  float* scale = (value ? p.v_scale : p.k_scale) + at;
  const int lane = threadIdx.x % (kWarps * 32);
  const int r0 = lane / kCols, col = (lane % kCols) * 8;
  const float before = live ? *scale : 1.f;

  uint4 raw[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    raw[i] = r0 + i * kStep < t.w ? load8(x + (r0 + i * kStep) * row_stride + col, p.vec)
                                  : make_uint4(0, 0, 0, 0);
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    float f[8];
    unpack8(raw[i], f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = fabsf(f[e]);
      amax = fmaxf(amax, a <= 3.4e38f ? a : 0.f);  // infinities and NaN have no say
    }
  }
  amax = warp_max(amax);
  if constexpr (kWarps > 1) {
    if ((threadIdx.x & 31) == 0) s_max[warp] = amax;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWarps; ++i) amax = fmaxf(amax, s_max[warp / kWarps * kWarps + i]);
  }
  const int old = kv::exponent_of(before);
  int e = kv::scale_exponent<INT8>(amax);
  if (t.z > 0) e = max(e, old);
  const float inv = kv::pow2i(-e);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = r0 + i * kStep;
    if (r < t.w) {
      float f[8];
      unpack8(raw[i], f);
      *reinterpret_cast<uint2*>(codes + (t.z + r) * D + col) =
          make_uint2(kv::encode4<INT8>(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv),
                     kv::encode4<INT8>(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
    }
  }
  if (t.z > 0 && e > old) {
    const float f = kv::pow2i(max(old - e, -126));
    for (int r = r0; r < t.z; r += kStep) {
      uint2* q = reinterpret_cast<uint2*>(codes + r * D + col);
      const uint2 c = *q;
      uint32_t w[4];
      kv::decode4<INT8>(c.x, w[0], w[1]);
      kv::decode4<INT8>(c.y, w[2], w[3]);
      float2 g[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) g[k] = kv::f16x2_to_float2(w[k]);
      *q = make_uint2(kv::encode4<INT8>(g[0].x * f, g[0].y * f, g[1].x * f, g[1].y * f),
                      kv::encode4<INT8>(g[2].x * f, g[2].y * f, g[3].x * f, g[3].y * f));
    }
  }
  if (live && lane == 0) *scale = kv::pow2i(e);
}

// -------------------------------------------------------------------------- cache read
// out[i] = codes[slot i] * scale as bf16 (exact: 8 significant bits or fewer). Eight codes an
// item, so that a warp's stores cover whole sectors; four items a thread in flight.
constexpr int kReadThreads = 256;
constexpr int kReadItems = 4;

struct ReadParams {
  const uint8_t *k_codes, *v_codes;
  const float *k_scale, *v_scale;
  uint4 *k_out, *v_out;
  const int* slots;
  int64_t n;          // slots * heads * (D / 8)
  int per_slot;       // heads * (D / 8)
  int H, col_shift, page_shift;
  int64_t num_slots;
};

template <bool INT8>
__global__ void __launch_bounds__(kReadThreads) read_kernel(const ReadParams p) {
  const uint8_t* codes = blockIdx.y ? p.v_codes : p.k_codes;
  const float* scale = blockIdx.y ? p.v_scale : p.k_scale;
  uint4* out = blockIdx.y ? p.v_out : p.k_out;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * (kReadThreads * kReadItems);
  const int64_t slot0 = base / p.per_slot;
  const unsigned rem = static_cast<unsigned>(base - slot0 * p.per_slot);
  uint2 v[kReadItems];
  float s[kReadItems];
#pragma unroll
  for (int k = 0; k < kReadItems; ++k) {
    const unsigned i = k * kReadThreads + threadIdx.x;
    v[k] = make_uint2(0, 0);
    s[k] = 0.f;
    if (base + i >= p.n) continue;
    const unsigned in = (rem + i) / p.per_slot, item = rem + i - in * p.per_slot;
    const int slot = __ldg(p.slots + slot0 + in);
    if (slot < 0 || slot >= p.num_slots) continue;
    const int h = item >> p.col_shift, c = item & ((1 << p.col_shift) - 1);
    const int64_t unit = static_cast<int64_t>(slot >> p.page_shift) * p.H + h;
    const int64_t row = (unit << p.page_shift) + (slot & ((1 << p.page_shift) - 1));
    v[k] = __ldg(reinterpret_cast<const uint2*>(codes) + (row << p.col_shift) + c);
    s[k] = __ldg(scale + unit);
  }
#pragma unroll
  for (int k = 0; k < kReadItems; ++k) {
    const int64_t i = base + k * kReadThreads + threadIdx.x;
    if (i >= p.n) continue;
    uint32_t w[4];
    kv::decode4<INT8>(v[k].x, w[0], w[1]);
    kv::decode4<INT8>(v[k].y, w[2], w[3]);
    uint32_t o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = kv::f16x2_to_float2(w[e]);
      o[e] = pack_bf16x2(f.x * s[k], f.y * s[k]);
    }
    out[i] = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// ------------------------------------------------------------------------- logit rules
// One block per (row, slice of the vocabulary). The block counts the row's history inside its
// slice in shared memory (integer counts: the order of the atomics does not matter), then
// passes once over the slice, eight logits at a time: repetition, frequency, presence, mask; the
// few biased tokens are finished after that. Bound by reading the logits and writing the scores;
// every slice rereads the history (from L2), so slices are as long as filling the GPU allows. 128 rows
// of 32768 with 4096 tokens of history take 9.9 us out of L2 and 17 from memory (27 MB: 4.1 at the copy
// rate).
constexpr int kLogitThreads = 256;
constexpr int kLogitSlice = 8192;   // the longest: 32 KB of counts, four loads a thread
constexpr int kMaxBias = 1024;
constexpr int kSeen = static_cast<int>(0x80000000u);  // top bit: occurs in the prompt

struct LogitParams {
  const void* logits;
  int64_t stride, out_stride;
  float* out;
  const int* history;
  int64_t history_stride;
  const int *lens, *prompts;
  const float *repetition, *presence, *frequency;
  const int* bias_ids;
  const float* bias;
  const int* allowed;
  int V, L, NB, words, slice, vec;
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// Eight logits in flight, as loaded.
template <typename T> struct Raw8;
template <> struct Raw8<__nv_bfloat16> {
  uint4 v;
  __device__ void load(const __nv_bfloat16* z) { v = __ldg(reinterpret_cast<const uint4*>(z)); }
  __device__ void get(float (&f)[8]) const { unpack8(v, f); }
};
template <> struct Raw8<float> {
  float4 a, b;
  __device__ void load(const float* z) {
    a = __ldg(reinterpret_cast<const float4*>(z));
    b = __ldg(reinterpret_cast<const float4*>(z) + 1);
  }
  __device__ void get(float (&f)[8]) const {
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
};

template <typename T>
__global__ void __launch_bounds__(kLogitThreads) logits_kernel(const LogitParams p) {
  extern __shared__ __align__(16) int s_count[];  // [slice] occurrences; see kSeen
  const int row = blockIdx.y, v0 = blockIdx.x * p.slice, n = min(p.slice, p.V - v0);
  for (int i = threadIdx.x; i < p.slice / 4; i += kLogitThreads)
    reinterpret_cast<int4*>(s_count)[i] = make_int4(0, 0, 0, 0);
  const int len = min(max(p.lens[row], 0), p.L), prompt = p.prompts[row];
  const float rep = p.repetition ? p.repetition[row] : 1.f;
  const float pre = p.presence ? p.presence[row] : 0.f, freq = p.frequency ? p.frequency[row] : 0.f;
  const T* z = static_cast<const T*>(p.logits) + row * p.stride + v0;
  float* o = p.out + row * p.out_stride + v0;
  // all of the slice's logits are on their way while the history is counted
  constexpr int kPasses = kLogitSlice / (kLogitThreads * 8);
  Raw8<T> raw[kPasses];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int c = (i * kLogitThreads + threadIdx.x) * 8;
    if (p.vec && c + 8 <= n) raw[i].load(z + c);
  }
  __syncthreads();
  const int* hist = p.history + row * p.history_stride;
  for (int i = threadIdx.x; i < len; i += 8 * kLogitThreads) {
    int id[8]; 
#pragma unroll
    for (int k = 0; k < 8; ++k) id[k] = i + k * kLogitThreads < len ? __ldg(hist + i + k * kLogitThreads) : -1;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const unsigned t = static_cast<unsigned>(id[k]) - static_cast<unsigned>(v0);
      if (id[k] >= 0 && t < static_cast<unsigned>(n)) {
        if (i + k * kLogitThreads >= prompt) atomicAdd(&s_count[t], 1);
        else atomicOr(&s_count[t], kSeen);
      }
    }
  }
  __syncthreads();
  // One reciprocal a row: x * (1 / rep) is within 1.5 ulp of x / rep and an eighth of its work (128
  // rows of 32768: 12.0 us a call, 13.1 with divisions).
  const float inv = 1.f / rep;
  auto rule = [&](float x, int count) {
    if (count != 0) x *= x > 0.f ? inv : rep;
    count &= ~kSeen;
    return count > 0 ? x - freq * count - pre : x;
  };
  const int* allowed = p.allowed ? p.allowed + static_cast<int64_t>(row) * p.words : nullptr;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int c = (i * kLogitThreads + threadIdx.x) * 8;
    if (c >= n) break;
    const unsigned bits = allowed ? static_cast<unsigned>(allowed[(v0 + c) >> 5]) >> ((v0 + c) & 31) : 255u;
    if (p.vec && c + 8 <= n) {
      float f[8];
      raw[i].get(f);
      const int4 n0 = reinterpret_cast<const int4*>(s_count + c)[0];
      const int4 n1 = reinterpret_cast<const int4*>(s_count + c)[1];
      const int cnt[8] = {n0.x, n0.y, n0.z, n0.w, n1.x, n1.y, n1.z, n1.w};
      if ((n0.x | n0.y | n0.z | n0.w | n1.x | n1.y | n1.z | n1.w) != 0) {  // few tokens occurred
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = rule(f[e], cnt[e]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = (bits >> e) & 1u ? f[e] : -INFINITY;
      reinterpret_cast<float4*>(o + c)[0] = make_float4(f[0], f[1], f[2], f[3]);
      reinterpret_cast<float4*>(o + c)[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
      for (int e = 0; e < 8 && c + e < n; ++e)
        o[c + e] = (bits >> e) & 1u ? rule(to_float(z[c + e]), s_count[c + e]) : -INFINITY;
    }
  }
  if (!(rep >= 0x1p-126f && rep <= 0x1p126f)) {  // not a normal reciprocal: the same with divisions
    __syncthreads();
    for (int t = threadIdx.x; t < n; t += kLogitThreads) {
      const int seen = s_count[t], count = seen & ~kSeen;
      if (seen == 0 || (allowed && !((allowed[(v0 + t) >> 5] >> ((v0 + t) & 31)) & 1))) continue;
      float x = to_float(z[t]);
      x = x > 0.f ? x / rep : x * rep;
      o[t] = count > 0 ? x - freq * count - pre : x;
    }
  }
  if (p.NB == 0) return;
  __syncthreads();
  // A warp per entry, its lanes looking for the same token in the list. A token listed more than
  // once gets the sum, in list order: its first entry adds them up.
  const int* ids = p.bias_ids + static_cast<int64_t>(row) * p.NB;
  const float* values = p.bias + static_cast<int64_t>(row) * p.NB;
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x / 32; i < p.NB; i += kLogitThreads / 32) {
    const int id = __ldg(ids + i);
    const unsigned t = static_cast<unsigned>(id) - static_cast<unsigned>(v0);
    if (id < 0 || t >= static_cast<unsigned>(n)) continue;
    if (allowed && !((allowed[id >> 5] >> (id & 31)) & 1)) continue;
    float s = 0.f;
    bool first = true;
    for (int j0 = 0; j0 < p.NB && first; j0 += 32) {
      const bool same = j0 + lane < p.NB && __ldg(ids + j0 + lane) == id;
      const float x = same ? __ldg(values + j0 + lane) : 0.f;
      unsigned hits = __ballot_sync(0xffffffffu, same);
      first = hits == 0 || j0 + __ffs(hits) - 1 >= i;
      for (; hits && first; hits &= hits - 1) s += __shfl_sync(0xffffffffu, x, __ffs(hits) - 1);
    }
    if (first && lane == 0) o[t] += s;
  }
}

}  // namespace serving
}  // namespace nmb

using namespace nmb;
using namespace nmb::serving;

namespace {

void check_ints(const at::Tensor& t, int64_t n, const at::Device& dev, const char* what) {
  TORCH_CHECK(t.device() == dev && t.scalar_type() == at::kInt && t.dim() == 1 &&
                  t.is_contiguous() && t.numel() == n,
              what, " must be a contiguous int32 tensor of ", num(n), " values on the same device");
}

int page_shift_of(int64_t page_size) {
  for (int s = 4; s <= 7; ++s)
    if (page_size == (1 << s)) return s;
  TORCH_CHECK(false, "page_size must be 16, 32, 64 or 128, got ", num(page_size));
}

void check_cache(const at::Tensor& codes, const at::Tensor& scale, const char* what) {
  TORCH_CHECK(codes.is_cuda() && codes.dim() == 4 && codes.is_contiguous() &&
                  (codes.scalar_type() == at::kFloat8_e4m3fn || codes.scalar_type() == at::kChar),
              what, " pages must be contiguous CUDA [pages, kv_heads, page_size, head_dim], e4m3 or int8");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16 == 0, what, " pages: 16-byte alignment");
  TORCH_CHECK(scale.device() == codes.device() && scale.scalar_type() == at::kFloat &&
                  scale.dim() == 2 && scale.is_contiguous() && scale.size(0) == codes.size(0) &&
                  scale.size(1) == codes.size(1),
              what, " scales must be contiguous fp32 [pages, kv_heads] on the pages' device");
  page_shift_of(codes.size(2));
  TORCH_CHECK(codes.size(3) == 64 || codes.size(3) == 128, "head_dim must be 64 or 128, got ",
              num(codes.size(3)));
  TORCH_CHECK(codes.size(0) * codes.size(2) < (1ll << 31), "the cache holds 2^31 tokens or more");
}

}  // namespace

void check_paged_cache(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_scale,
                       const at::Tensor& v_scale) {
  check_cache(k, k_scale, "key");
  check_cache(v, v_scale, "value");
  TORCH_CHECK(k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type() && k.device() == v.device(),
              "key and value pages must have the same shape, type and device");
}

// (q_starts, kv_lens, positions, slots, touched, free_count, missing); new entries of `tables`
// are written in place.
std::vector<at::Tensor> plan_step(at::Tensor context, at::Tensor fresh, at::Tensor tables,
                                  at::Tensor free_pages, at::Tensor free_count, int64_t page_size,
                                  int64_t num_tokens) {
  const at::Device dev = context.device();
  TORCH_CHECK(context.is_cuda() && context.dim() == 1, "context_lens must be a 1-D CUDA tensor");
  const int64_t B = context.numel();
  check_ints(context, B, dev, "context_lens");
  check_ints(fresh, B, dev, "new_lens");
  check_ints(free_pages, free_pages.numel(), dev, "free_pages");
  check_ints(free_count, 1, dev, "free_count");
  TORCH_CHECK(tables.device() == dev && tables.scalar_type() == at::kInt && tables.dim() == 2 &&
                  tables.stride(1) == 1 && tables.size(0) >= B,
              "tables must be int32 [>= ", num(B), " requests, pages] on the same device with contiguous rows");
  TORCH_CHECK(B <= kPlanMaxRequests, "at most ", num(kPlanMaxRequests), " requests in a step, got ", num(B));
  TORCH_CHECK(num_tokens >= 0 && num_tokens < (1ll << 30), "num_tokens out of range");
  PlanParams p{};
  p.page_shift = page_shift_of(page_size);
  p.B = static_cast<int>(B);
  p.T = static_cast<int>(num_tokens);
  p.U = static_cast<int>(std::min(num_tokens, num_tokens / page_size + 2 * B));
  p.width = static_cast<int>(tables.size(1));
  p.table_stride = tables.stride(0);
  p.num_free = static_cast<int>(free_pages.numel());
  const at::cuda::CUDAGuard guard(dev);
  // one allocation: [touched 4U | q_starts B+1 | kv_lens B | positions T | slots T | 2 counts]
  at::Tensor buf = at::empty({4ll * p.U + 2 * B + 1 + 2ll * p.T + 2}, context.options());
  int64_t at_ = 0;
  auto part = [&](at::IntArrayRef sizes) {  // a tensor over the next values (a third of a view's cost)
    auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(buf.storage()), buf.key_set(), buf.dtype());
    impl->set_storage_offset(at_);
    impl->set_sizes_contiguous(sizes);
    at_ += impl->numel();
    return at::Tensor(std::move(impl));
  };
  at::Tensor touched = part({p.U, 4}), q_starts = part({B + 1}), kv_lens = part({B}),
             positions = part({p.T}), slots = part({p.T}), free_out = part({1}), missing = part({1});
  p.context = context.data_ptr<int>();
  p.fresh = fresh.data_ptr<int>();
  p.tables = tables.data_ptr<int>();
  p.free_pages = free_pages.data_ptr<int>();
  p.free_count = free_count.data_ptr<int>();
  p.touched = reinterpret_cast<int4*>(touched.data_ptr<int>());
  p.q_starts = q_starts.data_ptr<int>();
  p.kv_lens = kv_lens.data_ptr<int>();
  p.positions = positions.data_ptr<int>();
  p.slots = slots.data_ptr<int>();
  p.free_out = free_out.data_ptr<int>();
  p.missing = missing.data_ptr<int>();
  const int blocks = std::max(1, (std::max(p.T, p.U) + kPlanThreads - 1) / kPlanThreads);
  const size_t smem = 3 * (B + 1) * sizeof(int);
  if (smem > 48 * 1024)
    C10_CUDA_CHECK(cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        3 * (kPlanMaxRequests + 1) * sizeof(int)));
  plan_kernel<<<blocks, kPlanThreads, smem, at::cuda::getCurrentCUDAStream()>>>(p);
  NMB_LAUNCHED(1);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {q_starts, kv_lens, positions, slots, touched, free_out, missing};
}

template <bool INT8, int D>
static void launch_append(const AppendParams& p, int ps, unsigned grid, cudaStream_t s) {
  switch (ps) {
    case 16: append_kernel<INT8, D, 16><<<grid, kAppendThreads, 0, s>>>(p); break;
    case 32: append_kernel<INT8, D, 32><<<grid, kAppendThreads, 0, s>>>(p); break;
    case 64: append_kernel<INT8, D, 64><<<grid, kAppendThreads, 0, s>>>(p); break;
    default: append_kernel<INT8, D, 128><<<grid, kAppendThreads, 0, s>>>(p); break;
  }
}

void append_kv(at::Tensor k_pages, at::Tensor v_pages, at::Tensor k_scale, at::Tensor v_scale,
               at::Tensor k, at::Tensor v, at::Tensor touched) {
  check_paged_cache(k_pages, v_pages, k_scale, v_scale);
  const int64_t H = k_pages.size(1), D = k_pages.size(3);
  const at::Device dev = k_pages.device();
  for (const at::Tensor* t : {&k, &v})
    TORCH_CHECK(t->device() == dev && t->scalar_type() == at::kBFloat16 && t->dim() == 3 &&
                    t->size(1) == H && t->size(2) == D && t->stride(2) == 1,
                "k and v must be bf16 [tokens, ", num(H), ", ", num(D), "] on the same device with contiguous rows");
  TORCH_CHECK(k.size(0) == v.size(0) && k.size(0) < (1ll << 31), "k and v must have the same tokens");
  TORCH_CHECK(touched.device() == dev && touched.scalar_type() == at::kInt && touched.dim() == 2 &&
                  touched.size(1) == 4 && touched.is_contiguous() &&
                  reinterpret_cast<uintptr_t>(touched.data_ptr()) % 16 == 0,
              "touched must be the plan's int32 [entries, 4] on the same device");
  if (touched.size(0) == 0) return;
  AppendParams p{};
  bool vec = true;
  for (const at::Tensor* x : {&k, &v})
    vec = vec && reinterpret_cast<uintptr_t>(x->data_ptr()) % 16 == 0 && x->stride(0) % 8 == 0 &&
          x->stride(1) % 8 == 0;
  p.k = reinterpret_cast<const __nv_bfloat16*>(k.data_ptr());
  p.v = reinterpret_cast<const __nv_bfloat16*>(v.data_ptr());
  p.k_row = k.stride(0);
  p.k_head = k.stride(1);
  p.v_row = v.stride(0);
  p.v_head = v.stride(1);
  p.k_codes = static_cast<uint8_t*>(k_pages.data_ptr());
  p.v_codes = static_cast<uint8_t*>(v_pages.data_ptr());
  p.k_scale = k_scale.data_ptr<float>();
  p.v_scale = v_scale.data_ptr<float>();
  p.touched = reinterpret_cast<const int4*>(touched.data_ptr<int>());
  p.entries = static_cast<int>(touched.size(0));
  p.rows = static_cast<int>(k.size(0));
  p.num_pages = static_cast<int>(k_pages.size(0));
  p.H = static_cast<int>(H);
  p.vec = vec;
  const at::cuda::CUDAGuard guard(dev);
  cudaStream_t s = at::cuda::getCurrentCUDAStream();
  const int ps = static_cast<int>(k_pages.size(2));
  const int64_t units = touched.size(0) * H * 2, warps = std::max<int64_t>(1, ps * D / 4096);
  TORCH_CHECK(units < (1ll << 31), "too many pages to write in one call");
  const unsigned grid = static_cast<unsigned>((units * warps + 3) / 4);
  const bool i8 = k_pages.scalar_type() == at::kChar;
  if (D == 64) i8 ? launch_append<true, 64>(p, ps, grid, s) : launch_append<false, 64>(p, ps, grid, s);
  else i8 ? launch_append<true, 128>(p, ps, grid, s) : launch_append<false, 128>(p, ps, grid, s);
  NMB_LAUNCHED(1);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

std::vector<at::Tensor> read_kv(at::Tensor k_pages, at::Tensor v_pages, at::Tensor k_scale,
                                at::Tensor v_scale, at::Tensor slots) {
  check_paged_cache(k_pages, v_pages, k_scale, v_scale);
  const int64_t H = k_pages.size(1), D = k_pages.size(3), n = slots.numel();
  check_ints(slots, n, k_pages.device(), "slots");
  const at::cuda::CUDAGuard guard(k_pages.device());
  at::Tensor k = at::empty({n, H, D}, k_scale.options().dtype(at::kBFloat16)), v = at::empty_like(k);
  if (n == 0) return {k, v};
  ReadParams p{};
  p.k_codes = static_cast<const uint8_t*>(k_pages.data_ptr());
  p.v_codes = static_cast<const uint8_t*>(v_pages.data_ptr());
  p.k_scale = k_scale.data_ptr<float>();
  p.v_scale = v_scale.data_ptr<float>();
  p.k_out = reinterpret_cast<uint4*>(k.data_ptr());
  p.v_out = reinterpret_cast<uint4*>(v.data_ptr());
  p.slots = slots.data_ptr<int>();
  p.H = static_cast<int>(H);
  p.col_shift = D == 64 ? 3 : 4;
  p.per_slot = static_cast<int>(H << p.col_shift);
  p.n = n * p.per_slot;
  p.page_shift = page_shift_of(k_pages.size(2));
  p.num_slots = k_pages.size(0) * k_pages.size(2);
  const int64_t per = kReadThreads * kReadItems;
  const dim3 grid(static_cast<unsigned>((p.n + per - 1) / per), 2);
  cudaStream_t s = at::cuda::getCurrentCUDAStream();
  if (k_pages.scalar_type() == at::kChar) read_kernel<true><<<grid, kReadThreads, 0, s>>>(p);
  else read_kernel<false><<<grid, kReadThreads, 0, s>>>(p);
  NMB_LAUNCHED(1);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {k, v};
}

at::Tensor adjust_logits(at::Tensor logits, at::Tensor history, at::Tensor lens, at::Tensor prompts,
                         c10::optional<at::Tensor> repetition, c10::optional<at::Tensor> presence,
                         c10::optional<at::Tensor> frequency, c10::optional<at::Tensor> bias_ids,
                         c10::optional<at::Tensor> bias, c10::optional<at::Tensor> allowed) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.stride(1) == 1 &&
                  (logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kFloat),
              "logits must be CUDA bf16 or fp32 [requests, vocabulary] with contiguous rows");
  const at::Device dev = logits.device();
  const int64_t B = logits.size(0), V = logits.size(1);
  TORCH_CHECK(V < (1ll << 30) && B <= 65535, "logits are too large: ", num(B), " x ", num(V));
  TORCH_CHECK(history.device() == dev && history.scalar_type() == at::kInt && history.dim() == 2 &&
                  history.size(0) == B && (history.size(1) == 0 || history.stride(1) == 1) &&
                  history.size(1) < (1ll << 31),
              "history must be int32 [", num(B), ", tokens] on the same device with contiguous rows");
  check_ints(lens, B, dev, "history_lens");
  check_ints(prompts, B, dev, "prompt_lens");
  LogitParams p{};
  auto param = [&](const c10::optional<at::Tensor>& t, const char* what) -> const float* {
    if (!t.has_value()) return nullptr;
    TORCH_CHECK(t->device() == dev && t->scalar_type() == at::kFloat && t->dim() == 1 &&
                    t->numel() == B && t->is_contiguous(),
                what, " must be a contiguous fp32 tensor of ", num(B), " values on the same device");
    return t->data_ptr<float>();
  };
  p.repetition = param(repetition, "repetition");
  p.presence = param(presence, "presence");
  p.frequency = param(frequency, "frequency");
  TORCH_CHECK(bias_ids.has_value() == bias.has_value(), "bias_ids and bias come together");
  if (bias.has_value()) {
    TORCH_CHECK(bias_ids->device() == dev && bias_ids->scalar_type() == at::kInt &&
                    bias_ids->dim() == 2 && bias_ids->size(0) == B && bias_ids->is_contiguous() &&
                    bias_ids->size(1) <= kMaxBias,
                "bias_ids must be contiguous int32 [", num(B), ", at most ", num(kMaxBias), "] on the same device");
    TORCH_CHECK(bias->device() == dev && bias->scalar_type() == at::kFloat &&
                    bias->sizes() == bias_ids->sizes() && bias->is_contiguous(),
                "bias must be contiguous fp32 of bias_ids' shape on the same device");
    p.NB = static_cast<int>(bias->size(1));
    p.bias_ids = bias_ids->data_ptr<int>();
    p.bias = bias->data_ptr<float>();
  }
  if (allowed.has_value()) {
    TORCH_CHECK(allowed->device() == dev && allowed->scalar_type() == at::kInt &&
                    allowed->dim() == 2 && allowed->size(0) == B && allowed->is_contiguous() &&
                    allowed->size(1) == (V + 31) / 32,
                "allowed must be contiguous int32 [", num(B), ", ", num((V + 31) / 32), "] on the same device");
    p.words = static_cast<int>(allowed->size(1));
    p.allowed = allowed->data_ptr<int>();
  }
  const at::cuda::CUDAGuard guard(dev);
  // rows padded to 32 bytes, so that every row takes wide stores
  const int64_t pitch = (V + 7) / 8 * 8;
  at::Tensor out = at::empty({B, pitch}, logits.options().dtype(at::kFloat));
  if (pitch != V) out = out.narrow(1, 0, V);
  if (B == 0 || V == 0) return out;
  p.logits = logits.data_ptr();
  p.stride = logits.stride(0);
  p.out_stride = pitch;
  p.vec = reinterpret_cast<uintptr_t>(p.logits) % 16 == 0 && (p.stride % 8 == 0 || B == 1);
  p.out = out.data_ptr<float>();
  p.history = history.data_ptr<int>();
  p.history_stride = history.stride(0);
  p.L = static_cast<int>(history.size(1));
  p.lens = lens.data_ptr<int>();
  p.prompts = prompts.data_ptr<int>();
  p.V = static_cast<int>(V);
  // longest slice that still gives every SM two blocks
  int slice = kLogitSlice;
  const int64_t want = 2ll * at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  while (slice > 512 && B * ((V + slice - 1) / slice) < want) slice /= 2;
  p.slice = slice;
  const dim3 grid(static_cast<unsigned>((V + slice - 1) / slice), static_cast<unsigned>(B));
  const size_t smem = slice * sizeof(int);
  cudaStream_t s = at::cuda::getCurrentCUDAStream();
  if (logits.scalar_type() == at::kFloat) logits_kernel<float><<<grid, kLogitThreads, smem, s>>>(p);
  else logits_kernel<__nv_bfloat16><<<grid, kLogitThreads, smem, s>>>(p);
  NMB_LAUNCHED(1);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return out;
}

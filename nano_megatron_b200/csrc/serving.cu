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
// another. Bound by latency: two dependent loads, three block scans, one binary search.
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
  int touch = 0, fresh = 0;
  for (int b = b0; b < b1; ++b) {
    // rows past the T that the outputs hold are dropped
    const int row = static_cast<int>(min(at, static_cast<int64_t>(p.T))), n = min(max(p.fresh[b], 0), p.T - row);
    at += min(max(p.fresh[b], 0), p.T);
    const int ctx = context_of(b);
    s_row[b] = row;
    s_touch[b] = n > 0 ? ((ctx + n - 1) >> p.page_shift) - (ctx >> p.page_shift) + 1 : 0;
    s_fresh[b] = ((ctx + n + ps - 1) >> p.page_shift) - ((ctx + ps - 1) >> p.page_shift);
    touch += s_touch[b];
    fresh += s_fresh[b];
  }
  int64_t touch_total, fresh_total;
  int touch_at = static_cast<int>(block_scan(touch, warp_sums, touch_total));
  int fresh_at = static_cast<int>(block_scan(fresh, warp_sums, fresh_total));
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
      *p.missing = max(need - have, 0);
    }
  }
}

// ------------------------------------------------------------------------- cache write
// One block per (touched page, kv head, K or V). The new rows are read once into registers,
// their largest finite magnitude gives the page's scale, and the codes leave as 8-byte
// stores; codes that were on the page before are rescaled only when the scale grows.
constexpr int kAppendThreads = 128;

struct AppendParams {
  const __nv_bfloat16 *x[2];
  int64_t row_stride[2], head_stride[2];
  uint8_t* codes[2];
  float* scale[2];
  const int4* touched;
  int rows, num_pages, H, ps, vec;
};

__device__ __forceinline__ void load8(const __nv_bfloat16* p, bool vec, float (&f)[8]) {
  if (vec) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    f[0] = bf16_lo(v.x); f[1] = bf16_hi(v.x); f[2] = bf16_lo(v.y); f[3] = bf16_hi(v.y);
    f[4] = bf16_lo(v.z); f[5] = bf16_hi(v.z); f[6] = bf16_lo(v.w); f[7] = bf16_hi(v.w);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = __bfloat162float(p[e]);
  }
}

template <bool INT8, int D, int PS>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const AppendParams p) {
  constexpr int kCols = D / 8;                                    // 8-value chunks of a row
  constexpr int kPer = (PS * kCols + kAppendThreads - 1) / kAppendThreads;
  constexpr int kRowStep = kAppendThreads / kCols;
  __shared__ float s_max[kAppendThreads / 32];
  const int4 t = p.touched[blockIdx.x];
  if (t.x < 0 || t.x >= p.num_pages || t.w <= 0 || t.z < 0 || t.z + t.w > PS || t.y < 0 ||
      t.y + t.w > p.rows)
    return;
  const int h = blockIdx.y, which = blockIdx.z;
  const __nv_bfloat16* x = p.x[which] + t.y * p.row_stride[which] + h * p.head_stride[which];
  const int64_t unit = static_cast<int64_t>(t.x) * p.H + h;
  uint8_t* codes = p.codes[which] + unit * (PS * D);
  const int r0 = threadIdx.x / kCols, col = (threadIdx.x % kCols) * 8;
  const float before = p.scale[which][unit];

  float v[kPer][8];
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = r0 + i * kRowStep;
    if (r < t.w) {
      load8(x + r * p.row_stride[which] + col, p.vec, v[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = fabsf(v[i][e]);
        if (a <= 3.4e38f) amax = fmaxf(amax, a);  // infinities and NaN have no say
      }
    }
  }
  amax = warp_max(amax);
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x / 32] = amax;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kAppendThreads / 32; ++i) amax = fmaxf(amax, s_max[i]);
  int e = kv::scale_exponent<INT8>(amax);
  if (t.z > 0) e = max(e, kv::exponent_of(before));
  const float inv = kv::pow2i(-e);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = r0 + i * kRowStep;
    if (r < t.w)
      *reinterpret_cast<uint2*>(codes + (t.z + r) * D + col) =
          make_uint2(kv::encode4<INT8>(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv),
                     kv::encode4<INT8>(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv));
  }
  if (t.z > 0 && e > kv::exponent_of(before)) {
    const float f = kv::pow2i(max(kv::exponent_of(before) - e, -126));
    for (int r = r0; r < t.z; r += kRowStep) {
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
  if (threadIdx.x == 0) p.scale[which][unit] = kv::pow2i(e);
}

// -------------------------------------------------------------------------- cache read
// out[i] = codes[slot i] * scale as bf16 (exact: 7 significant bits or fewer). 16 codes a thread.
struct ReadParams {
  const uint8_t* codes[2];
  const float* scale[2];
  __nv_bfloat16* out[2];
  const int* slots;
  int64_t n;          // slots * heads * (D / 16)
  int H, D16, page_shift;
  int64_t num_slots;
};

template <bool INT8>
__global__ void __launch_bounds__(256) read_kernel(const ReadParams p) {
  const int which = blockIdx.y;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < p.n;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    const int c = static_cast<int>(i % p.D16);
    const int64_t rest = i / p.D16;
    const int h = static_cast<int>(rest % p.H);
    const int slot = p.slots[rest / p.H];
    uint32_t o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (slot >= 0 && slot < p.num_slots) {
      const int64_t page = slot >> p.page_shift;
      const int off = slot & ((1 << p.page_shift) - 1);
      const int64_t unit = page * p.H + h;
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p.codes[which]) +
                            ((unit << p.page_shift) + off) * p.D16 + c);
      const float s = __ldg(p.scale[which] + unit);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t lo, hi;
        kv::decode4<INT8>(w[k], lo, hi);
        const float2 a = kv::f16x2_to_float2(lo), b = kv::f16x2_to_float2(hi);
        o[2 * k] = pack_bf16x2(a.x * s, a.y * s);
        o[2 * k + 1] = pack_bf16x2(b.x * s, b.y * s);
      }
    }
    uint4* dst = reinterpret_cast<uint4*>(p.out[which]) + i * 2;
    dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
    dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

// ------------------------------------------------------------------------- logit rules
// One block per (row, slice of the vocabulary). The block counts the row's history inside its
// slice in shared memory (integer counts: the order of the atomics does not matter), then
// passes once over the slice: repetition, frequency, presence, bias, allow-mask.
constexpr int kLogitThreads = 256;
constexpr int kLogitSlice = 4096;
constexpr int kMaxBias = 1024;

struct LogitParams {
  const void* logits;
  int64_t stride;
  float* out;
  const int* history;
  int64_t history_stride;
  const int *lens, *prompts;
  const float *repetition, *presence, *frequency;
  const int* bias_ids;
  const float* bias;
  const int* allowed;
  int V, L, NB, words;
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__global__ void __launch_bounds__(kLogitThreads) logits_kernel(const LogitParams p) {
  __shared__ int s_count[kLogitSlice];            // occurrences in the generated part
  __shared__ uint32_t s_seen[kLogitSlice / 32];   // occurs anywhere
  __shared__ float s_bias[kLogitSlice];
  const int row = blockIdx.y, v0 = blockIdx.x * kLogitSlice, n = min(kLogitSlice, p.V - v0);
  for (int i = threadIdx.x; i < kLogitSlice; i += kLogitThreads) {
    s_count[i] = 0;
    s_bias[i] = 0.f;
  }
  for (int i = threadIdx.x; i < kLogitSlice / 32; i += kLogitThreads) s_seen[i] = 0;
  __syncthreads();
  const int len = min(max(p.lens[row], 0), p.L), prompt = p.prompts[row];
  const int* hist = p.history + row * p.history_stride;
  for (int i = threadIdx.x; i < len; i += kLogitThreads) {
    const unsigned t = static_cast<unsigned>(hist[i]) - static_cast<unsigned>(v0);
    if (t < static_cast<unsigned>(n)) {
      atomicOr(&s_seen[t >> 5], 1u << (t & 31));
      if (i >= prompt) atomicAdd(&s_count[t], 1);
    }
  }
  // A token listed more than once gets the sum, in list order: its first entry adds them up.
  for (int i = threadIdx.x; i < p.NB; i += kLogitThreads) {
    const int* ids = p.bias_ids + static_cast<int64_t>(row) * p.NB;
    const int id = ids[i];
    const unsigned t = static_cast<unsigned>(id) - static_cast<unsigned>(v0);
    if (id >= 0 && t < static_cast<unsigned>(n)) {
      bool first = true;
      for (int j = 0; j < i; ++j) first = first && ids[j] != id;
      if (first) {
        float s = 0.f;
        for (int j = i; j < p.NB; ++j)
          if (ids[j] == id) s += p.bias[static_cast<int64_t>(row) * p.NB + j];
        s_bias[t] = s;
      }
    }
  }
  __syncthreads();
  const float rep = p.repetition ? p.repetition[row] : 1.f;
  const float pre = p.presence ? p.presence[row] : 0.f, freq = p.frequency ? p.frequency[row] : 0.f;
  const T* z = static_cast<const T*>(p.logits) + row * p.stride + v0;
  float* o = p.out + static_cast<int64_t>(row) * p.V + v0;
  for (int i = threadIdx.x; i < n; i += kLogitThreads) {
    float x = to_float(z[i]);
    if ((s_seen[i >> 5] >> (i & 31)) & 1u) x = x > 0.f ? x / rep : x * rep;
    const int c = s_count[i];
    if (c > 0) x = x - freq * c - pre;
    x += s_bias[i];
    if (p.allowed) {
      const int v = v0 + i;
      if (!((p.allowed[static_cast<int64_t>(row) * p.words + (v >> 5)] >> (v & 31)) & 1)) x = -INFINITY;
    }
    o[i] = x;
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
  auto view = [&](int64_t n) {
    at::Tensor t = buf.narrow(0, at_, n);
    at_ += n;
    return t;
  };
  at::Tensor touched = view(4ll * p.U).view({p.U, 4}), q_starts = view(B + 1), kv_lens = view(B),
             positions = view(p.T), slots = view(p.T), free_out = view(1), missing = view(1);
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
static void launch_append(const AppendParams& p, int ps, dim3 grid, cudaStream_t s) {
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
  for (int i = 0; i < 2; ++i) {
    const at::Tensor& x = i ? v : k;
    p.x[i] = reinterpret_cast<const __nv_bfloat16*>(x.data_ptr());
    p.row_stride[i] = x.stride(0);
    p.head_stride[i] = x.stride(1);
    p.codes[i] = static_cast<uint8_t*>((i ? v_pages : k_pages).data_ptr());
    p.scale[i] = (i ? v_scale : k_scale).data_ptr<float>();
    vec = vec && reinterpret_cast<uintptr_t>(p.x[i]) % 16 == 0 && x.stride(0) % 8 == 0 &&
          x.stride(1) % 8 == 0;
  }
  p.touched = reinterpret_cast<const int4*>(touched.data_ptr<int>());
  p.rows = static_cast<int>(k.size(0));
  p.num_pages = static_cast<int>(k_pages.size(0));
  p.H = static_cast<int>(H);
  p.vec = vec;
  const at::cuda::CUDAGuard guard(dev);
  cudaStream_t s = at::cuda::getCurrentCUDAStream();
  const int ps = static_cast<int>(k_pages.size(2));
  const dim3 grid(touched.size(0), H, 2);
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
  for (int i = 0; i < 2; ++i) {
    p.codes[i] = static_cast<const uint8_t*>((i ? v_pages : k_pages).data_ptr());
    p.scale[i] = (i ? v_scale : k_scale).data_ptr<float>();
    p.out[i] = reinterpret_cast<__nv_bfloat16*>((i ? v : k).data_ptr());
  }
  p.slots = slots.data_ptr<int>();
  p.H = static_cast<int>(H);
  p.D16 = static_cast<int>(D / 16);
  p.n = n * H * p.D16;
  p.page_shift = page_shift_of(k_pages.size(2));
  p.num_slots = k_pages.size(0) * k_pages.size(2);
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>((p.n + 255) / 256, 148 * 16)), 2);
  cudaStream_t s = at::cuda::getCurrentCUDAStream();
  if (k_pages.scalar_type() == at::kChar) read_kernel<true><<<grid, 256, 0, s>>>(p);
  else read_kernel<false><<<grid, 256, 0, s>>>(p);
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
  TORCH_CHECK(V < (1ll << 31) - kLogitSlice && B <= 65535, "logits are too large: ", num(B), " x ", num(V));
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
  at::Tensor out = at::empty({B, V}, logits.options().dtype(at::kFloat));
  if (B == 0 || V == 0) return out;
  p.logits = logits.data_ptr();
  p.stride = logits.stride(0);
  p.out = out.data_ptr<float>();
  p.history = history.data_ptr<int>();
  p.history_stride = history.stride(0);
  p.L = static_cast<int>(history.size(1));
  p.lens = lens.data_ptr<int>();
  p.prompts = prompts.data_ptr<int>();
  p.V = static_cast<int>(V);
  const dim3 grid((V + kLogitSlice - 1) / kLogitSlice, B);
  cudaStream_t s = at::cuda::getCurrentCUDAStream();
  if (logits.scalar_type() == at::kFloat) logits_kernel<float><<<grid, kLogitThreads, 0, s>>>(p);
  else logits_kernel<__nv_bfloat16><<<grid, kLogitThreads, 0, s>>>(p);
  NMB_LAUNCHED(1);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return out;
}

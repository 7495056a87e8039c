// Attention of a batched step over the 8-bit paged K/V cache.
//
//   o[row] = sum_j p_j vs_j c_j / sum_j p_j,   p_j = 2^(s_j - max),   s_j = log2e * scale * q.k_j
//
// with value codes c_j and value scales vs_j = 2^e_j (one per page and kv head). Because the
// scales are powers of two, vs_j joins the logit: t_j = s_j + e_j, M = running max of t, and
//   numerator += 2^(t_j - M) c_j,      denominator += 2^(t_j - M) 2^-e_j.
// The f16 probabilities stay at most 2^8 (see kLazy) whatever the scales of different pages.
// Codes of both formats are exact in f16, queries are scaled row by row by a power of two that
// brings their largest magnitude to [1, 2), so the f16 products are exact; sums are fp32.
//
// Decode kernel (few query rows per request: decoding, short continuations). Bound by reading
// the codes of K and V once.
//  * A unit is (request, kv head, block of 16 query rows = tokens x heads of the group). Its keys
//    are cut into tiles of 32; the tiles of all units, in order, are dealt evenly to the CTAs,
//    whatever the lengths (every CTA scans the B lengths for itself). A unit that is shared by
//    several CTAs is put together by the one that finishes last, in CTA order, so the result
//    does not depend on the schedule.
//  * The four warps of a CTA take every fourth tile of its share. Each has its own ring of TMA
//    loads (pages are contiguous [page_size, D] rectangles), its own softmax state, and no
//    barrier with the others until a unit ends.
//  * mma.m16n8k16 (f16): 16 rows are all there is to multiply with, too few for a 128-row
//    tcgen05 tile, and the kernel waits for memory anyway. Key order inside a tile and the
//    column order of V are permuted so that every shared-memory read is 16 bytes wide (8 for
//    D = 64 values) without bank conflicts and decoded codes are fragments in place.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cudaTypedefs.h>

#include <map>
#include <mutex>

#include "paged_kv.cuh"

// serving.cu: shapes, types and devices of a K/V cache.
void check_paged_cache(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_scale,
                       const at::Tensor& v_scale);

namespace nmb {
namespace paged {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 32;           // keys of a tile
constexpr int kMinTiles = kWarps;   // tiles of a CTA's share at least: one per warp
constexpr float kLog2e = 1.4426950408889634f;
// The running max only moves when a tile exceeds it by 2^8: most tiles then skip rescaling the
// accumulator, and P <= 256 keeps its 11 bits in f16.
constexpr float kLazy = 8.f;

template <int D>
struct Cfg {
  static constexpr int kStages = D == 128 ? 3 : 4;
  static constexpr int kStageBytes = 2 * kTile * D;
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kMerge = kWarps * 8 * D * 4;         // 8 rows at a time
  static constexpr int kStats = kWarps * 16 * 2 * 4 + 16 * 2 * 4;
  static constexpr int kInfo = kWarps * kStages * 16;
  static constexpr int kSmem = kRing + kMerge + kStats + kInfo + kWarps * kStages * 8 + 16;
  static constexpr int kCtasPerSm = D == 128 ? 2 : 3;
};

struct Params {
  const __nv_bfloat16* q;
  int64_t q_row, q_head;
  __nv_bfloat16* o;                 // [T, Hq, D]
  float* lse;                       // [T, Hq] or null
  const float *k_scale, *v_scale;
  const int *tables, *q_starts, *kv_lens;
  int64_t table_stride;
  int width, num_pages, ps, page_shift;
  int B, T, Hq, Hkv, G;
  int max_rows;                     // requests with more query rows than this are not handled here
  float scale_log2;
  float* part;                      // [grid][2][16][D] numerators of shared units
  float2* part_ml;                  // [grid][2][16] (M, denominator)
  int* counters;                    // tiles finished of each shared unit; zero between calls
  int* status;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// One request as this kernel sees it.
struct Request {
  int q0, nq, kv, blocks, tiles;    // blocks of 16 rows; tiles of one unit
  __device__ int64_t total(int Hkv) const { return static_cast<int64_t>(blocks) * Hkv * tiles; }
};

__device__ __forceinline__ Request load_request(const Params& p, int b) {
  Request r;
  r.q0 = min(max(__ldg(p.q_starts + b), 0), p.T);
  r.nq = min(max(__ldg(p.q_starts + b + 1) - r.q0, 0), p.T - r.q0);
  r.kv = min(max(__ldg(p.kv_lens + b), 0), p.width << p.page_shift);
  const int rows = r.nq <= p.max_rows / p.G ? r.nq * p.G : 0;
  r.blocks = (rows + 15) / 16;
  r.tiles = max(1, (r.kv + kTile - 1) / kTile);
  return r;
}

// A run of tiles of one unit: position in the CTA's share [g, end).
struct Cursor {
  int64_t g, end, base;   // base: global index of the request's first tile
  int b;
  Request r;
  int unit, tile, n;      // unit in the request, first tile, tiles in this run

  __device__ void set() {
    const int64_t at = g - base;
    unit = static_cast<int>(at / r.tiles);
    tile = static_cast<int>(at - static_cast<int64_t>(unit) * r.tiles);
    n = static_cast<int>(min(static_cast<int64_t>(r.tiles - tile), end - g));
  }
  __device__ bool done() const { return g >= end; }
  __device__ void next(const Params& p) {
    g += n;
    if (g >= end) return;
    while (g >= base + r.total(p.Hkv)) {  // a request with tiles left follows, since g < end
      if (b + 1 >= p.B) {                   // (only if the lengths changed under the kernel)
        g = end;
        return;
      }
      base += r.total(p.Hkv);
      r = load_request(p, ++b);
    }
    set();
  }
};

template <int D>
__device__ __forceinline__ int key_of(int n) {  // row inside an 8-key group of fragment column n
  return D == 128 ? ((n >> 1) | ((n & 1) << 2)) : (n ^ ((n >> 1) & 1));
}

template <int D>
__device__ __forceinline__ int chunk_at(int row, int c) {  // byte offset of 16-byte chunk c
  return D == 128 ? row * 128 + ((c ^ (row & 7)) << 4) : row * 64 + ((c ^ ((row >> 1) & 3)) << 4);
}

// Float4 slot of (row, 16-float block, i) in the merge area, spread over the banks.
template <int D>
__device__ __forceinline__ int merge_at(int row, int blk, int i) {
  return row * (D / 4) + blk * 4 + (i ^ (((blk >> 1) & 1) | ((row & 1) << 1)));
}

template <int D, bool INT8>
__global__ void __launch_bounds__(kThreads, Cfg<D>::kCtasPerSm)
    decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const Params p) {
  using C = Cfg<D>;
  constexpr int S = C::kStages;
  constexpr int kSteps = D / 16;
  constexpr int kCols = D / 8;      // n-tiles of the output
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* ring = smem;
  float4* s_merge = reinterpret_cast<float4*>(smem + C::kRing);
  float2* s_stat = reinterpret_cast<float2*>(smem + C::kRing + C::kMerge);   // [warp][16] (M, l)
  float2* s_tot = s_stat + kWarps * 16;                                      // [16]
  float4* s_info = reinterpret_cast<float4*>(s_tot + 16);                    // [warp][S]
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_info + kWarps * S);
  volatile int* s_flag = reinterpret_cast<volatile int*>(bars + kWarps * S); // abort, last

  const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32;
  const int g8 = lane >> 2, t4 = lane & 3;
  if (smem_u32(smem) & 1023u) {     // the swizzle pattern needs 1024-byte alignment
    if (tid == 0) record_status(p.status, kStatusSmemAlignment);
    return;
  }

  // Rows past the last request's (padding) are zero.
  {
    const int used = min(max(__ldg(p.q_starts + p.B), 0), p.T);
    const int64_t n = static_cast<int64_t>(p.T - used) * p.Hq * (D / 8);
    uint4* o4 = reinterpret_cast<uint4*>(p.o) + static_cast<int64_t>(used) * p.Hq * (D / 8);
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + tid; i < n;
         i += static_cast<int64_t>(gridDim.x) * kThreads)
      o4[i] = make_uint4(0, 0, 0, 0);
    if (p.lse != nullptr)
      for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + tid;
           i < static_cast<int64_t>(p.T - used) * p.Hq; i += static_cast<int64_t>(gridDim.x) * kThreads)
        p.lse[static_cast<int64_t>(used) * p.Hq + i] = -INFINITY;
  }

  // ---- this CTA's share of the tiles
  Cursor cur;
  int64_t total;
  int64_t ctas;
  {
    int64_t* s_scan = reinterpret_cast<int64_t*>(s_merge);  // free until the first merge
    const int per = (p.B + kThreads - 1) / kThreads;
    const int b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
    int64_t sum = 0;
    for (int b = b0; b < b1; ++b) sum += load_request(p, b).total(p.Hkv);
    int64_t x = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) s_scan[warp] = x;
    if (tid == 0) {
      for (int i = 0; i < kWarps * S; ++i) mbar_init(&bars[i], 1);
      s_flag[0] = 0;
      fence_mbar_init();
    }
    __syncthreads();
    int64_t before = x - sum;
    total = 0;
    for (int i = 0; i < kWarps; ++i) {
      if (i < warp) before += s_scan[i];
      total += s_scan[i];
    }
    ctas = min(static_cast<int64_t>(gridDim.x), (total + kMinTiles - 1) / kMinTiles);
    if (blockIdx.x >= ctas) return;
    cur.g = blockIdx.x * total / ctas;
    cur.end = (blockIdx.x + 1) * total / ctas;
    if (before <= cur.g && cur.g < before + sum) {
      int b = b0;
      int64_t base = before;
      for (;; ++b) {
        const int64_t t = load_request(p, b).total(p.Hkv);
        if (cur.g < base + t || b + 1 >= b1) break;
        base += t;
      }
      s_scan[4] = b;
      s_scan[5] = base;
    }
    __syncthreads();
    cur.b = static_cast<int>(s_scan[4]);
    cur.base = s_scan[5];
    cur.r = load_request(p, cur.b);
    cur.set();
    __syncthreads();  // the merge area is free again
  }

  // ---- this warp's loads, S tiles ahead of the math
  uint8_t* my_ring = ring + warp * S * C::kStageBytes;
  uint64_t* my_bars = bars + warp * S;
  float4* my_info = s_info + warp * S;
  Cursor ahead = cur;
  int ahead_i = warp;               // tile of the run
  int pages[2];                     // page ids of the next tile to load, fetched a step early
  bool more = true;
  int in_flight = 0;                // tiles loaded and not yet waited for
  float4 info = make_float4(0.f, 0.f, 0.f, 0.f);  // scales of the tile loaded last, on their way
  int info_stage = -1;
  const bool two = p.ps < kTile;
  const int box = two ? p.ps : kTile;

  auto fetch_pages = [&]() {        // moves `ahead` to this warp's next tile and asks for its pages
    while (ahead_i >= ahead.n) {
      ahead.next(p);
      ahead_i = warp;
      if (ahead.done()) {
        more = false;
        return;
      }
    }
    const int key0 = (ahead.tile + ahead_i) * kTile;
    const int* row = p.tables + ahead.b * p.table_stride;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int key = key0 + i * 16;
      pages[i] = key < ahead.r.kv && (i == 0 || two) ? __ldg(row + (key >> p.page_shift)) : -1;
    }
    if (!two) pages[1] = pages[0];
  };
  auto flush_info = [&]() {
    if (info_stage >= 0 && lane == 0) my_info[info_stage] = info;
    info_stage = -1;
  };
  auto issue = [&](int stage) {     // loads the tile of `pages` and moves on
    flush_info();
    if (!more) return;
    ++in_flight;
    info_stage = stage;
    const int h = ahead.unit / ahead.r.blocks;
    const int key0 = (ahead.tile + ahead_i) * kTile;
    const bool ok0 = pages[0] >= 0 && pages[0] < p.num_pages;
    const bool ok1 = pages[1] >= 0 && pages[1] < p.num_pages;
    const int64_t u0 = static_cast<int64_t>(pages[0]) * p.Hkv + h;
    const int64_t u1 = static_cast<int64_t>(pages[1]) * p.Hkv + h;
    if (lane == 0) {
      uint8_t* dst = my_ring + stage * C::kStageBytes;
      const uint32_t bytes = (ok0 ? 2u * box * D : 0u) + (two && ok1 ? 2u * box * D : 0u);
      if (bytes) mbar_arrive_expect_tx(&my_bars[stage], bytes);
      else mbar_arrive(&my_bars[stage]);
      if (ok0) {
        const int y = static_cast<int>(u0 << p.page_shift) + (key0 & (p.ps - 1));
        tma_load_2d(dst, &tmK, &my_bars[stage], 0, y);
        tma_load_2d(dst + kTile * D, &tmV, &my_bars[stage], 0, y);
      }
      if (two && ok1) {
        const int y = static_cast<int>(u1 << p.page_shift);
        tma_load_2d(dst + 16 * D, &tmK, &my_bars[stage], 0, y);
        tma_load_2d(dst + kTile * D + 16 * D, &tmV, &my_bars[stage], 0, y);
      }
    }
    // a value scale of 0 marks a page that does not exist
    info.x = ok0 ? __ldg(p.k_scale + u0) : 0.f;
    info.y = ok1 ? __ldg(p.k_scale + u1) : 0.f;
    info.z = ok0 ? __ldg(p.v_scale + u0) : 0.f;
    info.w = ok1 ? __ldg(p.v_scale + u1) : 0.f;
    ahead_i += kWarps;
    fetch_pages();
  };
  fetch_pages();
#pragma unroll 1
  for (int s = 0; s < S; ++s) issue(s);

  // ---- units
  int stage = 0;
  uint32_t phase = 0;
  bool first_run = true;
  for (; !cur.done(); cur.next(p), first_run = false) {
    const int h = cur.unit / cur.r.blocks, rb = cur.unit - h * cur.r.blocks;
    const int rows = min(16, cur.r.nq * p.G - rb * 16);
    // query fragments: rows g8 and g8 + 8, 16 consecutive values per 64 of D
    uint32_t qa[kSteps][4];
    float row_scale[2];
    int limit[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = g8 + 8 * i;
      const int tok = (rb * 16 + r) / p.G, head = (rb * 16 + r) - tok * p.G;
      const bool live = r < rows;
      limit[i] = live ? cur.r.kv - cur.r.nq + tok + 1 : 0;
      const __nv_bfloat16* src = p.q + (cur.r.q0 + tok) * p.q_row + (h * p.G + head) * p.q_head;
      uint4 raw[D / 32];
      float amax = 0.f;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        raw[c] = live ? __ldg(reinterpret_cast<const uint4*>(src + (c >> 1) * 64 + 16 * t4) + (c & 1))
                      : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          amax = fmaxf(amax, fmaxf(fabsf(bf16_lo(w[e])), fabsf(bf16_hi(w[e]))));
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      // exponent of the row's largest magnitude (fmaxf drops NaN; infinity keeps 127)
      const int e = min(max(kv::exponent_of(amax), -100), 126);
      const float down = kv::pow2i(-e);
      row_scale[i] = kv::pow2i(e) * p.scale_log2;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        const uint32_t w[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
        for (int e2 = 0; e2 < 4; ++e2)  // word e2 of half c: k-step 4 * (c / 2) + 2 * (c % 2) + e2 / 2
          qa[(c >> 1) * 4 + (c & 1) * 2 + (e2 >> 1)][(e2 & 1) * 2 + i] =
              f16x2(bf16_lo(w[e2]) * down, bf16_hi(w[e2]) * down);
      }
    }
    float acc[kCols][4];
#pragma unroll
    for (int j = 0; j < kCols; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
    const int free_keys = cur.r.kv - cur.r.nq + rb * 16 / p.G + 1;  // keys that every row sees

    for (int i = warp; i < cur.n; i += kWarps) {
      if (in_flight > 0) {
        --in_flight;
        if (!mbar_wait(&my_bars[stage], phase, p.status, kStatusAttnTimeout, s_flag)) {
          // give up: load no more, but wait (bounded) for what is still on its way
          more = false;
          mbar_wait(&my_bars[stage], phase, p.status, kStatusAttnTimeout, nullptr);
        }
      }
      const uint8_t* sk = my_ring + stage * C::kStageBytes;
      const uint8_t* sv = sk + kTile * D;
      __syncwarp();
      const float4 f = my_info[stage];
      const int key0 = (cur.tile + i) * kTile;
      const bool masked = key0 + kTile > free_keys || f.z == 0.f || f.w == 0.f;

      float s[4][4];
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) {
        s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
        const int row = nt * 8 + key_of<D>(g8);
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          const uint4 v = *reinterpret_cast<const uint4*>(sk + chunk_at<D>(row, c * 4 + t4));
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t lo, hi;
            kv::decode4<INT8>(w[e], lo, hi);
            mma_f16(s[nt], qa[c * 4 + e], lo, hi);
          }
        }
      }
      // logits in base 2 plus log2 of the value scale
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) {
        const float ks = nt < 2 ? f.x : f.y;
        const float vb = static_cast<float>(kv::exponent_of(nt < 2 ? f.z : f.w));
        const float f0 = ks * row_scale[0], f1 = ks * row_scale[1];
        s[nt][0] = fmaf(s[nt][0], f0, vb);
        s[nt][1] = fmaf(s[nt][1], f0, vb);
        s[nt][2] = fmaf(s[nt][2], f1, vb);
        s[nt][3] = fmaf(s[nt][3], f1, vb);
      }
      if (masked) {
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
          const bool page = (nt < 2 ? f.z : f.w) != 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + nt * 8 + key_of<D>(2 * t4 + (e & 1));
            if (!page || key >= limit[e >> 1]) s[nt][e] = -INFINITY;
          }
        }
      }
      float mx[2];
#pragma unroll
      for (int i2 = 0; i2 < 2; ++i2) {
        float m = s[0][2 * i2];
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) m = fmaxf(m, fmaxf(s[nt][2 * i2], s[nt][2 * i2 + 1]));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        mx[i2] = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      }
      if (__any_sync(0xffffffffu, mx[0] > m_run[0] + kLazy || mx[1] > m_run[1] + kLazy)) {
        float corr[2];
#pragma unroll
        for (int i2 = 0; i2 < 2; ++i2) {
          const float m = fmaxf(m_run[i2], mx[i2]);
          corr[i2] = m_run[i2] == -INFINITY ? (m == -INFINITY ? 1.f : 0.f) : ex2(m_run[i2] - m);
          l_run[i2] *= corr[i2];
          m_run[i2] = m;
        }
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
          acc[j][0] *= corr[0];
          acc[j][1] *= corr[0];
          acc[j][2] *= corr[1];
          acc[j][3] *= corr[1];
        }
      }
      const float ref0 = m_run[0] == -INFINITY ? 0.f : m_run[0];
      const float ref1 = m_run[1] == -INFINITY ? 0.f : m_run[1];
      float lt[2][2] = {{0.f, 0.f}, {0.f, 0.f}};  // [row][16-key half]
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) {
        s[nt][0] = ex2(s[nt][0] - ref0);
        s[nt][1] = ex2(s[nt][1] - ref0);
        s[nt][2] = ex2(s[nt][2] - ref1);
        s[nt][3] = ex2(s[nt][3] - ref1);
        lt[0][nt >> 1] += s[nt][0] + s[nt][1];
        lt[1][nt >> 1] += s[nt][2] + s[nt][3];
      }
      // a missing page has only zeros in lt; its 2^-(-127) = 2^127 stays finite
      const float iv0 = kv::pow2i(-kv::exponent_of(f.z)), iv1 = kv::pow2i(-kv::exponent_of(f.w));
#pragma unroll
      for (int i2 = 0; i2 < 2; ++i2)
        l_run[i2] = fmaf(lt[i2][0], iv0, fmaf(lt[i2][1], iv1, l_run[i2]));

      const bool tail = key0 + kTile > cur.r.kv || f.z == 0.f || f.w == 0.f;
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        const uint32_t pa[4] = {f16x2(s[2 * s2][0], s[2 * s2][1]), f16x2(s[2 * s2][2], s[2 * s2][3]),
                                f16x2(s[2 * s2 + 1][0], s[2 * s2 + 1][1]),
                                f16x2(s[2 * s2 + 1][2], s[2 * s2 + 1][3])};
        uint32_t v[4][D / 32];  // keys 2t, 2t+1 of the first 8-key group, then of the second
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = s2 * 16 + (e >> 1) * 8 + key_of<D>(2 * t4 + (e & 1));
          if constexpr (D == 128) {
            const uint4 x = *reinterpret_cast<const uint4*>(
                sv + chunk_at<D>(row, (g8 >> 1) | ((g8 & 1) << 2)));
            v[e][0] = x.x; v[e][1] = x.y; v[e][2] = x.z; v[e][3] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(sv + chunk_at<D>(row, g8 >> 1) + (g8 & 1) * 8);
            v[e][0] = x.x; v[e][1] = x.y;
          }
          // codes behind the last key or of a missing page are stale: 0 * NaN is NaN
          if (tail && (key0 + row >= cur.r.kv || (s2 == 0 ? f.z : f.w) == 0.f)) {
#pragma unroll
            for (int w = 0; w < D / 32; ++w) v[e][w] = 0;
          }
        }
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {
          uint32_t b0[4], b1[4];
          kv::decode4<INT8>(__byte_perm(v[0][w], v[1][w], 0x5140), b0[0], b0[1]);
          kv::decode4<INT8>(__byte_perm(v[0][w], v[1][w], 0x7362), b0[2], b0[3]);
          kv::decode4<INT8>(__byte_perm(v[2][w], v[3][w], 0x5140), b1[0], b1[1]);
          kv::decode4<INT8>(__byte_perm(v[2][w], v[3][w], 0x7362), b1[2], b1[3]);
#pragma unroll
          for (int e = 0; e < 4; ++e) mma_f16(acc[w * 4 + e], pa, b0[e], b1[e]);
        }
      }
      __syncwarp();
      issue(stage);
      if (++stage == S) {
        stage = 0;
        phase ^= 1u;
      }
    }

    // ---- the four warps' states into one
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 1);
      l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 2);
      if (t4 == 0) s_stat[warp * 16 + g8 + 8 * i] = make_float2(m_run[i], l_run[i]);
    }
    __syncthreads();
    float corr[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_stat[w * 16 + g8 + 8 * i].x);
      const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 st = s_stat[w * 16 + g8 + 8 * i];
        l = fmaf(st.y, ex2(st.x - ref), l);
      }
      corr[i] = ex2(m_run[i] - ref);
      if (warp == 0 && t4 == 0) s_tot[g8 + 8 * i] = make_float2(m, l);
    }
    const bool whole = cur.n == cur.r.tiles;
    const int slot = first_run ? 0 : 1;
    float* part = p.part + (static_cast<int64_t>(blockIdx.x) * 2 + slot) * (16 * D);
    for (int half = 0; half < (rows > 8 ? 2 : 1); ++half) {
      if (half) __syncthreads();    // the first half has been read
      float4* mine = s_merge + warp * 8 * (D / 4);
#pragma unroll
      for (int blk = 0; blk < D / 64; ++blk)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int d = i * 4 + e;  // of the 16 in this thread's block
            if constexpr (D == 128) x[e] = half ? acc[d][blk + 2] : acc[d][blk];
            else x[e] = d < 8 ? (half ? acc[d][2] : acc[d][0]) : (half ? acc[d - 8][3] : acc[d - 8][1]);
            x[e] *= corr[half];
          }
          mine[merge_at<D>(g8, blk * 4 + t4, i)] = make_float4(x[0], x[1], x[2], x[3]);
        }
      __syncthreads();
      for (int u = tid; u < 8 * (D / 4); u += kThreads) {
        const int r8 = u / (D / 4), q = u % (D / 4), row = half * 8 + r8;
        if (row >= rows) continue;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 y = s_merge[w * 8 * (D / 4) + merge_at<D>(r8, q >> 2, q & 3)];
          x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
        }
        const float2 tot = s_tot[row];
        if (whole) {
          const float inv = tot.y > 0.f || tot.y != tot.y ? 1.f / tot.y : 0.f;
          const int tok = (rb * 16 + row) / p.G, head = h * p.G + (rb * 16 + row) - tok * p.G;
          const int64_t at = static_cast<int64_t>(cur.r.q0 + tok) * p.Hq + head;
          *reinterpret_cast<uint2*>(p.o + at * D + q * 4) =
              make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
          if (p.lse != nullptr && q == 0)
            p.lse[at] = tot.y == 0.f ? -INFINITY : tot.x + log2f(tot.y);
        } else {
          *reinterpret_cast<float4*>(part + row * D + q * 4) = x;
          if (q == 0) p.part_ml[(blockIdx.x * 2 + slot) * 16 + row] = tot;
        }
      }
    }
    if (whole) continue;

    // ---- a unit shared with other CTAs: the last to finish adds the parts up in CTA order
    __threadfence();
    __syncthreads();
    const int rpt = (p.G + 15) / 16;
    if (tid == 0) {
      int* counter = p.counters + (static_cast<int64_t>(h) * p.T + cur.r.q0) * rpt + rb;
      const int before = atomicAdd(counter, cur.n);
      const bool last = before + cur.n == cur.r.tiles;
      if (last) *counter = 0;
      __threadfence();
      s_flag[1] = last;
    }
    __syncthreads();
    if (s_flag[1]) {
      const int64_t u0 = cur.base + static_cast<int64_t>(cur.unit) * cur.r.tiles;
      const int64_t u1 = u0 + cur.r.tiles;
      const int c0 = static_cast<int>(((u0 + 1) * ctas - 1) / total);
      const int c1 = static_cast<int>((u1 * ctas - 1) / total);
      auto slot_of = [&](int c) { return c * 2 + (c * total / ctas >= u0 ? 0 : 1); };
      for (int u = tid; u < rows * (D / 4); u += kThreads) {
        const int row = u / (D / 4), q = u % (D / 4);
        float m = -INFINITY, l = 0.f;
        for (int c = c0; c <= c1; ++c) m = fmaxf(m, __ldcg(&p.part_ml[slot_of(c) * 16 + row]).x);
        const float ref = m == -INFINITY ? 0.f : m;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int c = c0; c <= c1; ++c) {
          const int sl = slot_of(c);
          const float2 ml = __ldcg(&p.part_ml[sl * 16 + row]);
          const float4 y = __ldcg(reinterpret_cast<const float4*>(
              p.part + (static_cast<int64_t>(sl) * 16 + row) * D + q * 4));
          const float f = ex2(ml.x - ref);
          l = fmaf(ml.y, f, l);
          x.x = fmaf(y.x, f, x.x);
          x.y = fmaf(y.y, f, x.y);
          x.z = fmaf(y.z, f, x.z);
          x.w = fmaf(y.w, f, x.w);
        }
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
        const int tok = (rb * 16 + row) / p.G, head = h * p.G + (rb * 16 + row) - tok * p.G;
        const int64_t at = static_cast<int64_t>(cur.r.q0 + tok) * p.Hq + head;
        *reinterpret_cast<uint2*>(p.o + at * D + q * 4) =
            make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
        if (p.lse != nullptr && q == 0) p.lse[at] = l == 0.f ? -INFINITY : m + log2f(l);
      }
    }
  }
}

static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    cudaDriverEntryPointQueryResult q;
    void* ptr = nullptr;
    cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000,
                                                     cudaEnableDefault, &q);
    TORCH_CHECK(e == cudaSuccess && q == cudaDriverEntryPointSuccess && ptr != nullptr,
                "cuTensorMapEncodeTiled unavailable");
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }();
  return fn;
}

// Pages as rows of D bytes: box of `rows` keys, swizzled so that fragment reads are conflict-free.
static CUtensorMap page_map(const at::Tensor& t, int rows) {
  CUtensorMap m;
  const cuuint64_t D = t.size(3);
  cuuint64_t dims[2] = {D, static_cast<cuuint64_t>(t.size(0) * t.size(1) * t.size(2))};
  cuuint64_t strides[1] = {D};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(D), static_cast<cuuint32_t>(rows)};
  cuuint32_t estr[2] = {1u, 1u};
  CUresult r = encode_fn()(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, t.data_ptr(), dims, strides, box,
                           estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "paged_attention: tensor map encode failed (", num((int)r), ")");
  return m;
}

// Scratch of one stream: parts of shared units and their counters (zero between calls). Kept
// per (device, stream), so that calls on different streams never share it; while a graph is
// captured a private one is made, which the graph keeps and zeroes at every replay.
struct Scratch {
  at::Tensor part, counters;
};

static Scratch scratch_for(const at::Device& dev, cudaStream_t stream, int64_t part, int64_t counters) {
  static std::mutex mutex;
  static std::map<std::pair<int, cudaStream_t>, Scratch>* kept = new std::map<std::pair<int, cudaStream_t>, Scratch>();
  const auto f32 = at::TensorOptions().dtype(at::kFloat).device(dev);
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  C10_CUDA_CHECK(cudaStreamIsCapturing(stream, &capture));
  if (capture != cudaStreamCaptureStatusNone)
    return {at::empty({part}, f32), at::zeros({counters}, f32.dtype(at::kInt))};
  std::lock_guard<std::mutex> lock(mutex);
  Scratch& s = (*kept)[{dev.index(), stream}];
  if (!s.part.defined() || s.part.numel() < part) s.part = at::empty({part}, f32);
  if (!s.counters.defined() || s.counters.numel() < counters)
    s.counters = at::zeros({std::max<int64_t>(2 * counters, 4096)}, f32.dtype(at::kInt));
  return s;
}

template <int D, bool INT8>
static void launch_decode(const CUtensorMap& mk, const CUtensorMap& mv, const Params& p, int grid,
                          cudaStream_t stream) {
  static std::once_flag once[64];
  int dev = 0;
  C10_CUDA_CHECK(cudaGetDevice(&dev));
  std::call_once(once[dev & 63], [] {
    C10_CUDA_CHECK(cudaFuncSetAttribute(decode_kernel<D, INT8>,
                                        cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kSmem));
  });
  decode_kernel<D, INT8><<<grid, kThreads, Cfg<D>::kSmem, stream>>>(mk, mv, p);
  NMB_LAUNCHED(1);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace paged
}  // namespace nmb

using namespace nmb;
using namespace nmb::paged;

at::Tensor paged_attention(at::Tensor q, at::Tensor k_pages, at::Tensor v_pages,
                           at::Tensor k_scale, at::Tensor v_scale, at::Tensor tables,
                           at::Tensor q_starts, at::Tensor kv_lens, int64_t max_new,
                           double softmax_scale, c10::optional<at::Tensor> lse,
                           at::Tensor status) {
  check_paged_cache(k_pages, v_pages, k_scale, v_scale);
  const at::Device dev = k_pages.device();
  const int64_t Hkv = k_pages.size(1), ps = k_pages.size(2), D = k_pages.size(3);
  TORCH_CHECK(q.device() == dev && q.scalar_type() == at::kBFloat16 && q.dim() == 3 &&
                  q.size(2) == D && q.stride(2) == 1,
              "q must be bf16 [tokens, heads, ", num(D), "] on the same device with contiguous rows");
  const int64_t T = q.size(0), Hq = q.size(1), B = kv_lens.numel();
  TORCH_CHECK(Hkv > 0 && Hq > 0 && Hq % Hkv == 0, "query heads (", num(Hq),
              ") must be a multiple of kv heads (", num(Hkv), ")");
  TORCH_CHECK(kv_lens.device() == dev && kv_lens.scalar_type() == at::kInt && kv_lens.dim() == 1 &&
                  kv_lens.is_contiguous(),
              "kv_lens must be a contiguous int32 tensor on the same device");
  TORCH_CHECK(q_starts.device() == dev && q_starts.scalar_type() == at::kInt && q_starts.dim() == 1 &&
                  q_starts.is_contiguous() && q_starts.numel() == B + 1,
              "q_starts must be a contiguous int32 tensor of ", num(B + 1), " values on the same device");
  TORCH_CHECK(tables.device() == dev && tables.scalar_type() == at::kInt && tables.dim() == 2 &&
                  tables.stride(1) == 1 && tables.size(0) >= B,
              "tables must be int32 [>= ", num(B), " requests, pages] on the same device with contiguous rows");
  TORCH_CHECK(max_new >= 0, "max_new must be >= 0");
  TORCH_CHECK(tables.size(1) * ps < (1ll << 31) && T * Hq < (1ll << 31), "too many tokens");
  TORCH_CHECK(k_pages.size(0) * Hkv * ps < (1ll << 31), "the cache has 2^31 rows or more");
  const at::cuda::CUDAGuard guard(dev);
  // 16-byte loads of query rows; others are laid out anew
  if (reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 || q.stride(0) % 8 || q.stride(1) % 8)
    q = q.clone(at::MemoryFormat::Contiguous);
  at::Tensor o = at::empty({T, Hq, D}, q.options());
  if (lse.has_value())
    TORCH_CHECK(lse->device() == dev && lse->scalar_type() == at::kFloat && lse->is_contiguous() &&
                    lse->numel() == T * Hq,
                "lse must be contiguous fp32 [", num(T), ", ", num(Hq), "] on the same device");
  if (T == 0) return o;
  if (B == 0 || k_pages.size(0) == 0) {
    o.zero_();
    if (lse.has_value()) lse->fill_(-INFINITY);
    return o;
  }
  ensure_current_context(dev.index());
  const int box = static_cast<int>(std::min<int64_t>(ps, kTile));
  const CUtensorMap mk = page_map(k_pages, box), mv = page_map(v_pages, box);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  Params p{};
  p.q = reinterpret_cast<const __nv_bfloat16*>(q.data_ptr());
  p.q_row = q.stride(0);
  p.q_head = q.stride(1);
  p.o = reinterpret_cast<__nv_bfloat16*>(o.data_ptr());
  p.lse = lse.has_value() ? lse->data_ptr<float>() : nullptr;
  p.k_scale = k_scale.data_ptr<float>();
  p.v_scale = v_scale.data_ptr<float>();
  p.tables = tables.data_ptr<int>();
  p.table_stride = tables.stride(0);
  p.q_starts = q_starts.data_ptr<int>();
  p.kv_lens = kv_lens.data_ptr<int>();
  p.width = static_cast<int>(tables.size(1));
  p.num_pages = static_cast<int>(k_pages.size(0));
  p.ps = static_cast<int>(ps);
  p.page_shift = __builtin_ctz(p.ps);
  p.B = static_cast<int>(B);
  p.T = static_cast<int>(T);
  p.Hq = static_cast<int>(Hq);
  p.Hkv = static_cast<int>(Hkv);
  p.G = static_cast<int>(Hq / Hkv);
  p.max_rows = 1 << 30;
  p.scale_log2 = static_cast<float>(softmax_scale * 1.4426950408889634);
  p.status = status.data_ptr<int>();
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const int grid = sms * (D == 64 ? Cfg<64>::kCtasPerSm : Cfg<128>::kCtasPerSm);
  const int64_t part = static_cast<int64_t>(grid) * 2 * 16 * D, ml = static_cast<int64_t>(grid) * 2 * 16 * 2;
  Scratch scratch = scratch_for(dev, stream, part + ml, Hkv * T * ((p.G + 15) / 16));
  p.part = scratch.part.data_ptr<float>();
  p.part_ml = reinterpret_cast<float2*>(p.part + part);
  p.counters = scratch.counters.data_ptr<int>();
  const bool i8 = k_pages.scalar_type() == at::kChar;
  if (D == 64) i8 ? launch_decode<64, true>(mk, mv, p, grid, stream) : launch_decode<64, false>(mk, mv, p, grid, stream);
  else i8 ? launch_decode<128, true>(mk, mv, p, grid, stream) : launch_decode<128, false>(mk, mv, p, grid, stream);
  return o;
}

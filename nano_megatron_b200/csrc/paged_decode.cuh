// Attention of a batched step over the 8-bit paged K/V cache.
//
//   o[row] = sum_j p_j vs_j c_j / sum_j p_j,   p_j = 2^(s_j - max),   s_j = log2e * scale * q.k_j
//
// with value codes c_j and value scales vs_j = 2^e_j (one per page and kv head). Because the
// scales are powers of two, vs_j joins the logit: t_j = s_j + e_j, M = running max of t, and
//   numerator += 2^(t_j - M) c_j,      denominator += 2^(t_j - M) 2^-e_j.
// The f16 probabilities stay at most 2^15 whatever the scales of different pages (see kShift), and
// rows that they cannot resolve are computed again in fp32 (kResolved). Codes of both formats are
// exact in f16; queries are scaled row by row by a power of two that brings their largest magnitude
// to [2^14, 2^15), so that elements down to 2^-31 of it are exact and smaller ones are off by at most
// 2^-39 of it. Sums are fp32.
//
// Decode kernel (few query rows per request: decoding, short continuations). Bound by reading
// the codes of K and V once: 128 requests of 512 to 4096 tokens, 8 kv heads of 128, take 121 us, 5.7 TB/s
// or 87 % of the measured copy rate.
//  * A unit is (request, kv head, block of 8 or 16 query rows = tokens x heads of the group). Its
//    keys are cut into tiles of 32; the tiles of all units, in order, are dealt evenly to the
//    CTAs, whatever the lengths (every CTA scans the B lengths for itself). A unit that is shared
//    by several CTAs is put together by the one that finishes last, in CTA order, so the result
//    does not depend on the schedule.
//  * One warp of a CTA loads: its lanes look up page ids and scales of 32 tiles at a time, one
//    tile each, a batch ahead, and fill a ring by TMA (pages are contiguous [page_size, D]
//    rectangles). Four warps compute, each every fourth tile with a softmax state of its own and
//    no barrier with the others until a unit ends.
//  * The products are transposed, S^T = K Q^T and O^T = V^T P^T, with mma.m16n8k16 (f16): keys and
//    values fill the 16-row side and 8 query rows the other, half the accumulators and softmax
//    work of the untransposed form where a group has 8 heads or fewer. (A 128-row tcgen05 tile
//    would be 94% padding, and the kernel waits for memory anyway.) The order of keys in a
//    tile and of the value columns is permuted so that every shared-memory read is 16 bytes
//    (8 for values at D = 64) without bank conflicts and decoded codes are fragments in place;
//    movmatrix turns P^T into the second product's operand.
#pragma once

#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "paged_attention.cuh"

namespace nmb {
namespace paged {

// Scratch of one stream: parts of shared units and their counters (zero between calls).
struct Scratch {
  at::Tensor part, counters;
};
Scratch scratch_for(const at::Device& dev, cudaStream_t stream, int64_t part, int64_t counters);

constexpr int kTile = 32;           // keys of a tile
// Computing warps of a CTA; one more loads. (Twelve in one CTA an SM, for few units, gave 21.0 for
// 21.3 us at one request of 32k tokens and lost up to a quarter at 18 requests: 33.7 for 25 us at
// 2048 tokens. One CTA's unit ends are not hidden by others then.)
constexpr int kWarps = 4;
constexpr int kThreads = (kWarps + 1) * 32;
constexpr int kMinTiles = kWarps;   // tiles of a CTA's share at least (8: 11.4 for 10.0 us at 1 x 512)

// NT: 8-row tiles of query rows in a unit. The ring's length is a multiple of kWarps: tile j of a
// CTA goes through stage j % kStages to warp j % kWarps, so one warp sees all phases of a stage's
// barrier in order (loads land out of order, and a parity cannot tell a phase from the one
// before the last).
template <int D, int NT>
struct Cfg {
  static constexpr int kCtasPerSm = NT == 2 ? 2 : D == 128 ? 3 : 4;
  static constexpr int kStages = NT == 1 ? 8 : D == 128 ? 12 : 16;
  static_assert(kStages % kWarps == 0, "a stage belongs to one warp");
  static constexpr int kStageBytes = 2 * kTile * D;
  static constexpr int kRing = kStages * kStageBytes;
  static constexpr int kMerge = kWarps * 8 * 64 * 4;        // 8 rows by 64 columns at a time
  static constexpr int kStats = (kWarps + 1) * 8 * NT * 8;
  static constexpr int kSmem = kRing + kMerge + kStats + kStages * 16 + kStages * 16 + 16;
};

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Transposes an 8x8 matrix of f16: lane (g, t) gives [g][2t, 2t+1] and gets [2t, 2t+1][g].
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// One request as this kernel sees it.
struct Request {
  // rows q0, q0 + 1, .. are positions ctx, ctx + 1, ..; the table holds the first kv positions
  int q0, nq, ctx, kv, blocks, tiles;   // blocks of 8 * NT rows; tiles of one unit
  __device__ int64_t total(int Hkv) const { return static_cast<int64_t>(blocks) * Hkv * tiles; }
};

template <int NT>
__device__ __forceinline__ Request load_request(const Params& p, int b) {
  Request r;
  r.q0 = min(max(__ldg(p.q_starts + b), 0), p.T);
  r.nq = min(max(__ldg(p.q_starts + b + 1) - r.q0, 0), p.T - r.q0);
  const int len = max(__ldg(p.kv_lens + b), 0);
  r.ctx = len - r.nq;
  r.kv = min(len, p.width << p.page_shift);
  const int rows = r.nq <= p.max_rows / p.G ? r.nq * p.G : 0;
  r.blocks = (rows + 8 * NT - 1) / (8 * NT);
  r.tiles = max(1, (r.kv + kTile - 1) / kTile);
  return r;
}

// A run of tiles of one unit: position in the CTA's share [g, end).
template <int NT>
struct Cursor {
  int g, end, base;       // base: global index of the request's first tile
  int b;
  Request r;
  int unit, tile, n;      // unit in the request, first tile, tiles in this run

  __device__ void set() {
    unit = (g - base) / r.tiles;
    tile = (g - base) - unit * r.tiles;
    n = min(r.tiles - tile, end - g);
  }
  __device__ bool done() const { return g >= end; }
  __device__ void next(const Params& p) {
    g += n;
    if (g >= end) return;
    while (g >= base + static_cast<int>(r.total(p.Hkv))) {  // one with tiles left follows
      if (b + 1 >= p.B) {                   // (unless the lengths changed under the kernel)
        g = end;
        return;
      }
      base += static_cast<int>(r.total(p.Hkv));
      r = load_request<NT>(p, ++b);
    }
    set();
  }
};

template <int D>
__device__ __forceinline__ int key_of(int n) {  // row inside an 8-key group of fragment index n
  return D == 128 ? ((n >> 1) | ((n & 1) << 2)) : (n ^ ((n >> 1) & 1));
}

template <int D>
__device__ __forceinline__ int chunk_at(int row, int c) {  // byte offset of 16-byte chunk c
  return D == 128 ? row * 128 + ((c ^ (row & 7)) << 4) : row * 64 + ((c ^ ((row >> 1) & 3)) << 4);
}

// Float4 slot of column group u (4 of 64 columns) of a row in the merge area, spread over the
// banks: lanes with other rows or other blocks of columns write at the same time.
template <int D>
__device__ __forceinline__ int merge_at(int row, int u) {
  const int t = (row >> 1) & 3;
  return row * 16 + (u ^ (D == 128 ? t : (t & 1) | ((t >> 1) << 2)));
}

// exact_row in a function of its own: inlined, it took registers and instruction cache from the
// kernels that hardly ever need it (19 requests of 35 tokens, 8 heads of 128: 16.2 us, 14.4 with the call).
template <int D, bool INT8>
__device__ __noinline__ void exact_row_aside(const Params& p, int b, int q0, int ctx, int kv, int h, int row,
                                             bool look) {
  const int tok = row / p.G, head = h * p.G + row - tok * p.G;
  const int64_t at = static_cast<int64_t>(q0 + tok) * p.Hq + head;
  exact_row<D, INT8>(p, b, h, p.q + (q0 + tok) * p.q_row + head * p.q_head, min(kv, ctx + tok + 1), look,
                     p.o + at * D, p.lse == nullptr ? nullptr : p.lse + at);
}

// SEVERAL: requests may have several new tokens, so that a key can be hidden from some rows only
// (should one have several without it, its rows take the slow way of exact_row).
template <int D, bool INT8, int NT, bool SEVERAL>
__global__ void __launch_bounds__(kThreads, Cfg<D, NT>::kCtasPerSm)
    decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ Params p) {
  using C = Cfg<D, NT>;
  constexpr int S = C::kStages;
  constexpr int kSteps = D / 16;
  constexpr int kRows = 8 * NT;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* ring = smem;
  float4* s_merge = reinterpret_cast<float4*>(smem + C::kRing);
  float2* s_stat = reinterpret_cast<float2*>(smem + C::kRing + C::kMerge);   // [warp][row] (M, l)
  float2* s_tot = s_stat + kWarps * kRows;                                   // [row]
  float4* s_info = reinterpret_cast<float4*>(s_tot + kRows);                 // [S] scales
  uint64_t* full = reinterpret_cast<uint64_t*>(s_info + S);
  uint64_t* empty = full + S;
  volatile int* s_flag = reinterpret_cast<volatile int*>(empty + S);         // abort, last

  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid / 32, 0);
  if (smem_u32(smem) & 1023u) {     // the swizzle pattern needs 1024-byte alignment
    if (tid == 0) record_status(p.status, kStatusSmemAlignment);
    return;
  }

  // Rows before the first request's and past the last one's (padding) are zero; written at the end.
  const bool padded = __ldg(p.q_starts) > 0 || __ldg(p.q_starts + p.B) < p.T;
  auto zero_rows = [&](int from, int to) {
    constexpr int threads = kWarps * 32;
    const int64_t n = static_cast<int64_t>(to - from) * p.Hq * (D / 8);
    uint4* o4 = reinterpret_cast<uint4*>(p.o) + static_cast<int64_t>(from) * p.Hq * (D / 8);
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * threads + tid; i < n;
         i += static_cast<int64_t>(gridDim.x) * threads) {
      o4[i] = make_uint4(0, 0, 0, 0);
      if (p.lse != nullptr && i % (D / 8) == 0)
        p.lse[static_cast<int64_t>(from) * p.Hq + i / (D / 8)] = -INFINITY;
    }
  };
  auto zero_padding = [&] {
    if (!padded || tid >= kWarps * 32) return;
    const int first = min(max(__ldg(p.q_starts), 0), p.T);
    zero_rows(0, first);
    zero_rows(min(max(__ldg(p.q_starts + p.B), first), p.T), p.T);
  };

  // ---- this CTA's share of the tiles
  // Groups of `per` CTAs have `span` tiles each, the i-th of a group from i * share + min(i, extra)
  // on: equal to one tile. One group is all there is, but for a single request, whose units have
  // equal lengths: a group a unit then, so that no CTA merges two
  // (decode 1 x 32k: 22.7 -> 20.3 us).
  Cursor<NT> cur;
  int span, per_group, share, extra;
  auto start_of = [&](int c) {
    const int group = c / per_group, i = c - group * per_group;
    return group * span + i * share + min(i, extra);
  };
  {
    int64_t* s_scan = reinterpret_cast<int64_t*>(s_merge);  // free until the first merge
    int* s_found = reinterpret_cast<int*>(s_scan + 16);
    const int per = (p.B + kThreads - 1) / kThreads;
    const int b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
    int64_t sum = 0;
    Request r{0, 0, 0, 0, 0, 1};
    for (int b = b0; b < b1; ++b) {
      r = load_request<NT>(p, b);
      sum += r.total(p.Hkv);
    }
    int64_t x = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) s_scan[warp] = x;
    if (tid < S) {
      mbar_init(&full[tid], 1);
      mbar_init(&empty[tid], 1);
      fence_mbar_init();
    }
    if (tid == 0) s_flag[0] = 0;
    __syncthreads();
    int64_t before = x - sum, all = 0;
#pragma unroll
    for (int i = 0; i <= kWarps; ++i) {
      if (i < warp) before += s_scan[i];
      all += s_scan[i];
    }
    // Tiles are counted once per block of rows: groups over 128 heads, whose prompts come here too,
    // reach this with long ones (160 heads of a group, 4 groups, a prompt of 32k tokens).
    if (all > 0x3fffffff) {
      if (tid == 0) record_status(p.status, kStatusAttnTiles);
      return;
    }
    const int total = static_cast<int>(all);
    int ctas = min(static_cast<int>(gridDim.x), (total + kMinTiles - 1) / kMinTiles);
    span = total;
    per_group = ctas;
    if (p.B == 1 && total > 0) {
      const Request only = load_request<NT>(p, 0);
      const int units = only.blocks * p.Hkv;
      if (units <= ctas) {
        span = only.tiles;
        per_group = ctas / units;  // (at most 64, for fewer parts to join: no faster)
        ctas = per_group * units;
      }
    }
    const int cta = blockIdx.x;
    if (cta >= ctas) {
      zero_padding();
      return;
    }
    share = span / per_group;
    extra = span - share * per_group;
    cur.g = start_of(cta);
    cur.end = cur.g + share + (cta % per_group < extra ? 1 : 0);
    if (before <= cur.g && cur.g < before + sum) {
      int b = b0, base = static_cast<int>(before);
      if (per > 1) r = load_request<NT>(p, b);
      while (b + 1 < b1 && cur.g >= base + static_cast<int>(r.total(p.Hkv))) {
        base += static_cast<int>(r.total(p.Hkv));
        r = load_request<NT>(p, ++b);
      }
      s_found[0] = b;
      s_found[1] = base;
      s_found[2] = r.q0;
      s_found[3] = r.nq;
      s_found[4] = r.ctx;
      s_found[5] = r.kv;
      s_found[6] = r.blocks;
      s_found[7] = r.tiles;
    }
    __syncthreads();
    cur.b = s_found[0];
    cur.base = s_found[1];
    cur.r = Request{s_found[2], s_found[3], s_found[4], s_found[5], s_found[6], s_found[7]};
    cur.set();
    __syncthreads();  // the merge area is free again
  }

  // Bounded wait of a whole warp with one answer. The vote also brings the lanes together again:
  // they leave the polling loop one by one, and the matrix instructions need all of them at once.
  auto wait_warp = [&](uint64_t* bar, uint32_t parity) -> bool {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, p.status, kStatusAttnTimeout, s_flag));
  };

  if (warp == kWarps) {
    // ---------------------------------------------------------------- loading warp
    const bool two = p.ps < kTile;
    const int box = two ? p.ps : kTile;
    // one tile per lane: pages and, once those are here, scales
    struct Tile {
      int page0, page1, h, off;   // off: first key inside its page
    };
    int at = 0;                   // tiles of the run that were handed out
    auto batch = [&](int& count) {
      while (!cur.done() && at >= cur.n) {
        cur.next(p);
        at = 0;
      }
      count = cur.done() ? 0 : min(32, cur.n - at);
      Tile t{-1, -1, 0, 0};
      if (lane < count) {
        const int key0 = (cur.tile + at + lane) * kTile;
        const int* row = p.tables + cur.b * p.table_stride;
        if (key0 < cur.r.kv) t.page0 = __ldg(row + (key0 >> p.page_shift));
        if (two && key0 + 16 < cur.r.kv) t.page1 = __ldg(row + ((key0 + 16) >> p.page_shift));
        t.h = cur.unit / cur.r.blocks;
        t.off = key0 & (p.ps - 1);
      }
      at += count;
      return t;
    };
    int count, j = 0;
    Tile t = batch(count);
    bool ok = true;
    while (count > 0 && ok) {
      int next_count;
      const Tile next = batch(next_count);
      const bool ok0 = t.page0 >= 0 && t.page0 < p.num_pages;
      const bool ok1 = two ? t.page1 >= 0 && t.page1 < p.num_pages : ok0;
      const int64_t u0 = static_cast<int64_t>(t.page0) * p.Hkv + t.h;
      const int64_t u1 = two ? static_cast<int64_t>(t.page1) * p.Hkv + t.h : u0;
      // a value scale of 0 marks a page that does not exist
      float4 info;
      info.x = ok0 ? __ldg(p.k_scale + u0) : 0.f;
      info.y = ok1 ? __ldg(p.k_scale + u1) : 0.f;
      info.z = ok0 ? __ldg(p.v_scale + u0) : 0.f;
      info.w = ok1 ? __ldg(p.v_scale + u1) : 0.f;
      for (int i = 0; i < count; ++i, ++j) {
        const int stage = j % S;
        ok = wait_warp(&empty[stage], ((j / S) & 1) ^ 1);
        if (!ok) break;
        if (lane == i) {
          // The copies first: they need no scales. (Bytes may land before they are announced; the
          // phase cannot end before the arrival.)
          uint8_t* dst = ring + stage * C::kStageBytes;
          const uint32_t bytes = (ok0 ? 2u * box * D : 0u) + (two && ok1 ? 2u * box * D : 0u);
          if (ok0) {
            const int y = static_cast<int>(u0 << p.page_shift) + t.off;
            tma_load_2d(dst, &tmK, &full[stage], 0, y);
            tma_load_2d(dst + kTile * D, &tmV, &full[stage], 0, y);
          }
          if (two && ok1) {
            const int y = static_cast<int>(u1 << p.page_shift);
            tma_load_2d(dst + 16 * D, &tmK, &full[stage], 0, y);
            tma_load_2d(dst + kTile * D + 16 * D, &tmV, &full[stage], 0, y);
          }
          s_info[stage] = info;
          if (bytes) mbar_arrive_expect_tx(&full[stage], bytes);
          else mbar_arrive(&full[stage]);
        }
        __syncwarp();
      }
      t = next;
      count = next_count;
    }
    if (!ok)  // given up: wait (bounded) for what is still on its way
      for (int i = max(0, j - S); i < j; ++i)
        mbar_wait(&full[i % S], (i / S) & 1, p.status, kStatusAttnTimeout, nullptr);
    return;
  }

  // ------------------------------------------------------------------ computing warps
  const int g8 = lane >> 2, t4 = lane & 3;
  auto sync_all = [] {
    __syncwarp();
    asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory");
  };
  int j0 = 0;                       // tiles of this CTA before the run
  bool ok = true;
  bool first_run = true;
  for (; !cur.done(); j0 += cur.n, cur.next(p), first_run = false) {
    const int h = cur.unit / cur.r.blocks, rb = cur.unit - h * cur.r.blocks;
    const int rows = min(kRows, cur.r.nq * p.G - rb * kRows);
    // query fragments: row g8 of each 8, 16 consecutive values per 64 of D
    uint32_t qb[NT][kSteps][2];
    float row_scale[NT][2];         // of the rows 2 t4, 2 t4 + 1 whose scores this lane holds
    int limit[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = rb * kRows + nt * 8 + g8;
      const int tok = r / p.G, head = r - tok * p.G;
      const bool live = nt * 8 + g8 < rows;
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
      // the row's largest magnitude goes to [2^14, 2^15) (fmaxf drops NaN; infinity stays)
      const int e = min(max(kv::exponent_of(amax) - 14, -100), 113);
      const float down = kv::pow2i(-e), up = kv::pow2i(e) * p.scale_log2;
      const int see = live ? min(cur.r.ctx + tok + 1, cur.r.kv) : 0;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        row_scale[nt][i] = __shfl_sync(0xffffffffu, up, 8 * t4 + 4 * i);
        limit[nt][i] = __shfl_sync(0xffffffffu, see, 8 * t4 + 4 * i);
      }
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        const uint32_t w[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
        for (int e2 = 0; e2 < 4; ++e2)  // word e2 of half c: k-step 4 * (c / 2) + 2 * (c % 2) + e2 / 2
          qb[nt][(c >> 1) * 4 + (c & 1) * 2 + (e2 >> 1)][e2 & 1] =
              f16x2(bf16_lo(w[e2]) * down, bf16_hi(w[e2]) * down);
      }
    }
    float acc[NT][kSteps][4];       // O^T: columns 2j (c0, c1) and 2j + 1 (c2, c3) of this lane's 16
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < kSteps; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[nt][j][e] = 0.f;
    float m_run[NT][2], l_run[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        m_run[nt][i] = -INFINITY;
        l_run[nt][i] = 0.f;
      }
    const int free_keys = min(cur.r.ctx + rb * kRows / p.G + 1, cur.r.kv);  // keys that every row sees

#pragma unroll 1
    for (int i = (warp - j0) & (kWarps - 1); i < cur.n; i += kWarps) {
      const int stage = (j0 + i) % S;
      if (ok) ok = wait_warp(&full[stage], ((j0 + i) / S) & 1);
      if (!ok) break;
      const uint8_t* sk = ring + stage * C::kStageBytes;
      const uint8_t* sv = sk + kTile * D;
      const float4 f = s_info[stage];
      const int key0 = (cur.tile + i) * kTile;
      const bool masked = key0 + kTile > free_keys || f.z == 0.f || f.w == 0.f;

      // S^T: 16 keys (rows g8, g8 + 8) by 8 query rows
      float s[2][NT][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[mt][nt][0] = s[mt][nt][1] = s[mt][nt][2] = s[mt][nt][3] = 0.f;
        const int row = mt * 16 + key_of<D>(g8);
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          const uint4 x = *reinterpret_cast<const uint4*>(sk + chunk_at<D>(row, c * 4 + t4));
          const uint4 y = *reinterpret_cast<const uint4*>(sk + chunk_at<D>(row + 8, c * 4 + t4));
          const uint32_t w0[4] = {x.x, x.y, x.z, x.w}, w1[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t a[4];
            kv::decode4<INT8>(w0[e], a[0], a[2]);
            kv::decode4<INT8>(w1[e], a[1], a[3]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma_f16(s[mt][nt], a, qb[nt][c * 4 + e][0], qb[nt][c * 4 + e][1]);
          }
        }
      }
      // logits in base 2 plus log2 of the value scale; the first 16 keys may be another page
      const float vb[2] = {static_cast<float>(kv::exponent_of(f.z)),
                           static_cast<float>(kv::exponent_of(f.w))};
      float mx[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float f0 = f.x * row_scale[nt][c], f1 = f.y * row_scale[nt][c];
          s[0][nt][c] = fmaf(s[0][nt][c], f0, vb[0]);
          s[0][nt][c + 2] = fmaf(s[0][nt][c + 2], f0, vb[0]);
          s[1][nt][c] = fmaf(s[1][nt][c], f1, vb[1]);
          s[1][nt][c + 2] = fmaf(s[1][nt][c + 2], f1, vb[1]);
          if (masked) {
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
              const bool page = (mt == 0 ? f.z : f.w) != 0.f;
              const int key = key0 + mt * 16 + key_of<D>(g8);
              if (!page || key >= limit[nt][c]) s[mt][nt][c] = -INFINITY;
              if (!page || key + 8 >= limit[nt][c]) s[mt][nt][c + 2] = -INFINITY;
            }
          }
          float m = fmaxf(fmaxf(s[0][nt][c], s[0][nt][c + 2]), fmaxf(s[1][nt][c], s[1][nt][c + 2]));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
          mx[nt][c] = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
        }
      bool grow = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        grow = grow || mx[nt][0] > m_run[nt][0] + kLazy || mx[nt][1] > m_run[nt][1] + kLazy;
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float corr[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float m = fmaxf(m_run[nt][c], mx[nt][c]);
            corr[c] = m_run[nt][c] == -INFINITY ? (m == -INFINITY ? 1.f : 0.f) : ex2(m_run[nt][c] - m);
            l_run[nt][c] *= corr[c];
            m_run[nt][c] = m;
          }
#pragma unroll
          for (int j = 0; j < kSteps; ++j) {
            acc[nt][j][0] *= corr[0];
            acc[nt][j][1] *= corr[1];
            acc[nt][j][2] *= corr[0];
            acc[nt][j][3] *= corr[1];
          }
        }
      }
      // a missing page only adds zeros; its 2^-(-127) = 2^127 stays finite
      const float iv[2] = {kv::pow2i(-kv::exponent_of(f.z)), kv::pow2i(-kv::exponent_of(f.w))};
      uint32_t pb[2][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float r0 = m_run[nt][0] == -INFINITY ? 0.f : m_run[nt][0] - kShift;
        const float r1 = m_run[nt][1] == -INFINITY ? 0.f : m_run[nt][1] - kShift;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const float p0 = ex2(s[mt][nt][0] - r0), p1 = ex2(s[mt][nt][1] - r1);
          const float p2 = ex2(s[mt][nt][2] - r0), p3 = ex2(s[mt][nt][3] - r1);
          l_run[nt][0] = fmaf(p0 + p2, iv[mt], l_run[nt][0]);
          l_run[nt][1] = fmaf(p1 + p3, iv[mt], l_run[nt][1]);
          pb[mt][nt][0] = transpose8x8(f16x2(p0, p1));
          pb[mt][nt][1] = transpose8x8(f16x2(p2, p3));
        }
      }

      // NaN among the values of keys that some rows see and others do not: 0 * NaN would reach
      // the others. The rows that see one get NaN here, and the code becomes 0 in this stage.
      if (SEVERAL && !INT8 && masked && cur.r.nq > 1) {
        constexpr int kWords = D / 32;            // this lane's columns: D / 8 codes of each key
        uint32_t* mine = reinterpret_cast<uint32_t*>(const_cast<uint8_t*>(sv));
        auto word_at = [&](int r) {
          return (chunk_at<D>(r, D == 128 ? (g8 >> 1) | ((g8 & 1) << 2) : g8 >> 1) +
                  (D == 128 ? 0 : (g8 & 1) * 8)) / 4;
        };
        uint32_t any = 0;
#pragma unroll 1
        for (int r = 0; r < kTile; ++r)
#pragma unroll
          for (int w = 0; w < kWords; ++w) {
            const uint32_t bad = kv::nan_bytes(mine[word_at(r) + w]);
            any |= bad;
            if (bad == 0) continue;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int c = 0; c < 2; ++c)
                if (key0 + r < limit[nt][c] && (r < 16 ? f.z : f.w) != 0.f)
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    if ((bad >> (8 * e)) & 0x80u)
                      acc[nt][2 * w + e / 2][(e & 1) * 2 + c] = __int_as_float(0x7fffffff);
          }
        if (__any_sync(0xffffffffu, any != 0)) {
#pragma unroll 1
          for (int r = 0; r < kTile && t4 == 0; ++r)
            for (int w = 0; w < kWords; ++w) {
              uint32_t& x = mine[word_at(r) + w];
              x &= ~((kv::nan_bytes(x) >> 7) * 255u);
            }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the stage is TMA's next
          __syncwarp();
        }
      }

      // O^T += V^T P^T
      const bool tail = key0 + kTile > cur.r.kv || f.z == 0.f || f.w == 0.f;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        uint32_t v[4][D / 32];  // keys 2t, 2t+1 of the first 8-key group, then of the second
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = mt * 16 + (e >> 1) * 8 + key_of<D>(2 * t4 + (e & 1));
          if constexpr (D == 128) {
            const uint4 x = *reinterpret_cast<const uint4*>(
                sv + chunk_at<D>(row, (g8 >> 1) | ((g8 & 1) << 2)));
            v[e][0] = x.x; v[e][1] = x.y; v[e][2] = x.z; v[e][3] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(sv + chunk_at<D>(row, g8 >> 1) + (g8 & 1) * 8);
            v[e][0] = x.x; v[e][1] = x.y;
          }
          // codes behind the last key or of a missing page are stale: 0 * NaN is NaN
          if (tail && (key0 + row >= cur.r.kv || (mt == 0 ? f.z : f.w) == 0.f)) {
#pragma unroll
            for (int w = 0; w < D / 32; ++w) v[e][w] = 0;
          }
        }
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {
          uint32_t a[4], b[4];      // columns 4w, 4w + 1 and 4w + 2, 4w + 3
          kv::decode4<INT8>(__byte_perm(v[0][w], v[1][w], 0x5140), a[0], a[1]);
          kv::decode4<INT8>(__byte_perm(v[2][w], v[3][w], 0x5140), a[2], a[3]);
          kv::decode4<INT8>(__byte_perm(v[0][w], v[1][w], 0x7362), b[0], b[1]);
          kv::decode4<INT8>(__byte_perm(v[2][w], v[3][w], 0x7362), b[2], b[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_f16(acc[nt][2 * w], a, pb[mt][nt][0], pb[mt][nt][1]);
            mma_f16(acc[nt][2 * w + 1], b, pb[mt][nt][0], pb[mt][nt][1]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[stage]);
    }

    // ---- the warps' states into one
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float l = l_run[nt][c];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        if (g8 == 0) s_stat[warp * kRows + nt * 8 + 2 * t4 + c] = make_float2(m_run[nt][c], l);
      }
    sync_all();
    float corr[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int row = nt * 8 + 2 * t4 + c;
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_stat[w * kRows + row].x);
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float2 st = s_stat[w * kRows + row];
          l = fmaf(st.y, ex2(st.x - ref), l);
        }
        corr[nt][c] = ex2(m_run[nt][c] - ref);
        if (warp == 0 && g8 == 0) s_tot[row] = make_float2(m, l);
      }
    const bool whole = cur.n == cur.r.tiles;
    // A row is computed again unless one of its numerators reaches this. (kv bounds the keys it sees.
    // Without the NaN path, all rows of a request of several are: a `max_new` that is too small costs
    // speed only.)
    const float enough = !SEVERAL && cur.r.nq > 1 ? INFINITY : kResolved<INT8> * cur.r.kv;
    auto again = [&](int row) {
      exact_row_aside<D, INT8>(p, cur.b, cur.r.q0, cur.r.ctx, cur.r.kv, h, rb * kRows + row,
                               SEVERAL || cur.r.nq == 1);
    };
    const int slot = blockIdx.x * 2 + (first_run ? 0 : 1);
    float* part = p.part + static_cast<int64_t>(slot) * (kRows * D);
    constexpr int kParts = D / 64;  // 64 columns at a time; at D = 128 those of even, then odd g8
    static_assert(kWarps * 32 == 8 * 16, "16 lanes a row, the same ones in every part");
    float top = 0.f;                // of this thread's columns of its row
    uint32_t redo = 0;              // bit 2 * nt + i: row 8 * nt + 2 * warp + i
#pragma unroll
    for (int np = 0; np < NT * kParts; ++np) {
      const int nt = np / kParts, part_cols = np % kParts;
      if (nt * 8 >= rows) break;
      if (np) sync_all();           // what was there has been read
      float4* mine = s_merge + warp * 8 * 16;
      const int blk = D == 128 ? (g8 >> 1) * 4 : g8 * 2;
      if (D == 64 || (g8 & 1) == part_cols) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int u = 0; u < D / 32; ++u)
            mine[merge_at<D>(2 * t4 + c, blk + u)] =
                make_float4(acc[nt][2 * u][c] * corr[nt][c], acc[nt][2 * u][c + 2] * corr[nt][c],
                            acc[nt][2 * u + 1][c] * corr[nt][c], acc[nt][2 * u + 1][c + 2] * corr[nt][c]);
      }
      sync_all();
      const int in = min(8, rows - nt * 8);
      const int r8 = tid / 16, q = part_cols * 16 + tid % 16, row = nt * 8 + r8;
      if (part_cols == 0) top = r8 < in ? 0.f : INFINITY;
      if (r8 < in) {
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 y = s_merge[w * 8 * 16 + merge_at<D>(r8, tid % 16)];
          x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
        }
        const float2 tot = s_tot[row];
        if (whole) {
          const float inv = tot.y > 0.f || tot.y != tot.y ? 1.f / tot.y : 0.f;
          const int tok = (rb * kRows + row) / p.G, head = h * p.G + (rb * kRows + row) - tok * p.G;
          const int64_t at = static_cast<int64_t>(cur.r.q0 + tok) * p.Hq + head;
          *reinterpret_cast<uint2*>(p.o + at * D + q * 4) =
              make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
          top = fmaxf(top, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
          if (p.lse != nullptr && q == 0)
            p.lse[at] = tot.y == 0.f ? -INFINITY : tot.x - kShift + log2f(tot.y);
        } else {
          *reinterpret_cast<float4*>(part + row * D + q * 4) = x;
          if (q == 0) p.part_ml[slot * kRows + row] = tot;
        }
      }
      if (part_cols == kParts - 1) {
        const uint32_t fine = __ballot_sync(0xffffffffu, top >= enough);
        redo |= ((fine & 0xffffu ? 0u : 1u) | (fine >> 16 ? 0u : 2u)) << (2 * nt);
      }
    }
    if (whole) {
#pragma unroll 1
      for (; __builtin_expect(redo != 0, 0); redo &= redo - 1) {
        const int i = __ffs(redo) - 1;
        again(i / 2 * 8 + 2 * warp + (i & 1));
      }
      continue;
    }

    // ---- a unit shared with other CTAs: the last to finish adds the parts up in CTA order
    sync_all();
    const int rpt = (p.G + kRows - 1) / kRows;
    if (tid == 0) {
      int* counter = p.counters + (static_cast<int64_t>(h) * p.T + cur.r.q0) * rpt + rb;
      __threadfence();              // the barrier and this fence publish the whole CTA's part
      const int before = atomicAdd(counter, cur.n);
      const bool last = before + cur.n == cur.r.tiles;
      if (last) *counter = 0;
      __threadfence();
      s_flag[1] = last;
    }
    sync_all();
    if (s_flag[1]) {
      const int u0 = cur.base + cur.unit * cur.r.tiles, u1 = u0 + cur.r.tiles;
      auto owner = [&](int tile) {
        const int group = tile / span, longer = extra * (share + 1), t = tile - group * span;
        return group * per_group + (t < longer ? t / (share + 1) : extra + (t - longer) / share);
      };
      const int c0 = owner(u0), n = owner(u1 - 1) - c0 + 1;
      // only the first of them can have had another unit before this one
      const int first = c0 * 2 + (start_of(c0) >= u0 ? 0 : 1);
      auto slot_of = [&](int i) { return i == 0 ? first : (c0 + i) * 2; };
      // A warp, or several that share the parts, per row. Lanes hold the weights of 32 parts at a
      // time and 4 columns each (D = 64: the halves of the warp take every other part).
      constexpr int kHalves = 128 / D;
      const int col = (lane & (D / 4 - 1)) * 4, odd = lane / (D / 4);
      const int at_once = min(rows, kWarps), helpers = kWarps / at_once;   // rows, warps of a row
      for (int row0 = 0; row0 < rows; row0 += at_once) {
        const int row = row0 + warp % at_once, mine = warp / at_once;
        const bool live = row < rows && mine < helpers;
        const int from = live ? n * mine / helpers : 0, to = live ? n * (mine + 1) / helpers : 0;
        float m = -INFINITY, l = 0.f;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        constexpr int kBatch = 16 / kHalves;      // parts of a lane in flight
#pragma unroll 1
        for (int i0 = from; i0 < to; i0 += 16) {
          float4 y[kBatch];
#pragma unroll
          for (int k = 0; k < kBatch; ++k) {
            const int i = min(i0 + k * kHalves + odd, to - 1);
            y[k] = __ldcg(reinterpret_cast<const float4*>(
                p.part + (static_cast<int64_t>(slot_of(i)) * kRows + row) * D + col));
          }
          float2 ml = make_float2(-INFINITY, 0.f);
          if (lane < 16 && i0 + lane < to) ml = __ldcg(&p.part_ml[slot_of(i0 + lane) * kRows + row]);
          const float top = fmaxf(m, warp_max(ml.x)), ref = top == -INFINITY ? 0.f : top;
          const float w = ex2(ml.x - ref), down = ex2(m - ref);   // 0 past the last part
          m = top;
          l = fmaf(l, down, warp_sum(ml.y * w));
          x.x *= down; x.y *= down; x.z *= down; x.w *= down;
#pragma unroll
          for (int k = 0; k < kBatch; ++k) {
            const float f = __shfl_sync(0xffffffffu, w, k * kHalves + odd);
            const bool in = i0 + k * kHalves + odd < to;
            x.x = in ? fmaf(y[k].x, f, x.x) : x.x;
            x.y = in ? fmaf(y[k].y, f, x.y) : x.y;
            x.z = in ? fmaf(y[k].z, f, x.z) : x.z;
            x.w = in ? fmaf(y[k].w, f, x.w) : x.w;
          }
        }
        if constexpr (kHalves == 2) {
          x.x += __shfl_xor_sync(0xffffffffu, x.x, 16);
          x.y += __shfl_xor_sync(0xffffffffu, x.y, 16);
          x.z += __shfl_xor_sync(0xffffffffu, x.z, 16);
          x.w += __shfl_xor_sync(0xffffffffu, x.w, 16);
        }
        if (helpers > 1) {          // the row's first warp adds the others' sums, in order
          float* s_sum = reinterpret_cast<float*>(s_merge);
          if (odd == 0) *reinterpret_cast<float4*>(s_sum + warp * D + col) = x;
          if (lane == 0) s_stat[warp] = make_float2(m, l);
          sync_all();
          if (mine == 0) {
            float top = m;
            for (int k = 1; k < helpers; ++k) top = fmaxf(top, s_stat[warp + k * at_once].x);
            const float ref = top == -INFINITY ? 0.f : top, down = ex2(m - ref);
            m = top;
            l *= down;
            x.x *= down; x.y *= down; x.z *= down; x.w *= down;
            for (int k = 1; k < helpers; ++k) {
              const float2 st = s_stat[warp + k * at_once];
              const float f = ex2(st.x - ref);
              const float4 y = *reinterpret_cast<const float4*>(s_sum + (warp + k * at_once) * D + col);
              x.x = fmaf(y.x, f, x.x); x.y = fmaf(y.y, f, x.y);
              x.z = fmaf(y.z, f, x.z); x.w = fmaf(y.w, f, x.w);
              l = fmaf(st.y, f, l);
            }
          }
          sync_all();
        }
        if (!live || mine != 0) continue;
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
        const int tok = (rb * kRows + row) / p.G, head = h * p.G + (rb * kRows + row) - tok * p.G;
        const int64_t at = static_cast<int64_t>(cur.r.q0 + tok) * p.Hq + head;
        if (odd == 0)
          *reinterpret_cast<uint2*>(p.o + at * D + col) =
              make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
        if (p.lse != nullptr && lane == 0) p.lse[at] = l == 0.f ? -INFINITY : m - kShift + log2f(l);
        const float top = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
        if (!__any_sync(0xffffffffu, top >= enough)) again(row);
      }
    }
  }
  zero_padding();
}

template <int D, bool INT8, int NT, bool SEVERAL>
static void launch_decode_as(const CUtensorMap& mk, const CUtensorMap& mv, Params& p,
                          const at::Device& dev, cudaStream_t stream) {
  using C = Cfg<D, NT>;
  static std::once_flag once[64];
  std::call_once(once[dev.index() & 63], [] {
    C10_CUDA_CHECK(cudaFuncSetAttribute(decode_kernel<D, INT8, NT, SEVERAL>,
                                        cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
  });
  const int grid = at::cuda::getCurrentDeviceProperties()->multiProcessorCount * C::kCtasPerSm;
  const int64_t slots = 2ll * grid * 8 * NT;
  const Scratch scratch = scratch_for(dev, stream, slots * (D + 2),
                                      static_cast<int64_t>(p.Hkv) * p.T * ((p.G + 8 * NT - 1) / (8 * NT)));
  p.part = scratch.part.data_ptr<float>();
  p.part_ml = reinterpret_cast<float2*>(p.part + slots * D);
  p.counters = scratch.counters.data_ptr<int>();
  decode_kernel<D, INT8, NT, SEVERAL><<<grid, kThreads, C::kSmem, stream>>>(mk, mv, p);
  NMB_LAUNCHED(1);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// 8-row units unless some request can fill more: 16-row ones then read the cache once.
template <int D>
static void launch_decode_for(const CUtensorMap& mk, const CUtensorMap& mv, Params& p, int64_t max_new,
                              bool int8, const at::Device& dev, cudaStream_t stream) {
  if (max_new * p.G > 8)
    int8 ? launch_decode_as<D, true, 2, true>(mk, mv, p, dev, stream)
         : launch_decode_as<D, false, 2, true>(mk, mv, p, dev, stream);
  else if (int8)
    launch_decode_as<D, true, 1, true>(mk, mv, p, dev, stream);
  else if (max_new > 1)
    launch_decode_as<D, false, 1, true>(mk, mv, p, dev, stream);
  else
    launch_decode_as<D, false, 1, false>(mk, mv, p, dev, stream);
}

}  // namespace paged
}  // namespace nmb

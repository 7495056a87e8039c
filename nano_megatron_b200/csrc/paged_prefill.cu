// Attention over the 8-bit paged cache for requests with many new tokens (prompts and chunks of
// them) on the tensor cores (tcgen05 + TMEM). Same mathematics as the decode kernel
// (paged_decode.cuh): log2 of the power-of-two value scale joins the logit, codes and queries
// go to f16 (which holds both), sums are fp32.
//
// Bound by the tensor cores and the exponentials: 128 keys cost a pair of 128-row tiles about
// 2,100 cycles of tcgen05.mma at the nominal rate and as many of ex2. Measured: about 5,000, the chain
// softmax (2,500) -> products (2,000) -> softmax of a tile; chunks of up to 2048 tokens over as many
// cached ones, 32 / 8 heads of 128, run at 668 TFLOP/s, 41 % of the measured GEMM rate.
//
// A block takes two tiles of 128 query rows (tokens x the heads of one group, so grouped heads
// share every converted key) of one request and kv head, 512 threads:
//   warps 0-3, 4-7 : softmax of tile 0 / 1, a thread per row: loads S (tcgen05.ld), online softmax
//                    in base 2, writes P (f16) over S in TMEM, rescales O there when the maximum
//                    grows by more than 2^6, and stores the result at the end;
//   warps 8-11     : converters: cache codes from global memory (prefetched into registers one
//                    tile ahead) to f16 tiles in shared memory, in the K-major / MN-major
//                    128-byte-swizzled layouts that tcgen05.mma reads, two stages each of K and V;
//   warps 12, 13   : issue the products of tile 0 / 1: PV of the last keys, then QK of the next, so
//                    that one tile's softmax runs under the other's products (one warp for both
//                    was the bottleneck: about 140 cycles an instruction beside the others).
// Codes are converted once per block and used by 256 rows; a direct 8-bit product would need
// queries and probabilities in 8 bits.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <mutex>

#include "paged_attention.cuh"

namespace nmb {
namespace paged {

constexpr int kPfThreads = 512;
constexpr int kPfKeys = 128;
constexpr int kPfRows = 128;
// Floor of the logits' factor: keeps 0 * -inf out of masked places when the softmax scale is 0.
constexpr float kTinyScale = 1e-30f;
// setmaxnreg shares of the four warpgroups: 2 * 176 + 104 + 56 = 4 * 128, the launch's registers
constexpr int kRegSoftmax = 176, kRegConvert = 104, kRegIssue = 56;

template <int D>
struct PfCfg {
  static constexpr int kTile = kPfKeys * D * 2;              // one f16 tile of K, V or Q
  static constexpr int kInfo = 4 * 8 * 16;                   // [4 tiles][8 groups of 16 keys]
  static constexpr int kSmem = 6 * kTile + kInfo + 256;
};

__device__ __forceinline__ void tmem_st_32x32b_x32_f(uint32_t taddr, const uint32_t* r) {
  tmem_st_32x32b_x32(taddr, *reinterpret_cast<const uint32_t(*)[32]>(r));
}

__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 "
      "[%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)),
        "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}

// Shared-memory matrix descriptors (128-byte swizzle, 8-row groups 1024 bytes apart) as two words:
// the upper one is constant, and moving the start address adds to the lower one only.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(const void* p, uint32_t leading_bytes) {
  return ((smem_u32(p) >> 4) & 0x3FFFu) | ((leading_bytes >> 4) << 16);
}
// A whole warp runs the issuing loop, so that addresses stay in uniform registers, and one lane
// issues (a loop run by one lane alone spent 100 cycles a product moving them there).
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                       uint32_t accumulate, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(kDescHi), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t tmem_a, uint32_t b, uint32_t idesc,
                                       uint32_t accumulate, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
      "r"(tmem_a), "r"(b), "r"(kDescHi), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
          smem_u32(bar)),
      "r"(leader)
      : "memory");
}

// kind::f16 with f16 A and B, fp32 D.
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, bool b_mn) {
  return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}

template <int D, bool INT8>
__global__ void __launch_bounds__(kPfThreads, 1) prefill_kernel(const Params p) {
  using C = PfCfg<D>;
  constexpr int kHalf = kPfKeys * 128;                        // 64 columns of a tile
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;                                         // [2] tiles
  uint8_t* sK = sQ + 2 * C::kTile;                            // [2] stages
  uint8_t* sV = sK + 2 * C::kTile;                            // [2] stages
  float4* s_info = reinterpret_cast<float4*>(sV + 2 * C::kTile);  // (ks, log2 vs, 1 / vs, missing)
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_info + 4 * 8);
  uint64_t* q_full = bars;        // [2]
  uint64_t* k_full = bars + 2;    // [2]
  uint64_t* k_empty = bars + 4;   // [2]
  uint64_t* v_full = bars + 6;    // [2]
  uint64_t* v_empty = bars + 8;   // [2]
  uint64_t* s_full = bars + 10;   // [2]
  uint64_t* p_full = bars + 12;   // [2]
  uint64_t* o_full = bars + 14;   // [2]
  uint64_t* turn = bars + 16;     // [2] issuer r may start PV of the next tile
  int64_t* s_find = reinterpret_cast<int64_t*>(bars + 18);    // [2] + scan in s_info
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 20);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* s_nan = abort_flag + 1;           // NaN among values that only some rows see

  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid / 32, 0);
  if (smem_u32(smem) & 1023u) {
    if (tid == 0) record_status(p.status, kStatusSmemAlignment);
    return;
  }

  // ---- this block's request, head and rows; the last (longest) rows of a request first
  const int tpt = kPfRows / p.G;                  // tokens of a row tile
  auto blocks_of = [&](int b) -> int {
    const int q0 = min(max(__ldg(p.q_starts + b), 0), p.T);
    const int n = min(max(__ldg(p.q_starts + b + 1) - q0, 0), p.T - q0);
    return n > p.max_rows / p.G ? (n + 2 * tpt - 1) / (2 * tpt) : 0;
  };
  int b, blk, h;
  {
    int* s_scan = reinterpret_cast<int*>(s_info);
    const int per = (p.B + kPfThreads - 1) / kPfThreads;
    const int b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
    int sum = 0;
    for (int i = b0; i < b1; ++i) sum += blocks_of(i);
    int x = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) s_scan[warp] = x;
    __syncthreads();
    int before = x - sum, total = 0;
#pragma unroll
    for (int i = 0; i < kPfThreads / 32; ++i) {
      if (i < warp) before += s_scan[i];
      total += s_scan[i];
    }
    const int item = blockIdx.x / p.Hkv;
    if (item >= total) return;                    // the grid is an upper bound
    h = blockIdx.x - item * p.Hkv;
    if (before <= item && item < before + sum) {
      int i = b0, base = before;
      for (;; ++i) {
        const int t = blocks_of(i);
        if (item < base + t || i + 1 >= b1) break;
        base += t;
      }
      s_find[0] = i;
      s_find[1] = blocks_of(i) - 1 - (item - base);
    }
    __syncthreads();
    b = static_cast<int>(s_find[0]);
    blk = static_cast<int>(s_find[1]);
  }
  const int q0 = min(max(__ldg(p.q_starts + b), 0), p.T);
  const int n = min(max(__ldg(p.q_starts + b + 1) - q0, 0), p.T - q0);
  const int len = max(__ldg(p.kv_lens + b), 0);
  const int ctx = len - n;                        // position of the first row
  const int kv = min(len, p.width << p.page_shift);   // positions that the table holds
  const int tok0 = blk * 2 * tpt, toks = min(2 * tpt, n - tok0);
  // keys that the last row sees; the second row tile exists only if it has tokens
  const int keys = max(0, min(kv, ctx + tok0 + toks));
  const int tiles = (keys + kPfKeys - 1) / kPfKeys;
  const int rts = toks > tpt ? 2 : 1;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 4);
      mbar_init(&k_full[i], 4);
      mbar_init(&k_empty[i], rts);
      mbar_init(&v_full[i], 4);
      mbar_init(&v_empty[i], rts);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
      mbar_init(&turn[i], 1);
    }
    *abort_flag = 0;
    *s_nan = 0;
    fence_mbar_init();
  }
  if (warp == 12) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  // columns: S/P of tile 0, 1 at 0, 128; O of tile 0, 1 at 256, 384
  auto wait_warp = [&](uint64_t* bar, uint32_t parity) -> bool {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, p.status, kStatusAttnTimeout, abort_flag));
  };

  if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegIssue));
    const int r = warp - 12;
    if (r < rts && tiles > 0) {
      // ------------------------------------------------- product issuer of row tile r
      constexpr uint32_t id_s = idesc_f16(kPfRows, kPfKeys, false);
      constexpr uint32_t id_o = idesc_f16(kPfRows, D, true);
      const uint32_t leader = elect_one() ? 1u : 0u;
      const uint32_t q_lo = desc_lo(sQ, 16) + r * (C::kTile >> 4);
      const uint32_t k_lo = desc_lo(sK, 16), v_lo = desc_lo(sV, kHalf);
      const uint32_t tS = tmem + r * 128, tO = tmem + 256 + r * 128;
      bool ok = wait_warp(&q_full[r], 0);
      for (int j = 0; j <= tiles && ok; ++j) {
        if (j > 0) {                              // O += P V_{j-1}
          const int i = j - 1;
          ok = wait_warp(&v_full[i & 1], (i >> 1) & 1) && wait_warp(&p_full[r], i & 1) &&
               (rts == 1 || wait_warp(&turn[r], r == 0 ? (i & 1) ^ 1 : i & 1));
          if (!ok) break;
          tc_fence_after();
          const uint32_t v = v_lo + (i & 1) * (C::kTile >> 4);
#pragma unroll
          for (int kk = 0; kk < kPfKeys / 16; ++kk)
            mma_ts(tO, tS + kk * 8, v + kk * (2048 >> 4), id_o, i > 0 || kk > 0 ? 1u : 0u, leader);
          mma_commit(j == tiles ? &o_full[r] : &v_empty[i & 1], leader);
        }
        if (j == tiles) {
          if (r == 0 && leader) mbar_arrive(&turn[1]);
          break;
        }
        ok = wait_warp(&k_full[j & 1], (j >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        const uint32_t k = k_lo + (j & 1) * (C::kTile >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {     // S = Q K_j^T, over P of the last keys
          const uint32_t off = ((kk >> 2) * kHalf + (kk & 3) * 32) >> 4;
          mma_ss(tS, q_lo + off, k + off, id_s, kk > 0 ? 1u : 0u, leader);
        }
        mma_commit(&s_full[r], leader);
        mma_commit(&k_empty[j & 1], leader);
        if (j > 0 && leader) mbar_arrive(&turn[1 - r]);
      }
      if (!ok) {  // given up: wait (bounded) for the products on their way before TMEM is freed
        mma_commit(&o_full[r], leader);
        mbar_wait(&o_full[r], 0, p.status, kStatusAttnTimeout, nullptr);
        __syncwarp();
      }
    }
  } else if (warp >= 8) {
    // ------------------------------------------------------------------ converters
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegConvert));
    constexpr int kChunks = D / 16;               // 16-code chunks of a key
    constexpr int kStep = 128 / kChunks;          // keys of one pass
    constexpr int kPass = kPfKeys / kStep;
    // eight lanes that store together write four chunks of two rows: all banks once
    const int t = tid - 256;
    const int c = D == 128 ? (t & 3) | ((t >> 1) & 4) : t & 3;
    const int r0 = D == 128 ? ((t >> 4) << 1) | ((t >> 2) & 1) : t >> 2;
    const int* table = p.tables + b * p.table_stride;
    uint4 raw[2][kPass];
    // Lane l < 8 of each warp holds the page of the l-th 16 keys (-1: none), two tiles ahead, and,
    // in the first warp, their scales one tile ahead.
    auto page_of = [&](int j) {
      const int key = j * kPfKeys + lane * 16;
      return lane < 8 && key < kv ? __ldg(table + (key >> p.page_shift)) : -1;
    };
    auto fetch = [&](int which, int j, int page16) {   // stale and missing keys become code 0
      const uint8_t* codes = (which ? p.v_codes : p.k_codes) + c * 16;
#pragma unroll
      for (int i = 0; i < kPass; ++i) {
        const int in_tile = i * kStep + r0, key = j * kPfKeys + in_tile;
        const int page = __shfl_sync(0xffffffffu, page16, in_tile >> 4);
        const int64_t row = ((static_cast<int64_t>(page) * p.Hkv + h) << p.page_shift) + (key & (p.ps - 1));
        raw[which][i] = key < kv && page >= 0 && page < p.num_pages
                            ? __ldg(reinterpret_cast<const uint4*>(codes + row * D))
                            : make_uint4(0, 0, 0, 0);
      }
    };
    auto convert = [&](int which, uint8_t* dst) {
#pragma unroll
      for (int i = 0; i < kPass; ++i) {
        const int row = i * kStep + r0;
        const uint4 x = raw[which][i];
        uint32_t o[8];
        kv::decode4<INT8>(x.x, o[0], o[1]);
        kv::decode4<INT8>(x.y, o[2], o[3]);
        kv::decode4<INT8>(x.z, o[4], o[5]);
        kv::decode4<INT8>(x.w, o[6], o[7]);
        uint8_t* line = dst + (c >> 2) * kHalf + row * 128;
        const int c8 = (c & 3) * 2;
        *reinterpret_cast<uint4*>(line + ((c8 ^ (row & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
        *reinterpret_cast<uint4*>(line + (((c8 + 1) ^ (row & 7)) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
      }
    };
    auto publish = [&](uint64_t* bar) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    auto scales = [&](int page, int j) {
      float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
      if (t < 8) {
        if (page >= 0 && page < p.num_pages) {
          const int64_t u = static_cast<int64_t>(page) * p.Hkv + h;
          f.x = __ldg(p.k_scale + u);
          f.y = __ldg(p.v_scale + u);
        } else if (j * kPfKeys + t * 16 < kv) {
          f.w = 1.f;
        }
      }
      return f;
    };
    float4 sc = make_float4(0.f, 0.f, 0.f, 0.f);
    int page1 = page_of(1);
    if (tiles > 0) {
      const int page0 = page_of(0);
      sc = scales(page0, 0);
      fetch(0, 0, page0);
      fetch(1, 0, page0);
    }
    for (int j = 0; j < tiles; ++j) {
      const int st = j & 1;
      const uint32_t ph = (j >> 1) & 1;
      const float4 sc1 = scales(page1, j + 1);
      const int page2 = page_of(j + 2);
      if (!wait_warp(&k_empty[st], ph ^ 1)) break;
      convert(0, sK + st * C::kTile);
      if (t < 8) {
        const int e = kv::exponent_of(sc.y);      // -127 where there is no page
        s_info[(j & 3) * 8 + t] = make_float4(sc.x, static_cast<float>(e), kv::pow2i(-e), sc.w);
      }
      sc = sc1;
      publish(&k_full[st]);
      if (j + 1 < tiles) fetch(0, j + 1, page1);
      if (!wait_warp(&v_empty[st], ph ^ 1)) break;
      if (!INT8 && (j + 1) * kPfKeys > ctx + tok0 + 1) {
        // keys that some rows see and others do not: 0 * NaN would reach the others, so NaN
        // counts as 0 in the product and is put in at the end
        uint32_t bad = 0;
#pragma unroll
        for (int i = 0; i < kPass; ++i) {
          uint32_t* x = reinterpret_cast<uint32_t*>(&raw[1][i]);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t m = kv::nan_bytes(x[w]);
            bad |= m;
            x[w] &= ~((m >> 7) * 255u);
          }
        }
        if (bad) *s_nan = 1;
      }
      convert(1, sV + st * C::kTile);
      publish(&v_full[st]);
      if (j + 1 < tiles) fetch(1, j + 1, page1);
      page1 = page2;
    }
  } else {
    // --------------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegSoftmax));
    const int rt = warp / 4, row = (warp & 3) * 32 + lane;
    const uint32_t tS = tmem + rt * 128 + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t tO = tS - rt * 128 + 256 + rt * 128;
    const int tok = tok0 + rt * tpt + row / p.G, head = row % p.G;
    const bool live = row < tpt * p.G && tok < n;
    const int limit = live ? min(ctx + tok + 1, kv) : 0;
    const int first_limit = min(ctx + tok0 + rt * tpt + 1, kv);     // of the tile's first row
    float row_scale = 0.f;
    if (rt < rts) {
      // this row's query, scaled to [2^14, 2^15) by a power of two, as f16
      const __nv_bfloat16* src = p.q + (q0 + tok) * p.q_row + (h * p.G + head) * p.q_head;
      uint4 raw[D / 8];
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        raw[i] = live ? __ldg(reinterpret_cast<const uint4*>(src) + i) : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          amax = fmaxf(amax, fmaxf(fabsf(bf16_lo(w[e])), fabsf(bf16_hi(w[e]))));
      }
      const int e = min(max(kv::exponent_of(amax) - 14, -100), 113);
      const float down = p.scale_log2 < 0.f ? -kv::pow2i(-e) : kv::pow2i(-e);
      row_scale = kv::pow2i(e) * fabsf(p.scale_log2);
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        uint32_t o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = f16x2(bf16_lo(w[k]) * down, bf16_hi(w[k]) * down);
        *reinterpret_cast<uint4*>(sQ + rt * C::kTile + (i >> 3) * kHalf + row * 128 +
                                  (((i & 7) ^ (row & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[rt]);
    }
    float m_run = -INFINITY, l_run = 0.f;
    bool ok = true;
    for (int j = 0; j < tiles && rt < rts; ++j) {
      ok = wait_warp(&s_full[rt], j & 1);
      if (!ok) break;
      tc_fence_after();
      uint32_t r[kPfKeys];
#pragma unroll
      for (int c = 0; c < kPfKeys / 32; ++c)
        tmem_ld_32x32b_x32(tS + c * 32, *reinterpret_cast<uint32_t(*)[32]>(r + c * 32));
      tmem_wait_ld();
      const float4* info = s_info + (j & 3) * 8;
      const int key0 = j * kPfKeys;
      bool gap = false;
#pragma unroll
      for (int g = 0; g < 8; ++g) gap = gap || info[g].w != 0.f;
      if (gap || key0 + kPfKeys > first_limit) {
        const int see = limit - key0;
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          const int vis = info[g].w != 0.f ? 0 : see - g * 16;
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (e >= vis) r[g * 16 + e] = 0xff800000u;        // -inf
        }
      }
      // The key scale is positive: a group's largest logit is that of its largest product.
      float m_tile = -INFINITY;
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        const uint32_t* x = r + g * 16;
        float m = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
#pragma unroll
        for (int e = 2; e < 16; e += 2)
          m = fmaxf(fmaxf(m, __uint_as_float(x[e])), __uint_as_float(x[e + 1]));
        const float4 f = info[g];
        m_tile = fmaxf(m_tile, fmaf(m, fmaxf(f.x * row_scale, kTinyScale), f.y));
      }
      // (QK of this tile was issued after PV of the last one, so O is complete here.)
      if (__any_sync(0xffffffffu, m_tile > m_run + kLazy)) {
        const float m = fmaxf(m_run, m_tile);
        const float corr = m_run == -INFINITY ? (m == -INFINITY ? 1.f : 0.f) : ex2(m_run - m);
        l_run *= corr;
        m_run = m;
        if (j > 0) {
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_ld_32x32b_x16(tO + c * 16, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
            tmem_st_32x32b_x16(tO + c * 16, o);
          }
        }
      }
      const float ref = m_run == -INFINITY ? 0.f : m_run - kShift;
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        const float4 f = info[g];
        const float a = fmaxf(f.x * row_scale, kTinyScale), b = f.y - ref;
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          float2 x = fma2(make_float2(__uint_as_float(r[g * 16 + e]), __uint_as_float(r[g * 16 + e + 1])),
                          make_float2(a, a), make_float2(b, b));
          x.x = ex2(x.x);
          x.y = ex2(x.y);
          sum = add2(sum, x);
          r[g * 8 + e / 2] = f16x2(x.x, x.y);
        }
        // a missing page only adds zeros; its 2^-(-127) = 2^127 stays finite
        l_run = fmaf(sum.x + sum.y, f.z, l_run);
      }
#pragma unroll
      for (int c = 0; c < kPfKeys / 64; ++c) tmem_st_32x32b_x32_f(tS + c * 32, r + c * 32);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[rt]);
    }
    if (rt < rts) {
      if (tiles > 0) ok = ok && wait_warp(&o_full[rt], 0);
      tc_fence_after();
      const float inv = l_run > 0.f || l_run != l_run ? 1.f / l_run : 0.f;
      const int64_t at = static_cast<int64_t>(q0 + tok) * p.Hq + h * p.G + head;
      __nv_bfloat16* dst = p.o + at * D;
      uint32_t nan_cols[D / 32] = {};
      if (!INT8 && tiles > 0 && *s_nan) {         // which columns of the keys this row sees
        const int* table = p.tables + b * p.table_stride;
        for (int key = max(0, ctx + tok0 + 1) / kPfKeys * kPfKeys; key < limit; ++key) {
          const int page = __ldg(table + (key >> p.page_shift));
          if (page < 0 || page >= p.num_pages) continue;
          const uint8_t* x = p.v_codes + (((static_cast<int64_t>(page) * p.Hkv + h) << p.page_shift) +
                                          (key & (p.ps - 1))) * D;
#pragma unroll
          for (int c = 0; c < D / 32; ++c)
            for (int e = 0; e < 32; ++e)
              nan_cols[c] |= static_cast<uint32_t>((x[c * 32 + e] & 0x7F) == 0x7F) << e;
        }
      }
      if (ok) {
        float top = 0.f;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          if (tiles > 0) {
            tmem_ld_32x32b_x32(tO + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) top = fmaxf(top, fabsf(__uint_as_float(o[e])));
          }
          if (!INT8 && nan_cols[c] != 0)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if ((nan_cols[c] >> e) & 1u) o[e] = 0x7fffffffu;
          if (live) {
            // a row that saw nothing has 0 in O or, without any tile, nothing there
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                w[e] = tiles > 0 ? pack_bf16x2(__uint_as_float(o[q * 8 + 2 * e]) * inv,
                                               __uint_as_float(o[q * 8 + 2 * e + 1]) * inv)
                                 : 0u;
              reinterpret_cast<uint4*>(dst + c * 32)[q] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
        if (live && p.lse != nullptr)
          p.lse[at] = l_run == 0.f ? -INFINITY : m_run - kShift + log2f(l_run);
        // the last row first: if it sees no value but zeros, neither do the others
        uint32_t again = __ballot_sync(0xffffffffu, l_run > 0.f && l_run < INFINITY &&
                                                        top < kResolved<INT8> * limit);
#pragma unroll 1
        while (again) {
          const int i = 31 - __clz(again);
          again ^= 1u << i;
          const int64_t row_at = __shfl_sync(0xffffffffu, at, i);
          const int64_t row_q = __shfl_sync(0xffffffffu, (q0 + tok) * p.q_row + (h * p.G + head) * p.q_head, i);
          if (!exact_row<D, INT8>(p, b, h, p.q + row_q, __shfl_sync(0xffffffffu, limit, i), true,
                                  p.o + row_at * D, p.lse == nullptr ? nullptr : p.lse + row_at))
            break;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int D, bool INT8>
static void launch(const Params& p, const at::Device& dev, cudaStream_t stream) {
  static std::once_flag once[64];
  std::call_once(once[dev.index() & 63], [] {
    C10_CUDA_CHECK(cudaFuncSetAttribute(prefill_kernel<D, INT8>,
                                        cudaFuncAttributeMaxDynamicSharedMemorySize, PfCfg<D>::kSmem));
  });
  const int64_t per = 2 * (kPfRows / p.G);
  // every request has at most its tokens / per, rounded up, blocks
  const int64_t blocks = (p.T / per + std::min<int64_t>(p.B, p.T / (p.max_rows / p.G + 1))) * p.Hkv;
  if (blocks == 0) return;
  prefill_kernel<D, INT8><<<static_cast<unsigned>(blocks), kPfThreads, PfCfg<D>::kSmem, stream>>>(p);
  NMB_LAUNCHED(1);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

void launch_prefill(const Params& p, int64_t D, bool int8, const at::Device& dev, cudaStream_t stream) {
  if (D == 64) int8 ? launch<64, true>(p, dev, stream) : launch<64, false>(p, dev, stream);
  else int8 ? launch<128, true>(p, dev, stream) : launch<128, false>(p, dev, stream);
}

}  // namespace paged
}  // namespace nmb

// Entry point of attention over the 8-bit paged cache: checks, tensor maps, scratch, and which
// kernel serves which request (paged_decode.cuh, paged_prefill.cu).
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cudaTypedefs.h>

#include <map>
#include <mutex>

#include "paged_decode.cuh"

// serving.cu: shapes, types and devices of a K/V cache.
void check_paged_cache(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_scale,
                       const at::Tensor& v_scale);

namespace nmb {
namespace paged {

// paged_decode_64.cu, paged_decode_128.cu, paged_prefill.cu
void launch_decode_64(const CUtensorMap& mk, const CUtensorMap& mv, Params& p, int64_t max_new,
                      bool int8, const at::Device& dev, cudaStream_t stream);
void launch_decode_128(const CUtensorMap& mk, const CUtensorMap& mv, Params& p, int64_t max_new,
                       bool int8, const at::Device& dev, cudaStream_t stream);
void launch_prefill(const Params& p, int64_t D, bool int8, const at::Device& dev, cudaStream_t stream);

// Requests with more query rows (new tokens x heads of a group) than this go to the prefill
// kernel, the others to the decode kernel, which rereads the keys every 16 rows but splits them
// over the GPU. At 68 rows, 8 kv heads of 128: 32 requests of 256 / 4096 cached tokens take 79 / 308 us
// in the decode kernel and 37 / 199 in the other, 2 requests 33 / 42 and 21 / 91 us; at 256 rows
// the decode kernel only wins for the 2 long ones (73 for 102 us).
constexpr int kDecodeRows = 64;

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

// Kept per (device, stream), so that calls on different streams never share it; while a graph is
// captured a private one is made, which the graph keeps and zeroes at every replay.
Scratch scratch_for(const at::Device& dev, cudaStream_t stream, int64_t part, int64_t counters) {
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
  p.k_codes = static_cast<const uint8_t*>(k_pages.data_ptr());
  p.v_codes = static_cast<const uint8_t*>(v_pages.data_ptr());
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
  // all requests are decode's unless some may have more rows (a wrong `max_new` costs speed only)
  const bool prefill = p.G <= 128 && max_new * p.G > kDecodeRows;
  p.max_rows = prefill ? std::max<int>(kDecodeRows, p.G) : 1 << 30;
  p.scale_log2 = static_cast<float>(softmax_scale * 1.4426950408889634);
  p.status = status.data_ptr<int>();
  const bool i8 = k_pages.scalar_type() == at::kChar;
  if (prefill) launch_prefill(p, D, i8, dev, stream);
  // (prefill's requests have more rows than the decode kernel ever sees)
  const int64_t few = std::min<int64_t>(max_new, p.max_rows / p.G);
  D == 64 ? launch_decode_64(mk, mv, p, few, i8, dev, stream)
          : launch_decode_128(mk, mv, p, few, i8, dev, stream);
  return o;
}

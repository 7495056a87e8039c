// The decode kernels over the 8-bit paged cache for heads of 128 (a file for each size: they are
// compiled side by side).
#include "paged_decode.cuh"

namespace nmb {
namespace paged {

void launch_decode_128(const CUtensorMap& mk, const CUtensorMap& mv, Params& p, int64_t max_new,
                      bool int8, const at::Device& dev, cudaStream_t stream) {
  launch_decode_for<128>(mk, mv, p, max_new, int8, dev, stream);
}

}  // namespace paged
}  // namespace nmb

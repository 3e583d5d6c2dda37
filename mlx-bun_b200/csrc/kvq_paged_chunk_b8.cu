// kvq_paged_chunk_b8.cu — the chunk kernels for 8-bit pages, bf16.
#include "kvq_paged_chunk.cuh"

namespace kvq {
namespace paged {

template <>
int32_t launch_chunk<8, true>(const AttnArgs& a, const Work& ws, int ctas, int dev, cudaStream_t st) {
  return launch_chunk_impl<8, true>(a, ws, ctas, dev, st);
}

}  // namespace paged
}  // namespace kvq

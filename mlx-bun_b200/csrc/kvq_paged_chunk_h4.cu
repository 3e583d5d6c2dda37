// kvq_paged_chunk_h4.cu — the chunk kernels for 4-bit pages, fp16.
#include "kvq_paged_chunk.cuh"

namespace kvq {
namespace paged {

template <>
int32_t launch_chunk<4, false>(const AttnArgs& a, const Work& ws, int ctas, int dev, cudaStream_t st) {
  return launch_chunk_impl<4, false>(a, ws, ctas, dev, st);
}

}  // namespace paged
}  // namespace kvq

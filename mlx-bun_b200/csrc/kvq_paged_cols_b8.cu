// kvq_paged_cols_b8.cu — the column kernels for 8-bit pages, bf16.
#include "kvq_paged_cols.cuh"

namespace kvq {
namespace paged {

template <>
int32_t launch_cols<8, true>(const AttnArgs& a, const Work& ws, int NC, int ctas, int dev,
                          cudaStream_t st) {
  return launch_cols_impl<8, true>(a, ws, NC, ctas, dev, st);
}

}  // namespace paged
}  // namespace kvq

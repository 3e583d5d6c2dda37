// kvq_paged_cols_h4.cu — the column kernels for 4-bit pages, fp16.
#include "kvq_paged_cols.cuh"

namespace kvq {
namespace paged {

template <>
int32_t launch_cols<4, false>(const AttnArgs& a, const Work& ws, int NC, int ctas, int dev,
                          cudaStream_t st) {
  return launch_cols_impl<4, false>(a, ws, NC, ctas, dev, st);
}

}  // namespace paged
}  // namespace kvq

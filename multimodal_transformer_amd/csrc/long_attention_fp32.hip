// Attention over long rows: the fp32 kernels.
#include "long_attention_kernels.cuh"

namespace la {
template void forward<float>(Args &, DocRange *, hipStream_t);
template void backward<float>(Args &, DocRange *, f32x4 *, float *, float *, hipStream_t);
}  // namespace la

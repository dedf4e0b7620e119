// Attention over long rows: the bf16 kernels.
#include "long_attention_kernels.cuh"

namespace la {
template void forward<__bf16>(Args &, DocRange *, hipStream_t);
template void backward<__bf16>(Args &, DocRange *, f32x4 *, float *, float *, hipStream_t);
}  // namespace la

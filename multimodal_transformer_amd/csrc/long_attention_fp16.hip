// Attention over long rows: the fp16 kernels.
#include "long_attention_kernels.cuh"

namespace la {
template void forward<_Float16>(Args &, DocRange *, hipStream_t);
template void backward<_Float16>(Args &, DocRange *, f32x4 *, float *, float *, hipStream_t);
}  // namespace la

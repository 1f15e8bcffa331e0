#define CONVROT_NORM_KERNELS
#include "layer_norm.cuh"

namespace convrot {
namespace norm {
template int forward<__nv_bfloat16>(const NormParams&, cudaStream_t);
template int backward<__nv_bfloat16>(const NormParams&, cudaStream_t);
}  // namespace norm
}  // namespace convrot

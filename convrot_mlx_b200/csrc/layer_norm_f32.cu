#define CONVROT_NORM_KERNELS
#include "layer_norm.cuh"

namespace convrot {
namespace norm {
template int forward<float>(const NormParams&, cudaStream_t);
template int backward<float>(const NormParams&, cudaStream_t);
}  // namespace norm
}  // namespace convrot

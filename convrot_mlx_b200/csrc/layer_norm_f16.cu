#define CONVROT_NORM_KERNELS
#include "layer_norm.cuh"

namespace convrot {
namespace norm {
template int forward<__half>(const NormParams&, cudaStream_t);
template int backward<__half>(const NormParams&, cudaStream_t);
}  // namespace norm
}  // namespace convrot

// Pyramid group norm passes for __nv_bfloat16 features.
#include "msda_norm_kernels.cuh"
namespace msda {
template cudaError_t norm_launch<__nv_bfloat16>(const NormArgs&, int, bool, int, bool, bool,
                            cudaStream_t);
}  // namespace msda

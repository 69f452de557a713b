// Pyramid group norm passes for __half features.
#include "msda_norm_kernels.cuh"
namespace msda {
template cudaError_t norm_launch<__half>(const NormArgs&, int, bool, int, bool, bool,
                            cudaStream_t);
}  // namespace msda

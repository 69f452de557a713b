// Pyramid group norm passes for float features.
#include "msda_norm_kernels.cuh"
namespace msda {
template cudaError_t norm_launch<float>(const NormArgs&, int, bool, int, bool, bool,
                            cudaStream_t);
}  // namespace msda

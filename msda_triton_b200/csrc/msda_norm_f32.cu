// Pyramid group norm passes for float features.
#include "msda_norm_kernels.cuh"
namespace msda {
template cudaError_t norm_wave_t<float>(const NormArgs&, const NormWave&, int, int, bool, cudaStream_t);
}  // namespace msda

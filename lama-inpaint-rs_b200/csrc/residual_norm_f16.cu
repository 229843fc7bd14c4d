#include "residual_norm_kernels.cuh"

template cudaError_t lama::ops::run_forward<__half>(const Fwd&, cudaStream_t);
template cudaError_t lama::ops::run_backward<__half>(const Bwd&, cudaStream_t);

#include "residual_norm_kernels.cuh"

template cudaError_t lama::ops::run_forward<float>(const Fwd&, cudaStream_t);
template cudaError_t lama::ops::run_backward<float>(const Bwd&, cudaStream_t);

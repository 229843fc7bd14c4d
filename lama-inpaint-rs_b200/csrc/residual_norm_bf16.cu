#include "residual_norm_kernels.cuh"

template cudaError_t lama::ops::run_forward<__nv_bfloat16>(const Fwd&, cudaStream_t);
template cudaError_t lama::ops::run_backward<__nv_bfloat16>(const Bwd&, cudaStream_t);

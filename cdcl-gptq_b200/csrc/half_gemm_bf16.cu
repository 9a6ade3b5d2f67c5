// half_gemm_bf16.cu - the bf16 variants of the half-precision product.
#include "half_gemm_launch.cuh"

template int cdclq::hg::launch_form<true>(cdclq::HalfForm, int, int, const cdclq::hg::Maps&, const cdclq::hg::Params&, cudaStream_t);

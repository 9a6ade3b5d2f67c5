// half_gemm_f16.cu - the f16 variants of the half-precision product.
#include "half_gemm_launch.cuh"

template int cdclq::hg::launch_form<false>(cdclq::HalfForm, int, int, const cdclq::hg::Maps&, const cdclq::hg::Params&, cudaStream_t);

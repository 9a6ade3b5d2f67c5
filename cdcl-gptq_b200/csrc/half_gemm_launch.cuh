// half_gemm_launch.cuh - launches the variants of the half-precision product of one type; included by one .cu per type.
#pragma once

#include "half_gemm.cuh"
#include "half_gemm.h"

namespace cdclq {
namespace hg {

struct Maps {
    CUtensorMap a, b, u, x;
};

template <bool BF16, bool AMN, bool BMN, int BN, int ROWS, int EPI>
static int launch_one(const Maps& maps, const Params& p, cudaStream_t st) {
    auto kern = half_gemm_kernel<BF16, AMN, BMN, BN, ROWS, EPI>;
    static std::atomic<uint64_t> done{0};
    if (int rc = allow_smem(kern, smem_bytes(), done, "half_gemm_kernel shared memory")) return rc;
    const int64_t items = (int64_t)p.ntiles * p.splits;
    const int sms = sm_count();
    CDCLQ_LAUNCH(kern, (unsigned)(items < sms ? items : sms), THREADS, smem_bytes(), st, maps.a, maps.b, maps.u, maps.x, p);
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : cuda_error(e, "half_gemm_kernel launch");
}

template <bool BF16, bool AMN, bool BMN, int ROWS, int EPI>
static int launch_wide(int bn, const Maps& maps, const Params& p, cudaStream_t st) {
    if constexpr (ROWS == ROWS_GROUPED) {
        return launch_one<BF16, AMN, BMN, 64, ROWS, EPI>(maps, p, st);
    } else {
        if (bn == 256) return launch_one<BF16, AMN, BMN, 256, ROWS, EPI>(maps, p, st);
        if (bn == 128) return launch_one<BF16, AMN, BMN, 128, ROWS, EPI>(maps, p, st);
        if constexpr (EPI == EPI_STORE) return launch_one<BF16, AMN, BMN, 64, ROWS, EPI>(maps, p, st);
        return set_error(CDCLQ_ERR_ARG, "half product: no such tile");
    }
}

template <bool BF16>
int launch_form(HalfForm form, int bn, const Maps& maps, const Params& p, cudaStream_t st) {
    switch (form) {
        case HALF_STATS: return launch_wide<BF16, false, false, ROWS_PLAIN, EPI_STATS>(bn, maps, p, st);
        case HALF_GRAD: return launch_wide<BF16, false, false, ROWS_PLAIN, EPI_GRAD>(bn, maps, p, st);
        case HALF_NN: return launch_wide<BF16, false, true, ROWS_PLAIN, EPI_STORE>(bn, maps, p, st);
        case HALF_TN: return launch_wide<BF16, true, true, ROWS_PLAIN, EPI_STORE>(bn, maps, p, st);
        case HALF_NT_EXTEND: return launch_wide<BF16, false, false, ROWS_EXTEND, EPI_STORE>(bn, maps, p, st);
        case HALF_NN_EXTEND: return launch_wide<BF16, false, true, ROWS_EXTEND, EPI_STORE>(bn, maps, p, st);
        case HALF_NT_GROUPED: return launch_wide<BF16, false, false, ROWS_GROUPED, EPI_STORE>(bn, maps, p, st);
        case HALF_NN_GROUPED: return launch_wide<BF16, false, true, ROWS_GROUPED, EPI_STORE>(bn, maps, p, st);
    }
    return set_error(CDCLQ_ERR_ARG, "half product: no such form");
}

extern template int launch_form<true>(HalfForm, int, const Maps&, const Params&, cudaStream_t);
extern template int launch_form<false>(HalfForm, int, const Maps&, const Params&, cudaStream_t);

}  // namespace hg
}  // namespace cdclq

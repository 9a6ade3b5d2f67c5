// half_gemm_launch.cuh - launches the variants of the half-precision product of one type; included by one .cu per type.
#pragma once

#include "half_gemm.cuh"
#include "half_gemm.h"

namespace cdclq {
namespace hg {

struct Maps {
    CUtensorMap a, b, u, x;
};

template <bool BF16, bool AMN, bool BMN, int CG, int BN, int ROWS, int EPI>
static int launch_one(const Maps& maps, const Params& p, cudaStream_t st) {
    auto kern = half_gemm_kernel<BF16, AMN, BMN, CG, BN, ROWS, EPI>;
    static std::atomic<uint64_t> done{0};
    if (int rc = allow_smem(kern, smem_bytes(), done, "half_gemm_kernel shared memory")) return rc;
    const int64_t items = (int64_t)p.ntiles * p.splits;
    const int most = sm_count() / CG;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(CG * (items < most ? items : most)));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem_bytes();
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = CG;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = CG == 2 ? 1 : 0;
    g_launches.fetch_add(1, std::memory_order_relaxed);
    cudaError_t e = cudaLaunchKernelEx(&cfg, kern, maps.a, maps.b, maps.u, maps.x, p);
    return e == cudaSuccess ? 0 : cuda_error(e, "half_gemm_kernel launch");
}

template <bool BF16, bool AMN, bool BMN, int ROWS, int EPI>
static int launch_tile(int cg, int bn, const Maps& maps, const Params& p, cudaStream_t st) {
    if constexpr (EPI != EPI_STATS) {
        if (bn == 512) return launch_one<BF16, AMN, BMN, 2, 512, ROWS, EPI>(maps, p, st);
    }
    if (cg == 2 && bn == 256) return launch_one<BF16, AMN, BMN, 2, 256, ROWS, EPI>(maps, p, st);
    if (cg == 2) return launch_one<BF16, AMN, BMN, 2, 128, ROWS, EPI>(maps, p, st);
    if (bn == 128) return launch_one<BF16, AMN, BMN, 1, 128, ROWS, EPI>(maps, p, st);
    if constexpr (EPI == EPI_STORE) return launch_one<BF16, AMN, BMN, 1, 64, ROWS, EPI>(maps, p, st);
    return set_error(CDCLQ_ERR_ARG, "half product: no such tile");
}

template <bool BF16>
int launch_form(HalfForm form, int cg, int bn, const Maps& maps, const Params& p, cudaStream_t st) {
    switch (form) {
        case HALF_STATS: return launch_tile<BF16, false, false, ROWS_PLAIN, EPI_STATS>(cg, bn, maps, p, st);
        case HALF_GRAD: return launch_tile<BF16, false, false, ROWS_PLAIN, EPI_GRAD>(cg, bn, maps, p, st);
        case HALF_NN: return launch_tile<BF16, false, true, ROWS_PLAIN, EPI_STORE>(cg, bn, maps, p, st);
        case HALF_TN: return launch_tile<BF16, true, true, ROWS_PLAIN, EPI_STORE>(cg, bn, maps, p, st);
        case HALF_NT_EXTEND: return launch_tile<BF16, false, false, ROWS_EXTEND, EPI_STORE>(cg, bn, maps, p, st);
        case HALF_NN_EXTEND: return launch_tile<BF16, false, true, ROWS_EXTEND, EPI_STORE>(cg, bn, maps, p, st);
    }
    return set_error(CDCLQ_ERR_ARG, "half product: no such form");
}

extern template int launch_form<true>(HalfForm, int, int, const Maps&, const Params&, cudaStream_t);
extern template int launch_form<false>(HalfForm, int, int, const Maps&, const Params&, cudaStream_t);

}  // namespace hg
}  // namespace cdclq

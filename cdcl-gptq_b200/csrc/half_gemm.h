// half_gemm.h - host side of the half-precision tensor-core product (half_gemm.cuh) and what its callers share.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstddef>
#include <cstdint>

#include "cdclq.h"
#include "common.cuh"

namespace cdclq {

// The forms of the product the operators use.
enum HalfForm {
    HALF_STATS,       // K-major x K-major, running softmax statistics of the rows
    HALF_GRAD,        // K-major x K-major, softmax gradient
    HALF_NN,          // K-major x MN-major, stored
    HALF_TN,          // MN-major x MN-major, stored
    HALF_NT_EXTEND,   // K-major x K-major plus the rows' adapters, stored
    HALF_NN_EXTEND    // K-major x MN-major plus the rows' adapters, stored
};

// A 16-bit operand: `rows` x `cols` (cols contiguous), `ld` elements from row to row, `batch` of them `step` elements apart.
// Base, ld and step are whole multiples of 16 bytes.
struct HalfOperand {
    const void* p = nullptr;
    int64_t rows = 0, cols = 0, ld = 0, batch = 1, step = 0;
};

// What u lacks of the rows' factors in f16 (see RankArgs::past): past null: nothing.
struct FarRows {
    const int* past = nullptr;   // [m]
    const int* index = nullptr;  // [m]
    const float* u = nullptr;    // [m][rank]
    const uint16_t* x = nullptr; // as the operand x
    int64_t ld = 0, step = 0;
};

// The product's rows, columns and depth: a tile more is still an int.
constexpr size_t MOST_SIZE = 0x7fffff00;

struct HalfGemm {
    HalfForm form;
    bool bf16;
    int64_t m, n, k;
    HalfOperand a, b;
    HalfOperand u, x;            // extension: u (m x rank) times x[adapter]
    const uint32_t* lists = nullptr;  // the adapters of each tile's rows (RowLists), or null: no extension
    FarRows far;
    void* out = nullptr;         // 16-bit, ldo elements from row to row
    int64_t ldo = 0;
    float* f32out = nullptr;     // f32, ldf elements from row to row
    const float* f32in = nullptr;
    int64_t ldf = 0;
    const float* alpha = nullptr;
    const int64_t* target = nullptr;
    int64_t col0 = 0, vocab = 0;
    float2* stats = nullptr;
    float* label_logit = nullptr;
    const float *lse = nullptr, *dloss = nullptr, *gain = nullptr;
    float* partial = nullptr;    // workspace of the split plan
};

// Tile (cg CTAs of 128 rows, bn columns) and K splits of a product; partial_bytes of workspace when splits > 1.
struct HalfPlan {
    int cg, bn, splits;
    size_t partial_bytes;
};
HalfPlan plan_half_gemm(HalfForm form, int64_t m, int64_t n, int64_t k);

// (maximum, sum) pairs that the statistics form leaves for each row.
int64_t half_stats_parts(const HalfPlan& plan, int64_t n);

// The list of a tile's rows (R = 128 or 256), in words: the number of their adapters, padding to 4, R places for the adapters' ids,
// R places for R / 32 words each that have a bit for every row that is not the adapter's.
constexpr int ROW_LIST_IDS = 4;
__host__ __device__ constexpr int row_list_masks(int R) { return ROW_LIST_IDS + R; }
__host__ __device__ constexpr int row_list_words(int R) { return row_list_masks(R) + R * (R / 32); }

// The adapters of the rows of each of the plan's tiles, for the extended forms; words of them for m rows.
struct RowLists {
    const int* index = nullptr;  // [m], none if outside [0, adapters)
    int m = 0, adapters = 0;
    int rows = 0, tiles = 0;     // rows of a tile, tiles
    uint32_t* out = nullptr;
};
RowLists row_lists(const HalfPlan& plan, const int* index, int64_t m, int64_t adapters, void* out);
size_t row_lists_bytes(const HalfPlan& plan, int64_t m);

// Launches the product (and, when the plan splits K, the pass that adds the splits in order).
int launch_half_gemm(const HalfGemm& g, const HalfPlan& plan, cudaStream_t st);

// Launches a kernel.  overlap: it may start while the kernel before it in the stream still runs, once that one has let it
// (griddepcontrol.launch_dependents); what it needs of that one's results it waits for itself (griddepcontrol.wait).
template <typename... Params, typename... Args>
int launch_after(bool overlap, void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, const char* what, const Args&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = overlap ? 1 : 0;
    g_launches.fetch_add(1, std::memory_order_relaxed);
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    return e == cudaSuccess ? 0 : cuda_error(e, what);
}

// Lets a kernel use `bytes` of dynamic shared memory, once for each device; `done` is the kernel's own record.
template <typename Kernel>
int allow_smem(Kernel kernel, size_t bytes, std::atomic<uint64_t>& done, const char* what) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return cuda_error(e, what);
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (done.load(std::memory_order_relaxed) & bit) return 0;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != cudaSuccess) return cuda_error(e, what);
    done.fetch_or(bit, std::memory_order_relaxed);
    return 0;
}

// Number of SMs of the current device.
int sm_count();
// The current device's host word that a kernel sets when one of its bounded waits ran out; null on failure.
int* device_fail_word();
// CDCLQ_OK, or the error left by an earlier launch on the current device whose wait ran out (reported once).
int check_fail_word(const char* what);

}  // namespace cdclq

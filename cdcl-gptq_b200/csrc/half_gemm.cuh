// half_gemm.cuh - the half-precision tensor-core product behind the adapter, checkpoint and loss operators.
//
//   D[m][n] = sum_k A[m][k] B[n][k]        A, B both bf16 or both f16, D accumulated in f32 in tensor memory
//
// One persistent kernel, specialised at compile time on
//   AMN, BMN   whether an operand is contiguous along its rows' index (MN-major) or along k (K-major)
//   BN         tile columns (128 rows x BN columns): 256 where that fills the SMs, else 128 or 64
//   ROWS       what the adapters of the rows do (see RowMode)
//   EPI        what becomes of a finished tile (see Epilogue)
// TMA brings 64-deep K blocks into a ring of 128-byte-swizzled stages, one thread issues the MMAs, and eight warps
// work on the finished accumulator while the next tile's MMAs fill the other one.
#pragma once

#include "common.cuh"
#include "tcgen05.cuh"

namespace cdclq {
namespace hg {

using namespace tc;

constexpr int BM = 128;            // tile rows = tensor-memory lanes
constexpr int KB = 64;             // K block: 128 bytes of a 16-bit type
constexpr int EPI_WARPS = 8;       // two per lane quadrant, each with half of the tile's columns
constexpr int THREADS = (EPI_WARPS + 2) * 32;
constexpr int A_BYTES = BM * KB * 2;
constexpr int STAGE_WORDS = 32 * 33;  // one epilogue warp's transposition buffer, in floats
constexpr int RING_BYTES = 192 * 1024;
constexpr int BAND = 16;           // row blocks per band of the tile order: a wave's operands stay in L2

__host__ __device__ constexpr int b_bytes(int bn) { return bn * KB * 2; }
__host__ __device__ constexpr int stages(int bn) { return RING_BYTES / (A_BYTES + b_bytes(bn)); }
__host__ __device__ constexpr size_t smem_bytes() { return RING_BYTES + EPI_WARPS * STAGE_WORDS * 4 + 1024 /* alignment */ + 256 /* barriers */; }

// How the adapter of each row (index[m]; none if outside [0, adapters)) takes part.
enum RowMode {
    ROWS_PLAIN = 0,   // not at all
    ROWS_EXTEND = 1,  // D[m] += U[m] Bx[index[m]]: further K blocks, whose MMAs write the adapter's own rows only
    ROWS_GROUPED = 2  // D[m] = A[m] B[index[m]]: one pass over K for each adapter of the tile, for its own rows only
};
enum Epilogue {
    EPI_STORE = 0,  // a 16-bit matrix, and / or f32 partial sums
    EPI_STATS = 1,  // running maximum and sum of exp of each row, and the label's logit
    EPI_GRAD = 2    // (softmax - onehot) * dloss as a 16-bit matrix
};

struct Params {
    int m, n, nkb;             // rows, columns, K blocks
    int tiles_m, tiles_n, ntiles;
    int splits, kb_per_split;  // the K blocks of a tile, over several items
    // rows' adapters
    const int* index;
    int adapters;
    int rank;                  // ROWS_EXTEND: depth of the extension
    // EPI_STORE
    void* out;                 // 16-bit, or null
    int64_t ldo;
    int out_vec;               // rows of `out` start on 16 bytes
    float* f32out;             // f32 sums, or null; split s writes at s * split_stride
    const float* f32in;        // added to the sums first, or null
    int64_t ldf, split_stride;
    const float* alpha;        // multiplies the sums on their way to `out`, or null
    // EPI_STATS, EPI_GRAD
    const int64_t* target;     // label of each row, relative to the whole vocabulary
    int64_t col0;              // the first column's place in the vocabulary
    int64_t vocab;
    float2* stats;             // [2 * tiles_n][m]: maximum, sum of exp(v - maximum)
    float* label_logit;        // [m]
    const float* lse;          // [m]
    const float* dloss;        // [m]
    const float* gain;         // power of two on the gradient, or null
    int* fail;                 // host word, set when a wait ran out
};

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (BF16) {
        __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&v);
    } else {
        __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&v);
    }
}
template <bool BF16>
__device__ __forceinline__ uint16_t pack1(float a) {
    if constexpr (BF16)
        return __bfloat16_as_ushort(__float2bfloat16_rn(a));
    else
        return __half_as_ushort(__float2half_rn(a));
}

// Item -> (row block, column block, split): splits outermost; bands of BAND row blocks, column block by column block.
__device__ __forceinline__ void item_coords(const Params& P, int item, int& mb, int& nb, int& split) {
    split = item / P.ntiles;
    int t = item - split * P.ntiles;
    const int full = BAND * P.tiles_n;
    const int band = t / full;
    t -= band * full;
    const int rows = min(BAND, P.tiles_m - band * BAND);
    nb = t / rows;
    mb = band * BAND + t - nb * rows;
}

// The adapters of a tile's 128 rows, lowest first; a warp holds four rows in each lane.
struct RowAdapters {
    static constexpr int NONE = 0x7fffffff;
    int id[4];
    __device__ __forceinline__ void load(const Params& P, int m0, int lane) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int row = m0 + 32 * q + lane;
            const int v = (row < P.m && P.adapters > 0) ? P.index[row] : -1;
            id[q] = (v >= 0 && v < P.adapters) ? v : NONE;
        }
    }
    // the next adapter and the lanes that are not its rows; NONE after the last
    __device__ __forceinline__ int next(uint32_t (&off)[4]) {
        const int cur = __reduce_min_sync(0xffffffffu, min(min(id[0], id[1]), min(id[2], id[3])));
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const bool mine = id[q] == cur;
            off[q] = ~__ballot_sync(0xffffffffu, mine);
            if (mine) id[q] = NONE;
        }
        return cur;
    }
};

template <bool BF16, bool AMN, bool BMN, int BN, int ROWS, int EPI>
__global__ void __launch_bounds__(THREADS, 1)
half_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                 const __grid_constant__ CUtensorMap map_u, const __grid_constant__ CUtensorMap map_x, const Params P) {
    constexpr int NS = stages(BN);
    constexpr int B_BYTES = b_bytes(BN);
    constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
    constexpr uint32_t TMEM_COLS = 2 * BN;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    float* turn = reinterpret_cast<float*>(base + RING_BYTES);
    uint64_t* full = reinterpret_cast<uint64_t*>(turn + EPI_WARPS * STAGE_WORDS);
    uint64_t* empty = full + NS;
    uint64_t* accf = empty + NS;
    uint64_t* acce = accf + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acce + 2);
    int* flag = reinterpret_cast<int*>(tmem_slot + 1);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int s = 0; s < NS; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(&accf[b], 1);
            mbar_init(&acce[b], EPI_WARPS * 32);
        }
        *flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == EPI_WARPS + 1) tmem_alloc(tmem_slot, TMEM_COLS);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int items = P.ntiles * P.splits;
    const uint32_t ring = smem_u32(base);

    if (warp == EPI_WARPS) {
        // ---------------- TMA producer: the whole warp walks the items, lane 0 waits and issues
        int ctr = 0;
        bool ok = true;
        // waits for the next stage and announces its bytes; returns its address (0 when a wait ran out)
        auto stage = [&](uint64_t*& bar) -> uint32_t {
            const int s = ctr % NS;
            if (ctr >= NS && !mbar_wait(&empty[s], ((ctr / NS) - 1) & 1, flag)) {
                ok = false;
                return 0;
            }
            bar = &full[s];
            mbar_expect_tx(bar, STAGE_BYTES);
            ctr++;
            return ring + s * STAGE_BYTES;
        };
        auto load_a = [&](uint32_t dst, int m0, int kb, uint64_t* bar) {
            if constexpr (AMN) {
#pragma unroll
                for (int h = 0; h < BM / 64; h++) tma_load_2d(dst + h * (64 * KB * 2), &map_a, m0 + 64 * h, kb * KB, bar);
            } else {
                tma_load_2d(dst, &map_a, kb * KB, m0, bar);
            }
        };
        for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
            int mb, nb, split;
            item_coords(P, item, mb, nb, split);
            const int m0 = mb * BM, n0 = nb * BN;
            const int kb0 = split * P.kb_per_split, kb1 = min(P.nkb, kb0 + P.kb_per_split);
            if constexpr (ROWS != ROWS_GROUPED) {
                if (lane == 0) {
                    for (int kb = kb0; kb < kb1; kb++) {
                        uint64_t* bar;
                        const uint32_t st = stage(bar);
                        if (!ok) break;
                        load_a(st, m0, kb, bar);
                        if constexpr (BMN) {
#pragma unroll
                            for (int h = 0; h < BN / 64; h++)
                                tma_load_2d(st + A_BYTES + h * (64 * KB * 2), &map_b, n0 + 64 * h, kb * KB, bar);
                        } else {
                            tma_load_2d(st + A_BYTES, &map_b, kb * KB, n0, bar);
                        }
                    }
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
            }
            if constexpr (ROWS != ROWS_PLAIN) {
                if (ROWS == ROWS_EXTEND && split != P.splits - 1) continue;  // the last split extends
                RowAdapters who;
                who.load(P, m0, lane);
                uint32_t off[4];
                for (int j = who.next(off); j != RowAdapters::NONE && ok; j = who.next(off)) {
                    if (lane == 0) {
                        const int e0 = ROWS == ROWS_GROUPED ? kb0 : 0;
                        const int e1 = ROWS == ROWS_GROUPED ? kb1 : (P.rank + KB - 1) / KB;
                        for (int kb = e0; kb < e1; kb++) {
                            uint64_t* bar;
                            const uint32_t st = stage(bar);
                            if (!ok) break;
                            if constexpr (ROWS == ROWS_GROUPED)
                                load_a(st, m0, kb, bar);
                            else
                                tma_load_2d(st, &map_u, kb * KB, m0, bar);
                            if constexpr (BMN) {
#pragma unroll
                                for (int h = 0; h < BN / 64; h++)
                                    tma_load_3d(st + A_BYTES + h * (64 * KB * 2), &map_x, n0 + 64 * h, kb * KB, j, bar);
                            } else {
                                tma_load_3d(st + A_BYTES, &map_x, kb * KB, n0, j, bar);
                            }
                        }
                    }
                    ok = __shfl_sync(0xffffffffu, ok, 0);
                }
            }
        }
        // copies still in flight land before the CTA leaves (bounded)
        if (lane == 0)
            for (int k = (ctr > NS ? ctr - NS : 0); k < ctr; k++) mbar_wait(&full[k % NS], (k / NS) & 1, flag);
    } else if (warp == EPI_WARPS + 1) {
        // ---------------- MMA issuer
        int ctr = 0, acc = 0;
        bool ok = true;
        // the MMAs of one stage: `ks` steps of 16; A is MN-major only where `amn`
        auto multiply = [&](uint32_t d, bool amn, int ks, bool fresh, const uint32_t (&off)[4], bool rows) {
            const int s = ctr % NS;
            if (!mbar_wait(&full[s], (ctr / NS) & 1, flag)) {
                ok = false;
                return;
            }
            fence_after();
            const uint32_t sa = ring + s * STAGE_BYTES, sb = sa + A_BYTES;
#pragma unroll
            for (int k = 0; k < KB / 16; k++) {
                if (k < ks) {
                    const uint64_t da = amn ? smem_desc(sa + k * 2048, 64 * KB * 2, 1024) : smem_desc(sa + k * 32, 16, 1024);
                    const uint64_t db = BMN ? smem_desc(sb + k * 2048, 64 * KB * 2, 1024) : smem_desc(sb + k * 32, 16, 1024);
                    const uint32_t id = idesc_half(BF16, amn, BMN, BM, BN);
                    if (rows)
                        mma_half_rows(d, da, db, id, (fresh && k == 0) ? 0u : 1u, off);
                    else
                        mma_half(d, da, db, id, (fresh && k == 0) ? 0u : 1u);
                }
            }
            mma_commit(&empty[s]);  // the stage is free once these MMAs have read it
            ctr++;
        };
        for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
            int mb, nb, split;
            item_coords(P, item, mb, nb, split);
            const int kb0 = split * P.kb_per_split, kb1 = min(P.nkb, kb0 + P.kb_per_split);
            const int b = acc & 1;
            const uint32_t d = tmem_base + (uint32_t)(b * BN);
            if (lane == 0 && acc >= 2 && !mbar_wait(&acce[b], ((acc / 2) - 1) & 1, flag)) ok = false;
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (!ok) break;
            fence_after();
            uint32_t off[4] = {0, 0, 0, 0};
            if constexpr (ROWS != ROWS_GROUPED) {
                if (lane == 0)
                    for (int kb = kb0; kb < kb1 && ok; kb++) multiply(d, AMN, KB / 16, kb == kb0, off, false);
                ok = __shfl_sync(0xffffffffu, ok, 0);
            }
            if constexpr (ROWS != ROWS_PLAIN) {
                if (ROWS == ROWS_GROUPED || split == P.splits - 1) {
                    RowAdapters who;
                    who.load(P, mb * BM, lane);
                    for (int j = who.next(off); j != RowAdapters::NONE && ok; j = who.next(off)) {
                        if (lane == 0) {
                            const int e0 = ROWS == ROWS_GROUPED ? kb0 : 0;
                            const int e1 = ROWS == ROWS_GROUPED ? kb1 : (P.rank + KB - 1) / KB;
                            for (int kb = e0; kb < e1 && ok; kb++) {
                                if constexpr (ROWS == ROWS_GROUPED)
                                    multiply(d, AMN, KB / 16, kb == kb0, off, true);
                                else
                                    multiply(d, false, min(KB / 16, (P.rank - kb * KB + 15) / 16), false, off, true);
                            }
                        }
                        ok = __shfl_sync(0xffffffffu, ok, 0);
                    }
                }
            }
            if (lane == 0) mma_commit(&accf[b]);  // accumulator b is complete (or tracks what was issued)
            acc++;
        }
        // every issued MMA has completed before the tensor memory is released (bounded)
        if (lane == 0 && acc > 0) mbar_wait(&accf[(acc - 1) & 1], ((acc - 1) / 2) & 1, flag);
    } else {
        // ---------------- epilogue: warps 0..7; lanes 32 * (warp % 4) .., columns BN / 2 * (warp / 4) ..
        const int quad = warp & 3, half = warp >> 2;
        float* buf = turn + warp * STAGE_WORDS;
        int acc = 0;
        for (int item = blockIdx.x; item < items; item += gridDim.x, acc++) {
            int mb, nb, split;
            item_coords(P, item, mb, nb, split);
            const int b = acc & 1, row0 = mb * BM + quad * 32, row = row0 + lane;
            const bool live = row < P.m;
            // what the row's epilogue needs, read while the MMAs run
            float factor = 1.0f, lse = 0.0f, dl = 0.0f, top = -INFINITY, sum = 0.0f;
            int64_t label = -1;  // relative to this piece's column 0
            bool none = false;
            if constexpr (EPI == EPI_STORE) {
                if constexpr (ROWS == ROWS_GROUPED) {
                    const int id = live ? P.index[row] : -1;
                    none = id < 0 || id >= P.adapters;
                }
                if (P.alpha) factor = *P.alpha;
            } else {
                const int64_t t = live ? P.target[row] : -1;
                const bool labelled = t >= 0 && t < P.vocab;
                label = labelled ? t - P.col0 : -1;
                if constexpr (EPI == EPI_GRAD) {
                    none = !labelled;
                    if (labelled) {
                        lse = P.lse[row];
                        dl = P.dloss[row];
                        if (P.gain) dl *= *P.gain;
                    }
                }
            }
            if (!mbar_wait(&accf[b], (acc / 2) & 1, flag)) break;
            fence_after();
#pragma unroll 1
            for (int cb = half * (BN / 64); cb < (half + 1) * (BN / 64); cb++) {
                const int c0 = nb * BN + cb * 32;
                float v[32];
                tmem_ld32(tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(b * BN + cb * 32), v);
                if (c0 >= P.n || row0 >= P.m) continue;
                const int cols = min(32, P.n - c0);
                if constexpr (EPI == EPI_STATS) {
                    float hi = top;
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        if (i < cols) hi = fmaxf(hi, v[i]);
                    // exp2((v - hi) log2 e); a row of -inf alone keeps sum 0
                    constexpr float L2E = 1.4426950408889634f;
                    const float ref = hi == -INFINITY ? 0.0f : hi;
                    float part = sum * exp2f((top - ref) * L2E);
                    if (top == -INFINITY) part = sum;
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        if (i < cols) part += exp2f((v[i] - ref) * L2E);
                    sum = part;
                    top = hi;
                    if (label >= c0 && label < c0 + cols) {
                        float mine = 0.0f;
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            if (c0 + i == label) mine = v[i];
                        P.label_logit[row] = mine;
                    }
                    continue;
                }
                if constexpr (EPI == EPI_GRAD) {
                    constexpr float L2E = 1.4426950408889634f;
#pragma unroll
                    for (int i = 0; i < 32; i++) {
                        float p = exp2f((v[i] - lse) * L2E);
                        if (c0 + i == label) p -= 1.0f;
                        v[i] = none ? 0.0f : p * dl;
                    }
                }
                if constexpr (EPI == EPI_STORE) {
                    if (P.f32in && live) {
                        const float* src = P.f32in + (int64_t)row * P.ldf + c0;
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            if (i < cols) v[i] += src[i];
                    }
#pragma unroll
                    for (int i = 0; i < 32; i++) v[i] = (ROWS == ROWS_GROUPED && none) ? 0.0f : v[i] * factor;
                    if (P.f32out && live) {
                        float* dst = P.f32out + (int64_t)split * P.split_stride + (int64_t)row * P.ldf + c0;
                        if (cols == 32) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4)
                                *reinterpret_cast<float4*>(dst + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; i++)
                                if (i < cols) dst[i] = v[i];
                        }
                    }
                    if (!P.out) continue;
                }
                uint16_t* out = reinterpret_cast<uint16_t*>(P.out);
                if (P.out_vec && cols == 32) {
                    if (live) {
                        uint16_t* dst = out + (int64_t)row * P.ldo + c0;
#pragma unroll
                        for (int i = 0; i < 32; i += 8)
                            *reinterpret_cast<uint4*>(dst + i) =
                                make_uint4(pack2<BF16>(v[i], v[i + 1]), pack2<BF16>(v[i + 2], v[i + 3]),
                                           pack2<BF16>(v[i + 4], v[i + 5]), pack2<BF16>(v[i + 6], v[i + 7]));
                    }
                } else {
                    // rows that start anywhere: turned in shared memory so that a warp writes along one row
#pragma unroll
                    for (int i = 0; i < 32; i++) buf[lane * 33 + i] = v[i];
                    __syncwarp();
                    const int rows = min(32, P.m - row0);
                    for (int r = 0; r < rows; r++)
                        if (lane < cols) out[(int64_t)(row0 + r) * P.ldo + c0 + lane] = pack1<BF16>(buf[r * 33 + lane]);
                    __syncwarp();
                }
            }
            if constexpr (EPI == EPI_STATS) {
                if (live) P.stats[(int64_t)(nb * 2 + half) * P.m + row] = make_float2(top, sum);
            }
            fence_before();
            mbar_arrive(&acce[b]);
        }
    }

    // teardown: every role is done with the tensor memory
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == EPI_WARPS + 1) tmem_free(tmem_base, TMEM_COLS);
    if (tid == 0 && *(volatile int*)flag) {
        *(volatile int*)P.fail = 1;
        __threadfence_system();
    }
}

}  // namespace hg
}  // namespace cdclq

// half_gemm.cuh - the half-precision tensor-core product behind the adapter, checkpoint and loss operators.
//
//   D[m][n] = sum_k A[m][k] B[n][k]        A, B both bf16 or both f16, D accumulated in f32 in tensor memory
//
// One persistent kernel, specialised at compile time on
//   AMN, BMN   whether an operand is contiguous along its rows' index (MN-major) or along k (K-major)
//   CG, BN     a tile is 128 CG rows x BN columns.  CG = 2: a pair of CTAs shares it, each with half of A's and half of
//              B's rows in its shared memory and half of D's rows in its tensor memory, so that a product of 256 x 256
//              reads 64 bytes a clock and SM through L2 (96 with CG = 1 and 128 x 256), one of 256 x 512 48; 47 is what
//              L2 was measured to give.  CG = 1, narrow, where there are few tiles
//   ROWS       what the adapters of the rows do (see RowMode)
//   EPI        what becomes of a finished tile (see Epilogue)
// TMA brings 64-deep K blocks into a ring of 128-byte-swizzled stages, one thread issues the MMAs, and sixteen warps take
// a finished accumulator into registers and work on it while the next MMAs run.  Tensor memory holds two accumulators of
// up to 256 columns: two tiles' in turn, or the halves of a tile of 512, where the next tile's first MMAs go to the half
// that is free first.
// Bound by the tensor cores, and over milliseconds by the power limit.  Measured: 4096 x 4096 x 4096 in bf16 with 8 adapters
// of rank 32, 103 us (1.34 PFLOP/s, 82 % of what a library product of bf16 gives in a burst); the three products of a training
// step of 8191 x 32000 x 2048 in f16, 1.18-1.23 PFLOP/s (86-90 % of the library's lasting rate).  With 57 rows it reads its
// other operand, 206 MB, at 5.0 TB/s (76 % of a copy): 393 tiles make 2.7 rounds over 148 SMs.
#pragma once

#include "common.cuh"
#include "half_gemm.h"
#include "tcgen05.cuh"

namespace cdclq {
namespace hg {

using namespace tc;

constexpr int BM = 128;            // tile rows of a CTA = tensor-memory lanes
constexpr int KB = 64;             // K block: 128 bytes of a 16-bit type
constexpr int A_BYTES = BM * KB * 2;
constexpr int EPI_WARPS = 16;      // four per lane quadrant, each with a quarter of the accumulator's columns
constexpr int THREADS = (EPI_WARPS + 2) * 32;
constexpr int TURN_BYTES = 32 * 64;   // one epilogue warp's transposition buffer: 64 bytes of each of its 32 rows
constexpr int RING_BYTES = 192 * 1024;  // deep enough: eight stages of 57 rows of A, in place of six of 128, gave the same time
constexpr int LEAD = 2;            // tiles of 512: stages whose MMAs go to the first half before the second half's
constexpr int BAND = 16;           // row blocks per band of the tile order: a wave's operands stay in L2

// Each sum of at most this many K blocks leaves tensor memory and is added up in registers (EPI_STATS): the tensor core
// cuts its f32 sums off instead of rounding them, which over 4096 products moved a loss of 10 by 1e-5; 1024 at a time
// keep it within a few 1e-6.
constexpr int STATS_KB = 16;

__host__ __device__ constexpr int b_bytes(int cg, int bn) { return bn / cg * KB * 2; }

// How the adapter of each row (none if outside [0, adapters)) takes part.
enum RowMode {
    ROWS_PLAIN = 0,   // not at all
    ROWS_EXTEND = 1   // D[m] += U[m] Bx[index[m]]: further K blocks, whose MMAs write the adapter's own rows only
};
enum Epilogue {
    EPI_STORE = 0,  // a 16-bit matrix, and / or f32 partial sums
    EPI_STATS = 1,  // running maximum and sum of exp of each row, and the label's logit
    EPI_GRAD = 2    // (softmax - onehot) * dloss as a 16-bit matrix
};

__host__ __device__ constexpr size_t smem_bytes() {
    return RING_BYTES + EPI_WARPS * TURN_BYTES + 1024 /* alignment */ + 256 /* barriers */;
}
// Parts of a tile's columns for which EPI_STATS keeps a (maximum, sum) pair of each row.
constexpr int STATS_PARTS = EPI_WARPS / 4;

struct Params {
    int m, n, nkb;             // rows, columns, K blocks
    int tiles_m, tiles_n, ntiles;
    int splits, kb_per_split;  // the K blocks of a tile, over several items
    int stage_bytes;           // that the copies of a K block bring, to all CTAs of the tile
    // rows' adapters (see RowLists): null where there are none
    const uint32_t* lists;
    int rank;                  // ROWS_EXTEND: depth of the extension
    FarRows far;
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
    float2* stats;             // [STATS_PARTS * tiles_n][m]: maximum, sum of exp(v - maximum)
    float* label_logit;        // [m]
    const float* lse;          // [m]
    const float* dloss;        // [m]
    const float* gain;         // on the gradient
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

// 2^v; results below 2^-126 are 0, nothing beside a sum of 1 or more or in a gradient of 16 bits.
__device__ __forceinline__ float exp2_normal(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// (v - ref) * factor, two at a time, each operation rounded: the difference of near numbers stays exact.
__device__ __forceinline__ void scale_off(float (&v)[16], float ref, float factor) {
    uint64_t minus, by;
    asm("mov.b64 %0, {%1, %1};" : "=l"(minus) : "f"(-ref));
    asm("mov.b64 %0, {%1, %1};" : "=l"(by) : "f"(factor));
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
        uint64_t x;
        asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(v[i]), "f"(v[i + 1]));
        asm("add.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(minus));
        asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(by));
        asm("mov.b64 {%0, %1}, %2;" : "=f"(v[i]), "=f"(v[i + 1]) : "l"(x));
    }
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


// The part of a row's extension whose factors are past f16's range, in f32, to 16 of its columns.  Few rows ever have one: a function
// of its own keeps it out of the epilogue's registers.
template <bool BMN>
__device__ __noinline__ void add_far(const FarRows far, int rank, int n, int row, int col, float* z) {
    const float* u = far.u + (int64_t)row * rank;
    const uint16_t* x = far.x + far.index[row] * far.step + col * (BMN ? (int64_t)1 : far.ld);
    for (int k = 0; k < rank; k++) {
        const float v = u[k];
        if (!(fabsf(v) >= 65520.0f && fabsf(v) < INFINITY)) continue;  // what rounds to an infinity
        for (int i = 0; i < 16 && col + i < n; i++)
            z[i] = fmaf(v, __half2float(__ushort_as_half(x[BMN ? k * far.ld + i : i * far.ld + k])), z[i]);
    }
}

template <bool BF16, bool AMN, bool BMN, int CG, int BN, int ROWS, int EPI>
__global__ void __launch_bounds__(THREADS, 1)
half_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                 const __grid_constant__ CUtensorMap map_u, const __grid_constant__ CUtensorMap map_x, const Params P) {
    constexpr bool WIDE = BN == 512;
    constexpr int AC = WIDE ? 256 : BN;  // columns of an accumulator
    constexpr int STAGE_BYTES = A_BYTES + b_bytes(CG, BN);
    constexpr int NS = RING_BYTES / STAGE_BYTES;
    constexpr int BC = AC / CG;  // B's rows of an accumulator in this CTA
    constexpr int HALF_BYTES = BC * KB * 2;
    constexpr uint32_t TMEM_COLS = 2 * AC;
    static_assert(!WIDE || (CG == 2 && EPI != EPI_STATS), "tiles of 512 columns");
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* turn = base + RING_BYTES;
    uint64_t* full = reinterpret_cast<uint64_t*>(turn + EPI_WARPS * TURN_BYTES);  // of the pair's first CTA
    uint64_t* empty = full + NS;
    uint64_t* accf = empty + NS;
    uint64_t* acce = accf + 2;  // of the pair's first CTA
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acce + 2);
    int* flag = reinterpret_cast<int*>(tmem_slot + 1);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = CG == 2 ? (int)cluster_rank() : 0;

    // a later kernel that needs nothing of this one may take the SMs that run out of tiles
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (tid == 0) {
        for (int s = 0; s < NS; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(&accf[b], 1);
            mbar_init(&acce[b], CG * EPI_WARPS);
        }
        *flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == EPI_WARPS + 1) tmem_alloc<CG>(tmem_slot, TMEM_COLS);
    fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();
    fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int items = P.ntiles * P.splits;
    const int step = gridDim.x / CG, first = blockIdx.x / CG;
    const uint32_t ring = smem_u32(base);

    if (warp == EPI_WARPS) {
        // ---------------- TMA producer: one thread waits and issues (a loop that takes the whole warp along, to share a word of it
        // now and then, pays 200 clocks for each)
        int ctr = 0;
        bool ok = true;
        // waits for the next stage and, in the first CTA, announces the pair's bytes; returns its address
        auto stage = [&](uint32_t& bar) -> uint32_t {
            const int s = ctr % NS;
            if (ctr >= NS && !mbar_wait(&empty[s], ((ctr / NS) - 1) & 1, flag)) {
                ok = false;
                return 0;
            }
            bar = smem_u32(&full[s]);
            if constexpr (CG == 2) bar = first_cta(bar);
            if (rank == 0) mbar_expect_tx(&full[s], (uint32_t)P.stage_bytes);
            ctr++;
            return ring + s * STAGE_BYTES;
        };
        auto load2 = [&](uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
            if constexpr (CG == 2)
                tma_load_2d_pair(dst, map, x, y, bar);
            else
                tma_load_2d(dst, map, x, y, bar);
        };
        auto load3 = [&](uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
            if constexpr (CG == 2)
                tma_load_3d_pair(dst, map, x, y, z, bar);
            else
                tma_load_3d(dst, map, x, y, z, bar);
        };
        auto load_a = [&](uint32_t dst, int m0, int kb, uint32_t bar) {
            if constexpr (AMN) {
#pragma unroll
                for (int h = 0; h < BM / 64; h++) load2(dst + h * (64 * KB * 2), &map_a, m0 + 64 * h, kb * KB, bar);
            } else {
                load2(dst, &map_a, kb * KB, m0, bar);
            }
        };
        for (int item = lane == 0 ? first : items; item < items && ok; item += step) {
            int mb, nb, split;
            item_coords(P, item, mb, nb, split);
            const int m0 = (mb * CG + rank) * BM, n0 = nb * BN + rank * BC;
            const int kb0 = split * P.kb_per_split, kb1 = min(P.nkb, kb0 + P.kb_per_split);
            for (int kb = kb0; kb < kb1; kb++) {
                uint32_t bar;
                const uint32_t st = stage(bar);
                if (!ok) break;
                load_a(st, m0, kb, bar);
#pragma unroll
                for (int w = 0; w < BN / AC; w++) {
                    const uint32_t sb = st + A_BYTES + w * HALF_BYTES;
                    if constexpr (BMN) {
#pragma unroll
                        for (int h = 0; h < BC / 64; h++) load2(sb + h * (64 * KB * 2), &map_b, n0 + w * AC + 64 * h, kb * KB, bar);
                    } else {
                        load2(sb, &map_b, kb * KB, n0 + w * AC, bar);
                    }
                }
            }
            if constexpr (ROWS == ROWS_EXTEND) {
                if (split != P.splits - 1 || !P.lists) continue;  // the last split extends
                const uint32_t* list = P.lists + (int64_t)mb * row_list_words(CG * BM);
                const int count = (int)list[0];
                for (int e = 0; e < count && ok; e++) {
                    const int j = (int)list[ROW_LIST_IDS + e];
                    for (int kb = 0; kb < (P.rank + KB - 1) / KB; kb++) {
                        uint32_t bar;
                        const uint32_t st = stage(bar);
                        if (!ok) break;
                        load2(st, &map_u, kb * KB, m0, bar);
#pragma unroll
                        for (int w = 0; w < BN / AC; w++) {
                            const uint32_t sb = st + A_BYTES + w * HALF_BYTES;
                            if constexpr (BMN) {
#pragma unroll
                                for (int h = 0; h < BC / 64; h++)
                                    load3(sb + h * (64 * KB * 2), &map_x, n0 + w * AC + 64 * h, kb * KB, j, bar);
                            } else {
                                load3(sb, &map_x, kb * KB, n0 + w * AC, j, bar);
                            }
                        }
                    }
                }
            }
        }
        // the last stages have been read before the pair leaves, so nothing is on its way to either CTA; where the MMA
        // issuer gave up, the copies in flight land (bounded)
        if (lane == 0)
            for (int k = (ctr > NS ? ctr - NS : 0); k < ctr; k++)
                if (!mbar_wait(&empty[k % NS], (k / NS) & 1, flag) && rank == 0) mbar_wait(&full[k % NS], (k / NS) & 1, flag);
        __syncwarp();
    } else if (warp == EPI_WARPS + 1) {
        // ---------------- MMA issuer, one thread of the pair's first CTA
        int acc = 0;
        bool ok = rank == 0 && lane == 0;
        int slot = 0;        // of the next stage
        uint32_t phase = 0;  // parity of its barrier
        // the next stage's operands are there (false: the wait ran out); a look at the barrier may have shown it already
        auto arrived = [&](bool seen) -> bool {
            if (!seen && !mbar_wait(&full[slot], phase, flag)) {
                ok = false;
                return false;
            }
            fence_after();
            return true;
        };
        auto advance = [&](int& s, uint32_t& p) {
            if (++s == NS) s = 0, p ^= 1;
        };
        // the stage is free once the MMAs issued so far have read it; a look at the next one while they run
        auto done = [&]() -> bool {
            mma_commit<CG>(&empty[slot]);
            advance(slot, phase);
            return mbar_test(&full[slot], phase);
        };
        // descriptors of the first stage's operands; a stage, a half and a step of 16 further are added to their addresses
        constexpr uint64_t A_STEP = (AMN ? 2048 : 32) >> 4, B_STEP = (BMN ? 2048 : 32) >> 4;
        const uint64_t desc_a = AMN ? smem_desc(ring, 64 * KB * 2, 1024) : smem_desc(ring, 16, 1024);
        [[maybe_unused]] const uint64_t desc_u = smem_desc(ring, 16, 1024);  // the extension's first operand is K-major
        const uint64_t desc_b = BMN ? smem_desc(ring + A_BYTES, 64 * KB * 2, 1024) : smem_desc(ring + A_BYTES, 16, 1024);
        constexpr uint32_t ID = idesc_half(BF16, AMN, BMN, CG * BM, AC);
        [[maybe_unused]] constexpr uint32_t ID_U = idesc_half(BF16, false, BMN, CG * BM, AC);
        // the four MMAs of a stage's operands into d
        auto multiply = [&](uint32_t d, int s, int half, bool fresh) {
            const uint64_t da = desc_a + (uint64_t)(s * (STAGE_BYTES >> 4)), db = desc_b + (uint64_t)(s * (STAGE_BYTES >> 4) + half * (HALF_BYTES >> 4));
#pragma unroll
            for (int k = 0; k < KB / 16; k++) mma_half<CG>(d, da + k * A_STEP, db + k * B_STEP, ID, (fresh && k == 0) ? 0u : 1u);
        };
        // `ks` of them, of the extension, for some rows only
        [[maybe_unused]] auto extend = [&](uint32_t d, int s, int half, int ks, const uint32_t (&off)[4 * CG]) {
            const uint64_t da = desc_u + (uint64_t)(s * (STAGE_BYTES >> 4)), db = desc_b + (uint64_t)(s * (STAGE_BYTES >> 4) + half * (HALF_BYTES >> 4));
#pragma unroll
            for (int k = 0; k < KB / 16; k++)
                if (k < ks) mma_half_rows(d, da + k * 2, db + k * B_STEP, ID_U, 1u, off);
        };
        // the K blocks k0 .. k1 into accumulator d
        auto plain = [&](uint32_t d, int k0, int k1) {
            bool seen = false;
            for (int kb = k0; kb < k1; kb++) {
                if (!arrived(seen)) break;
                multiply(d, slot, 0, kb == k0);
                seen = done();
            }
        };
        // the same into both halves of a tile of 512; the second is waited for after the first stages' MMAs into the first
        auto plain_wide = [&](int item_no, int k0, int k1) {
            const int lead = min(LEAD, k1 - k0);
            const int slot0 = slot;
            const uint32_t phase0 = phase;
            for (int q = 0; q < lead; q++) {
                if (!arrived(false)) return;
                multiply(tmem_base, slot, 0, q == 0);
                advance(slot, phase);
            }
            slot = slot0;
            phase = phase0;
            if (item_no > 0 && !mbar_wait(&acce[1], (item_no - 1) & 1, flag)) {
                ok = false;
                return;
            }
            fence_after();
            bool seen = true;
            for (int kb = k0; kb < k1; kb++) {
                if (!arrived(seen)) return;
                if (kb >= k0 + lead) multiply(tmem_base, slot, 0, false);
                multiply(tmem_base + AC, slot, 1, kb == k0);
                seen = done();
            }
        };
        // accumulator `acc & 1` (of a tile of 512: the first half), once its last contents have been read
        auto accumulator = [&]() -> uint32_t {
            const int b = WIDE ? 0 : acc & 1, use = WIDE ? acc : acc / 2;
            if (use > 0 && !mbar_wait(&acce[b], (use - 1) & 1, flag)) ok = false;
            fence_after();
            return tmem_base + (uint32_t)(b * AC);
        };
        auto finished = [&]() {
            mma_commit<CG>(&accf[WIDE ? 0 : acc & 1]);  // the accumulator is complete (or tracks what was issued)
            if (WIDE) mma_commit<CG>(&accf[1]);
            acc++;
        };
        for (int item = first; item < items && ok; item += step) {
            int mb, nb, split;
            item_coords(P, item, mb, nb, split);
            const int kb0 = split * P.kb_per_split, kb1 = min(P.nkb, kb0 + P.kb_per_split);
            if constexpr (EPI == EPI_STATS) {
                for (int c0 = kb0; c0 < kb1 && ok; c0 += STATS_KB) {
                    const uint32_t d = accumulator();
                    if (!ok) break;
                    plain(d, c0, min(kb1, c0 + STATS_KB));
                    finished();
                }
                continue;
            }
            const uint32_t d = accumulator();
            if (!ok) break;
            if constexpr (WIDE)
                plain_wide(acc, kb0, kb1);
            else
                plain(d, kb0, kb1);
            if constexpr (ROWS == ROWS_EXTEND) {
                if (split == P.splits - 1 && P.lists) {
                    const uint32_t* list = P.lists + (int64_t)mb * row_list_words(CG * BM);
                    const int count = (int)list[0];
                    const uint4* masks = reinterpret_cast<const uint4*>(list + row_list_masks(CG * BM));
                    for (int e = 0; e < count && ok; e++) {
                        uint32_t off[4 * CG];
#pragma unroll
                        for (int q = 0; q < CG; q++) *reinterpret_cast<uint4*>(off + 4 * q) = masks[e * CG + q];
                        for (int kb = 0; kb < (P.rank + KB - 1) / KB; kb++) {
                            if (!arrived(false)) break;
#pragma unroll
                            for (int w = 0; w < BN / AC; w++)
                                extend(d + w * AC, slot, w, min(KB / 16, (P.rank - kb * KB + 15) / 16), off);
                            done();
                        }
                    }
                }
            }
            finished();
        }
        // every issued MMA has completed before the tensor memory is released (bounded)
        if (lane == 0 && acc > 0) {
            if (WIDE)
                mbar_wait(&accf[1], (acc - 1) & 1, flag);
            else
                mbar_wait(&accf[(acc - 1) & 1], ((acc - 1) / 2) & 1, flag);
        }
        __syncwarp();
    } else {
        // ---------------- epilogue: lanes 32 * (warp % 4) .., quarter warp / 4 of the accumulator's columns
        constexpr int COLS = AC / 4;  // a thread's: 64, 32 or 16 of one row
        const int quad = warp & 3, part = warp >> 2;
        // A thread holds one row, so 32 rows' pieces of 64 bytes are turned in shared memory: a warp then reads or writes whole
        // sectors, eight rows at a time (piece by piece of 16 bytes and row, a tile's stores took 8000 clocks).  Chunk c of
        // row r lies at c ^ (r / 2) % 4: neither side meets a bank twice.
        [[maybe_unused]] unsigned char* buf = turn + warp * TURN_BYTES;
        [[maybe_unused]] auto chunk = [&](int r, int c) { return reinterpret_cast<uint4*>(buf + r * 64 + ((c ^ (r >> 1)) & 3) * 16); };
        const uint32_t mine = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(part * COLS);
        int acc = 0;
        // the accumulator has been read: tell the MMA issuer
        auto release = [&](int b) {
            fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (CG == 2)
                    mbar_arrive_cluster(first_cta(smem_u32(&acce[b])));
                else
                    mbar_arrive(&acce[b]);
            }
        };
        // writes `cols` of `piece` columns from c0 of the rows in the buffer
        [[maybe_unused]] auto put_rows = [&](int piece, int c0, int cols, int rows, int row0) {
            uint16_t* out = reinterpret_cast<uint16_t*>(P.out);
            const int ch = piece / 8;
            if (P.out_vec && cols == piece) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int r = i * (32 / ch) + lane / ch, c = lane % ch;
                    if (i < ch && r < rows) *reinterpret_cast<uint4*>(out + (int64_t)(row0 + r) * P.ldo + c0 + c * 8) = *chunk(r, c);
                }
            } else {
                // rows that start anywhere: a warp writes along one row
                for (int r = 0; r < rows; r++)
                    if (lane < cols) out[(int64_t)(row0 + r) * P.ldo + c0 + lane] = reinterpret_cast<const uint16_t*>(chunk(r, lane / 8))[lane & 7];
            }
            __syncwarp();
        };
        bool ok = true;
        for (int item = first; item < items && ok; item += step) {
            int mb, nb, split;
            item_coords(P, item, mb, nb, split);
            const int row0 = (mb * CG + rank) * BM + quad * 32, row = row0 + lane;
            const bool live = row < P.m;
            if constexpr (EPI == EPI_STATS) {
                const int64_t t = live ? P.target[row] : -1;
                const int chunks = (P.nkb + STATS_KB - 1) / STATS_KB;
                const int c0 = nb * BN + part * COLS, cols = min(COLS, P.n - c0);
                // the label's place among the thread's columns, -1 where it is not
                const int at = (t >= P.col0 + c0 && t < P.col0 + c0 + cols && t < P.vocab) ? (int)(t - P.col0 - c0) : -1;
                float top = -INFINITY, sum = 0.0f;
                float z[COLS];
#pragma unroll
                for (int i = 0; i < COLS; i++) z[i] = 0.0f;
                for (int c = 0; c < chunks; c++, acc++) {
                    if (!mbar_wait_warp(&accf[acc & 1], (acc / 2) & 1, flag)) {
                        ok = false;
                        break;
                    }
                    fence_after();
                    if (c + 1 < chunks) {
#pragma unroll
                        for (int q = 0; q < COLS; q += 16) {
                            float v[16];
                            tmem_ld16(mine + (uint32_t)((acc & 1) * AC + q), v);
#pragma unroll
                            for (int i = 0; i < 16; i++) z[q + i] += v[i];
                        }
                    } else {
                        // the logits are complete, 16 columns at a time: exp2((v - top) log2 e), the sum so far brought to the new
                        // maximum; a row of -inf alone keeps sum 0, one with +inf gets the sum inf (nothing is taken off an infinite maximum)
                        constexpr float L2E = 1.4426950408889634f;
#pragma unroll
                        for (int q = 0; q < COLS; q += 16) {
                            float v[16];
                            tmem_ld16(mine + (uint32_t)((acc & 1) * AC + q), v);
                            float most = top;
#pragma unroll
                            for (int i = 0; i < 16; i++) v[i] += z[q + i];
                            if (cols < COLS) {
#pragma unroll
                                for (int i = 0; i < 16; i++)
                                    if (q + i >= cols) v[i] = -INFINITY;
                            }
#pragma unroll
                            for (int i = 0; i < 16; i++) most = fmaxf(most, v[i]);
                            if (at >= q && at < q + 16) {
                                float own = 0.0f;
#pragma unroll
                                for (int i = 0; i < 16; i++)
                                    if (q + i == at) own = v[i];
                                P.label_logit[row] = own;
                            }
                            const float ref = fabsf(most) == INFINITY ? 0.0f : most;
                            scale_off(v, ref, L2E);
                            float some = 0.0f;
#pragma unroll
                            for (int i = 0; i < 16; i++) some += exp2_normal(v[i]);
                            sum = sum * exp2_normal((top - ref) * L2E) + some;
                            top = most;
                        }
                    }
                    release(acc & 1);
                }
                if (!ok) break;
                if (live) P.stats[(int64_t)(nb * STATS_PARTS + part) * P.m + row] = make_float2(top, sum);
                continue;
            }
            // what the row's epilogue needs, read while the MMAs run
            float factor = 1.0f, lse = 0.0f, dl = 0.0f;
            int64_t label = -1;  // relative to this piece's column 0
            bool none = false;
            if constexpr (EPI == EPI_STORE) {
                if (P.alpha) factor = *P.alpha;
            } else {
                const int64_t t = live ? P.target[row] : -1;
                none = !(t >= 0 && t < P.vocab);
                if (!none) {
                    label = t - P.col0;
                    lse = P.lse[row];
                    dl = P.dloss[row];
                    dl *= *P.gain;
                }
            }
            const int rows = min(32, P.m - row0);
            bool far = false;  // whether the row has factors that U lacks
            if constexpr (!BF16 && ROWS == ROWS_EXTEND) far = live && P.far.past && split == P.splits - 1 && P.far.past[row];
            // waits for the accumulator of the tile's half `w` (or the whole tile)
            auto complete = [&]() -> bool {
                if (!mbar_wait_warp(&accf[acc & 1], (acc / 2) & 1, flag)) ok = false;
                fence_after();
                return ok;
            };
            if constexpr (EPI == EPI_STORE) {
                if (P.f32in || P.f32out || __any_sync(0xffffffffu, far)) {
                    // f32 sums (or what of them is to be added to), 16 columns at a time
#pragma unroll 1
                    for (int w = 0; w < BN / AC; w++, acc++) {
                        if (!complete()) break;
#pragma unroll 1
                        for (int q = 0; q < COLS; q += 16) {
                            float z[16];
                            tmem_ld16(mine + (uint32_t)((acc & 1) * AC + q), z);
                            const int c0 = nb * BN + w * AC + part * COLS + q, cols = min(16, P.n - c0);
                            if (cols <= 0 || rows <= 0) continue;
                            if constexpr (!BF16 && ROWS == ROWS_EXTEND) {
                                if (far) {
                                    float some[16];
#pragma unroll
                                    for (int i = 0; i < 16; i++) some[i] = z[i];
                                    add_far<BMN>(P.far, P.rank, P.n, row, c0, some);
#pragma unroll
                                    for (int i = 0; i < 16; i++) z[i] = some[i];
                                }
                                __syncwarp();
                            }
                            if (P.f32in) {
#pragma unroll
                                for (int i = 0; i < 4; i++) {
                                    const int r = i * 8 + lane / 4, c = (lane & 3) * 4;
                                    const float* src = P.f32in + (int64_t)(row0 + r) * P.ldf + c0 + c;
                                    float4 f = make_float4(0, 0, 0, 0);
                                    if (r < rows && c < cols) f = *reinterpret_cast<const float4*>(src);  // ldf is a multiple of 4
                                    *reinterpret_cast<float4*>(chunk(r, lane & 3)) = f;
                                }
                                __syncwarp();
#pragma unroll
                                for (int i = 0; i < 4; i++) {
                                    const float4 f = *reinterpret_cast<const float4*>(chunk(lane, i));
                                    z[4 * i] += f.x, z[4 * i + 1] += f.y, z[4 * i + 2] += f.z, z[4 * i + 3] += f.w;
                                }
                                __syncwarp();
                            }
                            if (P.f32out) {
#pragma unroll
                                for (int i = 0; i < 4; i++)
                                    *reinterpret_cast<float4*>(chunk(lane, i)) = make_float4(z[4 * i], z[4 * i + 1], z[4 * i + 2], z[4 * i + 3]);
                                __syncwarp();
#pragma unroll
                                for (int i = 0; i < 4; i++) {
                                    const int r = i * 8 + lane / 4, c = (lane & 3) * 4;
                                    float* dst = P.f32out + (int64_t)split * P.split_stride + (int64_t)(row0 + r) * P.ldf + c0 + c;
                                    if (r < rows && c < cols) *reinterpret_cast<float4*>(dst) = *reinterpret_cast<const float4*>(chunk(r, lane & 3));
                                }
                                __syncwarp();
                            }
                            if (P.out) {
#pragma unroll
                                for (int i = 0; i < 2; i++)
                                    *chunk(lane, i) = make_uint4(pack2<BF16>(z[8 * i] * factor, z[8 * i + 1] * factor),
                                                                 pack2<BF16>(z[8 * i + 2] * factor, z[8 * i + 3] * factor),
                                                                 pack2<BF16>(z[8 * i + 4] * factor, z[8 * i + 5] * factor),
                                                                 pack2<BF16>(z[8 * i + 6] * factor, z[8 * i + 7] * factor));
                                __syncwarp();
                                put_rows(16, c0, cols, rows, row0);
                            }
                        }
                        release(acc & 1);
                    }
                    continue;
                }
            }
            // A tile of 512 leaves tensor memory as 16-bit numbers, both halves, before any is written: all CTAs finish their
            // tiles at about the same time, and 64 KB a half then wait 3000 clocks for L2.
            uint32_t packed[BN / AC][COLS / 2];
#pragma unroll
            for (int w = 0; w < BN / AC; w++, acc++) {
                if (!complete()) break;
                const int first_col = nb * BN + w * AC + part * COLS;
#pragma unroll
                for (int q = 0; q < COLS; q += 16) {
                    float z[16];
                    tmem_ld16(mine + (uint32_t)((acc & 1) * AC + q), z);
                    if constexpr (EPI == EPI_GRAD) {
                        constexpr float L2E = 1.4426950408889634f;
                        const int c0 = first_col + q, at = (label >= c0 && label < c0 + 16) ? (int)(label - c0) : -1;
                        scale_off(z, lse, L2E);
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            float p = exp2_normal(z[i]);
                            if (i == at) p -= 1.0f;
                            z[i] = none ? 0.0f : p * dl;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 8; i++) packed[w][q / 2 + i] = pack2<BF16>(z[2 * i] * factor, z[2 * i + 1] * factor);
                }
                release(acc & 1);
            }
            if (!ok || rows <= 0 || !P.out) continue;
#pragma unroll
            for (int w = 0; w < BN / AC; w++) {
                // 32 columns at a time (16 where the thread has no more)
                constexpr int PIECE = COLS < 32 ? COLS : 32;
#pragma unroll
                for (int q = 0; q < COLS; q += PIECE) {
                    const int c0 = nb * BN + w * AC + part * COLS + q, cols = min(PIECE, P.n - c0);
                    if (cols <= 0) break;
#pragma unroll
                    for (int i = 0; i < PIECE / 8; i++)
                        *chunk(lane, i) = make_uint4(packed[w][q / 2 + 4 * i], packed[w][q / 2 + 4 * i + 1], packed[w][q / 2 + 4 * i + 2],
                                                     packed[w][q / 2 + 4 * i + 3]);
                    __syncwarp();
                    put_rows(PIECE, c0, cols, rows, row0);
                }
            }
        }
    }

    // teardown: every role of the pair is done with the tensor memory, the stages and the barriers
    fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();
    fence_after();
    if (warp == EPI_WARPS + 1) tmem_free<CG>(tmem_base, TMEM_COLS);
    if (tid == 0 && *(volatile int*)flag) {
        *(volatile int*)P.fail = 1;
        __threadfence_system();
    }
}

}  // namespace hg
}  // namespace cdclq

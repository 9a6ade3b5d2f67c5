// rank.cu - products of tokens with their own adapters' low-rank factors: u = A_i x and v = B_i^T dy.
//
// A cluster of up to 8 CTAs takes 64 (16) neighbouring tokens, whatever their adapters, and up to 64 ranks; each CTA a share of
// k.  The tokens pass through a ring in shared memory once for every two adapters among them, beside the two adapters' factors;
// each adapter has sums of its own for all the tokens, and a token takes those of its adapter: what another adapter or another
// token holds never enters them.  The cluster's CTAs then add up one another's sums, each for its share of the tokens, in
// order, and write the results.
// Bound by reading the tokens (r products for each value read): mma.sync keeps up with memory at any rank of up to 64.
#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "half_gemm.h"
#include "mma16.cuh"
#include "rank.h"
#include "tcgen05.cuh"

namespace cdclq {

namespace {

constexpr int THREADS = 128, KB = 64, STAGES = 4, PAIR = 2, MOST_RANK = 64;
constexpr int X_PITCH = KB + 8;  // halves: 16-byte pieces of eight rows fall into different banks

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Halves of a stage: the tokens' K block, then PAIR factors' (r x k, or k x r where transposed).
__host__ __device__ constexpr int factor_halves(int rp, bool transposed) { return transposed ? KB * (rp + 8) : rp * X_PITCH; }
__host__ __device__ constexpr int stage_halves(int tokens, int rp, bool transposed) {
    return tokens * X_PITCH + PAIR * factor_halves(rp, transposed);
}
size_t smem_bytes(int tokens, int rp, bool transposed) {
    // the sums of the CTA reuse the ring
    return std::max((size_t)STAGES * stage_halves(tokens, rp, transposed) * 2, (size_t)4 * 16 * (MOST_RANK + 2) * 4);
}

// The tokens of one adapter, ascending; start[id] = tokens of lower adapters.
__device__ __forceinline__ void token_list(const RankArgs& P, int id) {
    __shared__ int below[THREADS / 32], mine[THREADS / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int lower = 0;
#pragma unroll 4
    for (int i = threadIdx.x; i < P.t; i += THREADS) {
        const int v = P.index[i];
        lower += v >= 0 && v < id;
    }
    lower = __reduce_add_sync(0xffffffffu, lower);
    if (lane == 0) below[warp] = lower;
    __syncthreads();
    int at = 0;
    for (int w = 0; w < THREADS / 32; w++) at += below[w];
    if (threadIdx.x == 0) P.start[id] = at;
    for (int base = 0; base < P.t; base += 4 * THREADS) {
        // four neighbouring tokens a thread
        int hits = 0, which = 0;
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int i = base + threadIdx.x * 4 + q;
            if (i < P.t && P.index[i] == id) hits++, which |= 1 << q;
        }
        int sum = hits;  // inclusive prefix sum over the warp
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        if (lane == 31) mine[warp] = sum;
        __syncthreads();
        int place = at + sum - hits, all = 0;
        for (int w = 0; w < THREADS / 32; w++) {
            if (w < warp) place += mine[w];
            all += mine[w];
        }
#pragma unroll
        for (int q = 0; q < 4; q++)
            if (which >> q & 1) P.order[place++] = base + threadIdx.x * 4 + q;
        at += all;
        __syncthreads();
    }
    if (id == P.n - 1 && threadIdx.x == 0) P.start[P.n] = at;
}

// TOKENS: 64, a warp for each 16 of them, or 16, a warp for each 16 of the K block's columns.  NT: the ranks' tiles of 8, at
// most; fewer leave registers for a fourth CTA on the SM.
template <bool BF16, bool TRANSPOSED, int TOKENS, int NT>
__global__ void __launch_bounds__(THREADS, NT == 8 ? 3 : 4) rank_kernel(const RankArgs P) {
    extern __shared__ __align__(16) uint16_t ring[];
    __shared__ int id_of[TOKENS], who[TOKENS], found;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int products = P.compute ? P.tiles * P.cut : 0;
    if ((int)blockIdx.x >= products) {
        if (blockIdx.y == 0 && (int)blockIdx.x - products < P.n) token_list(P, blockIdx.x - products);
        return;
    }
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = blockIdx.x % P.cut, t0 = blockIdx.x / P.cut * TOKENS, r0 = blockIdx.y * MOST_RANK, ranks = min(MOST_RANK, P.r - r0);
    const int nkb = (P.k + KB - 1) / KB, per = (nkb + P.cut - 1) / P.cut, kb0 = min(nkb, rank * per), kb1 = min(nkb, kb0 + per);
    if (tid < TOKENS) {
        const int v = t0 + tid < P.t ? P.index[t0 + tid] : -1;
        id_of[tid] = v >= 0 && v < P.n ? v : 0x7fffffff;
    }
    __syncthreads();
    if (warp == 0) {  // the adapters among the tokens, lowest first
        int a = lane < TOKENS ? id_of[lane] : 0x7fffffff, b = TOKENS > 32 ? id_of[(lane + 32) % TOKENS] : 0x7fffffff, n = 0;
        for (int least = __reduce_min_sync(0xffffffffu, min(a, b)); least != 0x7fffffff; least = __reduce_min_sync(0xffffffffu, min(a, b))) {
            if (lane == 0) who[n] = least;
            if (a == least) a = 0x7fffffff;
            if (b == least) b = 0x7fffffff;
            n++;
        }
        if (lane == 0) found = n;
    }
    __syncthreads();
    const int m0 = TOKENS == 64 ? warp * 16 : 0;
    const int pitch = TRANSPOSED ? P.rp + 8 : X_PITCH, fh = factor_halves(P.rp, TRANSPOSED), sh = stage_halves(TOKENS, P.rp, TRANSPOSED);
    const int mine0 = id_of[m0 + lane / 4], mine1 = id_of[m0 + lane / 4 + 8];
    float sums[NT][4];
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) sums[j][i] = 0.0f;

    // This thread's copies of a stage: XC pieces of 16 bytes of the tokens, up to FC of each factor.  A whole K block needs only
    // their offsets; the last one, cut short, is looked at piece by piece.
    constexpr int XC = TOKENS * 8 / THREADS, FC = NT / 2;
    const int pieces = TRANSPOSED ? KB * P.rp / 8 : P.rp * 8;  // of a factor
    const uint16_t* x_from[XC];
    bool x_live[XC];
#pragma unroll
    for (int i = 0; i < XC; i++) {
        const int t = t0 + (tid >> 3) + i * (THREADS / 8);
        x_live[i] = t < P.t;
        x_from[i] = P.x + (int64_t)min(t, P.t - 1) * P.ldx + (tid & 7) * 8;
    }
    int f_row[FC], f_col[FC];
#pragma unroll
    for (int i = 0; i < FC; i++) {
        const int n = tid + i * THREADS, wide = TRANSPOSED ? P.rp / 8 : 8;
        f_row[i] = n < pieces ? n / wide : -1;
        f_col[i] = n % wide * 8;
    }
    const int64_t f_step = TRANSPOSED ? (int64_t)KB * P.ldm : KB;
    // 8 values of a row to shared memory: those from c on, as far as `last`
    auto piece = [&](uint16_t* dst, const uint16_t* row, int c, int last, bool live) {
        if (!live || c >= last || c + 8 <= last) {
            const bool all = live && c + 8 <= last;
            copy16(dst, all ? row + c : P.x, all);
        } else {
            for (int i = 0; i < 8; i++) dst[i] = c + i < last ? row[c + i] : (uint16_t)0;
        }
    };
    for (int g0 = 0; g0 < found; g0 += PAIR) {
        const int pair = min(PAIR, found - g0);
        bool use[PAIR];  // some token of this warp has the adapter
        float acc[PAIR][NT][4];
#pragma unroll
        for (int q = 0; q < PAIR; q++) {
            const int j = q < pair ? who[g0 + q] : -1;
            use[q] = __any_sync(0xffffffffu, mine0 == j || mine1 == j);
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) acc[q][n][i] = 0.0f;
        }
        const uint16_t* factor[PAIR];
        int64_t f_from[FC];
#pragma unroll
        for (int q = 0; q < PAIR; q++) factor[q] = P.m + (int64_t)who[g0 + min(q, pair - 1)] * (TRANSPOSED ? P.k : P.r) * P.ldm;
#pragma unroll
        for (int i = 0; i < FC; i++)
            f_from[i] = TRANSPOSED ? f_row[i] * P.ldm + r0 + f_col[i] : (int64_t)min(r0 + f_row[i], P.r - 1) * P.ldm + f_col[i];
        auto load = [&](int kb, int slot) {
            uint16_t* st = ring + slot * sh;
            uint16_t* to = st + (tid >> 3) * X_PITCH + (tid & 7) * 8;
            uint16_t* fs = st + TOKENS * X_PITCH;
            if ((kb + 1) * KB <= P.k) {
#pragma unroll
                for (int i = 0; i < XC; i++) copy16(to + i * (THREADS / 8) * X_PITCH, x_from[i] + kb * KB, x_live[i]);
                const int64_t further = kb * f_step;
#pragma unroll
                for (int i = 0; i < FC; i++) {
                    if (f_row[i] < 0) break;
                    // where the rank ends inside a piece of 8, or a row is past it
                    const bool whole = TRANSPOSED ? f_col[i] + 8 <= ranks : true, live = TRANSPOSED ? f_col[i] < ranks : f_row[i] < ranks;
                    uint16_t* dst = fs + f_row[i] * pitch + f_col[i];
#pragma unroll
                    for (int q = 0; q < PAIR; q++) {
                        if (q >= pair) break;
                        const uint16_t* src = factor[q] + f_from[i] + further;
                        if (whole || !live)
                            copy16(dst + q * fh, live ? src : P.x, live);
                        else
                            for (int e = 0; e < 8; e++) dst[q * fh + e] = f_col[i] + e < ranks ? src[e] : (uint16_t)0;
                    }
                }
                return;
            }
#pragma unroll
            for (int i = 0; i < XC; i++)
                piece(to + i * (THREADS / 8) * X_PITCH, x_from[i] - (tid & 7) * 8, kb * KB + (tid & 7) * 8, P.k, x_live[i]);
            for (int q = 0; q < pair; q++) {
#pragma unroll
                for (int i = 0; i < FC; i++) {
                    if (f_row[i] < 0) break;
                    uint16_t* dst = fs + q * fh + f_row[i] * pitch + f_col[i];
                    if (TRANSPOSED) {
                        const int k = kb * KB + f_row[i];
                        piece(dst, factor[q] + (int64_t)min(k, P.k - 1) * P.ldm + r0, f_col[i], ranks, k < P.k);
                    } else {
                        piece(dst, factor[q] + (int64_t)min(r0 + f_row[i], P.r - 1) * P.ldm, kb * KB + f_col[i], P.k, f_row[i] < ranks);
                    }
                }
            }
        };
#pragma unroll 1
        for (int s = 0; s < STAGES - 1; s++) {
            if (kb0 + s < kb1) load(kb0 + s, s);
            copy_commit();
        }
        int slot = 0;
#pragma unroll 1
        for (int kb = kb0; kb < kb1; kb++, slot = (slot + 1) % STAGES) {
            copy_wait<STAGES - 2>();
            __syncthreads();  // stage kb is there, and the one before it has been used by every warp
            if (kb + STAGES - 1 < kb1) load(kb + STAGES - 1, (slot + STAGES - 1) % STAGES);
            copy_commit();
            const uint16_t* st = ring + slot * sh;
#pragma unroll
            for (int q4 = 0; q4 < (TOKENS == 64 ? 4 : 1); q4++) {
                const int kk = (TOKENS == 64 ? q4 : warp) * 16;
                uint32_t a[4];
                load_pieces<false>(a, st + (m0 + (lane & 15)) * X_PITCH + kk + (lane >> 4) * 8);
#pragma unroll
                for (int q = 0; q < PAIR; q++) {
                    if (!use[q]) continue;
                    const uint16_t* f = st + TOKENS * X_PITCH + q * fh;
#pragma unroll
                    for (int j = 0; j < NT; j += 2) {
                        if (NT == 8 && j * 8 >= P.rp) break;
                        uint32_t b[4];
                        if (TRANSPOSED)
                            load_pieces<true>(b, f + (kk + (lane & 15)) * pitch + j * 8 + (lane >> 4) * 8);
                        else
                            load_pieces<false>(b, f + (j * 8 + (lane & 7) + (lane >> 4) * 8) * pitch + kk + (lane >> 3 & 1) * 8);
                        mma16816<BF16>(acc[q][j], a, b[0], b[1]);
                        mma16816<BF16>(acc[q][j + 1], a, b[2], b[3]);
                    }
                }
            }
        }
        copy_wait<0>();
        __syncthreads();  // the ring is free
#pragma unroll
        for (int q = 0; q < PAIR; q++) {
            const int j = q < pair ? who[g0 + q] : -1;
#pragma unroll
            for (int n = 0; n < NT; n++) {
                if (mine0 == j) sums[n][0] = acc[q][n][0], sums[n][1] = acc[q][n][1];
                if (mine1 == j) sums[n][2] = acc[q][n][2], sums[n][3] = acc[q][n][3];
            }
        }
    }
    // [warp's tokens, or the token's parts of the K block][16][MOST_RANK + 2]
    float* part = reinterpret_cast<float*>(ring);
    constexpr int PITCH = MOST_RANK + 2;
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) part[(warp * 16 + lane / 4 + (i >> 1) * 8) * PITCH + n * 8 + (lane & 3) * 2 + (i & 1)] = sums[n][i];
    __syncthreads();
    if (TOKENS == 16) {
        for (int i = tid; i < 16 * ranks; i += THREADS) {
            const int at = i / ranks * PITCH + i % ranks;
            part[at] = (part[at] + part[at + 16 * PITCH]) + (part[at + 32 * PITCH] + part[at + 48 * PITCH]);
        }
        __syncthreads();
    }
    if (P.cut > 1) tc::cluster_sync();
    const int share = (TOKENS + P.cut - 1) / P.cut, first = rank * share, rows = min(share, min(TOKENS - first, P.t - t0 - first));
    for (int i = tid; i < rows * ranks; i += THREADS) {
        const int row = first + i / ranks, c = i % ranks;
        const uint32_t at = tc::smem_u32(part + row * PITCH + c);
        float s = 0.0f;
        for (int q = 0; q < P.cut; q++) s += tc::cluster_load(at, q);
        const int64_t t = t0 + row, k = r0 + c;
        if (P.u16) P.u16[t * P.ldu + k] = half_bits<BF16>(s);
        if (P.su16 || P.su32) {
            const int id = id_of[row];
            const float v = id != 0x7fffffff ? P.scale[id] * s : 0.0f;
            const uint16_t h = half_bits<BF16>(v);
            if (P.su16) P.su16[t * P.lds + k] = h;
            if (P.rest16) P.rest16[t * P.lds + k] = rest_bits<BF16>(v, h);
            if (P.su32) P.su32[t * P.r + k] = v;
        }
    }
    if (P.cut > 1) {
        __syncwarp();
        tc::cluster_sync();  // nobody leaves while its sums may be read
    }
}

template <bool BF16, bool TRANSPOSED, int TOKENS, int NT>
int launch(const RankArgs& p, cudaStream_t st) {
    auto kern = rank_kernel<BF16, TRANSPOSED, TOKENS, NT>;
    static std::atomic<uint64_t> done{0};
    if (int rc = allow_smem(kern, smem_bytes(TOKENS, MOST_RANK, TRANSPOSED), done, "rank_kernel shared memory")) return rc;
    const int64_t lists = p.start ? ceil_div(p.n, p.cut) * p.cut : 0;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)((p.compute ? (int64_t)p.tiles * p.cut : 0) + lists), (unsigned)ceil_div(p.r, MOST_RANK));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem_bytes(TOKENS, p.rp, TRANSPOSED);
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = p.cut;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = p.cut > 1 ? 1 : 0;
    g_launches.fetch_add(1, std::memory_order_relaxed);
    cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
    return e == cudaSuccess ? 0 : cuda_error(e, "rank_kernel launch");
}

template <bool BF16, bool TRANSPOSED, int TOKENS>
int launch_ranks(const RankArgs& p, cudaStream_t st) {
    if (p.rp == 16) return launch<BF16, TRANSPOSED, TOKENS, 2>(p, st);
    return p.rp == 32 ? launch<BF16, TRANSPOSED, TOKENS, 4>(p, st) : launch<BF16, TRANSPOSED, TOKENS, 8>(p, st);
}
template <bool BF16, bool TRANSPOSED>
int launch_tokens(const RankArgs& p, bool few, cudaStream_t st) {
    return few ? launch_ranks<BF16, TRANSPOSED, 16>(p, st) : launch_ranks<BF16, TRANSPOSED, 64>(p, st);
}

}  // namespace

int launch_rank(bool bf16, bool transposed, RankArgs p, cudaStream_t st) {
    p.compute = p.u16 || p.su16 || p.su32;
    if (!p.compute && !p.start) return 0;
    // 16 tokens to a cluster where 64 leave SMs idle even with 8 CTAs each; K blocks over as many CTAs as make four to an SM,
    // four blocks at least for each
    const int sms = sm_count(), nkb = (int)ceil_div(p.k, KB);
    const bool few = ceil_div(p.t, 64) * 8 < sms;
    p.tiles = (int)ceil_div(p.t, few ? 16 : 64);
    p.cut = 1;
    while (p.cut < 8 && (int64_t)p.tiles * p.cut * ceil_div(p.r, MOST_RANK) < 4 * sms && nkb / (p.cut * 2) >= 4) p.cut *= 2;
    p.rp = (int)ceil_div(std::min(p.r, MOST_RANK), 16) * 16;
    if (bf16) return transposed ? launch_tokens<true, true>(p, few, st) : launch_tokens<true, false>(p, few, st);
    return transposed ? launch_tokens<false, true>(p, few, st) : launch_tokens<false, false>(p, few, st);
}

}  // namespace cdclq

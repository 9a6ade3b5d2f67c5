// rank.cu - products of tokens with their own adapters' low-rank factors: u = A_i x and v = B_i^T dy.
//
// A first kernel sorts the tokens by adapter.  Then a cluster of up to 8 CTAs takes 64 (16) tokens of one adapter and up to 64
// ranks; each CTA a share of k.  The tokens' rows, gathered by the list, and the factor's pass through a ring in shared memory
// once; the cluster's CTAs add up one another's sums, each for its share of the tokens, in order, and write the results.
// Bound by reading the tokens (r products for each value read): mma.sync keeps up with memory at any rank of up to 64.
// 4096 tokens of 4096 values, 8 adapters of rank 32: 18 us (1.8 TB/s) beside the weight's expansion, after 4 us of sorting;
// 4100, 6 of rank 64: 34 us.  Tokens as they come, one pass over them for every two adapters of a tile, took 28 and 49 us, and
// 76 us for 3005 tokens of 8256 values and 32 adapters of rank 64 (now 40); it saved the sorting, 2 us for 333 tokens.
#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "half_gemm.h"
#include "mma16.cuh"
#include "rank.h"
#include "tcgen05.cuh"

namespace cdclq {

namespace {

constexpr int THREADS = 128, LIST_THREADS = 512, KB = 64, STAGES = 4, MOST_RANK = 64, MOST_CUT = 8;
constexpr int X_PITCH = KB + 8;  // halves: 16-byte pieces of eight rows fall into different banks

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Halves of a stage: the tokens' K block, then the factor's (r x k, or k x r where transposed).
__host__ __device__ constexpr int factor_halves(int rp, bool transposed) { return transposed ? KB * (rp + 8) : rp * X_PITCH; }
__host__ __device__ constexpr int stage_halves(int tokens, int rp, bool transposed) {
    return tokens * X_PITCH + factor_halves(rp, transposed);
}
size_t smem_bytes(int tokens, int rp, bool transposed) {
    // the sums of the CTA reuse the ring
    return std::max((size_t)STAGES * stage_halves(tokens, rp, transposed) * 2, (size_t)4 * 16 * (MOST_RANK + 2) * 4);
}

// A CTA for each adapter and one for the tokens without: its tokens, ascending, after those of lower adapters.
__global__ void __launch_bounds__(LIST_THREADS) token_list_kernel(const int* __restrict__ index, int t, int n, int* start, int* order,
                                                                  int* past, uint32_t* top) {
    constexpr int WARPS = LIST_THREADS / 32;
    __shared__ int below[WARPS], mine[WARPS];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, id = blockIdx.x;
    auto key = [&](int i) {
        const int v = index[i];
        return v >= 0 && v < n ? v : n;
    };
    int lower = 0;
#pragma unroll 4
    for (int i = threadIdx.x; i < t; i += LIST_THREADS) lower += key(i) < id;
    lower = __reduce_add_sync(0xffffffffu, lower);
    if (lane == 0) below[warp] = lower;
    __syncthreads();
    int at = 0;
#pragma unroll
    for (int w = 0; w < WARPS; w++) at += below[w];
    if (threadIdx.x == 0) {
        start[id] = at;
        if (id == n) start[n + 1] = t;
        if (top && id < n) top[id] = 0;
    }
    for (int base = 0; base < t; base += 4 * LIST_THREADS) {
        // four neighbouring tokens a thread
        int hits = 0, which = 0;
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int i = base + threadIdx.x * 4 + q;
            if (i < t && key(i) == id) hits++, which |= 1 << q;
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
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            if (w < warp) place += mine[w];
            all += mine[w];
        }
#pragma unroll
        for (int q = 0; q < 4; q++)
            if (which >> q & 1) {
                const int i = base + threadIdx.x * 4 + q;
                order[place++] = i;
                if (past) past[i] = 0;
            }
        at += all;
        __syncthreads();
    }
}

// The `g`-th group of up to `tokens` tokens of one adapter (or of none: id = n); false past the last.
struct Group {
    int id, first, count;
};
__device__ __forceinline__ bool find_group(const RankArgs& P, int g, int tokens, Group* out) {
    __shared__ int sums[THREADS / 32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int before = 0;
    for (int base = 0; base <= P.n; base += THREADS) {
        const int id = base + tid, from = id <= P.n ? P.start[id] : 0, to = id <= P.n ? P.start[id + 1] : 0;
        const int groups = (to - from + tokens - 1) / tokens;
        int sum = groups;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        if (lane == 31) sums[warp] = sum;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int w = 0; w < THREADS / 32; w++) {
            if (w < warp) sum += sums[w];
            all += sums[w];
        }
        const int mine = g - before - (sum - groups);
        if (mine >= 0 && mine < groups) *out = {id, from + mine * tokens, min(tokens, to - from - mine * tokens)};
        __syncthreads();
        before += all;
        if (g < before) return true;
    }
    return false;
}

// TOKENS: 64, a warp for each 16 of them, or 16, a warp for each 16 of the K block's columns.  NT: the ranks' tiles of 8, at
// most; fewer leave registers for a fourth CTA on the SM.
template <bool BF16, bool TRANSPOSED, int TOKENS, int NT>
__global__ void __launch_bounds__(THREADS, NT == 8 ? 3 : 4) rank_kernel(const RankArgs P) {
    extern __shared__ __align__(16) uint16_t ring[];
    __shared__ int token[TOKENS];
    __shared__ Group group;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = blockIdx.x % P.cut, r0 = blockIdx.y * MOST_RANK, ranks = min(MOST_RANK, P.r - r0);
    const int nkb = (P.k + KB - 1) / KB, per = (nkb + P.cut - 1) / P.cut, kb0 = min(nkb, rank * per);
    wait_for_previous();  // the lists
    if (!find_group(P, blockIdx.x / P.cut, TOKENS, &group)) return;  // the whole cluster
    const int id = group.id, count = group.count;
    const bool bare = id == P.n;
    const int kb1 = bare ? kb0 : min(nkb, kb0 + per);
    if (tid < TOKENS) token[tid] = P.order[group.first + min(tid, count - 1)];
    __syncthreads();
    const int m0 = TOKENS == 64 ? warp * 16 : 0;
    const int pitch = TRANSPOSED ? P.rp + 8 : X_PITCH, sh = stage_halves(TOKENS, P.rp, TRANSPOSED);
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
        const int row = (tid >> 3) + i * (THREADS / 8);
        x_live[i] = row < count;
        x_from[i] = P.x + (int64_t)token[row] * P.ldx + (tid & 7) * 8;
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
    const uint16_t* factor = P.m + (int64_t)min(id, P.n - 1) * (TRANSPOSED ? P.k : P.r) * P.ldm;
    int64_t f_from[FC];
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
                const uint16_t* src = factor + f_from[i] + further;
                if (whole || !live)
                    copy16(dst, live ? src : P.x, live);
                else
                    for (int e = 0; e < 8; e++) dst[e] = f_col[i] + e < ranks ? src[e] : (uint16_t)0;
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < XC; i++)
            piece(to + i * (THREADS / 8) * X_PITCH, x_from[i] - (tid & 7) * 8, kb * KB + (tid & 7) * 8, P.k, x_live[i]);
#pragma unroll
        for (int i = 0; i < FC; i++) {
            if (f_row[i] < 0) break;
            uint16_t* dst = fs + f_row[i] * pitch + f_col[i];
            if (TRANSPOSED) {
                const int k = kb * KB + f_row[i];
                piece(dst, factor + (int64_t)min(k, P.k - 1) * P.ldm + r0, f_col[i], ranks, k < P.k);
            } else {
                piece(dst, factor + (int64_t)min(r0 + f_row[i], P.r - 1) * P.ldm, kb * KB + f_col[i], P.k, f_row[i] < ranks);
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
        if (m0 >= count) continue;
        const uint16_t* st = ring + slot * sh;
        const uint16_t* f = st + TOKENS * X_PITCH;
#pragma unroll
        for (int q4 = 0; q4 < (TOKENS == 64 ? 4 : 1); q4++) {
            const int kk = (TOKENS == 64 ? q4 : warp) * 16;
            uint32_t a[4];
            load_pieces<false>(a, st + (m0 + (lane & 15)) * X_PITCH + kk + (lane >> 4) * 8);
#pragma unroll
            for (int j = 0; j < NT; j += 2) {
                if (NT == 8 && j * 8 >= P.rp) break;
                uint32_t b[4];
                if (TRANSPOSED)
                    load_pieces<true>(b, f + (kk + (lane & 15)) * pitch + j * 8 + (lane >> 4) * 8);
                else
                    load_pieces<false>(b, f + (j * 8 + (lane & 7) + (lane >> 4) * 8) * pitch + kk + (lane >> 3 & 1) * 8);
                mma16816<BF16>(sums[j], a, b[0], b[1]);
                mma16816<BF16>(sums[j + 1], a, b[2], b[3]);
            }
        }
    }
    copy_wait<0>();
    __syncthreads();  // the ring is free
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
    const int share = (TOKENS + P.cut - 1) / P.cut, first = rank * share, rows = min(share, count - first);
    uint32_t most = 0;
    for (int i = tid; i < rows * ranks; i += THREADS) {
        const int row = first + i / ranks, c = i % ranks;
        const uint32_t at = tc::smem_u32(part + row * PITCH + c);
        float v8[MOST_CUT], s = 0.0f;  // all on their way at once
#pragma unroll
        for (int q = 0; q < MOST_CUT; q++) v8[q] = q < P.cut ? tc::cluster_load(at, q) : 0.0f;
#pragma unroll
        for (int q = 0; q < MOST_CUT; q++) s += v8[q];
        const int64_t t = token[row], k = r0 + c;
        if (P.u16) P.u16[t * P.ldu + k] = half_bits<BF16>(s);
        if (P.su16 || P.su32) {
            const float v = bare ? 0.0f : P.scale[id] * s;
            const uint32_t size = __float_as_uint(fabsf(v));
            if (size < 0x7f800000u) most = max(most, size);
            uint16_t h = half_bits<BF16>(v);
            if (!BF16 && P.past && (h & 0x7fffu) == 0x7c00u && size < 0x7f800000u) h = 0, P.past[t] = 1;
            if (P.su16) P.su16[t * P.lds + k] = h;
            if (P.rest16) P.rest16[t * P.lds + k] = rest_bits<BF16>(v, h);
            if (P.su32) P.su32[t * P.r + k] = v;
        }
    }
    if (P.top && !bare) {  // a maximum does not depend on the order
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0 && most) atomicMax(P.top + id, most);
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
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(p.groups * p.cut), (unsigned)ceil_div(p.r, MOST_RANK));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem_bytes(TOKENS, p.rp, TRANSPOSED);
    cfg.stream = st;
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.cut;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.cut > 1 ? 2 : 1;
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

__global__ void __launch_bounds__(256) rank_split_kernel(const RankSplit S) { rank_split(S, blockIdx.x); }

}  // namespace

int rank_split_ctas(const RankSplit& s, int threads) {
    return (int)std::min<int64_t>(ceil_div((int64_t)s.t * (s.ld / 8), threads), 2 * sm_count());
}

int launch_rank_split(RankSplit s, cudaStream_t st) {
    s.ctas = rank_split_ctas(s, 256);
    CDCLQ_LAUNCH(rank_split_kernel, (unsigned)s.ctas, 256, 0, st, s);
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : cuda_error(e, "rank_split_kernel launch");
}

int launch_rank(bool bf16, bool transposed, RankArgs p, cudaStream_t st) {
    CDCLQ_LAUNCH(token_list_kernel, (unsigned)(p.n + 1), LIST_THREADS, 0, st, p.index, p.t, p.n, p.start, p.order, p.past, p.top);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_error(e, "token_list_kernel launch");
    if (!p.u16 && !p.su16 && !p.su32) return 0;
    // Each adapter (and those without) may leave one group that is not full.  16 tokens to a cluster where 64 leave SMs idle
    // even with 8 CTAs each; K blocks over as many CTAs as run at once, four blocks at least for each.
    const int64_t sms = sm_count(), nkb = ceil_div(p.k, KB);
    auto most = [&](int64_t tokens) { return p.t / tokens + std::min<int64_t>(p.n + 1, p.t); };
    auto likely = [&](int64_t tokens) { return ceil_div(p.t, tokens) + std::min<int64_t>(p.n, p.t / tokens); };
    const bool few = likely(64) * 8 < sms;
    const int tokens = few ? 16 : 64;
    p.groups = (int)most(tokens);
    p.cut = 1;
    const int64_t at_once = (p.r > 32 ? 3 : 4) * sms;
    while (p.cut < MOST_CUT && likely(tokens) * p.cut * 2 * ceil_div(p.r, MOST_RANK) <= at_once && nkb / (p.cut * 2) >= 4) p.cut *= 2;
    p.rp = (int)ceil_div(std::min(p.r, MOST_RANK), 16) * 16;
    if (bf16) return transposed ? launch_tokens<true, true>(p, few, st) : launch_tokens<true, false>(p, few, st);
    return transposed ? launch_tokens<false, true>(p, few, st) : launch_tokens<false, false>(p, few, st);
}

}  // namespace cdclq

// adapters.cu - low-rank adapters of many requests beside a shared packed projection.
//
//   u_t = A_i x_t        y_t = W x_t + s_i B_i u_t                               i = index[t], none for an index outside [0, n)
//   v_t = s_i B_i^T dy_t     dx_t = W^T dy_t + A_i^T v_t     dA_i = sum_{t in i} v_t x_t^T     dB_i = s_i sum_{t in i} dy_t u_t^T
//
// A few tokens (packed.cu): the codes are read once, W is never formed.  More tokens: W is expanded once to 16 bits, which
// stays in L2 for the layers of a model, and multiplied on the tensor cores; the adapters ride in the same accumulators as
// further K blocks, whose MMAs write only the tensor-memory lanes of the adapter's own tokens.  So a request never meets
// another one's adapter, not even as a product with zero: a NaN in one adapter or one request stays there.  In f16 what of s_i u_t
// or v_t is past 65504 stays f32 and meets its factor in the product's epilogue, so that y and dx are as large as they are.
// dA and dB gather the adapter's tokens by a list, for the same reason.
#include <algorithm>
#include <exception>

#include "half_gemm.h"
#include "mma16.cuh"
#include "packed.h"
#include "rank.h"

namespace cdclq {

namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t align_up(size_t b) { return (b + 255) & ~(size_t)255; }

// ---------------------------------------------------------------------------------------------------------------------
// Outer products of an adapter's tokens: out[c][k] = factor * sum_t wide[t][c] narrow[t][k], c over the wide matrix'
// columns, k over the rank: dA (wide = x, narrow = v) and dB (wide = dy, narrow = u) in one launch.  Work item: 128 columns,
// 64 ranks, one adapter, a chunk of its tokens.  An adapter of one chunk writes its result; the chunks of others go to f32
// slots that a second kernel adds in order.  Tokens are gathered by list into a ring in shared memory (asynchronous copies;
// a checkpoint's codes through registers) and transposed into fragments by ldmatrix; what lies past the chunk is zero.
// v is f32: it enters as the sum of two 16-bit numbers, so that dA's rounding is the one of its output: in bf16 off by 2^-17 of
// it at most; in f16, whose pairs end at 2^-24 and 2^16, under a gain that makes the adapter's largest |v| about 2^13 and comes
// off the sums (without it v of 3e-6 cost dA 5e-3 of its norm, v past 65504 everything): off by 2^-22, or 2^-38 of the largest.
// Bound by reading `wide`: the rank is small, so mma.sync keeps up with memory.  4100 tokens, x and dy of 4096 columns, rank 64
// in f16: 41 us alone (67 MB, 1.6 TB/s: at rank 64 the fragments' loads from shared memory take their share); it starts on the
// SMs that dx's product leaves first.  A second kernel of 8 us adds the chunks.
constexpr int OUTER_COLS = 128, OUTER_TOK = 32, OUTER_MOST = 1024, OUTER_RANK = 64, OUTER_STAGES = 4;

struct OuterArgs {
    const uint16_t* wide;      // [t][ldw] 16-bit, or null:
    const int8_t* codes;       // [t][cols] with
    const float* scales;       // [t][ceil(cols / 128)]
    int64_t ldw;
    int cols;
    int wide16;                // its rows can be read 16 bytes at a time
    const uint16_t* narrow;    // [t][ldn] 16-bit, and
    const uint16_t* rest;      // what is added to it, or null; with codes both are null:
    const float* narrow32;     // [t][r]
    const uint32_t* top;       // [n]: of the gain that narrow and rest have in f16 (rank_gain)
    int64_t ldn;
    int narrow16;              // its rows can be read 16 bytes at a time
    const float* factor;       // [n] or null
    uint16_t* out;             // dA: [n][r][cols], dB: [n][cols][r]
    int by_rank;               // the rank is the last index (dB)
    float* slots;              // [slot][r * cols], in the output's order
    int tiles;                 // column tiles; 0: not wanted
};
struct OuterPair {
    OuterArgs a, b;
    int r, n, t, chunk;
    const int* start;          // [n + 1] and more
    const int* order;
};

// Item -> (adapter, chunk, its chunks); slot: the item's place among those of adapters with several chunks.  A warp looks
// at 32 adapters at a time.
__device__ __forceinline__ bool outer_item(const OuterPair& P, int item, int lane, int& id, int& chunk, int& chunks, int& slot) {
    int at = 0, s = 0;
    for (int base = 0; base < P.n; base += 32) {
        const int i = base + lane;
        const int mine = i < P.n ? max(1, (P.start[i + 1] - P.start[i] + P.chunk - 1) / P.chunk) : 0;
        const int many = mine > 1 ? mine : 0;
        int sum = mine, msum = many;  // inclusive prefix sums
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o), w = __shfl_up_sync(0xffffffffu, msum, o);
            if (lane >= o) sum += v, msum += w;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, item < at + sum && i < P.n);
        if (past) {
            const int l = __ffs(past) - 1;
            id = base + l;
            chunks = __shfl_sync(0xffffffffu, mine, l);
            chunk = item - at - (__shfl_sync(0xffffffffu, sum, l) - chunks);
            slot = s + __shfl_sync(0xffffffffu, msum - many, l) + chunk;
            return true;
        }
        at += __shfl_sync(0xffffffffu, sum, 31);
        s += __shfl_sync(0xffffffffu, msum, 31);
    }
    return false;
}

// rows of 128 + 8 and 64 + 8 halves: 16-byte pieces of eight rows fall into different banks
struct OuterStage {
    uint16_t wide[OUTER_TOK][OUTER_COLS + 8];
    uint16_t high[OUTER_TOK][OUTER_RANK + 8];
    uint16_t low[OUTER_TOK][OUTER_RANK + 8];
};

// LOW: the narrow factor is high + low.  A checkpoint's codes and its v meet as bf16 whatever the type: codes are exact in it,
// and v times a block's scale keeps 16 bits however small or large it is.  (As f16 the pair ends at 2^-24: with v of 3e-6 da was
// off by a quarter of its norm.)
template <bool BF16, bool CODES, bool LOW>
__device__ __forceinline__ void outer_tile(const OuterPair& P, const OuterArgs& Q, OuterStage* ring, const int* list, int count, int id,
                                           int chunks, int slot, int tile, int k0) {
    constexpr bool AS_BF16 = BF16 || CODES, GAIN = LOW && !AS_BF16;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int c0 = tile * OUTER_COLS, ranks = min(OUTER_RANK, P.r - k0);
    const int steps = (count + OUTER_TOK - 1) / OUTER_TOK;
    const int row = tid >> 3, part = tid & 7, c = c0 + part * 16;  // 8 threads a token, with 16 columns and 8 ranks each
    const int in = min(8, ranks - part * 8);                       // of this thread's ranks
    // a warp's share: 32 columns, one half of a stage's tokens; the halves are added at the end
    const int m0 = (warp & 3) * 32, kk = (warp >> 2) * 16;
    float acc[2][8][4];
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int j = 0; j < 8; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[m][j][i] = 0.0f;

    auto token = [&](int s) {
        const int k = s * OUTER_TOK + row;
        return k < count ? list[k] : -1;
    };
    // 16-bit matrices: copies on their way to stage s
    auto copy = [&](int s) {
        const int tok = token(s);
        OuterStage& st = ring[s % OUTER_STAGES];
        const uint16_t* src = Q.wide + (int64_t)max(tok, 0) * Q.ldw + c;
        uint16_t* dst = &st.wide[row][part * 16];
        if (Q.wide16) {
            const bool first = tok >= 0 && c + 8 <= Q.cols, second = tok >= 0 && c + 16 <= Q.cols;
            copy16(dst, first ? src : Q.wide, first);
            copy16(dst + 8, second ? src + 8 : Q.wide, second);
        } else {
            for (int i = 0; i < 16; i++) dst[i] = (tok >= 0 && c + i < Q.cols) ? src[i] : (uint16_t)0;
        }
        const int64_t at = (int64_t)max(tok, 0) * Q.ldn + k0 + part * 8;
        uint16_t* high = &st.high[row][part * 8];
        uint16_t* low = &st.low[row][part * 8];
        if (Q.narrow16 && (in <= 0 || in == 8)) {
            const bool live = tok >= 0 && in > 0;
            // an address that is not read is on 16 bytes all the same, as `wide` may not be
            copy16(high, live ? Q.narrow + at : Q.narrow, live);
            if constexpr (LOW) copy16(low, live ? Q.rest + at : Q.rest, live);
        } else {
            for (int i = 0; i < 8; i++) {
                high[i] = (tok >= 0 && i < in) ? Q.narrow[at + i] : (uint16_t)0;
                if constexpr (LOW) low[i] = (tok >= 0 && i < in) ? Q.rest[at + i] : (uint16_t)0;
            }
        }
    };
    // a checkpoint: a thread's 16 codes and 8 ranks of its token, through registers
    float nv[8];
    uint4 qv = make_uint4(0, 0, 0, 0);
    auto fetch = [&](int s) {
        const int tok = token(s);
        const float f = tok >= 0 ? Q.scales[(int64_t)tok * ((Q.cols + 127) / 128) + tile] : 0.0f;
        const int8_t* src = Q.codes + (int64_t)max(tok, 0) * Q.cols + c;
        if (tok >= 0 && Q.wide16 && c + 16 <= Q.cols) {
            qv = *reinterpret_cast<const uint4*>(src);
        } else {
            alignas(16) int8_t q[16];
#pragma unroll
            for (int i = 0; i < 16; i++) q[i] = (tok >= 0 && c + i < Q.cols) ? src[i] : (int8_t)0;
            qv = *reinterpret_cast<uint4*>(q);
        }
        // a checkpoint's values are code * scale, one scale for these 128 columns: it joins the narrow factor, so that the
        // codes enter the tensor instruction exactly
        const float* v = Q.narrow32 + (int64_t)max(tok, 0) * P.r + k0 + part * 8;
#pragma unroll
        for (int i = 0; i < 8; i++) nv[i] = (tok >= 0 && i < in) ? v[i] * f : 0.0f;
    };
    auto put = [&](int s) {
        OuterStage& st = ring[s % OUTER_STAGES];
        alignas(16) uint16_t h[8], l[8], w[16];
        alignas(16) int8_t q[16];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            h[i] = half_bits<AS_BF16>(nv[i]);
            l[i] = rest_bits<AS_BF16>(nv[i], h[i]);
        }
        *reinterpret_cast<uint4*>(&st.high[row][part * 8]) = *reinterpret_cast<uint4*>(h);
        *reinterpret_cast<uint4*>(&st.low[row][part * 8]) = *reinterpret_cast<uint4*>(l);
        *reinterpret_cast<uint4*>(q) = qv;
#pragma unroll
        for (int i = 0; i < 16; i++) w[i] = half_bits<AS_BF16>((float)q[i]);
        uint16_t* dst = &st.wide[row][part * 16];
        reinterpret_cast<uint4*>(dst)[0] = reinterpret_cast<uint4*>(w)[0];
        reinterpret_cast<uint4*>(dst)[1] = reinterpret_cast<uint4*>(w)[1];
    };
    constexpr int AHEAD = OUTER_STAGES - 1;
#pragma unroll 1
    for (int s = 0; s < AHEAD; s++) {
        if (s < steps) {
            if constexpr (CODES) {
                fetch(s);
                put(s);
            } else {
                copy(s);
            }
        }
        copy_commit();
    }
    if constexpr (CODES) {
        if (AHEAD < steps) fetch(AHEAD);
    }
#pragma unroll 1
    for (int s = 0; s < steps; s++) {
        copy_wait<OUTER_STAGES - 2>();
        __syncthreads();  // stage s is there, and stage s - 1 has been used by every warp
        if constexpr (CODES) {
            if (s + AHEAD < steps) put(s + AHEAD);
            if (s + AHEAD + 1 < steps) fetch(s + AHEAD + 1);
        } else {
            if (s + AHEAD < steps) copy(s + AHEAD);
        }
        copy_commit();
        const OuterStage& st = ring[s % OUTER_STAGES];
        // A (16 columns x 16 tokens, twice) from token rows: transposed 8 x 8 pieces
        uint32_t a[2][4];
#pragma unroll
        for (int m = 0; m < 2; m++)
            load_pieces<true>(a[m], &st.wide[kk + (lane & 7) + ((lane >> 4) & 1) * 8][m0 + m * 16 + ((lane >> 3) & 1) * 8]);
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            if (j * 8 >= ranks) break;
#pragma unroll
            for (int low = 0; low < (LOW ? 2 : 1); low++) {
                uint32_t q[4];  // ranks j * 8 .. + 8, and the next 8
                load_pieces<true>(q, &(low ? st.low : st.high)[kk + (lane & 15)][j * 8 + (lane >> 4) * 8]);
#pragma unroll
                for (int m = 0; m < 2; m++) {
                    mma16816<AS_BF16>(acc[m][j], a[m], q[0], q[1]);
                    mma16816<AS_BF16>(acc[m][j + 1], a[m], q[2], q[3]);
                }
            }
        }
    }
    copy_wait<0>();
    __syncthreads();
    // both halves' sums in the ring's memory, in the output's order (dA: 128 columns a rank, dB: the ranks a column), so that
    // the CTA writes along the output's rows
    float* sum = reinterpret_cast<float*>(ring);
    const int ncols = min(OUTER_COLS, Q.cols - c0);
    const int pitch = Q.by_rank ? OUTER_RANK + 1 : OUTER_COLS + 4;
#pragma unroll
    for (int half = 1; half >= 0; half--) {
        if ((warp >> 2) == half) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (j * 8 >= ranks) break;
#pragma unroll
                for (int q = 0; q < 8; q++) {
                    const int cc = m0 + q / 4 * 16 + lane / 4 + (q >> 1 & 1) * 8, k = j * 8 + (lane & 3) * 2 + (q & 1);
                    float& v = sum[Q.by_rank ? cc * pitch + k : k * pitch + cc];
                    v = half ? acc[q / 4][j][q % 4] : v + acc[q / 4][j][q % 4];
                }
            }
        }
        __syncthreads();
    }
    const bool whole = chunks == 1;
    const float f = GAIN ? 1.0f / rank_gain(Q.top[id]) : (whole && Q.factor) ? Q.factor[id] : 1.0f;
    const int64_t base = (int64_t)(whole ? id : slot) * P.r * Q.cols;
    // rows of the output's piece, `len` long, `stride` apart; two neighbours a thread where rows start even
    const int lines = Q.by_rank ? ncols : ranks, len = Q.by_rank ? ranks : ncols;
    const int64_t stride = Q.by_rank ? P.r : Q.cols, origin = base + (Q.by_rank ? (int64_t)c0 * P.r + k0 : (int64_t)k0 * Q.cols + c0);
    const bool even = stride % 2 == 0 && len % 2 == 0 && (base & 1) == 0 && (reinterpret_cast<uintptr_t>(Q.out) & 3) == 0;
    const int per = even ? len / 2 : len;
    for (int i = tid; i < lines * per; i += 256) {
        const int line = i / per, e = (i - line * per) * (even ? 2 : 1);
        const float* v = sum + line * pitch + e;
        const int64_t at = origin + line * stride + e;
        if (whole) {
            if (even)
                *reinterpret_cast<uint32_t*>(Q.out + at) = (uint32_t)half_bits<BF16>(v[0] * f) | (uint32_t)half_bits<BF16>(v[1] * f) << 16;
            else
                Q.out[at] = half_bits<BF16>(v[0] * f);
        } else {
            Q.slots[at] = v[0] * f;
            if (even) Q.slots[at + 1] = v[1] * f;
        }
    }
}

template <bool BF16, bool CODES>
__global__ void __launch_bounds__(256) outer_kernel(const OuterPair P) {
    extern __shared__ __align__(16) unsigned char smem[];
    OuterStage* ring = reinterpret_cast<OuterStage*>(smem);
    __shared__ int list[OUTER_MOST];
    __shared__ int which[4];
    if (threadIdx.x < 32) {
        int id = 0, chunk = 0, chunks = 0, slot = 0;
        const bool any = outer_item(P, blockIdx.y, threadIdx.x, id, chunk, chunks, slot);
        if (threadIdx.x == 0) which[0] = any ? id : -1, which[1] = chunk, which[2] = chunks, which[3] = slot;
    }
    __syncthreads();
    const int id = which[0], chunks = which[2], slot = which[3];
    if (id < 0) return;
    const int first = P.start[id] + which[1] * P.chunk, count = max(0, min(P.start[id + 1] - first, P.chunk));
    for (int i = threadIdx.x; i < count; i += 256) list[i] = P.order[first + i];
    __syncthreads();
    const int k0 = blockIdx.z * OUTER_RANK;
    if ((int)blockIdx.x < P.a.tiles)
        outer_tile<BF16, CODES, true>(P, P.a, ring, list, count, id, chunks, slot, blockIdx.x, k0);
    else
        outer_tile<BF16, false, false>(P, P.b, ring, list, count, id, chunks, slot, blockIdx.x - P.a.tiles, k0);
    if (blockIdx.x + blockIdx.y + blockIdx.z == 0) wait_for_previous();
}

// The adapters of several chunks: out = factor * (slot 0 + slot 1 + ...), four neighbouring values a thread.
template <bool BF16>
__global__ void __launch_bounds__(256) outer_finish_kernel(const OuterPair P) {
    const OuterArgs& Q = blockIdx.z ? P.b : P.a;
    if (!Q.tiles) return;
    const int id = blockIdx.y;
    __shared__ int before;
    if (threadIdx.x < 32) {
        int s = 0;
        for (int i = threadIdx.x; i < id; i += 32) {
            const int chunks = (P.start[i + 1] - P.start[i] + P.chunk - 1) / P.chunk;
            s += chunks > 1 ? chunks : 0;
        }
        s = __reduce_add_sync(0xffffffffu, s);
        if (threadIdx.x == 0) before = s;
    }
    __syncthreads();
    const int chunks = (P.start[id + 1] - P.start[id] + P.chunk - 1) / P.chunk;
    if (chunks <= 1) return;
    const float f = Q.factor ? Q.factor[id] : 1.0f;
    const int64_t total = (int64_t)P.r * Q.cols;
    const float* src = Q.slots + before * total;
    uint16_t* out = Q.out + id * total;
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        float s = 0.0f;
#pragma unroll 4
        for (int q = 0; q < chunks; q++) s += src[q * total + i];
        out[i] = half_bits<BF16>(s * f);
    }
}

// Tokens of a chunk: as many as leave two CTAs to an SM over both products' column tiles, 128 at least (a shorter chunk's sums
// would weigh as much as its tokens), OUTER_MOST at most.  Backward of 4100 tokens, rank 64: 191 us so, 190 with three CTAs to an
// SM and 201 with four; 2048 tokens, rank 16: 81.6, 81.5 and 86.
int outer_chunk(int64_t t, int64_t tiles, int64_t r) {
    int chunk = OUTER_MOST;
    while (chunk > 128 && ceil_div(t, chunk) * tiles * ceil_div(r, OUTER_RANK) < 2 * sm_count()) chunk /= 2;
    return chunk;
}
// Slots of adapters with several chunks: each such adapter has over `chunk` tokens, so it has fewer than 2 tokens / chunk.
int64_t outer_slots(int64_t t, int chunk) { return 2 * t / chunk; }

// beside: the launch before this one is not the one that made its factors or lists.
int launch_outer(bool bf16, const OuterPair& p, bool beside, cudaStream_t st) {
    // an adapter without tokens still writes its zeros: one item each
    const int64_t items = ceil_div(p.t, p.chunk) + p.n, tiles = p.a.tiles + p.b.tiles;
    if (items > 65535) return set_error(CDCLQ_ERR_ARG, "adapters: too many tokens or adapters for one call");
    const dim3 grid((unsigned)tiles, (unsigned)items, (unsigned)ceil_div(p.r, OUTER_RANK));
    const size_t smem = OUTER_STAGES * sizeof(OuterStage);
    static std::atomic<uint64_t> done[4];
    const int which = (bf16 ? 2 : 0) + (p.a.codes ? 1 : 0);
    auto kern = bf16 ? (p.a.codes ? outer_kernel<true, true> : outer_kernel<true, false>)
                     : (p.a.codes ? outer_kernel<false, true> : outer_kernel<false, false>);
    if (int rc = allow_smem(kern, smem, done[which], "outer_kernel shared memory")) return rc;
    if (int rc = launch_after(beside, kern, grid, dim3(256), smem, st, "outer_kernel launch", p)) return rc;
    if (outer_slots(p.t, p.chunk) > 0) {
        const int64_t most = (int64_t)p.r * std::max(p.a.cols, p.b.cols);
        const unsigned gx = (unsigned)std::max<int64_t>(1, std::min<int64_t>(ceil_div(most, 256), sm_count() * 4));
        auto fin = bf16 ? outer_finish_kernel<true> : outer_finish_kernel<false>;
        CDCLQ_LAUNCH(fin, dim3(gx, p.n, 2), 256, 0, st, p);
    }
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : cuda_error(e, "adapters' outer products launch");
}

// ---------------------------------------------------------------------------------------------------------------------

struct Space {
    size_t at = 0;
    size_t take(size_t bytes) {
        const size_t here = at;
        at += align_up(bytes);
        return here;
    }
};

struct ForwardLayout {
    size_t expanded = 0, ranked = 0, ranked32 = 0, past = 0, lists = 0, start = 0, order = 0, partial = 0, decode = 0, total = 0;
};
ForwardLayout forward_layout(const PackedView& w, int64_t t, int64_t n, int64_t r) {
    ForwardLayout l;
    Space s;
    if (t <= DECODE_TOKENS) {
        l.decode = s.take(packed_decode_workspace(w, (int)t, n ? (int)r : 0));
    } else {
        l.expanded = s.take((size_t)w.d_out * ceil_div(w.d_in, 8) * 8 * 2);
        const HalfPlan plan = plan_half_gemm(HALF_NT_EXTEND, t, w.d_out, w.d_in);
        if (n) l.ranked = s.take((size_t)t * ceil_div(r, 8) * 8 * 2);
        if (n) l.ranked32 = s.take((size_t)t * r * sizeof(float));
        if (n) l.past = s.take((size_t)t * sizeof(int));
        if (n) l.lists = s.take(row_lists_bytes(plan, t));
        if (n) l.start = s.take((size_t)(n + 2) * sizeof(int));
        if (n) l.order = s.take((size_t)t * sizeof(int));
        l.partial = s.take(plan.partial_bytes);
    }
    l.total = s.at;
    return l;
}

struct BackwardLayout {
    size_t expanded = 0, ranked = 0, lists = 0, high = 0, rest = 0, ranked32 = 0, past = 0, top = 0, partial = 0, start = 0, order = 0, slots_a = 0, slots_b = 0, total = 0;
};
BackwardLayout backward_layout(const PackedView& w, int64_t t, int64_t n, int64_t r, bool need_dx) {
    BackwardLayout l;
    Space s;
    size_t partial = 0;
    if (need_dx) {
        l.expanded = s.take((size_t)w.d_out * ceil_div(w.d_in, 8) * 8 * 2);
        const HalfPlan plan = plan_half_gemm(HALF_NN_EXTEND, t, w.d_in, w.d_out);
        if (n) l.lists = s.take(row_lists_bytes(plan, t));
        partial = plan.partial_bytes;
    }
    if (n) {
        l.ranked = s.take((size_t)t * ceil_div(r, 8) * 8 * 2);
        l.start = s.take((size_t)(n + 2) * sizeof(int));
        l.order = s.take((size_t)t * sizeof(int));
        l.high = s.take((size_t)t * ceil_div(r, 8) * 8 * 2);
        l.rest = s.take((size_t)t * ceil_div(r, 8) * 8 * 2);
        l.ranked32 = s.take((size_t)t * r * sizeof(float));
        l.past = s.take((size_t)t * sizeof(int));
        l.top = s.take((size_t)n * sizeof(uint32_t));
        // fewer column tiles, where only one of the two is wanted, may shorten the chunk and so make more slots
        const int chunk = outer_chunk(t, ceil_div(w.d_in, OUTER_COLS) + ceil_div(w.d_out, OUTER_COLS), r);
        const size_t slots = (size_t)outer_slots(t, std::min(chunk, outer_chunk(t, ceil_div(std::min(w.d_in, w.d_out), OUTER_COLS), r)));
        l.slots_a = s.take(slots * r * w.d_in * sizeof(float));
        l.slots_b = s.take(slots * r * w.d_out * sizeof(float));
    }
    l.partial = s.take(partial);
    l.total = s.at;
    return l;
}

HalfOperand operand(const void* p, int64_t rows, int64_t cols, int64_t ld, int64_t batch = 1) {
    HalfOperand o;
    o.p = p;
    o.rows = rows;
    o.cols = cols;
    o.ld = ld;
    o.batch = batch;
    o.step = batch > 1 ? rows * ld : 0;
    return o;
}

FarRows far_rows(const void* past, const int* index, const void* u32, const HalfOperand& x) {
    FarRows f;
    f.past = static_cast<const int*>(past);
    f.index = index;
    f.u = static_cast<const float*>(u32);
    f.x = static_cast<const uint16_t*>(x.p);
    f.ld = x.ld, f.step = x.step;
    return f;
}

bool aligned(const void* p, size_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0; }

constexpr size_t MOST_ADAPTERS = 32767, MOST_RANK = 4096;

// Whether a call of these sizes is refused: it has no workspace.
bool refused(const cdclq_packed_layer* w, size_t t, size_t n, size_t r) {
    return !w || !t || !w->d_out || !w->d_in || t > MOST_SIZE || n > MOST_ADAPTERS || (n && (!r || r > MOST_RANK));
}

int check_call(const char* what, const cdclq_packed_layer* w, int dtype, size_t t, const cdclq_adapters* ad) {
    const std::string s(what);
    if (!w || !w->layout || !w->d_out || !w->d_in) return set_error(CDCLQ_ERR_ARG, s + ": no packed layer");
    if (dtype != CDCLQ_DTYPE_F16 && dtype != CDCLQ_DTYPE_BF16) return set_error(CDCLQ_ERR_ARG, s + ": dtype must be f16 or bf16");
    if (t > MOST_SIZE) return set_error(CDCLQ_ERR_ARG, s + ": too many tokens");
    if (ad && ad->n) {
        if (!ad->r) return set_error(CDCLQ_ERR_ARG, s + ": the adapters' rank must be > 0");
        if (ad->n > MOST_ADAPTERS || ad->r > MOST_RANK) return set_error(CDCLQ_ERR_ARG, s + ": too many adapters, or too high a rank");
        if (!ad->a || !ad->b || !ad->scale || (t && !ad->index)) return set_error(CDCLQ_ERR_ARG, s + ": null pointer");
        if (ad->lda < w->d_in || ad->ldb < ad->r || !aligned(ad->a, ad->lda) || !aligned(ad->b, ad->ldb))
            return set_error(CDCLQ_ERR_ARG, s + ": rows of a and b must start on 16 bytes and not overlap");
    }
    return check_fail_word(what);
}

}  // namespace

}  // namespace cdclq

using namespace cdclq;

extern "C" size_t cdclq_projection_forward_workspace(const cdclq_packed_layer* w, size_t t, size_t n, size_t r) {
    if (refused(w, t, n, r)) return 0;
    return forward_layout(packed_view(*w), t, n, n ? r : 0).total;
}

extern "C" int cdclq_projection_forward_device(const cdclq_packed_layer* w, const void* x, size_t ldx, int dtype, size_t t,
                                               const cdclq_adapters* ad, void* y, size_t ldy, void* u, void* workspace,
                                               size_t workspace_bytes, void* stream) {
    int rc = check_call("projection_forward", w, dtype, t, ad);
    if (rc || !t) return rc;
    if (!x || !y || ldy < w->d_out) return set_error(CDCLQ_ERR_ARG, "projection_forward: null pointer, or rows of y overlap");
    if (ldx < w->d_in || !aligned(x, ldx)) return set_error(CDCLQ_ERR_ARG, "projection_forward: rows of x must start on 16 bytes");
    const int64_t n = ad ? (int64_t)ad->n : 0, r = n ? (int64_t)ad->r : 0;
    const PackedView v = packed_view(*w);
    const ForwardLayout l = forward_layout(v, t, n, r);
    if (!workspace || workspace_bytes < l.total) return set_error(CDCLQ_ERR_ARG, "projection_forward: the workspace is too small");
    char* ws = static_cast<char*>(workspace);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool bf16 = dtype == CDCLQ_DTYPE_BF16;
    if (t <= DECODE_TOKENS) {
        AdapterArgs a{};
        if (n) a = {ad->a, ad->b, (int64_t)ad->lda, (int64_t)ad->ldb, ad->scale, ad->index, (int)n, (int)r};
        return launch_packed_decode(v, bf16, x, ldx, (int)t, a, y, ldy, n ? u : nullptr, ws + l.decode, st);
    }
    const int64_t ldw = ceil_div(v.d_in, 8) * 8, ldr = ceil_div(r, 8) * 8;
    float* partial = reinterpret_cast<float*>(ws + l.partial);
    if (n) {
        RankArgs p{};
        p.x = static_cast<const uint16_t*>(x);
        p.ldx = ldx;
        p.t = (int)t, p.k = v.d_in;
        p.m = static_cast<const uint16_t*>(ad->a);
        p.ldm = ad->lda;
        p.index = ad->index;
        p.n = (int)n, p.r = (int)r;
        p.scale = ad->scale;
        p.u16 = static_cast<uint16_t*>(u);
        p.ldu = r;
        p.su16 = reinterpret_cast<uint16_t*>(ws + l.ranked);
        p.lds = ldr;
        if (!bf16) {
            p.su32 = reinterpret_cast<float*>(ws + l.ranked32);
            p.past = reinterpret_cast<int*>(ws + l.past);
        }
        p.start = reinterpret_cast<int*>(ws + l.start);
        p.order = reinterpret_cast<int*>(ws + l.order);
        if ((rc = launch_rank(bf16, false, p, st))) return rc;
    }
    const HalfPlan plan = plan_half_gemm(HALF_NT_EXTEND, t, v.d_out, v.d_in);
    const RowLists lists = n ? row_lists(plan, ad->index, t, n, ws + l.lists) : RowLists();
    if ((rc = launch_packed_expand(v, bf16, ws + l.expanded, ldw, lists, RankSplit(), n > 0, st))) return rc;  // beside u's products
    HalfGemm g{};
    g.form = HALF_NT_EXTEND;
    g.bf16 = bf16;
    g.m = t, g.n = v.d_out, g.k = v.d_in;
    g.a = operand(x, t, v.d_in, ldx);
    g.b = operand(ws + l.expanded, v.d_out, v.d_in, ldw);
    if (n) {
        g.u = operand(ws + l.ranked, t, r, ldr);
        g.x = operand(ad->b, v.d_out, r, ad->ldb, n);
        g.lists = lists.out;
        if (!bf16) g.far = far_rows(ws + l.past, ad->index, ws + l.ranked32, g.x);
    }
    g.out = y;
    g.ldo = ldy;
    g.partial = partial;
    return launch_half_gemm(g, plan, st);
}

extern "C" size_t cdclq_projection_backward_workspace(const cdclq_packed_layer* w, size_t t, size_t n, size_t r, int need_dx) {
    if (refused(w, t, n, r)) return 0;
    return backward_layout(packed_view(*w), t, n, n ? r : 0, need_dx != 0).total;
}

extern "C" int cdclq_projection_backward_device(const cdclq_packed_layer* w, const void* dy, size_t lddy, int dtype, size_t t,
                                                const cdclq_adapters* ad, const void* x, size_t ldx, const int8_t* x_codes,
                                                const float* x_scales, const void* u, void* dx, size_t lddx, void* da, void* db,
                                                void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_call("projection_backward", w, dtype, t, ad);
    if (rc) return rc;
    const int64_t n = ad ? (int64_t)ad->n : 0, r = n ? (int64_t)ad->r : 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const PackedView v = packed_view(*w);
    if (dx && lddx < w->d_in) return set_error(CDCLQ_ERR_ARG, "projection_backward: rows of dx overlap");
    if (!t) {
        if (n && da) CDCLQ_CUDA_TRY(cudaMemsetAsync(da, 0, (size_t)n * r * v.d_in * 2, st));
        if (n && db) CDCLQ_CUDA_TRY(cudaMemsetAsync(db, 0, (size_t)n * r * v.d_out * 2, st));
        return 0;
    }
    if (!dy || lddy < w->d_out || !aligned(dy, lddy)) return set_error(CDCLQ_ERR_ARG, "projection_backward: rows of dy must start on 16 bytes");
    if (n && da && !x && !(x_codes && x_scales)) return set_error(CDCLQ_ERR_ARG, "projection_backward: the gradient of a needs x");
    if (n && da && x && ldx < w->d_in) return set_error(CDCLQ_ERR_ARG, "projection_backward: rows of x overlap");
    if (n && db && !u) return set_error(CDCLQ_ERR_ARG, "projection_backward: the gradient of b needs u");
    const BackwardLayout l = backward_layout(v, t, n, r, dx != nullptr);
    if (!workspace || workspace_bytes < l.total) return set_error(CDCLQ_ERR_ARG, "projection_backward: the workspace is too small");
    char* ws = static_cast<char*>(workspace);
    const bool bf16 = dtype == CDCLQ_DTYPE_BF16;
    const int64_t ldw = ceil_div(v.d_in, 8) * 8, ldr = ceil_div(r, 8) * 8;
    float* partial = reinterpret_cast<float*>(ws + l.partial);
    RankSplit split;  // dA's v in f16
    if (n) {
        RankArgs p{};
        p.x = static_cast<const uint16_t*>(dy);
        p.ldx = lddy;
        p.t = (int)t, p.k = v.d_out;
        p.m = static_cast<const uint16_t*>(ad->b);
        p.ldm = ad->ldb;
        p.index = ad->index;
        p.n = (int)n, p.r = (int)r;
        p.scale = ad->scale;
        p.lds = ldr;
        if (dx || da) p.su16 = reinterpret_cast<uint16_t*>(ws + l.ranked);
        if (da && x && bf16) p.rest16 = reinterpret_cast<uint16_t*>(ws + l.rest);
        if ((da && !x) || ((dx || da) && !bf16)) p.su32 = reinterpret_cast<float*>(ws + l.ranked32);
        if (dx && !bf16) p.past = reinterpret_cast<int*>(ws + l.past);
        if (da && x && !bf16) {
            p.top = reinterpret_cast<uint32_t*>(ws + l.top);
            split.v = p.su32, split.top = p.top, split.index = ad->index;
            split.t = (int)t, split.n = (int)n, split.r = (int)r;
            split.high = reinterpret_cast<uint16_t*>(ws + l.high), split.low = reinterpret_cast<uint16_t*>(ws + l.rest);
            split.ld = ldr;
        }
        p.start = reinterpret_cast<int*>(ws + l.start);
        p.order = reinterpret_cast<int*>(ws + l.order);
        if ((rc = launch_rank(bf16, true, p, st))) return rc;
        if (!dx && split.v && (rc = launch_rank_split(split, st))) return rc;
    }
    const HalfPlan plan = plan_half_gemm(HALF_NN_EXTEND, t, v.d_in, v.d_out);
    if (dx) {
        const RowLists lists = n ? row_lists(plan, ad->index, t, n, ws + l.lists) : RowLists();
        if ((rc = launch_packed_expand(v, bf16, ws + l.expanded, ldw, lists, split, n > 0, st))) return rc;  // beside v's products
        HalfGemm g{};
        g.form = HALF_NN_EXTEND;
        g.bf16 = bf16;
        g.m = t, g.n = v.d_in, g.k = v.d_out;
        g.a = operand(dy, t, v.d_out, lddy);
        g.b = operand(ws + l.expanded, v.d_out, v.d_in, ldw);
        if (n) {
            g.u = operand(ws + l.ranked, t, r, ldr);
            g.x = operand(ad->a, r, v.d_in, ad->lda, n);
            g.lists = lists.out;
            if (!bf16) g.far = far_rows(ws + l.past, ad->index, ws + l.ranked32, g.x);
        }
        g.out = dx;
        g.ldo = lddx;
        g.partial = partial;
        if ((rc = launch_half_gemm(g, plan, st))) return rc;
    }
    if (!n || !(da || db)) return 0;
    OuterPair o{};
    o.r = (int)r, o.n = (int)n, o.t = (int)t;
    o.start = reinterpret_cast<const int*>(ws + l.start);
    o.order = reinterpret_cast<const int*>(ws + l.order);
    if (da) {
        o.a.wide = static_cast<const uint16_t*>(x);
        if (!x) o.a.codes = x_codes, o.a.scales = x_scales;
        o.a.ldw = ldx;
        o.a.cols = v.d_in;
        o.a.wide16 = x ? ldx % 8 == 0 && v.d_in % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0
                       : v.d_in % 16 == 0 && (reinterpret_cast<uintptr_t>(x_codes) & 15) == 0;
        if (x) {
            o.a.narrow = split.v ? split.high : reinterpret_cast<const uint16_t*>(ws + l.ranked);
            o.a.top = split.top;
            o.a.rest = reinterpret_cast<const uint16_t*>(ws + l.rest);
            o.a.ldn = ldr;
            o.a.narrow16 = r % 8 == 0;
        } else {
            o.a.narrow32 = reinterpret_cast<const float*>(ws + l.ranked32);
        }
        o.a.out = static_cast<uint16_t*>(da);
        o.a.slots = reinterpret_cast<float*>(ws + l.slots_a);
        o.a.tiles = (int)ceil_div(v.d_in, OUTER_COLS);
    }
    if (db) {
        o.b.wide = static_cast<const uint16_t*>(dy);
        o.b.ldw = lddy;
        o.b.cols = v.d_out;
        o.b.wide16 = v.d_out % 8 == 0;  // the rows start on 16 bytes
        o.b.narrow = static_cast<const uint16_t*>(u);
        o.b.ldn = r;
        o.b.narrow16 = r % 8 == 0 && (reinterpret_cast<uintptr_t>(u) & 15) == 0;
        o.b.factor = ad->scale;
        o.b.out = static_cast<uint16_t*>(db);
        o.b.by_rank = 1;
        o.b.slots = reinterpret_cast<float*>(ws + l.slots_b);
        o.b.tiles = (int)ceil_div(v.d_out, OUTER_COLS);
    }
    o.chunk = outer_chunk(t, o.a.tiles + o.b.tiles, r);
    // dx's product stands between them, unless its sums were split: then the kernel that joins them does
    return launch_outer(bf16, o, dx && plan.splits == 1, st);
}

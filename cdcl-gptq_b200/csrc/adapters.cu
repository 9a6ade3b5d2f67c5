// adapters.cu - low-rank adapters of many requests beside a shared packed projection.
//
//   u_t = A_i x_t        y_t = W x_t + s_i B_i u_t                               i = index[t], none for an index outside [0, n)
//   v_t = s_i B_i^T dy_t     dx_t = W^T dy_t + A_i^T v_t     dA_i = sum_{t in i} v_t x_t^T     dB_i = s_i sum_{t in i} dy_t u_t^T
//
// A few tokens (packed.cu): the codes are read once, W is never formed.  More tokens: W is expanded once to 16 bits, which
// stays in L2 for the layers of a model, and multiplied on the tensor cores; the adapters ride in the same accumulators as
// further K blocks, whose MMAs write only the tensor-memory lanes of the adapter's own tokens.  So a request never meets
// another one's adapter, not even as a product with zero: a NaN in one adapter or one request stays there.
// dA and dB gather the adapter's tokens by a list, for the same reason.
#include <algorithm>
#include <exception>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "half_gemm.h"
#include "packed.h"

namespace cdclq {

namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t align_up(size_t b) { return (b + 255) & ~(size_t)255; }

template <bool BF16>
__device__ __forceinline__ uint16_t half_bits(float v) {
    return BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}

// The f32 sums of a grouped product, splits in order: u16 = sum, su16 = scale of the row's adapter times sum (either may be
// null; ldu and lds elements from row to row).
template <bool BF16>
__global__ void __launch_bounds__(256) rank_finish_kernel(const float* __restrict__ partial, int splits, int t, int r, int ldp,
                                                          const int* __restrict__ index, int n, const float* __restrict__ scale,
                                                          uint16_t* __restrict__ u16, int ldu, uint16_t* __restrict__ su16, int lds) {
    const int64_t total = (int64_t)t * r;
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t row = i / r;
        const int c = (int)(i - row * r);
        float s = 0.0f;
        for (int k = 0; k < splits; k++) s += partial[((int64_t)k * t + row) * ldp + c];
        if (u16) u16[row * ldu + c] = half_bits<BF16>(s);
        if (su16) {
            const int id = index[row];
            su16[row * lds + c] = half_bits<BF16>((id >= 0 && id < n) ? scale[id] * s : 0.0f);
        }
    }
}

// Each adapter's tokens in ascending order, one CTA an adapter: start[i] = tokens of lower adapters.
__global__ void __launch_bounds__(1024) token_lists_kernel(const int* __restrict__ index, int t, int n, int* __restrict__ start,
                                                           int* __restrict__ order) {
    __shared__ int below[32], mine[32];
    const int id = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int lower = 0;
    for (int i = threadIdx.x; i < t; i += 1024) {
        const int v = index[i];
        lower += v >= 0 && v < id;
    }
    lower = __reduce_add_sync(0xffffffffu, lower);
    if (lane == 0) below[warp] = lower;
    __syncthreads();
    int at = 0;
    for (int w = 0; w < 32; w++) at += below[w];
    if (threadIdx.x == 0) start[id] = at;
    for (int base = 0; base < t; base += 1024) {
        const int i = base + threadIdx.x;
        const bool hit = i < t && index[i] == id;
        const uint32_t m = __ballot_sync(0xffffffffu, hit);
        if (lane == 0) mine[warp] = __popc(m);
        __syncthreads();
        int before = at, all = 0;
        for (int w = 0; w < 32; w++) {
            if (w < warp) before += mine[w];
            all += mine[w];
        }
        if (hit) order[before + __popc(m & ((1u << lane) - 1u))] = i;
        at += all;
        __syncthreads();
    }
    if (id == n - 1 && threadIdx.x == 0) start[n] = at;
}

// ---------------------------------------------------------------------------------------------------------------------
// Outer products of an adapter's tokens: out[c][k] = factor * sum_t wide[t][c] narrow[t][k], c over the wide matrix'
// columns, k over the rank.  Work item: 128 columns of c, one adapter, up to OUTER_CHUNK of its tokens.  An adapter of one
// chunk writes its result; the chunks of others go to f32 slots that a second kernel adds in order.  Tokens are gathered by
// list into shared memory (transposed into fragments by ldmatrix); a token past the chunk's end is a row of zeros.
// Bound by reading `wide`: the rank is small, so mma.sync keeps up with memory.
constexpr int OUTER_COLS = 128, OUTER_TOK = 32, OUTER_CHUNK = 512, OUTER_RANK = 64;

struct OuterArgs {
    const uint16_t* wide;      // [t][ldw] 16-bit, or null:
    const int8_t* codes;       // [t][cols] with
    const float* scales;       // [t][ceil(cols / 128)]
    int64_t ldw;
    int cols;
    const uint16_t* narrow;    // [t][ldn]
    int64_t ldn;
    int r, n, t;
    const int* start;          // [n + 1]
    const int* order;
    const float* factor;       // [n] or null
    uint16_t* out;             // element (i, c, k) at i * out_i + c * out_c + k * out_k
    int64_t out_i, out_c, out_k;
    float* slots;              // [slot][r rounded up to 64][cols]
    int slot_rank;
};

// The chunk items of all adapters in order; item -> (adapter, chunk).  slot: the item's place among those of adapters with
// several chunks.
__device__ __forceinline__ bool outer_item(const OuterArgs& P, int item, int& id, int& chunk, int& chunks, int& slot) {
    int at = 0, s = 0;
    for (id = 0; id < P.n; id++) {
        const int count = P.start[id + 1] - P.start[id];
        chunks = max(1, (count + OUTER_CHUNK - 1) / OUTER_CHUNK);
        if (item < at + chunks) {
            chunk = item - at;
            slot = s + chunk;
            return true;
        }
        at += chunks;
        if (chunks > 1) s += chunks;
    }
    return false;
}

template <bool BF16, bool CODES>
__global__ void __launch_bounds__(256) outer_kernel(const OuterArgs P) {
    // rows of 128 + 8 and 64 + 8 halves: 16-byte pieces of eight rows fall into different banks
    __shared__ __align__(16) uint16_t wide[2][OUTER_TOK][OUTER_COLS + 8];
    __shared__ __align__(16) uint16_t narrow[2][OUTER_TOK][OUTER_RANK + 8];
    __shared__ int which[4];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        int id = 0, chunk = 0, chunks = 0, slot = 0;
        which[0] = outer_item(P, blockIdx.y, id, chunk, chunks, slot) ? id : -1;
        which[1] = chunk, which[2] = chunks, which[3] = slot;
    }
    __syncthreads();
    const int id = which[0], chunk = which[1], chunks = which[2], slot = which[3];
    if (id < 0) return;
    const int c0 = blockIdx.x * OUTER_COLS, k0 = blockIdx.z * OUTER_RANK;
    const int first = P.start[id] + chunk * OUTER_CHUNK, last = min(P.start[id + 1], first + OUTER_CHUNK);
    const int ranks = min(OUTER_RANK, P.r - k0);
    const int nb = (P.cols + 127) / 128;
    float acc[8][4];
#pragma unroll
    for (int j = 0; j < 8; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[j][i] = 0.0f;

    auto load = [&](int b, int at) {
        // wide: 8 threads a token, 16 columns each; narrow: 8 columns each
        const int row = tid >> 3, part = tid & 7, k = at + row;
        const int tok = k < last ? P.order[k] : -1;
        float s = 1.0f;
        uint16_t* dst = &wide[b][row][part * 16];
        const int c = c0 + part * 16;
        if constexpr (CODES) {
            if (tok >= 0) s = P.scales[(int64_t)tok * nb + c0 / 128];
            const int8_t* src = P.codes + (int64_t)(tok < 0 ? 0 : tok) * P.cols + c;
            alignas(16) uint16_t v[16];
            if (tok >= 0 && c + 16 <= P.cols && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
                alignas(16) int8_t q[16];
                *reinterpret_cast<uint4*>(q) = *reinterpret_cast<const uint4*>(src);
#pragma unroll
                for (int i = 0; i < 16; i++) v[i] = half_bits<BF16>((float)q[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 16; i++) v[i] = (tok >= 0 && c + i < P.cols) ? half_bits<BF16>((float)src[i]) : (uint16_t)0;
            }
            reinterpret_cast<uint4*>(dst)[0] = reinterpret_cast<uint4*>(v)[0];
            reinterpret_cast<uint4*>(dst)[1] = reinterpret_cast<uint4*>(v)[1];
        } else {
            const uint16_t* src = P.wide + (int64_t)(tok < 0 ? 0 : tok) * P.ldw + c;
            if (tok >= 0 && c + 16 <= P.cols && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
                reinterpret_cast<uint4*>(dst)[0] = reinterpret_cast<const uint4*>(src)[0];
                reinterpret_cast<uint4*>(dst)[1] = reinterpret_cast<const uint4*>(src)[1];
            } else {
                for (int i = 0; i < 16; i++) dst[i] = (tok >= 0 && c + i < P.cols) ? src[i] : (uint16_t)0;
            }
        }
        const uint16_t* nsrc = P.narrow + (int64_t)(tok < 0 ? 0 : tok) * P.ldn + k0 + part * 8;
        uint16_t* ndst = &narrow[b][row][part * 8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            uint16_t v = (tok >= 0 && part * 8 + i < ranks) ? nsrc[i] : (uint16_t)0;
            if constexpr (CODES) {
                // a checkpoint's values are code * scale, one scale for these 128 columns: it joins the narrow factor, so
                // that the codes enter the tensor instruction exactly
                const float f = BF16 ? __uint_as_float((uint32_t)v << 16) : __half2float(__ushort_as_half(v));
                v = tok >= 0 ? half_bits<BF16>(f * s) : (uint16_t)0;
            }
            ndst[i] = v;
        }
    };

    int b = 0;
    if (first < last) load(0, first);
    __syncthreads();
    for (int at = first; at < last; at += OUTER_TOK, b ^= 1) {
        if (at + OUTER_TOK < last) load(b ^ 1, at + OUTER_TOK);
        const int m0 = warp * 16;
#pragma unroll
        for (int kk = 0; kk < OUTER_TOK; kk += 16) {
            // A (16 columns x 16 tokens) from token rows: transposed 8 x 8 pieces
            uint32_t a[4];
            const uint32_t pa = (uint32_t)__cvta_generic_to_shared(&wide[b][kk + (lane & 7) + ((lane >> 4) & 1) * 8][m0 + ((lane >> 3) & 1) * 8]);
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                         : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
                         : "r"(pa));
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (j * 8 >= ranks) break;
                uint32_t q0, q1;
                const uint32_t pb = (uint32_t)__cvta_generic_to_shared(&narrow[b][kk + (lane & 15)][j * 8]);
                asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];" : "=r"(q0), "=r"(q1) : "r"(pb));
                if constexpr (BF16)
                    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                                 : "+f"(acc[j][0]), "+f"(acc[j][1]), "+f"(acc[j][2]), "+f"(acc[j][3])
                                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(q0), "r"(q1));
                else
                    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                                 : "+f"(acc[j][0]), "+f"(acc[j][1]), "+f"(acc[j][2]), "+f"(acc[j][3])
                                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(q0), "r"(q1));
            }
        }
        __syncthreads();
    }
    const float f = (chunks == 1 && P.factor) ? P.factor[id] : 1.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int c = c0 + warp * 16 + lane / 4 + (i >> 1) * 8, k = j * 8 + (lane & 3) * 2 + (i & 1);
            if (k >= ranks || c >= P.cols) continue;
            if (chunks == 1)
                P.out[id * P.out_i + c * P.out_c + (k0 + k) * P.out_k] = half_bits<BF16>(acc[j][i] * f);
            else
                P.slots[((int64_t)slot * P.slot_rank + k0 + k) * P.cols + c] = acc[j][i];
        }
    }
}

// The adapters of several chunks: out = factor * (slot 0 + slot 1 + ...).
template <bool BF16>
__global__ void __launch_bounds__(256) outer_finish_kernel(const OuterArgs P) {
    const int id = blockIdx.y;
    int slot = 0;
    for (int i = 0; i < id; i++) {
        const int chunks = (P.start[i + 1] - P.start[i] + OUTER_CHUNK - 1) / OUTER_CHUNK;
        if (chunks > 1) slot += chunks;
    }
    const int chunks = (P.start[id + 1] - P.start[id] + OUTER_CHUNK - 1) / OUTER_CHUNK;
    if (chunks <= 1) return;
    const float f = P.factor ? P.factor[id] : 1.0f;
    const int64_t total = (int64_t)P.r * P.cols;
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        // neighbouring threads along the output's contiguous index
        const int64_t k = P.out_k == 1 ? i % P.r : i / P.cols, c = P.out_k == 1 ? i / P.r : i % P.cols;
        float s = 0.0f;
        for (int q = 0; q < chunks; q++) s += P.slots[((int64_t)(slot + q) * P.slot_rank + k) * P.cols + c];
        P.out[id * P.out_i + c * P.out_c + k * P.out_k] = half_bits<BF16>(s * f);
    }
}

// Slots of adapters with several chunks: each such adapter has over OUTER_CHUNK tokens, so chunks <= 2 tokens / OUTER_CHUNK.
int64_t outer_slots(int64_t t) { return 2 * t / OUTER_CHUNK; }

size_t outer_bytes(int64_t t, int64_t cols, int64_t r) { return (size_t)outer_slots(t) * ceil_div(r, 64) * 64 * cols * sizeof(float); }

int launch_outer(bool bf16, const OuterArgs& p, cudaStream_t st) {
    // an adapter without tokens still writes its zeros: one item each
    const int64_t items = ceil_div(p.t, OUTER_CHUNK) + p.n;
    if (items > 65535) return set_error(CDCLQ_ERR_ARG, "adapters: too many tokens or adapters for one call");
    const dim3 grid((unsigned)ceil_div(p.cols, OUTER_COLS), (unsigned)items, (unsigned)ceil_div(p.r, OUTER_RANK));
    if (p.codes) {
        auto kern = bf16 ? outer_kernel<true, true> : outer_kernel<false, true>;
        CDCLQ_LAUNCH(kern, grid, 256, 0, st, p);
    } else {
        auto kern = bf16 ? outer_kernel<true, false> : outer_kernel<false, false>;
        CDCLQ_LAUNCH(kern, grid, 256, 0, st, p);
    }
    if (outer_slots(p.t) > 0) {
        const unsigned gx = (unsigned)std::max<int64_t>(1, std::min<int64_t>(ceil_div((int64_t)p.r * p.cols, 1024), sm_count() * 4));
        auto kern = bf16 ? outer_finish_kernel<true> : outer_finish_kernel<false>;
        CDCLQ_LAUNCH(kern, dim3(gx, p.n), 256, 0, st, p);
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
    size_t expanded = 0, ranked = 0, partial = 0, decode = 0, total = 0;
};
ForwardLayout forward_layout(const PackedView& w, int64_t t, int64_t n, int64_t r) {
    ForwardLayout l;
    Space s;
    if (t <= DECODE_TOKENS) {
        l.decode = s.take(packed_decode_workspace(w, (int)t, n ? (int)r : 0));
    } else {
        l.expanded = s.take((size_t)w.d_out * ceil_div(w.d_in, 8) * 8 * 2);
        size_t partial = plan_half_gemm(HALF_NT_EXTEND, t, w.d_out, w.d_in).partial_bytes;
        if (n) {
            l.ranked = s.take((size_t)t * ceil_div(r, 8) * 8 * 2);
            partial = std::max(partial, plan_half_gemm(HALF_NT_GROUPED, t, r, w.d_in).partial_bytes);
        }
        l.partial = s.take(partial);
    }
    l.total = s.at;
    return l;
}

struct BackwardLayout {
    size_t expanded = 0, ranked = 0, partial = 0, start = 0, order = 0, slots = 0, total = 0;
};
BackwardLayout backward_layout(const PackedView& w, int64_t t, int64_t n, int64_t r, bool need_dx) {
    BackwardLayout l;
    Space s;
    size_t partial = 0;
    if (need_dx) {
        l.expanded = s.take((size_t)w.d_out * ceil_div(w.d_in, 8) * 8 * 2);
        partial = plan_half_gemm(HALF_NN_EXTEND, t, w.d_in, w.d_out).partial_bytes;
    }
    if (n) {
        l.ranked = s.take((size_t)t * ceil_div(r, 8) * 8 * 2);
        partial = std::max(partial, plan_half_gemm(HALF_NN_GROUPED, t, r, w.d_out).partial_bytes);
        l.start = s.take((size_t)(n + 1) * sizeof(int));
        l.order = s.take((size_t)t * sizeof(int));
        l.slots = s.take(outer_bytes(t, std::max(w.d_in, w.d_out), r));
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

bool aligned(const void* p, size_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0; }

int check_call(const char* what, const cdclq_packed_layer* w, int dtype, size_t t, const cdclq_adapters* ad) {
    const std::string s(what);
    if (!w || !w->layout || !w->d_out || !w->d_in) return set_error(CDCLQ_ERR_ARG, s + ": no packed layer");
    if (dtype != CDCLQ_DTYPE_F16 && dtype != CDCLQ_DTYPE_BF16) return set_error(CDCLQ_ERR_ARG, s + ": dtype must be f16 or bf16");
    if (t > 0x7fffff00) return set_error(CDCLQ_ERR_ARG, s + ": too many tokens");
    if (ad && ad->n) {
        if (!ad->r) return set_error(CDCLQ_ERR_ARG, s + ": the adapters' rank must be > 0");
        if (ad->n > 32767 || ad->r > 4096) return set_error(CDCLQ_ERR_ARG, s + ": too many adapters, or too high a rank");
        if (!ad->a || !ad->b || !ad->scale || (t && !ad->index)) return set_error(CDCLQ_ERR_ARG, s + ": null pointer");
        if (ad->lda < w->d_in || ad->ldb < ad->r || !aligned(ad->a, ad->lda) || !aligned(ad->b, ad->ldb))
            return set_error(CDCLQ_ERR_ARG, s + ": rows of a and b must start on 16 bytes and not overlap");
    }
    return check_fail_word(what);
}

// The f32 sums of a grouped product, turned into u and scale * u.
int finish_rank(bool bf16, const HalfGemm& g, const HalfPlan& plan, const float* scale, void* u, int64_t ldu, void* su, int64_t lds,
                cudaStream_t st) {
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(g.m * g.n, 256), sm_count() * 8);
    auto kern = bf16 ? rank_finish_kernel<true> : rank_finish_kernel<false>;
    CDCLQ_LAUNCH(kern, grid, 256, 0, st, g.partial, plan.splits, (int)g.m, (int)g.n, (int)(ceil_div(g.n, 4) * 4), g.index, g.adapters, scale,
                 static_cast<uint16_t*>(u), (int)ldu, static_cast<uint16_t*>(su), (int)lds);
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : cuda_error(e, "rank_finish_kernel launch");
}

}  // namespace

}  // namespace cdclq

using namespace cdclq;

extern "C" size_t cdclq_projection_forward_workspace(const cdclq_packed_layer* w, size_t t, size_t n, size_t r) {
    if (!w || !t) return 0;
    return forward_layout(packed_view(*w), t, n, r).total;
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
        HalfGemm g{};
        g.form = HALF_NT_GROUPED;
        g.bf16 = bf16;
        g.m = t, g.n = r, g.k = v.d_in;
        g.a = operand(x, t, v.d_in, ldx);
        g.x = operand(ad->a, r, v.d_in, ad->lda, n);
        g.index = ad->index;
        g.adapters = (int)n;
        g.partial = partial;
        const HalfPlan plan = plan_half_gemm(HALF_NT_GROUPED, t, r, v.d_in);
        if ((rc = launch_half_gemm(g, plan, st))) return rc;
        if ((rc = finish_rank(bf16, g, plan, ad->scale, u, r, ws + l.ranked, ldr, st))) return rc;
    }
    if ((rc = launch_packed_expand(v, bf16, ws + l.expanded, ldw, st))) return rc;
    HalfGemm g{};
    g.form = HALF_NT_EXTEND;
    g.bf16 = bf16;
    g.m = t, g.n = v.d_out, g.k = v.d_in;
    g.a = operand(x, t, v.d_in, ldx);
    g.b = operand(ws + l.expanded, v.d_out, v.d_in, ldw);
    if (n) {
        g.u = operand(ws + l.ranked, t, r, ldr);
        g.x = operand(ad->b, v.d_out, r, ad->ldb, n);
        g.index = ad->index;
        g.adapters = (int)n;
    }
    g.out = y;
    g.ldo = ldy;
    g.partial = partial;
    return launch_half_gemm(g, plan_half_gemm(HALF_NT_EXTEND, t, v.d_out, v.d_in), st);
}

extern "C" size_t cdclq_projection_backward_workspace(const cdclq_packed_layer* w, size_t t, size_t n, size_t r, int need_dx) {
    if (!w || !t) return 0;
    return backward_layout(packed_view(*w), t, n, r, need_dx != 0).total;
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
    if (n && (dx || da)) {
        HalfGemm g{};
        g.form = HALF_NN_GROUPED;
        g.bf16 = bf16;
        g.m = t, g.n = r, g.k = v.d_out;
        g.a = operand(dy, t, v.d_out, lddy);
        g.x = operand(ad->b, v.d_out, r, ad->ldb, n);
        g.index = ad->index;
        g.adapters = (int)n;
        g.partial = partial;
        const HalfPlan plan = plan_half_gemm(HALF_NN_GROUPED, t, r, v.d_out);
        if ((rc = launch_half_gemm(g, plan, st))) return rc;
        if ((rc = finish_rank(bf16, g, plan, ad->scale, nullptr, 0, ws + l.ranked, ldr, st))) return rc;
    }
    if (dx) {
        if ((rc = launch_packed_expand(v, bf16, ws + l.expanded, ldw, st))) return rc;
        HalfGemm g{};
        g.form = HALF_NN_EXTEND;
        g.bf16 = bf16;
        g.m = t, g.n = v.d_in, g.k = v.d_out;
        g.a = operand(dy, t, v.d_out, lddy);
        g.b = operand(ws + l.expanded, v.d_out, v.d_in, ldw);
        if (n) {
            g.u = operand(ws + l.ranked, t, r, ldr);
            g.x = operand(ad->a, r, v.d_in, ad->lda, n);
            g.index = ad->index;
            g.adapters = (int)n;
        }
        g.out = dx;
        g.ldo = lddx;
        g.partial = partial;
        if ((rc = launch_half_gemm(g, plan_half_gemm(HALF_NN_EXTEND, t, v.d_in, v.d_out), st))) return rc;
    }
    if (!n || !(da || db)) return 0;
    OuterArgs o{};
    o.r = (int)r, o.n = (int)n, o.t = (int)t;
    o.start = reinterpret_cast<const int*>(ws + l.start);
    o.order = reinterpret_cast<const int*>(ws + l.order);
    o.slots = reinterpret_cast<float*>(ws + l.slots);
    o.slot_rank = (int)(ceil_div(r, 64) * 64);
    CDCLQ_LAUNCH(token_lists_kernel, (unsigned)n, 1024, 0, st, ad->index, (int)t, (int)n, reinterpret_cast<int*>(ws + l.start),
                 reinterpret_cast<int*>(ws + l.order));
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_error(e, "token_lists_kernel launch");
    if (da) {
        OuterArgs p = o;
        p.wide = static_cast<const uint16_t*>(x);
        if (!x) p.codes = x_codes, p.scales = x_scales;
        p.ldw = ldx;
        p.cols = v.d_in;
        p.narrow = reinterpret_cast<const uint16_t*>(ws + l.ranked);
        p.ldn = ldr;
        p.out = static_cast<uint16_t*>(da);
        p.out_i = r * v.d_in, p.out_c = 1, p.out_k = v.d_in;
        if ((rc = launch_outer(bf16, p, st))) return rc;
    }
    if (db) {
        OuterArgs p = o;
        p.wide = static_cast<const uint16_t*>(dy);
        p.ldw = lddy;
        p.cols = v.d_out;
        p.narrow = static_cast<const uint16_t*>(u);
        p.ldn = r;
        p.factor = ad->scale;
        p.out = static_cast<uint16_t*>(db);
        p.out_i = r * v.d_out, p.out_c = r, p.out_k = 1;
        if ((rc = launch_outer(bf16, p, st))) return rc;
    }
    return 0;
}

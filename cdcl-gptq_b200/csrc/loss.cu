// loss.cu - softmax cross entropy of a linear head over a large vocabulary, without its logits.
//
//   z = h W^T      lse_t = log sum_v exp z_tv      loss_t = lse_t - z_t,label      (0 for a token without a label)
//   g_tv = (exp(z_tv - lse_t) - [v = label]) dloss_t      dh = g W      dW = g^T h
//
// Forward: the product's epilogue keeps each row's running maximum and sum of exponentials over the tile's columns and
// picks the label's logit; a small kernel joins the tiles.  Backward: the logits are computed again, a piece of the
// vocabulary at a time; the epilogue turns a piece into g, rounded once to the inputs' type as the operand of the two
// gradient products under a gain that makes the largest |dloss| 2^13, taken off again where dh and dW are written: a label's
// entry, of nearly that size in every row, is then not rounded where all tokens weigh alike (as 1 / t it was off by up to
// 2^-9 in bf16, for all rows alike, and so were the gradients), and f16 keeps small probabilities.  dh is summed over the pieces
// in f32.  Memory does not grow with the vocabulary beyond GRAD_BYTES for g.
//
// Bound by the tensor cores: 2 t d v operations forward, 4 or 6 backward; with few tokens by reading W.  Forward and
// backward, 2048 tokens x 32000 words of 4096 in bf16, no dW: 1.04 ms (1.54 PFLOP/s in a burst, 1.28 under the power limit);
// 8191 x 32000 of 2048 in f16, all gradients: 3.28 ms (1.31 PFLOP/s; 1.17 under the limit).
// Forward of 57 tokens x 50257 words of 2048 in bf16: 50 us.  With words of 232 the exponentials and additions of the
// epilogue take most of the time (4069 x 68034: 185 us, 1.5 T logits a second).
#include <algorithm>

#include "half_gemm.h"

namespace cdclq {

namespace {

constexpr size_t GRAD_BYTES = 256u << 20;  // one piece of g
constexpr int JOIN_THREADS = 512;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t align_up(size_t b) { return (b + 255) & ~(size_t)255; }

// Joins the (maximum, sum) pairs of a row's column tiles: JOIN_ROWS rows to a CTA, a row's threads each with every (threads to
// a row)-th pair; the maximum of all first, so that a pair costs one exponential.  A pair's maximum is -inf where its logits
// all are; its sum is then 0, or NaN with a NaN among them.  Where it is +inf the sum is inf, or NaN, and lse with it.
template <int JOIN_ROWS>
__global__ void __launch_bounds__(JOIN_THREADS)
loss_join_kernel(const float2* __restrict__ stats, int parts, int t, int64_t vocab, const int64_t* __restrict__ target,
                 const float* __restrict__ label_logit, float* loss, float* lse) {
    constexpr int STEP = JOIN_THREADS / JOIN_ROWS, WARPS = JOIN_THREADS / 32, BATCH = 8;
    constexpr float L2E = 1.4426950408889634f;
    __shared__ float s[JOIN_ROWS][WARPS + 1];
    const int tx = threadIdx.x % JOIN_ROWS, ty = threadIdx.x / JOIN_ROWS, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = blockIdx.x * JOIN_ROWS + tx;
    const float2* mine = stats + row;
    // a row's value over its threads: over the lanes of each warp, then over the warps
    auto over_row = [&](float v, auto join) {
#pragma unroll
        for (int o = 16; o >= JOIN_ROWS; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
        __syncthreads();
        if (lane < JOIN_ROWS) s[tx][warp] = v;
        __syncthreads();
        v = s[tx][0];
#pragma unroll
        for (int w = 1; w < WARPS; w++) v = join(v, s[tx][w]);
        return v;
    };
    float top = -INFINITY, sum = 0.0f;
    if (row < t) {
        for (int p = ty; p < parts; p += BATCH * STEP) {
            float v[BATCH];
#pragma unroll
            for (int q = 0; q < BATCH; q++) v[q] = p + q * STEP < parts ? mine[(int64_t)(p + q * STEP) * t].x : -INFINITY;
#pragma unroll
            for (int q = 0; q < BATCH; q++) top = fmaxf(top, v[q]);
        }
    }
    top = over_row(top, [](float a, float b) { return fmaxf(a, b); });
    const float ref = fabsf(top) == INFINITY ? 0.0f : top;
    if (row < t) {
        for (int p = ty; p < parts; p += BATCH * STEP) {
            float2 v[BATCH];
#pragma unroll
            for (int q = 0; q < BATCH; q++)
                v[q] = p + q * STEP < parts ? mine[(int64_t)(p + q * STEP) * t] : make_float2(-INFINITY, 0.0f);
#pragma unroll
            for (int q = 0; q < BATCH; q++) sum += v[q].y * exp2f((v[q].x - ref) * L2E);
        }
    }
    sum = over_row(sum, [](float a, float b) { return a + b; });
    if (ty == 0 && row < t) {
        const float l = ref + logf(sum);
        const int64_t label = target[row];
        lse[row] = l;
        loss[row] = (label >= 0 && label < vocab) ? l - label_logit[row] : 0.0f;
    }
}

// gain[0] = 2^13 / the largest finite |dloss| of a labelled token, gain[1] = 1 / it; powers of two where that leaves the range.
__global__ void __launch_bounds__(1024) loss_gain_kernel(const float* __restrict__ dloss, const int64_t* __restrict__ target,
                                                         int t, int64_t vocab, float* gain) {
    __shared__ float part[32];
    float top = 0.0f;
    for (int i = threadIdx.x; i < t; i += 1024) {
        const float v = fabsf(dloss[i]);
        if (target[i] >= 0 && target[i] < vocab && v < INFINITY) top = fmaxf(top, v);
    }
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 32; w++) top = fmaxf(top, part[w]);
        const bool normal = top > 7.8886091e-31f && top < 1.2676506e30f;  // 2^-100, 2^100
        const float g = top == 0.0f ? 1.0f : top < 1.0f ? 1.2676506e30f : 7.8886091e-31f;
        gain[0] = normal ? 8192.0f / top : g;
        gain[1] = normal ? top * (1.0f / 8192.0f) : 1.0f / g;
    }
}

// The rows of h with a label; the others are zero, so that what they hold (a NaN among it) stays out of dW.
__global__ void __launch_bounds__(256) labelled_rows_kernel(const uint16_t* __restrict__ h, int64_t ld,
                                                            const int64_t* __restrict__ target, int64_t vocab, int64_t t,
                                                            int64_t d, int64_t d8, uint4* out) {
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < t * d8; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t row = i / d8, c = (i - row * d8) * 8;
        const int64_t label = target[row];
        const uint16_t* src = h + row * ld + c;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (label >= 0 && label < vocab) {
            if (c + 8 <= d) {
                v = *reinterpret_cast<const uint4*>(src);
            } else {  // the row's last columns: nothing is read past them
                uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
                for (int q = 0; q < 8; q++)
                    if (c + q < d) w[q >> 1] |= (uint32_t)src[q] << (16 * (q & 1));
                v = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        out[i] = v;
    }
}

struct Piece {
    int64_t cols;  // columns of the vocabulary in a piece
    int64_t count;
};
Piece pieces(int64_t t, int64_t v) {
    const int64_t most = std::max<int64_t>(256, (int64_t)(GRAD_BYTES / 2) / t / 256 * 256);
    const int64_t count = ceil_div(v, most);
    const int64_t cols = ceil_div(ceil_div(v, count), 256) * 256;
    return {cols, ceil_div(v, cols)};
}

struct Layout {
    size_t grad = 0, acc = 0, rows = 0, gain = 0, partial = 0, total = 0;
};
Layout backward_layout(int64_t t, int64_t d, int64_t v, bool need_dh, bool need_dw) {
    const Piece pc = pieces(t, v);
    Layout l;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += align_up(bytes);
        return here;
    };
    l.grad = take((size_t)t * pc.cols * 2);
    l.gain = take(2 * sizeof(float));
    size_t partial = 0;
    if (need_dh) {
        if (pc.count > 1) l.acc = take((size_t)t * ceil_div(d, 4) * 4 * sizeof(float));
        // a shorter last piece may be planned otherwise
        partial = std::max(plan_half_gemm(HALF_NN, t, d, pc.cols).partial_bytes,
                           plan_half_gemm(HALF_NN, t, d, v - (pc.count - 1) * pc.cols).partial_bytes);
    }
    if (need_dw) {
        l.rows = take((size_t)t * ceil_div(d, 8) * 8 * 2);
        partial = std::max(partial, std::max(plan_half_gemm(HALF_TN, std::min(pc.cols, v), d, t).partial_bytes,
                                             plan_half_gemm(HALF_TN, v - (pc.count - 1) * pc.cols, d, t).partial_bytes));
    }
    l.partial = take(partial);
    l.total = at;
    return l;
}

int check_head(const char* what, const void* h, size_t ldh, const void* w, size_t ldw, int dtype, size_t t, size_t d, size_t v) {
    const std::string s(what);
    if (dtype != CDCLQ_DTYPE_F16 && dtype != CDCLQ_DTYPE_BF16) return set_error(CDCLQ_ERR_ARG, s + ": dtype must be f16 or bf16");
    if (d == 0 || v == 0) return set_error(CDCLQ_ERR_ARG, s + ": the head has no rows or no columns");
    if (t > MOST_SIZE || d > MOST_SIZE || v > MOST_SIZE) return set_error(CDCLQ_ERR_ARG, s + ": too large");
    if (t && (!h || !w)) return set_error(CDCLQ_ERR_ARG, s + ": null pointer");
    if (ldh < d || ldw < d) return set_error(CDCLQ_ERR_ARG, s + ": rows overlap");
    if (t && ((ldh % 8) || (ldw % 8) || (reinterpret_cast<uintptr_t>(h) & 15) || (reinterpret_cast<uintptr_t>(w) & 15)))
        return set_error(CDCLQ_ERR_ARG, s + ": rows of h and w must start on 16 bytes");
    return check_fail_word(what);
}

HalfOperand operand(const void* p, int64_t rows, int64_t cols, int64_t ld) {
    HalfOperand o;
    o.p = p;
    o.rows = rows;
    o.cols = cols;
    o.ld = ld;
    return o;
}

}  // namespace

}  // namespace cdclq

using namespace cdclq;

extern "C" size_t cdclq_linear_cross_entropy_workspace(size_t t, size_t d, size_t v) {
    if (!t || !d || !v || t > MOST_SIZE || d > MOST_SIZE || v > MOST_SIZE) return 0;
    return align_up(sizeof(float2) * half_stats_parts(plan_half_gemm(HALF_STATS, t, v, d), v) * t) + align_up(sizeof(float) * t);
}

extern "C" int cdclq_linear_cross_entropy_device(const void* h, size_t ldh, const void* w, size_t ldw, int dtype, size_t t,
                                                 size_t d, size_t v, const int64_t* target, float* loss, float* lse,
                                                 void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_head("linear_cross_entropy", h, ldh, w, ldw, dtype, t, d, v);
    if (rc || !t) return rc;
    if (!target || !loss || !lse) return set_error(CDCLQ_ERR_ARG, "linear_cross_entropy: null pointer");
    if (!workspace || workspace_bytes < cdclq_linear_cross_entropy_workspace(t, d, v))
        return set_error(CDCLQ_ERR_ARG, "linear_cross_entropy: the workspace is too small");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    HalfGemm g{};
    g.form = HALF_STATS;
    g.bf16 = dtype == CDCLQ_DTYPE_BF16;
    g.m = t, g.n = v, g.k = d;
    g.a = operand(h, t, d, ldh);
    g.b = operand(w, v, d, ldw);
    g.target = target;
    g.vocab = v;
    const HalfPlan plan = plan_half_gemm(HALF_STATS, t, v, d);
    const int parts = (int)half_stats_parts(plan, v);
    g.stats = static_cast<float2*>(workspace);
    g.label_logit = reinterpret_cast<float*>(static_cast<char*>(workspace) + align_up(sizeof(float2) * parts * t));
    if ((rc = launch_half_gemm(g, plan, st))) return rc;
    // 32 rows read whole lines; fewer where that leaves SMs idle (57 tokens x 4008 pairs: 8 rows 11.8 us, 1 row 4.4 us)
    const int rows = t >= 32 * (size_t)sm_count() ? 32 : t >= 2 * (size_t)sm_count() ? 8 : 1;
    auto join = rows == 32 ? loss_join_kernel<32> : rows == 8 ? loss_join_kernel<8> : loss_join_kernel<1>;
    CDCLQ_LAUNCH(join, (unsigned)ceil_div(t, rows), JOIN_THREADS, 0, st, g.stats, parts, (int)t, (int64_t)v, target, g.label_logit, loss,
                 lse);
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : cuda_error(e, "loss_join_kernel launch");
}

extern "C" size_t cdclq_linear_cross_entropy_backward_workspace(size_t t, size_t d, size_t v, int need_dh, int need_dw) {
    if (!t || !d || !v || t > MOST_SIZE || d > MOST_SIZE || v > MOST_SIZE) return 0;
    return backward_layout(t, d, v, need_dh != 0, need_dw != 0).total;
}

extern "C" int cdclq_linear_cross_entropy_backward_device(const void* h, size_t ldh, const void* w, size_t ldw, int dtype,
                                                          size_t t, size_t d, size_t v, const int64_t* target,
                                                          const float* lse, const float* dloss, void* dh, size_t lddh,
                                                          void* dw, size_t lddw, void* workspace, size_t workspace_bytes,
                                                          void* stream) {
    int rc = check_head("linear_cross_entropy_backward", h, ldh, w, ldw, dtype, t, d, v);
    if (rc) return rc;
    if ((dh && lddh < d) || (dw && lddw < d)) return set_error(CDCLQ_ERR_ARG, "linear_cross_entropy_backward: rows overlap");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!t) {
        if (dw) CDCLQ_CUDA_TRY(cudaMemset2DAsync(dw, lddw * 2, 0, d * 2, v, st));
        return 0;
    }
    if (!dh && !dw) return 0;
    if (!target || !lse || !dloss) return set_error(CDCLQ_ERR_ARG, "linear_cross_entropy_backward: null pointer");
    const Layout l = backward_layout(t, d, v, dh != nullptr, dw != nullptr);
    if (!workspace || workspace_bytes < l.total)
        return set_error(CDCLQ_ERR_ARG, "linear_cross_entropy_backward: the workspace is too small");
    char* ws = static_cast<char*>(workspace);
    const bool bf16 = dtype == CDCLQ_DTYPE_BF16;
    float* gain = reinterpret_cast<float*>(ws + l.gain);
    CDCLQ_LAUNCH(loss_gain_kernel, 1, 1024, 0, st, dloss, target, (int)t, (int64_t)v, gain);
    const int64_t d8 = ceil_div(d, 8);
    if (dw) {
        const int64_t blocks = ceil_div((int64_t)t * d8, 256);
        CDCLQ_LAUNCH(labelled_rows_kernel, (unsigned)std::min<int64_t>(blocks, sm_count() * 16), 256, 0, st,
                     static_cast<const uint16_t*>(h), (int64_t)ldh, target, (int64_t)v, (int64_t)t, (int64_t)d, d8,
                     reinterpret_cast<uint4*>(ws + l.rows));
    }
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_error(e, "linear_cross_entropy_backward launch");
    const Piece pc = pieces(t, v);
    float* acc = reinterpret_cast<float*>(ws + l.acc);
    for (int64_t i = 0; i < pc.count; i++) {
        const int64_t v0 = i * pc.cols, cols = std::min<int64_t>(pc.cols, (int64_t)v - v0);
        const char* piece = static_cast<const char*>(w) + v0 * ldw * 2;
        HalfGemm g{};
        g.form = HALF_GRAD;
        g.bf16 = bf16;
        g.m = t, g.n = cols, g.k = d;
        g.a = operand(h, t, d, ldh);
        g.b = operand(piece, cols, d, ldw);
        g.out = ws + l.grad;
        g.ldo = pc.cols;
        g.target = target;
        g.col0 = v0;
        g.vocab = v;
        g.lse = lse;
        g.dloss = dloss;
        g.gain = gain;
        if ((rc = launch_half_gemm(g, plan_half_gemm(HALF_GRAD, t, cols, d), st))) return rc;
        if (dh) {
            HalfGemm q{};
            q.form = HALF_NN;
            q.bf16 = bf16;
            q.m = t, q.n = d, q.k = cols;
            q.a = operand(ws + l.grad, t, cols, pc.cols);
            q.b = operand(piece, cols, d, ldw);
            q.ldf = ceil_div(d, 4) * 4;
            q.f32in = i ? acc : nullptr;
            if (i + 1 < pc.count) {
                q.f32out = acc;
            } else {
                q.out = dh;
                q.ldo = lddh;
                q.alpha = gain + 1;
            }
            q.partial = reinterpret_cast<float*>(ws + l.partial);
            if ((rc = launch_half_gemm(q, plan_half_gemm(HALF_NN, t, d, cols), st))) return rc;
        }
        if (dw) {
            HalfGemm q{};
            q.form = HALF_TN;
            q.bf16 = bf16;
            q.m = cols, q.n = d, q.k = t;
            q.a = operand(ws + l.grad, t, cols, pc.cols);
            q.b = operand(ws + l.rows, t, d, d8 * 8);
            q.out = static_cast<char*>(dw) + v0 * lddw * 2;
            q.ldo = lddw;
            q.alpha = gain + 1;
            q.partial = reinterpret_cast<float*>(ws + l.partial);
            if ((rc = launch_half_gemm(q, plan_half_gemm(HALF_TN, cols, d, t), st))) return rc;
        }
    }
    return 0;
}

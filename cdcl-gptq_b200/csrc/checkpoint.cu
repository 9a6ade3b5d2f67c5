// checkpoint.cu - activations kept in 8 bits between the forward and the backward pass.
//
//   s = max |x| / 127 over a block of 128 columns of a row      q = round(x / s), to nearest, ties to even      x^ = q s
//
// A block of zeros has s = 0; one that holds a NaN or an infinity has s = NaN and is restored as NaN, so that an
// overflow in the forward pass is not hidden.  q fits 8 signed bits, and the error is at most s / 2 for each value.
// Saving and restoring are bound by memory: the 16-bit matrix once, the codes once.
//
// The weight gradient dW = dy^T x^ restores a piece of tokens at a time into a buffer that stays in L2 and multiplies it
// on the tensor cores; pieces are added in f32.
#include <algorithm>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "half_gemm.h"

namespace cdclq {

namespace {

constexpr int BLOCK = 128;                  // columns of a scale
constexpr size_t PIECE_BYTES = 32u << 20;   // restored tokens of the weight gradient

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t align_up(size_t b) { return (b + 255) & ~(size_t)255; }

template <int DT>
struct Type;
template <>
struct Type<CDCLQ_DTYPE_F32> {
    typedef float T;
    static __device__ __forceinline__ float up(float v) { return v; }
    static __device__ __forceinline__ float down(float v) { return v; }
};
template <>
struct Type<CDCLQ_DTYPE_F16> {
    typedef __half T;
    static __device__ __forceinline__ float up(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half down(float v) { return __float2half_rn(v); }
};
template <>
struct Type<CDCLQ_DTYPE_BF16> {
    typedef __nv_bfloat16 T;
    static __device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 down(float v) { return __float2bfloat16_rn(v); }
};

// The absolute values' largest bits over 8 values: as whole numbers they order like the values, infinities and NaN above.
__device__ __forceinline__ uint32_t top_bits(const float (&raw)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) m = max(m, __float_as_uint(raw[i]) & 0x7fffffffu);
    return m;
}
template <typename T>
__device__ __forceinline__ uint32_t top_bits(const T (&raw)[8]) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(raw);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
    return max(m & 0xffffu, m >> 16);
}
__device__ __forceinline__ float value_of_bits(uint32_t b, const float*) { return __uint_as_float(b); }
__device__ __forceinline__ float value_of_bits(uint32_t b, const __half*) { return __half2float(__ushort_as_half((uint16_t)b)); }
__device__ __forceinline__ float value_of_bits(uint32_t b, const __nv_bfloat16*) { return __uint_as_float(b << 16); }

// 16 lanes to a block of 128 columns, 8 values a lane: one wide load of a 16-bit type.  A CTA has 16 such groups: `across`
// of them (a power of two) side by side along a row, 16 / across rows; it takes two such sets of rows at a time.
//
// Rounding x / s: p = x * (1 / s) is within 127 * 2^-23 of the quotient, so it rounds to the same number unless it lies
// within 2^-15 of a half; a thread with such a value divides.  Adding 1.5 * 2^23 rounds p to the nearest whole number, ties
// to even, and leaves it in the sum's low byte.  |p| <= 127 (1 + 2^-22), so no code is out of range.
template <int DT, bool WIDE>
__global__ void __launch_bounds__(256) checkpoint_save_kernel(const typename Type<DT>::T* __restrict__ x, int64_t ldx, int64_t t,
                                                              int64_t d, int across, int8_t* __restrict__ codes,
                                                              float* __restrict__ scales) {
    typedef typename Type<DT>::T T;
    constexpr int UNROLL = 2;
    constexpr float MAGIC = 12582912.0f;
    const int lane = threadIdx.x & 15, group = threadIdx.x >> 4;
    const int64_t nb = (d + BLOCK - 1) / BLOCK;
    const int64_t b = (int64_t)blockIdx.x * across + (group & (across - 1));
    const int64_t c = b * BLOCK + lane * 8;
    const int down = 16 / across;
    const int n = (int)max((int64_t)0, min((int64_t)8, d - c));
    // every thread of a warp walks the same number of rows (the shuffles need them all)
    for (int64_t r0 = (int64_t)blockIdx.y * down * UNROLL; r0 < t; r0 += (int64_t)gridDim.y * down * UNROLL) {
        alignas(16) T raw[UNROLL][8];
        int64_t row[UNROLL];
#pragma unroll
        for (int k = 0; k < UNROLL; k++) {
            row[k] = r0 + k * down + group / across;
            const int m = row[k] < t ? n : 0;
            const T* src = x + row[k] * ldx + c;
            if (WIDE) {
#pragma unroll
                for (int i = 0; i < (int)sizeof(raw[0]) / 16; i++)
                    reinterpret_cast<uint4*>(raw[k])[i] = m ? __ldcs(reinterpret_cast<const uint4*>(src) + i) : make_uint4(0, 0, 0, 0);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) raw[k][i] = i < m ? src[i] : Type<DT>::down(0.0f);
            }
        }
#pragma unroll
        for (int k = 0; k < UNROLL; k++) {
            uint32_t bits = top_bits(raw[k]);
#pragma unroll
            for (int o = 8; o; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
            const float top = value_of_bits(bits, static_cast<const T*>(nullptr));
            const bool finite = top < INFINITY;
            const float s = finite ? __fdiv_rn(top, 127.0f) : __int_as_float(0x7fffffff);
            const bool normal = finite && s >= 1.1754944e-38f;  // 1 / s is then finite
            const float inv = normal ? __fdiv_rn(1.0f, s) : 0.0f;
            uint32_t q[8];
            float near = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float p = normal ? Type<DT>::up(raw[k][i]) * inv : 0.0f;
                const float m = p + MAGIC;
                near = fmaxf(near, fabsf(p - (m - MAGIC)));
                q[i] = __float_as_uint(m);
            }
            if (near > 0.5f - 1.0f / 32768.0f || (finite && !normal && s > 0.0f)) {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    q[i] = (uint32_t)(int)fminf(fmaxf(rintf(__fdiv_rn(Type<DT>::up(raw[k][i]), s)), -127.0f), 127.0f);
            }
            if (row[k] >= t || n == 0) continue;
            if (lane == 0) scales[row[k] * nb + b] = s;
            int8_t* dst = codes + row[k] * d + c;
            if (WIDE) {
                const uint32_t lo = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
                const uint32_t hi = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
                *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (i < n) dst[i] = (int8_t)q[i];
            }
        }
    }
}

// 16 values a thread; a CTA has `across` (a power of two) threads along a row.  ld: elements from row to row of the output;
// columns d..ld of it are left as they are.
template <int DT, bool WIDE>
__global__ void __launch_bounds__(256) checkpoint_restore_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scales,
                                                                 int64_t t, int64_t d, int across, typename Type<DT>::T* __restrict__ out,
                                                                 int64_t ld) {
    typedef typename Type<DT>::T T;
    const int64_t nb = (d + BLOCK - 1) / BLOCK;
    const int64_t c = ((int64_t)blockIdx.x * across + (threadIdx.x & (across - 1))) * 16;
    if (c >= d) return;
    const int down = 256 / across;
    for (int64_t row = (int64_t)blockIdx.y * down + threadIdx.x / across; row < t; row += (int64_t)gridDim.y * down) {
        const float s = scales[row * nb + c / BLOCK];
        const int8_t* src = codes + row * d + c;
        T* dst = out + row * ld + c;
        if (WIDE && c + 16 <= d) {
            alignas(16) int8_t q[16];
            alignas(16) T r[16];
            *reinterpret_cast<uint4*>(q) = __ldcs(reinterpret_cast<const uint4*>(src));
#pragma unroll
            for (int k = 0; k < 16; k++) r[k] = Type<DT>::down(__fmul_rn((float)q[k], s));
#pragma unroll
            for (int k = 0; k < (int)sizeof(r) / 16; k++) reinterpret_cast<uint4*>(dst)[k] = reinterpret_cast<uint4*>(r)[k];
        } else {
            for (int k = 0; k < 16 && c + k < d; k++) dst[k] = Type<DT>::down(__fmul_rn((float)src[k], s));
        }
    }
}

int power_of_two(int64_t want, int most) {
    int p = 1;
    while (p < most && p < want) p *= 2;
    return p;
}

// Rows' CTAs: enough for 32 to an SM over the whole grid, at most what a grid's second dimension holds.
unsigned grid_rows(int64_t rows, int64_t columns) {
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>({rows, ceil_div((int64_t)sm_count() * 32, columns), 65535}));
}

template <int DT>
int save(const void* x, int64_t ldx, int64_t t, int64_t d, int8_t* codes, float* scales, cudaStream_t st) {
    typedef typename Type<DT>::T T;
    const bool wide = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ldx * sizeof(T)) % 16 == 0 &&
                      (reinterpret_cast<uintptr_t>(codes) & 7) == 0 && d % 8 == 0;
    const int64_t nb = ceil_div(d, BLOCK);
    const int across = power_of_two(nb, 16);
    const int64_t gx = ceil_div(nb, across);
    auto kern = wide ? checkpoint_save_kernel<DT, true> : checkpoint_save_kernel<DT, false>;
    CDCLQ_LAUNCH(kern, dim3((unsigned)gx, grid_rows(ceil_div(t, 2 * (16 / across)), gx)), 256, 0, st, static_cast<const T*>(x), ldx, t, d,
                 across, codes, scales);
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : cuda_error(e, "checkpoint_save_kernel launch");
}

template <int DT>
int restore(const int8_t* codes, const float* scales, int64_t t, int64_t d, void* out, int64_t ld, cudaStream_t st) {
    typedef typename Type<DT>::T T;
    const bool wide = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && (ld * sizeof(T)) % 16 == 0 &&
                      (reinterpret_cast<uintptr_t>(codes) & 15) == 0 && d % 16 == 0;
    const int across = power_of_two(ceil_div(d, 16), 256);
    const int64_t gx = ceil_div(d, 16 * across);
    auto kern = wide ? checkpoint_restore_kernel<DT, true> : checkpoint_restore_kernel<DT, false>;
    CDCLQ_LAUNCH(kern, dim3((unsigned)gx, grid_rows(ceil_div(t, 256 / across), gx)), 256, 0, st, codes, scales, t, d, across,
                 static_cast<T*>(out), ld);
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : cuda_error(e, "checkpoint_restore_kernel launch");
}

int restore_half(bool bf16, const int8_t* codes, const float* scales, int64_t t, int64_t d, void* out, int64_t ld, cudaStream_t st) {
    return bf16 ? restore<CDCLQ_DTYPE_BF16>(codes, scales, t, d, out, ld, st)
                : restore<CDCLQ_DTYPE_F16>(codes, scales, t, d, out, ld, st);
}

struct Grad {
    int64_t rows, count;  // tokens of a piece, pieces
    size_t acc, partial, total;
};
Grad grad_layout(int64_t t, int64_t d, int64_t n) {
    Grad g{};
    const int64_t ld = ceil_div(d, 8) * 8;
    const int64_t most = std::max<int64_t>(64, (int64_t)(PIECE_BYTES / 2) / ld / 64 * 64);
    g.count = ceil_div(t, most);
    g.rows = ceil_div(ceil_div(t, g.count), 64) * 64;
    g.count = ceil_div(t, g.rows);
    size_t at = align_up((size_t)std::min(g.rows, t) * ld * 2);
    g.acc = at;
    if (g.count > 1) at += align_up((size_t)n * ceil_div(d, 4) * 4 * sizeof(float));
    g.partial = at;
    at += align_up(std::max(plan_half_gemm(HALF_TN, n, d, std::min(g.rows, t)).partial_bytes,
                            plan_half_gemm(HALF_TN, n, d, t - (g.count - 1) * g.rows).partial_bytes));
    g.total = at;
    return g;
}

bool known(int dtype) { return dtype == CDCLQ_DTYPE_F32 || dtype == CDCLQ_DTYPE_F16 || dtype == CDCLQ_DTYPE_BF16; }

}  // namespace

}  // namespace cdclq

using namespace cdclq;

extern "C" int cdclq_checkpoint_save_device(const void* x, size_t ldx, int dtype, size_t t, size_t d, int8_t* codes, float* scales,
                                            void* stream) {
    if (!known(dtype)) return set_error(CDCLQ_ERR_ARG, "checkpoint_save: dtype must be f32, f16 or bf16");
    if (!t || !d) return 0;
    if (!x || !codes || !scales) return set_error(CDCLQ_ERR_ARG, "checkpoint_save: null pointer");
    if (ldx < d) return set_error(CDCLQ_ERR_ARG, "checkpoint_save: rows overlap");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == CDCLQ_DTYPE_F32) return save<CDCLQ_DTYPE_F32>(x, ldx, t, d, codes, scales, st);
    if (dtype == CDCLQ_DTYPE_F16) return save<CDCLQ_DTYPE_F16>(x, ldx, t, d, codes, scales, st);
    return save<CDCLQ_DTYPE_BF16>(x, ldx, t, d, codes, scales, st);
}

extern "C" int cdclq_checkpoint_restore_device(const int8_t* codes, const float* scales, size_t t, size_t d, void* out, size_t ldo,
                                               int dtype, void* stream) {
    if (!known(dtype)) return set_error(CDCLQ_ERR_ARG, "checkpoint_restore: dtype must be f32, f16 or bf16");
    if (!t || !d) return 0;
    if (!codes || !scales || !out) return set_error(CDCLQ_ERR_ARG, "checkpoint_restore: null pointer");
    if (ldo < d) return set_error(CDCLQ_ERR_ARG, "checkpoint_restore: rows overlap");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == CDCLQ_DTYPE_F32) return restore<CDCLQ_DTYPE_F32>(codes, scales, t, d, out, ldo, st);
    return restore_half(dtype == CDCLQ_DTYPE_BF16, codes, scales, t, d, out, ldo, st);
}

extern "C" size_t cdclq_checkpoint_weight_grad_workspace(size_t t, size_t d, size_t n) {
    return t && d && n ? grad_layout(t, d, n).total : 0;
}

extern "C" int cdclq_checkpoint_weight_grad_device(const void* dy, size_t lddy, int dtype, const int8_t* codes, const float* scales,
                                                   size_t t, size_t d, size_t n, void* dw, size_t lddw, void* workspace,
                                                   size_t workspace_bytes, void* stream) {
    if (dtype != CDCLQ_DTYPE_F16 && dtype != CDCLQ_DTYPE_BF16)
        return set_error(CDCLQ_ERR_ARG, "checkpoint_weight_grad: dtype must be f16 or bf16");
    if (!d || !n) return 0;
    if (!dw || lddw < d) return set_error(CDCLQ_ERR_ARG, "checkpoint_weight_grad: null pointer, or rows overlap");
    if (t > 0x7fffff00 || d > 0x7fffff00 || n > 0x7fffff00) return set_error(CDCLQ_ERR_ARG, "checkpoint_weight_grad: too large");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!t) {
        CDCLQ_CUDA_TRY(cudaMemset2DAsync(dw, lddw * 2, 0, d * 2, n, st));
        return 0;
    }
    if (!dy || !codes || !scales) return set_error(CDCLQ_ERR_ARG, "checkpoint_weight_grad: null pointer");
    if (lddy < n || lddy % 8 || (reinterpret_cast<uintptr_t>(dy) & 15))
        return set_error(CDCLQ_ERR_ARG, "checkpoint_weight_grad: rows of dy must start on 16 bytes");
    const Grad l = grad_layout(t, d, n);
    if (!workspace || workspace_bytes < l.total) return set_error(CDCLQ_ERR_ARG, "checkpoint_weight_grad: the workspace is too small");
    int rc = check_fail_word("checkpoint_weight_grad");
    if (rc) return rc;
    char* ws = static_cast<char*>(workspace);
    const bool bf16 = dtype == CDCLQ_DTYPE_BF16;
    const int64_t ld = ceil_div(d, 8) * 8, nb = ceil_div(d, BLOCK);
    for (int64_t i = 0; i < l.count; i++) {
        const int64_t r0 = i * l.rows, rows = std::min<int64_t>(l.rows, (int64_t)t - r0);
        if ((rc = restore_half(bf16, codes + r0 * d, scales + r0 * nb, rows, d, ws, ld, st))) return rc;
        HalfGemm g{};
        g.form = HALF_TN;
        g.bf16 = bf16;
        g.m = n, g.n = d, g.k = rows;
        g.a.p = static_cast<const char*>(dy) + r0 * lddy * 2;
        g.a.rows = rows, g.a.cols = n, g.a.ld = lddy;
        g.b.p = ws;
        g.b.rows = rows, g.b.cols = d, g.b.ld = ld;
        g.ldf = ceil_div(d, 4) * 4;
        float* acc = reinterpret_cast<float*>(ws + l.acc);
        g.f32in = i ? acc : nullptr;
        if (i + 1 < l.count) {
            g.f32out = acc;
        } else {
            g.out = dw;
            g.ldo = lddw;
        }
        g.partial = reinterpret_cast<float*>(ws + l.partial);
        if ((rc = launch_half_gemm(g, plan_half_gemm(HALF_TN, n, d, rows), st))) return rc;
    }
    return 0;
}

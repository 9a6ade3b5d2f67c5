// checkpoint.cu - activations kept in 8 bits between the forward and the backward pass.
//
//   s = max |x| / 127 over a block of 128 columns of a row      q = round(x / s), to nearest, ties to even      x^ = q s
//
// A block of zeros has s = 0; one that holds a NaN or an infinity has s = NaN and is restored as NaN, so that an
// overflow in the forward pass is not hidden.  q fits 8 signed bits, and the error is at most s / 2 for each value, or 127 2^-150
// where that is more: s below f32's normal range (a maximum below 1.5e-36) is itself rounded to a multiple of 2^-149.
// Saving and restoring are bound by memory: the 16-bit matrix once, the codes once.  16384 x 4096 in bf16: save 42 us
// (4.9 TB/s, the division in the way), restore 31 us (6.6 TB/s, what a copy gets); with 4091 columns, rows that start anywhere,
// 5717 rows of f32 take 51 and 31 us (2.3 and 3.8 TB/s), single values in place of pieces.
//
// The weight gradient dW = dy^T x^ restores a piece of tokens at a time into a buffer that stays in L2 and multiplies it
// on the tensor cores; pieces are added in f32.  Its operand is x^ rounded to dy's type, as the tensor cores take 16 bits.
// 4096 tokens, 2048 x 5632 in bf16: 6 us restoring, 80 us multiplying (1.18 PFLOP/s).
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

// The largest f32 over 127, rounded up, is the one scale of save whose 127-fold passes f32's range: the number below it stands in
// for it, so that finite values come back finite (one compare for a scale; bounding every product took 3 % of a restore in f32).
template <int DT>
__device__ __forceinline__ float scale_of(float s) {
    return DT == CDCLQ_DTYPE_F32 && __float_as_uint(s) == 0x7c010204u ? __uint_as_float(0x7c010203u) : s;
}

// Two f32 operations at a time, each rounded on its own.
struct Pair {
    float x, y;
};
__device__ __forceinline__ uint64_t bits(Pair v) { return (uint64_t)__float_as_uint(v.y) << 32 | __float_as_uint(v.x); }
__device__ __forceinline__ Pair pair(uint64_t v) { return {__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32))}; }
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
    return pair(r);
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
    return pair(r);
}

__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
    return pair(r);
}

// The absolute values' largest bits over N values: as whole numbers they order like the values, infinities and NaN above.
template <int N>
__device__ __forceinline__ uint32_t top_bits(const float (&raw)[N]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; i++) m = max(m, __float_as_uint(raw[i]) & 0x7fffffffu);
    return m;
}
template <int N, typename T>
__device__ __forceinline__ uint32_t top_bits(const T (&raw)[N]) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(raw);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N / 2; i++) asm("max.u16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i] & 0x7fff7fffu));
    return max(m & 0xffffu, m >> 16);
}
__device__ __forceinline__ float value_of_bits(uint32_t b, const float*) { return __uint_as_float(b); }
__device__ __forceinline__ float value_of_bits(uint32_t b, const __half*) { return __half2float(__ushort_as_half((uint16_t)b)); }
__device__ __forceinline__ float value_of_bits(uint32_t b, const __nv_bfloat16*) { return __uint_as_float(b << 16); }

constexpr int SAVE_LANES = 8, SAVE_VALUES = BLOCK / SAVE_LANES;  // lanes of a block, values of a lane
constexpr int SAVE_GROUPS = 256 / SAVE_LANES;

// 8 lanes to a block of 128 columns, 16 values a lane: two pieces of eight where x's rows start on 16 bytes and the codes' on
// 8 (WIDE), else every eighth value, so that the lanes' pieces or values lie side by side.  A CTA has 32 such groups: `across` of them (a power of two)
// along a row, 32 / across rows.
//
// x / s to the nearest whole number of the rounded quotient, ties to even (values of few bits meet ties often: with a block's
// largest value a power of two, in one of two).  With y = 1 / s rounded, q = x y and its remainder e = x - q s, which one FMA
// gives exactly, q + e y rounded is the quotient rounded (Markstein, IBM J. Res. Dev. 34, 1990) - as long as nothing
// underflows: below a scale of 2^-100 a thread divides.  Adding 1.5 * 2^23 rounds to a whole number and leaves it in the
// sum's low byte; |x / s| <= 127 (1 + 2^-23), so no code is out of range.
template <int DT, bool WIDE>
__global__ void __launch_bounds__(256, 4) checkpoint_save_kernel(const typename Type<DT>::T* __restrict__ x, int64_t ldx, int64_t t,
                                                              int64_t d, int across, int8_t* __restrict__ codes,
                                                              float* __restrict__ scales) {
    typedef typename Type<DT>::T T;
    constexpr int N = SAVE_VALUES;
    constexpr float MAGIC = 12582912.0f;
    const int lane = threadIdx.x % SAVE_LANES, group = threadIdx.x / SAVE_LANES;
    const int64_t nb = (d + BLOCK - 1) / BLOCK;
    const int64_t b = (int64_t)blockIdx.x * across + (group & (across - 1));
    constexpr int PIECE = WIDE ? 8 : 1, STRIDE = SAVE_LANES * PIECE;  // neighbouring values, from a lane's piece to its next
    const int64_t c = b * BLOCK + lane * PIECE;
    const int down = SAVE_GROUPS / across;
    const int n = (int)max((int64_t)0, min((int64_t)(N / PIECE), (d - c + STRIDE - 1) / STRIDE));  // pieces
    const int64_t first = (int64_t)blockIdx.y * down + group / across, step = (int64_t)gridDim.y * down;
    const T* src = x + first * ldx + c;
    int8_t* dst = codes + first * d + c;
    float* to = scales + first * nb + b;
    alignas(16) T next[N];
    auto load = [&](int m) {
        if (WIDE) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(next) / 16; i++) {
                constexpr int IN_PIECE = PIECE * (int)sizeof(T) / 16;
                reinterpret_cast<uint4*>(next)[i] = i / IN_PIECE < m ? __ldcs(reinterpret_cast<const uint4*>(src + i / IN_PIECE * STRIDE) + i % IN_PIECE)
                                                                     : make_uint4(0, 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) next[i] = i < m ? __ldcs(src + i * STRIDE) : Type<DT>::down(0.0f);
        }
        src += step * ldx;
    };
    load(first < t ? n : 0);
    // every thread of a warp walks the same number of rows (the shuffles need them all); the next row is on its way meanwhile
    for (int64_t r0 = (int64_t)blockIdx.y * down; r0 < t; r0 += step, dst += step * d, to += step * nb) {
        const int64_t row = r0 + group / across;
        const int m = row < t ? n : 0;
        alignas(16) T raw[N];
#pragma unroll
        for (int i = 0; i < N; i++) raw[i] = next[i];
        load(row + step < t ? n : 0);
        uint32_t most = top_bits(raw);
#pragma unroll
        for (int o = SAVE_LANES / 2; o; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        const float top = value_of_bits(most, static_cast<const T*>(nullptr));
        const bool finite = top < INFINITY;
        const float s = finite ? __fdiv_rn(top, 127.0f) : __int_as_float(0x7fffffff);
        const bool normal = finite && s >= 7.8886091e-31f;  // 2^-100
        const float inv = normal ? __fdiv_rn(1.0f, s) : 0.0f;
        uint32_t q[N];
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const Pair v = {Type<DT>::up(raw[i]), Type<DT>::up(raw[i + 1])};
            const Pair p = mul2(v, {inv, inv});
            const Pair r = add2(fma2(fma2(p, {-s, -s}, v), {inv, inv}, p), {MAGIC, MAGIC});
            q[i] = __float_as_uint(r.x), q[i + 1] = __float_as_uint(r.y);
        }
        if (!normal) {
#pragma unroll
            for (int i = 0; i < N; i++)
                q[i] = finite && s > 0.0f ? (uint32_t)(int)fminf(fmaxf(rintf(__fdiv_rn(Type<DT>::up(raw[i]), s)), -127.0f), 127.0f) : 0u;
        }
        if (m == 0) continue;
        if (lane == 0) *to = s;  // lane 0 has the block's first value
        if (WIDE) {
            uint32_t w[N / 4];
#pragma unroll
            for (int i = 0; i < N / 4; i++)
                w[i] = __byte_perm(__byte_perm(q[4 * i], q[4 * i + 1], 0x0040), __byte_perm(q[4 * i + 2], q[4 * i + 3], 0x0040), 0x5410);
#pragma unroll
            for (int i = 0; i < N / PIECE; i++)
                if (i < m) *reinterpret_cast<uint2*>(dst + i * STRIDE) = make_uint2(w[2 * i], w[2 * i + 1]);
        } else {
#pragma unroll
            for (int i = 0; i < N; i++)
                if (i < m) dst[i * STRIDE] = (int8_t)q[i];
        }
    }
}

// 16 values a thread; a CTA has `across` (a power of two) threads along a row.  WIDE: two pieces of eight, where the output's
// rows start on 16 bytes and the codes' on 8; else single values (8 <= across <= 32).  Either way the threads' pieces lie side
// by side.  ld: elements from row to row of the output; columns d..ld of it are left as they are.  A code's byte, its sign bit
// turned, in the low byte of 2^23 is the number 2^23 + 128 + code.
template <int DT, bool WIDE>
__global__ void __launch_bounds__(256) checkpoint_restore_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scales,
                                                                 int64_t t, int64_t d, int across, typename Type<DT>::T* __restrict__ out,
                                                                 int64_t ld) {
    typedef typename Type<DT>::T T;
    const int64_t nb = (d + BLOCK - 1) / BLOCK;
    const int lane = threadIdx.x & (across - 1);
    const int64_t c = (int64_t)blockIdx.x * across * 16 + lane * (WIDE ? 8 : 1);
    if (c >= d) return;
    const int down = 256 / across;
    const bool both = c + across * 8 < d;
    for (int64_t row = (int64_t)blockIdx.y * down + threadIdx.x / across; row < t; row += (int64_t)gridDim.y * down) {
        const int8_t* src = codes + row * d + c;
        T* dst = out + row * ld + c;
        if constexpr (WIDE) {
            const float* scale = scales + row * nb;
            const uint2 w[2] = {__ldcs(reinterpret_cast<const uint2*>(src)), both ? __ldcs(reinterpret_cast<const uint2*>(src + across * 8)) : make_uint2(0, 0)};
            const float s[2] = {scale_of<DT>(scale[c / BLOCK]), both ? scale_of<DT>(scale[(c + across * 8) / BLOCK]) : 0.0f};
#pragma unroll
            for (int i = 0; i < 2; i++) {
                alignas(16) T r[8];
#pragma unroll
                for (int k = 0; k < 8; k += 2) {
                    const uint32_t v = (k < 4 ? w[i].x : w[i].y) ^ 0x80808080u;
                    const Pair q = add2({__uint_as_float(__byte_perm(v, 0x4b000000u, 0x7540 + k % 4)), __uint_as_float(__byte_perm(v, 0x4b000000u, 0x7540 + k % 4 + 1))},
                                        {-8388736.0f, -8388736.0f});
                    const Pair p = mul2(q, {s[i], s[i]});
                    r[k] = Type<DT>::down(p.x), r[k + 1] = Type<DT>::down(p.y);
                }
                if (i == 0 || both) {
#pragma unroll
                    for (int k = 0; k < (int)sizeof(r) / 16; k++) reinterpret_cast<uint4*>(dst + i * across * 8)[k] = reinterpret_cast<uint4*>(r)[k];
                }
            }
        } else {
            const int n = (int)min((int64_t)16, (d - c + across - 1) / across);
            const float* scale = scales + row * nb + (c - lane) / BLOCK;  // a CTA's first column begins a block
            int8_t q[16];
#pragma unroll
            for (int k = 0; k < 16; k++) q[k] = k < n ? __ldcs(src + k * across) : (int8_t)0;
#pragma unroll
            for (int k = 0; k < 16; k += 4) {  // four values of a thread lie in one block
                const float s = k < n ? scale_of<DT>(scale[k * across / BLOCK]) : 0.0f;
#pragma unroll
                for (int i = k; i < k + 4; i++)
                    if (i < n) dst[i * across] = Type<DT>::down(__fmul_rn((float)q[i], s));
            }
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
    const int across = power_of_two(nb, SAVE_GROUPS);
    const int64_t gx = ceil_div(nb, across);
    auto kern = wide ? checkpoint_save_kernel<DT, true> : checkpoint_save_kernel<DT, false>;
    CDCLQ_LAUNCH(kern, dim3((unsigned)gx, grid_rows(ceil_div(t, SAVE_GROUPS / across), gx)), 256, 0, st, static_cast<const T*>(x), ldx, t, d,
                 across, codes, scales);
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : cuda_error(e, "checkpoint_save_kernel launch");
}

template <int DT>
int restore(const int8_t* codes, const float* scales, int64_t t, int64_t d, void* out, int64_t ld, cudaStream_t st) {
    typedef typename Type<DT>::T T;
    const bool wide = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && (ld * sizeof(T)) % 16 == 0 &&
                      (reinterpret_cast<uintptr_t>(codes) & 7) == 0 && d % 8 == 0;
    const int across = wide ? power_of_two(ceil_div(d, 16), 256) : std::max(8, power_of_two(ceil_div(d, 16), 32));
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
    if (int rc = check_fail_word("checkpoint_save")) return rc;
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
    if (int rc = check_fail_word("checkpoint_restore")) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == CDCLQ_DTYPE_F32) return restore<CDCLQ_DTYPE_F32>(codes, scales, t, d, out, ldo, st);
    return restore_half(dtype == CDCLQ_DTYPE_BF16, codes, scales, t, d, out, ldo, st);
}

extern "C" size_t cdclq_checkpoint_weight_grad_workspace(size_t t, size_t d, size_t n) {
    if (!t || !d || !n || t > MOST_SIZE || d > MOST_SIZE || n > MOST_SIZE) return 0;
    return grad_layout(t, d, n).total;
}

extern "C" int cdclq_checkpoint_weight_grad_device(const void* dy, size_t lddy, int dtype, const int8_t* codes, const float* scales,
                                                   size_t t, size_t d, size_t n, void* dw, size_t lddw, void* workspace,
                                                   size_t workspace_bytes, void* stream) {
    if (dtype != CDCLQ_DTYPE_F16 && dtype != CDCLQ_DTYPE_BF16)
        return set_error(CDCLQ_ERR_ARG, "checkpoint_weight_grad: dtype must be f16 or bf16");
    if (!d || !n) return 0;
    if (!dw || lddw < d) return set_error(CDCLQ_ERR_ARG, "checkpoint_weight_grad: null pointer, or rows overlap");
    if (t > MOST_SIZE || d > MOST_SIZE || n > MOST_SIZE) return set_error(CDCLQ_ERR_ARG, "checkpoint_weight_grad: too large");
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

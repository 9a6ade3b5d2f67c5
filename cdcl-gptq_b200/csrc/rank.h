// rank.h - products of tokens with their own adapters' low-rank factors.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "mma16.cuh"

namespace cdclq {

// p_t = x_t M_i^T (M_i: r x k) or, transposed, x_t M_i (M_i: k x r) for the adapter i = index[t] of each token, f32 sums.
// A token without an adapter has 0.
struct RankArgs {
    const uint16_t* x;      // [t][ldx], rows on 16 bytes
    int64_t ldx;
    int t, k;
    const uint16_t* m;      // [n][r][ldm] or [n][k][ldm], rows on 16 bytes
    int64_t ldm;
    const int* index;
    int n, r;
    const float* scale;     // [n]
    uint16_t* u16;          // p, rounded, [t][ldu], or null
    int64_t ldu;
    uint16_t* su16;         // scale p, rounded, [t][lds], or null
    int* past;              // [t], written, or null: whether some of the token's scale p are past f16, which are then 0 in su16 and
                            // in su32 alone (an infinity or a NaN is in both)
    uint16_t* rest16;       // what that rounding took off, rounded, [t][lds], or null
    int64_t lds;
    float* su32;            // scale p, [t][r], or null
    uint32_t* top;          // [n], written: the bits of each adapter's largest finite |scale p|, or null
    int* start;             // [n + 2], written: the adapters' token lists (and that of the tokens without), each one's first place in
    int* order;             // [t], written: ascending tokens, adapter by adapter
    // the launch's own
    int groups, cut, rp;
};
int launch_rank(bool bf16, bool transposed, RankArgs p, cudaStream_t st);

// su32 under each adapter's gain as the sum of two f16 numbers: 22 bits of every value that is within 2^-15 of the largest, and
// 2^-38 of that one where smaller.  Without the gain they end at 2^-24 and 65504.  The expansion's last CTAs do it, which takes the
// backward pass of 4100 tokens, rank 64, no longer; done by the outer products for each of their tiles it took 13 us of 203.
struct RankSplit {
    const float* v = nullptr;       // su32
    const uint32_t* top = nullptr;  // as RankArgs leaves it
    const int* index = nullptr;
    int t = 0, n = 0, r = 0;
    int64_t ld = 0;                 // of high and low: r rounded up to 8; past r they hold zeros
    uint16_t *high = nullptr, *low = nullptr;  // rows of tokens without an adapter are left as they are
    int ctas = 0;                   // that share the work
};
// 2^13 / 2^floor(log2 top), between 2^-114 and 2^100
__device__ __forceinline__ float rank_gain(uint32_t top) {
    return __uint_as_float((uint32_t)(127 + min(140 - (int)(top >> 23), 100)) << 23);
}
// CTA `part` of S.ctas.
__device__ __forceinline__ void rank_split(const RankSplit& S, int part) {
    const int across = (int)(S.ld / 8);
    for (int64_t i = (int64_t)part * blockDim.x + threadIdx.x; i < (int64_t)S.t * across; i += (int64_t)S.ctas * blockDim.x) {
        const int64_t row = i / across;
        const int c = (int)(i - row * across) * 8, id = S.index[row];
        if (id < 0 || id >= S.n) continue;
        const float gain = rank_gain(S.top[id]);
        const float* v = S.v + row * S.r + c;
        alignas(16) uint16_t h[8], l[8];
#pragma unroll
        for (int q = 0; q < 8; q++) {
            const float x = c + q < S.r ? v[q] * gain : 0.0f;
            h[q] = half_bits<false>(x);
            l[q] = rest_bits<false>(x, h[q]);
        }
        *reinterpret_cast<uint4*>(S.high + row * S.ld + c) = *reinterpret_cast<uint4*>(h);
        *reinterpret_cast<uint4*>(S.low + row * S.ld + c) = *reinterpret_cast<uint4*>(l);
    }
}
// Its CTAs, for a launch of its own or beside other work.
int rank_split_ctas(const RankSplit& s, int threads);
int launch_rank_split(RankSplit s, cudaStream_t st);

}  // namespace cdclq

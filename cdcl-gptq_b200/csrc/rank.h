// rank.h - products of tokens with their own adapters' low-rank factors.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

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
    uint16_t* rest16;       // what that rounding took off, rounded, [t][lds], or null
    int64_t lds;
    float* su32;            // scale p, [t][r], or null
    int* start;             // [n + 2], written: the adapters' token lists (and that of the tokens without), each one's first place in
    int* order;             // [t], written: ascending tokens, adapter by adapter
    // the launch's own
    int groups, cut, rp;
};
int launch_rank(bool bf16, bool transposed, RankArgs p, cudaStream_t st);

}  // namespace cdclq

// packed.h - a packed layer laid out for products with activations, and the kernels that read it.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "cdclq.h"
#include "common.cuh"
#include "half_gemm.h"
#include "rank.h"

namespace cdclq {

// The layout.  Rows in tiles of 16; the permuted columns in k-steps of 16 (each column group padded to whole steps), four
// k-steps of one code width to a unit.  A (row tile, unit) is `bits` words for each of 32 lanes, word-major: lane l holds
// the 8 codes of each k-step that the m16n8k16 tensor instruction wants of it, rows l / 4 and l / 4 + 8, columns
// 2 (l % 4) + {0, 1, 8, 9}.  The width is cut into planes of 4, 2 and 1 bits (3 = 2 + 1, 8 = 4 + 4), low bits first; a plane
// keeps the codes of a column pair 16 bits apart, so that one shift and one AND give both.
struct PackedUnit {
    uint32_t word;     // first word of the unit in a row tile, in units of 32 lanes
    uint32_t bits;
    uint16_t group[4]; // column group of each k-step (repeated for padding)
};

struct PackedView {
    int d_out, d_in, groups, units, tiles;
    int tile_words;            // words of a row tile, in units of 32 lanes
    int max_bits;
    int bits;                  // the width of every group, 0 where they differ
    const PackedUnit* unit;    // [units]
    const int* column;         // [64 * units]: original column of a padded place, -1 for padding
    const uint32_t* place;     // [d_in, rounded up to 4 with zeros]: padded place of an original column
    const uint32_t* grid;      // [tiles][groups][16]: f16 scale in the low half, zero point in the high half
    const uint32_t* codes;     // [tiles][32 * tile_words]
};

// Points into the layout buffer of `w`.
PackedView packed_view(const cdclq_packed_layer& w);

// W (d_out x d_in, original column order, ldw elements from row to row: d_in rounded up to 8, rows on 16 bytes; what lies past
// d_in holds anything) rounded once to f16 or bf16.  beside: the launch before
// it in the stream neither writes what it reads nor reads what it writes, so that they may run side by side.
// lists: built along the way, by CTAs of their own; split: done by others, once the launch before it has ended.
int launch_packed_expand(const PackedView& w, bool bf16, void* out, int64_t ldw, const RowLists& lists, RankSplit split, bool beside,
                         cudaStream_t st);

// Largest number of tokens of the single-token form.  It costs a pass over the codes for every 32 tokens, the expanded form one
// expansion: 2048 x 2048 in 3 bits 12.3 us for 32 tokens and 28 us for 33, 4096 x 4096 in 4 bits 20.6 and 38 us, 11008 x 4096
// 45 and 73 us.  A second pass would bring it level with the expansion.
constexpr int DECODE_TOKENS = 32;
size_t packed_decode_workspace(const PackedView& w, int t, int rank);

struct AdapterArgs {
    const void* a;      // [n][r][lda]
    const void* b;      // [n][d_out][ldb]
    int64_t lda, ldb;
    const float* scale; // [n]
    const int* index;   // [t]
    int n, r;
};
// y = W x + scale B A x for up to DECODE_TOKENS tokens; u (t x r) = A x where wanted.
int launch_packed_decode(const PackedView& w, bool bf16, const void* x, int64_t ldx, int t, const AdapterArgs& ad, void* y,
                         int64_t ldy, void* u, void* workspace, cudaStream_t st);

}  // namespace cdclq

// packed.cu - the packed format (src/quant.rs:106-151) laid out for products with activations: the layout itself, its
// expansion to a 16-bit matrix, and the product with a few tokens.
#include <algorithm>
#include <exception>
#include <type_traits>
#include <vector>

#include "half_gemm.h"
#include "mma16.cuh"
#include "packed.h"
#include "tcgen05.cuh"

namespace cdclq {

namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t align_up(size_t b) { return (b + 255) & ~(size_t)255; }

struct Sections {
    size_t unit, column, place, grid, codes, total;
};
Sections sections(uint64_t d_out, uint64_t d_in, uint64_t groups, uint64_t units, uint64_t tile_words) {
    const uint64_t tiles = (d_out + 15) / 16;
    Sections s;
    size_t at = 0;
    s.unit = at, at += align_up(units * sizeof(PackedUnit));
    s.column = at, at += align_up(units * 64 * sizeof(int));
    s.place = at, at += align_up((d_in + 3) / 4 * 4 * sizeof(uint32_t));
    s.grid = at, at += align_up(tiles * groups * 16 * sizeof(uint32_t));
    s.codes = at, at += align_up(tiles * tile_words * 32 * sizeof(uint32_t));
    s.total = at;
    return s;
}

// The units of a layer; false when the groups' widths are not 2..8.
bool plan_units(size_t d_in, size_t g, const uint8_t* gbits, std::vector<PackedUnit>* unit, std::vector<int>* column,
                uint64_t* units, uint64_t* tile_words, int* max_bits, int* min_bits) {
    const size_t ng = (d_in + g - 1) / g;
    uint64_t n = 0, words = 0;
    int most = 0, least = 8;
    for (size_t i = 0; i < ng;) {
        const int bits = gbits[i];
        if (bits < 2 || bits > 8) return false;
        most = std::max(most, bits);
        least = std::min(least, bits);
        size_t steps = 0;
        for (; i < ng && gbits[i] == bits; i++) {
            const size_t c0 = i * g, width = std::min(g, d_in - c0);
            for (size_t k = 0; k < width; k += 16, steps++) {
                if (!unit) continue;
                if (steps % 4 == 0) {
                    PackedUnit u;
                    u.word = (uint32_t)(words + steps / 4 * bits);
                    u.bits = (uint32_t)bits;
                    for (int q = 0; q < 4; q++) u.group[q] = (uint16_t)i;
                    unit->push_back(u);
                    column->resize(column->size() + 64, -1);
                }
                for (size_t q = steps % 4; q < 4; q++) unit->back().group[q] = (uint16_t)i;
                int* place = column->data() + column->size() - 64 + steps % 4 * 16;
                for (size_t c = 0; c < std::min<size_t>(16, width - k); c++) place[c] = (int)(c0 + k + c);
            }
        }
        const uint64_t here = (steps + 3) / 4;
        n += here;
        words += here * bits;
    }
    *units = n;
    *tile_words = words;
    *max_bits = most;
    *min_bits = least;
    return true;
}

// Planes of a code width, low bits first: bits of each (0: none).
__host__ __device__ constexpr int plane_bits(int bits, int p) {
    const int first = bits >= 4 ? 4 : bits >= 2 ? 2 : 1;
    if (p == 0) return first;
    const int rest = bits - first;
    if (rest == 0) return 0;
    const int second = rest >= 4 ? 4 : rest >= 2 ? 2 : 1;
    if (p == 1) return second;
    return rest - second;
}

// One thread for each word of the layout.  `column` still holds permuted places here.
__global__ void __launch_bounds__(256) packed_layout_kernel(const uint8_t* __restrict__ q, int64_t row_bytes, int d_out, int g,
                                                            const uint64_t* __restrict__ group_bit, const PackedUnit* __restrict__ unit,
                                                            const int* __restrict__ column, int tiles, int tile_words,
                                                            const int* __restrict__ unit_of, uint32_t* codes) {
    const int64_t total = (int64_t)tiles * tile_words * 32;
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int lane = (int)(i & 31);
        const int64_t wi = (i >> 5) % tile_words, tile = (i >> 5) / tile_words;
        const int u = unit_of[wi], bits = (int)unit[u].bits;
        int w = (int)(wi - unit[u].word), shift = 0, pb = 0;
        for (int p = 0; p < 3; p++) {
            pb = plane_bits(bits, p);
            if (w < pb) break;
            w -= pb;
            shift += pb;
        }
        const int per = 16 / pb;
        uint32_t out = 0;
        for (int s = 0; s < per; s++) {
            const int slot = w * per + s, ks = slot / 4, pair = slot % 4;
            const int row = (int)(tile * 16) + lane / 4 + (pair & 1) * 8;
            for (int odd = 0; odd < 2; odd++) {
                const int k = (lane & 3) * 2 + odd + (pair & 2) * 4;
                const int j = column[u * 64 + ks * 16 + k];
                if (j < 0 || row >= d_out) continue;
                const uint64_t bit = group_bit[j / g] + (uint64_t)(j % g) * bits;
                const uint8_t* src = q + row * row_bytes + (bit >> 3);
                uint32_t v = src[0];
                if ((bit & 7) + bits > 8) v |= (uint32_t)src[1] << 8;
                const uint32_t code = (v >> (bit & 7)) & ((1u << bits) - 1u);
                out |= ((code >> shift) & ((1u << pb) - 1u)) << (pb * s + 16 * odd);
            }
        }
        codes[i] = out;
    }
}

// column: permuted place -> original column; place: its inverse.  A perm that is not one raises *bad.
__global__ void __launch_bounds__(256) packed_columns_kernel(const int* __restrict__ perm, int places, int d_in, int* column,
                                                             uint32_t* place, int* seen, int* bad) {
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < places; i += gridDim.x * blockDim.x) {
        const int j = column[i];
        int c = -1;
        if (j >= 0) {
            c = perm[j];
            if (c < 0 || c >= d_in || atomicAdd(&seen[c], 1)) {
                *bad = 1;
                c = -1;
            }
            column[i] = c;
            if (c >= 0) place[c] = i;
        }
    }
}

__global__ void __launch_bounds__(256) packed_grid_kernel(const uint16_t* __restrict__ scales, const uint8_t* __restrict__ zeros,
                                                          const uint8_t* __restrict__ gbits, int d_out, int groups, int tiles,
                                                          uint32_t* grid, int* bad) {
    const int64_t total = (int64_t)tiles * groups * 16;
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int r = (int)(i & 15), g = (int)((i >> 4) % groups);
        const int64_t row = (i >> 4) / groups * 16 + r;
        uint32_t v = 0;
        if (row < d_out) {
            const uint32_t z = zeros[row * groups + g];
            if (z >> gbits[g]) *bad = 2;
            v = scales[row * groups + g] | z << 16;
        }
        grid[i] = v;
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Expansion to a 16-bit matrix in the original column order.

// A pair of small whole numbers (16 bits each) as f16 or bf16, minus a zero point, exactly: the numbers go into the low
// bits of a float whose last place is 1 (f16 1024, bf16 128), and the same offset plus the zero point comes off.
template <bool BF16>
__device__ __forceinline__ uint32_t minus_zero(uint32_t q, uint32_t offset_zero) {
    if constexpr (BF16) {
        const uint32_t v = q | 0x43004300u;
        __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&offset_zero));
        return *reinterpret_cast<uint32_t*>(&r);
    } else {
        const uint32_t v = q | 0x64006400u;
        __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&offset_zero));
        return *reinterpret_cast<uint32_t*>(&r);
    }
}
template <bool BF16>
__device__ __forceinline__ uint32_t pair_of(float v) {
    const uint32_t h = half_bits<BF16>(v);
    return h | h << 16;
}
// What minus_zero (or, for 8 bits in bf16, decode_pair) takes off for the zero point of a grid word: its 16 high bits are
// the zero point, which lies in the low bits of the offset's significand.
template <bool BF16, int BITS>
__device__ __forceinline__ uint32_t zero_pair(uint32_t scale_zero) {
    if constexpr (BF16 && BITS == 8) return pair_of<BF16>((float)(scale_zero >> 16));
    return __byte_perm(scale_zero | (BF16 ? 0x43000000u : 0x64000000u), 0, 0x3232);
}

// Code minus zero point, exactly, of pair p (0..3) of a k-step: rows l / 4 (even pairs) and l / 4 + 8.  For 8 bits in bf16,
// which holds whole numbers to 256 only, the two nibbles are brought in one by one.
template <bool BF16, int BITS>
__device__ __forceinline__ uint32_t decode_pair(const uint32_t (&w)[BITS], int ks, int p, uint32_t zero) {
    const int slot = ks * 4 + p;
    if constexpr (BITS == 8 && BF16) {
        const uint32_t lo = (w[slot / 4] >> (4 * (slot % 4))) & 0x000f000fu, hi = (w[4 + slot / 4] >> (4 * (slot % 4))) & 0x000f000fu;
        const uint32_t h = hi | 0x45004500u, h0 = 0x45004500u;  // 2048 + 16 hi, 2048
        const uint32_t l = lo | 0x43004300u, l0 = 0x43004300u;  // 128 + lo, 128
        typedef __nv_bfloat162 B2;
        const B2 high = __hsub2(*reinterpret_cast<const B2*>(&h), *reinterpret_cast<const B2*>(&h0));
        const B2 low = __hsub2(*reinterpret_cast<const B2*>(&l), *reinterpret_cast<const B2*>(&l0));
        B2 r = __hadd2(__hsub2(high, *reinterpret_cast<const B2*>(&zero)), low);
        return *reinterpret_cast<uint32_t*>(&r);
    } else {
        uint32_t q = 0;
        int at = 0, shift = 0;
#pragma unroll
        for (int plane = 0; plane < 3; plane++) {
            const int pb = plane_bits(BITS, plane);
            if (pb) {
                const int per = 16 / pb;
                const uint32_t m = (1u << pb) - 1u;
                q |= ((w[at + slot / per] >> (pb * (slot % per))) & (m | m << 16)) << shift;
                at += pb;
                shift += pb;
            }
        }
        return minus_zero<BF16>(q, zero);
    }
}

// scale * (code - zero point) of a pair, rounded once: the product of an 11-bit and an 8-bit significand is exact in f32, and
// f16's own product is that product rounded.
template <bool BF16>
__device__ __forceinline__ uint32_t scaled_pair(uint32_t d, uint32_t scale_f16) {
    if constexpr (BF16) {
        const uint32_t s = __float_as_uint(__half2float(__ushort_as_half((uint16_t)scale_f16)));
        uint64_t p;
        asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(p) : "l"((uint64_t)(d & 0xffff0000u) << 32 | d << 16), "l"((uint64_t)s << 32 | s));
        __nv_bfloat162 r = __floats2bfloat162_rn(__uint_as_float((uint32_t)p), __uint_as_float((uint32_t)(p >> 32)));
        return *reinterpret_cast<uint32_t*>(&r);
    } else {
        const uint32_t ss = scale_f16 | scale_f16 << 16;
        __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&d), *reinterpret_cast<const __half2*>(&ss));
        return *reinterpret_cast<uint32_t*>(&r);
    }
}

constexpr int EXPAND_WARPS = 16;
constexpr size_t EXPAND_SMEM = 220 * 1024;
constexpr size_t EXPAND_LIST_BYTES = (512 + EXPAND_WARPS) * sizeof(int);  // of a tile's list of adapters

// The unit's codes of one half of the tile's rows, scaled, to their places; sz: the first k-step's grid word, `at`: the lane's
// row of its first place of the unit.
template <bool BF16, int BITS, int R>
__device__ __forceinline__ void expand_unit(const uint16_t (&group)[4], uint32_t (&w)[BITS], const uint32_t* __restrict__ g,
                                            uint32_t sz, int half, bool live, uint16_t* at) {
    // the upper rows' codes follow the lower rows' in every plane
    int word = 0;
#pragma unroll
    for (int plane = 0; plane < 3; plane++) {
        const int pb = plane_bits(BITS, plane);
#pragma unroll
        for (int i = 0; i < pb; i++) w[word + i] >>= half * pb;
        word += pb;
    }
    auto step = [&](int ks, uint32_t sz, uint32_t zero) {
        const uint32_t lo = scaled_pair<BF16>(decode_pair<BF16, BITS>(w, ks, 0, zero), sz & 0xffffu);
        const uint32_t hi = scaled_pair<BF16>(decode_pair<BF16, BITS>(w, ks, 2, zero), sz & 0xffffu);
        if (R == 8 || live) {
            at[(ks * 16 + 0) * R] = (uint16_t)lo;
            at[(ks * 16 + 1) * R] = (uint16_t)(lo >> 16);
            at[(ks * 16 + 8) * R] = (uint16_t)hi;
            at[(ks * 16 + 9) * R] = (uint16_t)(hi >> 16);
        }
    };
    if (group[0] == group[3]) {
        const uint32_t zero = zero_pair<BF16, BITS>(sz);
#pragma unroll
        for (int ks = 0; ks < 4; ks++) step(ks, sz, zero);
    } else {
#pragma unroll
        for (int ks = 0; ks < 4; ks++) {
            const uint32_t s = ks ? g[(int64_t)group[ks] * 16] : sz;
            step(ks, s, zero_pair<BF16, BITS>(s));
        }
    }
}

// The adapters of the rows of one tile, in order of their first rows (see row_list_words).  Small integers at a CTA's leisure
// while others expand the weight: of the product's loop it would be the longest part, 2000 clocks an adapter.
__device__ void build_row_list(const RowLists& L, int tile, int* ids) {
    const int R = L.rows, i = threadIdx.x, row = tile * R + i, lane = i & 31;
    int* place = ids + 256;   // of an adapter's first row
    int* before = ids + 512;  // first rows of each warp
    uint32_t* out = L.out + (int64_t)tile * row_list_words(R);
    int id = i < R && row < L.m ? L.index[row] : -1;
    if (id >= L.adapters) id = -1;
    if (i < R) ids[i] = id;
    __syncthreads();
    int first = i;
    if (i < R && id >= 0)
        for (int j = R - 1; j >= 0; j--)
            if (ids[j] == id) first = j;
    const bool leads = i < R && id >= 0 && first == i;
    const uint32_t leaders = __ballot_sync(0xffffffffu, leads);
    if (lane == 0) before[i >> 5] = __popc(leaders);
    __syncthreads();
    int at = __popc(leaders & ((1u << lane) - 1u)), count = 0;
    for (int w = 0; w < R / 32; w++) {
        if (w < (i >> 5)) at += before[w];
        count += before[w];
    }
    if (leads) place[i] = at, out[ROW_LIST_IDS + at] = id;
    if (i == 0) out[0] = count;
    uint32_t* mask = out + row_list_masks(R);
    for (int k = i; k < count * (R / 32); k += blockDim.x) mask[k] = 0xffffffffu;
    __syncthreads();
    const uint32_t same = __match_any_sync(0xffffffffu, id);
    if (i < R && id >= 0 && lane == __ffs(same) - 1) mask[place[first] * (R / 32) + (i >> 5)] = ~same;
}

// R values of neighbouring rows at one place.
template <int R>
struct Rows;
template <>
struct Rows<8> { typedef uint4 T; };
template <>
struct Rows<4> { typedef uint2 T; };
template <>
struct Rows<2> { typedef uint32_t T; };
template <>
struct Rows<1> { typedef uint16_t T; };

// A CTA expands R of a tile's 16 rows (8, unless they do not fit).  Warps decode unit by unit into shared memory, the R rows'
// values of a place side by side: no two lanes meet in a bank, and addresses are constants.  Then every thread gathers four
// neighbouring columns, a place of R values at once, and the warps write along the rows.  BITS: the width of every group, or 0
// where they differ.  A weight is rounded to 16 bits here, as the tensor cores take them.
// 4096 x 4096 in 4 bits to bf16: 14.8 us (2.8 TB/s; values scattered by 2 bytes took 17.4).  Two rounds of CTAs, in each of
// which decoding waits for the codes and writing for the whole row: latency, not a unit that is full.
template <bool BF16, int BITS, int R>
__global__ void __launch_bounds__(EXPAND_WARPS * 32) packed_expand_kernel(const PackedView W, uint16_t* __restrict__ out, int64_t ldw,
                                                                          const RowLists lists, const RankSplit split) {
    extern __shared__ __align__(16) uint16_t places[];
    if ((int)blockIdx.x < lists.tiles) {
        build_row_list(lists, blockIdx.x, reinterpret_cast<int*>(places));
        if (blockIdx.x == 0) wait_for_previous();
        return;
    }
    if ((int)(gridDim.x - blockIdx.x) <= split.ctas) {
        wait_for_previous();
        rank_split(split, gridDim.x - 1 - blockIdx.x);
        return;
    }
    constexpr int PARTS = 16 / R;
    const int here = blockIdx.x - lists.tiles, tile = here / PARTS, first = here % PARTS * R;  // rows first .. first + R of the tile
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int half = first >> 3, r0 = lane / 4 - (first & 7);
    const bool live = r0 >= 0 && r0 < R;
    uint16_t* mine = places + (lane & 3) * 2 * R + (live ? r0 : 0);
    const uint32_t* codes = W.codes + (int64_t)tile * W.tile_words * 32 + lane;
    const uint32_t* g = W.grid + (int64_t)tile * W.groups * 16 + half * 8 + lane / 4;
    if constexpr (BITS) {
        // the next unit's codes and scale, and the groups of the one after it, are on their way while this one is decoded; units
        // of one width follow one another
        const int last = W.units - 1;
        uint32_t ahead[BITS], sz_ahead;
        uint2 group_ahead;
        auto groups = [&](int ui) { return *reinterpret_cast<const uint2*>(W.unit[min(ui, last)].group); };
        uint2 group_next = groups(warp);
#pragma unroll
        for (int i = 0; i < BITS; i++) ahead[i] = codes[(min(warp, last) * BITS + i) * 32];
        group_ahead = groups(warp + EXPAND_WARPS);
        sz_ahead = g[(int64_t)(group_next.x & 0xffffu) * 16];
        for (int ui = warp; ui <= last; ui += EXPAND_WARPS) {
            uint32_t w[BITS];
            alignas(8) uint16_t group[4];
            *reinterpret_cast<uint2*>(group) = group_next;
            const uint32_t sz = sz_ahead;
#pragma unroll
            for (int i = 0; i < BITS; i++) w[i] = ahead[i];
            const int next = min(ui + EXPAND_WARPS, last) * BITS;
#pragma unroll
            for (int i = 0; i < BITS; i++) ahead[i] = codes[(next + i) * 32];
            group_next = group_ahead;
            sz_ahead = g[(int64_t)(group_next.x & 0xffffu) * 16];
            group_ahead = groups(ui + 2 * EXPAND_WARPS);
            expand_unit<BF16, BITS, R>(group, w, g, sz, half, live, mine + (int64_t)ui * 64 * R);
        }
    } else {
        auto unit = [&](auto width, const PackedUnit& u, int ui) {
            constexpr int B = decltype(width)::value;
            uint32_t w[B];
#pragma unroll
            for (int i = 0; i < B; i++) w[i] = codes[(u.word + i) * 32];
            expand_unit<BF16, B, R>(u.group, w, g, g[(int64_t)u.group[0] * 16], half, live, mine + (int64_t)ui * 64 * R);
        };
        PackedUnit after = W.unit[min(warp, W.units - 1)];
        for (int ui = warp; ui < W.units; ui += EXPAND_WARPS) {
            const PackedUnit u = after;
            after = W.unit[min(ui + EXPAND_WARPS, W.units - 1)];
            switch (u.bits) {
                case 2: unit(std::integral_constant<int, 2>(), u, ui); break;
                case 3: unit(std::integral_constant<int, 3>(), u, ui); break;
                case 4: unit(std::integral_constant<int, 4>(), u, ui); break;
                case 5: unit(std::integral_constant<int, 5>(), u, ui); break;
                case 6: unit(std::integral_constant<int, 6>(), u, ui); break;
                case 7: unit(std::integral_constant<int, 7>(), u, ui); break;
                default: unit(std::integral_constant<int, 8>(), u, ui); break;
            }
        }
    }
    __syncthreads();
    const int rows_here = min(R, W.d_out - tile * 16 - first);
    uint16_t* dst = out + ((int64_t)tile * 16 + first) * ldw;
    for (int c = threadIdx.x * 4; c < W.d_in; c += EXPAND_WARPS * 32 * 4) {
        typedef typename Rows<R>::T T;
        const uint4 p = *reinterpret_cast<const uint4*>(W.place + c);
        alignas(16) T v[4] = {reinterpret_cast<const T*>(places)[p.x], reinterpret_cast<const T*>(places)[p.y],
                              reinterpret_cast<const T*>(places)[p.z], reinterpret_cast<const T*>(places)[p.w]};
        const uint16_t* h = reinterpret_cast<const uint16_t*>(v);
#pragma unroll
        for (int r = 0; r < R; r++)
            if (r < rows_here)
                *reinterpret_cast<uint2*>(dst + r * ldw + c) =
                    make_uint2((uint32_t)h[r] | (uint32_t)h[R + r] << 16, (uint32_t)h[2 * R + r] | (uint32_t)h[3 * R + r] << 16);
    }
    if (blockIdx.x == 0) wait_for_previous();
}

template <bool BF16, int BITS, int R>
int expand(const PackedView& w, void* out, int64_t ldw, const RowLists& lists, const RankSplit& split, bool beside, cudaStream_t st) {
    static std::atomic<uint64_t> done{0};
    auto kern = packed_expand_kernel<BF16, BITS, R>;
    if (int rc = allow_smem(kern, EXPAND_SMEM, done, "packed_expand_kernel shared memory")) return rc;
    return launch_after(beside, kern, dim3(lists.tiles + w.tiles * (16 / R) + split.ctas), dim3(EXPAND_WARPS * 32),
                        std::max((size_t)w.units * 64 * R * 2, EXPAND_LIST_BYTES), st, "packed_expand_kernel launch", w,
                        static_cast<uint16_t*>(out), ldw, lists, split);
}

// The widths of configurations that quantize every group alike have a kernel of their own; the others, and rows too long for
// eight of them, share those that branch by unit.
template <bool BF16>
int expand_any(const PackedView& w, void* out, int64_t ldw, const RowLists& lists, const RankSplit& split, bool beside, cudaStream_t st) {
    const size_t row = (size_t)w.units * 64 * 2;
    if (row > EXPAND_SMEM) return set_error(CDCLQ_ERR_ARG, "packed layer: a row of over 112000 columns cannot be expanded");
    if (row * 8 > EXPAND_SMEM) {
        if (row * 4 <= EXPAND_SMEM) return expand<BF16, 0, 4>(w, out, ldw, lists, split, beside, st);
        return row * 2 <= EXPAND_SMEM ? expand<BF16, 0, 2>(w, out, ldw, lists, split, beside, st) : expand<BF16, 0, 1>(w, out, ldw, lists, split, beside, st);
    }
    switch (w.bits) {
        case 2: return expand<BF16, 2, 8>(w, out, ldw, lists, split, beside, st);
        case 3: return expand<BF16, 3, 8>(w, out, ldw, lists, split, beside, st);
        case 4: return expand<BF16, 4, 8>(w, out, ldw, lists, split, beside, st);
        case 8: return expand<BF16, 8, 8>(w, out, ldw, lists, split, beside, st);
        default: return expand<BF16, 0, 8>(w, out, ldw, lists, split, beside, st);
    }
}

}  // namespace

PackedView packed_view(const cdclq_packed_layer& w) {
    const Sections s = sections(w.d_out, w.d_in, w.groups, w.units, w.tile_words);
    const char* base = static_cast<const char*>(w.layout);
    PackedView v;
    v.d_out = (int)w.d_out, v.d_in = (int)w.d_in, v.groups = (int)w.groups, v.units = (int)w.units;
    v.tiles = (v.d_out + 15) / 16;
    v.tile_words = (int)w.tile_words;
    v.max_bits = (int)w.max_bits;
    v.bits = (int)w.bits;
    v.unit = reinterpret_cast<const PackedUnit*>(base + s.unit);
    v.column = reinterpret_cast<const int*>(base + s.column);
    v.place = reinterpret_cast<const uint32_t*>(base + s.place);
    v.grid = reinterpret_cast<const uint32_t*>(base + s.grid);
    v.codes = reinterpret_cast<const uint32_t*>(base + s.codes);
    return v;
}

int launch_packed_expand(const PackedView& w, bool bf16, void* out, int64_t ldw, const RowLists& lists, RankSplit split, bool beside,
                         cudaStream_t st) {
    if (split.v) split.ctas = rank_split_ctas(split, EXPAND_WARPS * 32);
    return bf16 ? expand_any<true>(w, out, ldw, lists, split, beside, st) : expand_any<false>(w, out, ldw, lists, split, beside, st);
}

// ---------------------------------------------------------------------------------------------------------------------
// The product with a few tokens.

namespace {

using namespace tc;

constexpr int DEC_GROUPS = 8, DEC_WARPS = 16, DEC_THREADS = DEC_WARPS * 32;
// shared memory: two slots of codes (at least one row tile of 8 bits), sums, the units' table, the grid
constexpr int DEC_RING = 160 * 1024, DEC_SUMS = 44 * 1024, DEC_TABLE = 4 * 1024, DEC_SMEM = 226 * 1024;

// First launch: x in the tensor instruction's order (its columns gathered through the permutation, padding zero), and
// u_t = A_i x_t, some warps for each (token, rank).
template <bool BF16>
__global__ void __launch_bounds__(256) packed_tokens_kernel(const PackedView W, const uint16_t* __restrict__ x, int64_t ldx, int t,
                                                            int token_tiles, uint2* __restrict__ xf, int frag_blocks, int cut,
                                                            const AdapterArgs ad, float* __restrict__ u32, uint16_t* __restrict__ u16) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if ((int)blockIdx.x >= frag_blocks) {
        // `cut` warps (a power of two) to a product, each with 2048 neighbouring columns at a time
        __shared__ float part[8];
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        const int w = (blockIdx.x - frag_blocks) * (8 / cut) + warp / cut;
        const int tok = w / ad.r, r = w - tok * ad.r, id = w < t * ad.r ? ad.index[tok] : -1;
        float s = 0.0f;
        if (id >= 0 && id < ad.n) {
            const uint16_t* a = static_cast<const uint16_t*>(ad.a) + ((int64_t)id * ad.r + r) * ad.lda;
            const uint16_t* xr = x + tok * ldx;
            float p[8] = {};
            for (int c0 = (warp & (cut - 1)) * 2048; c0 < W.d_in; c0 += cut * 2048) {
                uint4 av[8], xv[8];
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const int c = c0 + k * 256 + lane * 8;
                    av[k] = xv[k] = make_uint4(0, 0, 0, 0);
                    if (c + 8 <= W.d_in) {
                        av[k] = *reinterpret_cast<const uint4*>(a + c);
                        xv[k] = *reinterpret_cast<const uint4*>(xr + c);
                    } else {
                        for (int q = c; q < W.d_in; q++) p[0] = fmaf(half_value<BF16>(a[q]), half_value<BF16>(xr[q]), p[0]);
                    }
                }
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const uint32_t aw[4] = {av[k].x, av[k].y, av[k].z, av[k].w}, xw[4] = {xv[k].x, xv[k].y, xv[k].z, xv[k].w};
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        p[2 * q] = fmaf(half_value<BF16>((uint16_t)aw[q]), half_value<BF16>((uint16_t)xw[q]), p[2 * q]);
                        p[2 * q + 1] = fmaf(half_value<BF16>((uint16_t)(aw[q] >> 16)), half_value<BF16>((uint16_t)(xw[q] >> 16)), p[2 * q + 1]);
                    }
                }
            }
            s = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
            for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        }
        if (lane == 0) part[warp] = s;
        __syncthreads();
        if (lane == 0 && (warp & (cut - 1)) == 0 && w < t * ad.r) {
            for (int k = 1; k < cut; k++) s += part[warp + k];
            u32[w] = s;
            if (u16) u16[w] = half_bits<BF16>(s);
        }
        return;
    }
    const int i = blockIdx.x * 256 + threadIdx.x, total = W.units * 4 * token_tiles * 32;
    if (i >= total) return;
    const int lane = i & 31, nt = (i >> 5) % token_tiles, step = (i >> 5) / token_tiles;
    const int tok = nt * 8 + lane / 4;
    const int2* column = reinterpret_cast<const int2*>(W.column + step * 16) + (lane & 3);
    const int2 c0 = column[0], c1 = column[4];
    const uint16_t* xr = x + (int64_t)min(tok, t - 1) * ldx;
    const uint32_t a = c0.x >= 0 ? xr[c0.x] : 0, b = c0.y >= 0 ? xr[c0.y] : 0, c = c1.x >= 0 ? xr[c1.x] : 0, d = c1.y >= 0 ? xr[c1.y] : 0;
    xf[i] = tok < t ? make_uint2(a | b << 16, c | d << 16) : make_uint2(0, 0);
}

// One unit of a row tile times NT token tiles.  codes: the unit's words; grid: the tile's, one word for each (group, row).
template <bool BF16, int BITS, int NT>
__device__ __forceinline__ void decode_unit(const PackedUnit& u, const uint32_t* codes, const uint32_t* grid, const uint2 (&x)[4][NT],
                                            int lane, float (&acc)[NT][4]) {
    uint32_t w[BITS];
#pragma unroll
    for (int i = 0; i < BITS; i++) w[i] = codes[i * 32 + lane];
    const uint32_t* g = grid + lane / 4;
    if (u.group[0] == u.group[3]) {  // one column group: its four k-steps share a scale
        const uint32_t s0 = g[u.group[0] * 16], s1 = g[u.group[0] * 16 + 8];
        const uint32_t zero[2] = {zero_pair<BF16, BITS>(s0), zero_pair<BF16, BITS>(s1)};
        float part[NT][4] = {};
#pragma unroll
        for (int ks = 0; ks < 4; ks++) {
            uint32_t a[4];
#pragma unroll
            for (int p = 0; p < 4; p++) a[p] = decode_pair<BF16, BITS>(w, ks, p, zero[p & 1]);
#pragma unroll
            for (int n = 0; n < NT; n++) mma16816<BF16>(part[n], a, x[ks][n].x, x[ks][n].y);
        }
        const float f0 = __half2float(__ushort_as_half((uint16_t)s0)), f1 = __half2float(__ushort_as_half((uint16_t)s1));
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[n][i] = fmaf(i < 2 ? f0 : f1, part[n][i], acc[n][i]);
    } else {
#pragma unroll
        for (int ks = 0; ks < 4; ks++) {
            const uint32_t s0 = g[u.group[ks] * 16], s1 = g[u.group[ks] * 16 + 8];
            const uint32_t zero[2] = {zero_pair<BF16, BITS>(s0), zero_pair<BF16, BITS>(s1)};
            const float f0 = __half2float(__ushort_as_half((uint16_t)s0)), f1 = __half2float(__ushort_as_half((uint16_t)s1));
            uint32_t a[4];
#pragma unroll
            for (int p = 0; p < 4; p++) a[p] = decode_pair<BF16, BITS>(w, ks, p, zero[p & 1]);
#pragma unroll
            for (int n = 0; n < NT; n++) {
                float part[4] = {};
                mma16816<BF16>(part, a, x[ks][n].x, x[ks][n].y);
#pragma unroll
                for (int i = 0; i < 4; i++) acc[n][i] = fmaf(i < 2 ? f0 : f1, part[i], acc[n][i]);
            }
        }
    }
}

struct DecodeArgs {
    const uint2* xf;
    const float* u32;
    uint16_t* y;
    int64_t ldy;
    int t;
    int tiles;        // row tiles of a CTA
    int pass_tiles;   // of them at a time
    int table_staged; // the units' table in shared memory
    int grid_staged;  // the grid of all the CTA's row tiles in shared memory
    int* fail;
};

// Units of a pass through shared memory: DEC_GROUPS groups of warps with DEC_UNITS units each, whose tokens stay in registers
// for all the row tiles.
__host__ __device__ constexpr int dec_units(int nt) { return nt == 4 ? 2 : 4; }
__host__ __device__ constexpr int dec_chunk(int nt) { return DEC_GROUPS * dec_units(nt); }
// Sums of a group of warps: [row tile of the pass][token][16 rows + 1].
__host__ __device__ constexpr int dec_sums(int nt) { return nt * 8 * 17; }

// Second launch: one CTA to an SM, each with its share of the row tiles.  Bulk copies bring a chunk of the units' codes for
// all row tiles of a pass into one of two slots, the first two before the first launch has finished (they do not depend on
// it): at 4 bits a layer of 4096 x 11008 is then in flight at once.  Warp w has the units of group w % 8 and the row tiles of
// parity w / 8; a token's bytes cross L2 once for all rows of a CTA.  The scale of a (row, group) multiplies the group's f32
// sum, so the codes minus their zero points enter the tensor instruction exactly and no weight is rounded.
// Bound by the codes' bytes and, below some MB, by latency; mma.sync because 16 rows and a few tokens leave most of tcgen05's
// 128 rows empty.  2048 x 2048 in 3 bits, 1 token: 4.7 us after the first launch's 3.0; 11008 x 4096 in 4 bits, 12 tokens of
// 12 adapters: 16.8 us (27 MB, 1.6 TB/s) after 3.8.
template <bool BF16, int BITS, int NT>
__global__ void __launch_bounds__(DEC_THREADS, 1) packed_decode_kernel(const PackedView W, const AdapterArgs ad, const DecodeArgs P) {
    extern __shared__ __align__(128) uint32_t smem[];
    constexpr int UNITS = dec_units(NT), CHUNK = dec_chunk(NT);
    __shared__ uint64_t ready[2];
    __shared__ int flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = warp % DEC_GROUPS, parity = warp / DEC_GROUPS;
    const int tile0 = blockIdx.x * P.tiles, tiles = min(P.tiles, W.tiles - tile0);
    const int chunks = (W.units + CHUNK - 1) / CHUNK, passes = (tiles + P.pass_tiles - 1) / P.pass_tiles, fills = chunks * passes;
    const int tile_words = CHUNK * W.max_bits * 32, slot_words = P.pass_tiles * tile_words;
    uint32_t* table_s = smem + 2 * slot_words;
    uint32_t* grid_s = table_s + (P.table_staged ? W.units * 4 : 0);
    float* sums = reinterpret_cast<float*>(grid_s + (P.grid_staged ? P.tiles * W.groups * 16 : 0));
    const uint32_t* grid = P.grid_staged ? grid_s : W.grid + (int64_t)tile0 * W.groups * 16;
    const PackedUnit* table = P.table_staged ? reinterpret_cast<const PackedUnit*>(table_s) : W.unit;
    auto word_of = [&](int u) -> uint32_t { return u >= W.units ? (uint32_t)W.tile_words : BITS ? (uint32_t)(u * BITS) : W.unit[u].word; };
    auto fetch = [&](int f, uint32_t more) {
        const int t0 = f / chunks * P.pass_tiles, n = min(P.pass_tiles, tiles - t0), u0 = f % chunks * CHUNK;
        const uint32_t w0 = word_of(u0), bytes = (word_of(u0 + CHUNK) - w0) * 128;
        mbar_expect_tx(&ready[f & 1], n * bytes + more);
        for (int i = 0; i < n; i++)
            bulk_load(smem_u32(smem + (f & 1) * slot_words + i * tile_words), W.codes + ((int64_t)(tile0 + t0 + i) * W.tile_words + w0) * 32,
                      bytes, &ready[f & 1]);
    };
    if (threadIdx.x == 0) {
        mbar_init(&ready[0], 1);
        mbar_init(&ready[1], 1);
        flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        const uint32_t tb = P.table_staged ? W.units * 16 : 0, gb = P.grid_staged ? tiles * W.groups * 64 : 0;
        fetch(0, tb + gb);
        if (tb) bulk_load(smem_u32(table_s), W.unit, tb, &ready[0]);
        if (gb) bulk_load(smem_u32(grid_s), W.grid + (int64_t)tile0 * W.groups * 16, gb, &ready[0]);
        if (fills > 1) fetch(1, 0);
    }
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int f = 0; f < fills; f++) {
        const int t0 = f / chunks * P.pass_tiles, n = min(P.pass_tiles, tiles - t0), c = f % chunks;
        const int u0 = c * CHUNK + group * UNITS;
        uint2 x[UNITS][4][NT];
#pragma unroll
        for (int q = 0; q < UNITS; q++)
#pragma unroll
            for (int ks = 0; ks < 4; ks++)
#pragma unroll
                for (int k = 0; k < NT; k++)
                    x[q][ks][k] = u0 + q < W.units ? P.xf[((int64_t)((u0 + q) * 4 + ks) * NT + k) * 32 + lane] : make_uint2(0, 0);
        const bool there = mbar_wait_warp(&ready[f & 1], (f >> 1) & 1, &flag);
        const uint32_t w0 = word_of(c * CHUNK);
        for (int tl = there ? parity : n; tl < n; tl += DEC_WARPS / DEC_GROUPS) {
            const uint32_t* codes = smem + (f & 1) * slot_words + tl * tile_words;
            const uint32_t* g = grid + (t0 + tl) * W.groups * 16;
            float acc[NT][4];
            float* mine = sums + (group * P.pass_tiles + tl) * dec_sums(NT) + (lane & 3) * 34 + lane / 4;
#pragma unroll
            for (int k = 0; k < NT; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) acc[k][i] = c ? mine[(k * 8 + (i & 1)) * 17 + (i >> 1) * 8] : 0.0f;
#pragma unroll
            for (int q = 0; q < UNITS; q++) {
                if (u0 + q >= W.units) break;
                const PackedUnit u = table[u0 + q];
                const uint32_t* cw = codes + (u.word - w0) * 32;
                if constexpr (BITS) {
                    decode_unit<BF16, BITS, NT>(u, cw, g, x[q], lane, acc);
                } else {
                    switch (u.bits) {
                        case 2: decode_unit<BF16, 2, NT>(u, cw, g, x[q], lane, acc); break;
                        case 3: decode_unit<BF16, 3, NT>(u, cw, g, x[q], lane, acc); break;
                        case 4: decode_unit<BF16, 4, NT>(u, cw, g, x[q], lane, acc); break;
                        case 5: decode_unit<BF16, 5, NT>(u, cw, g, x[q], lane, acc); break;
                        case 6: decode_unit<BF16, 6, NT>(u, cw, g, x[q], lane, acc); break;
                        case 7: decode_unit<BF16, 7, NT>(u, cw, g, x[q], lane, acc); break;
                        default: decode_unit<BF16, 8, NT>(u, cw, g, x[q], lane, acc); break;
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < NT; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) mine[(k * 8 + (i & 1)) * 17 + (i >> 1) * 8] = acc[k][i];
        }
        // the slot is free, the sums are there; where a wait ran out all leave together, the copies on their way first (bounded)
        if (__syncthreads_or(!there)) {
            if (threadIdx.x == 0) {
                int own = 0;
                mbar_wait(&ready[f & 1], (f >> 1) & 1, &own);
                if (f + 1 < fills) mbar_wait(&ready[(f + 1) & 1], ((f + 1) >> 1) & 1, &own);
            }
            __syncthreads();
            break;
        }
        if (threadIdx.x == 0 && f + 2 < fills) fetch(f + 2, 0);
        if (c + 1 < chunks) continue;
        for (int i = threadIdx.x; i < n * 16 * P.t; i += DEC_THREADS) {
            const int r = i & 15, tl = i / 16 % n, tok = i / 16 / n, row = (tile0 + t0 + tl) * 16 + r;
            if (row >= W.d_out) continue;
            float s = 0.0f;
#pragma unroll
            for (int q = 0; q < DEC_GROUPS; q++) s += sums[(q * P.pass_tiles + tl) * dec_sums(NT) + tok * 17 + r];
            const int id = ad.n > 0 ? ad.index[tok] : -1;
            if (id >= 0 && id < ad.n) {
                const uint16_t* b = static_cast<const uint16_t*>(ad.b) + ((int64_t)id * W.d_out + row) * ad.ldb;
                const float* u = P.u32 + tok * ad.r;
                float v = 0.0f;
                int k = 0;
                for (; k + 8 <= ad.r; k += 8) {
                    const uint4 q = *reinterpret_cast<const uint4*>(b + k);
                    const uint32_t bw[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        v = fmaf(half_value<BF16>((uint16_t)bw[j]), u[k + 2 * j], v);
                        v = fmaf(half_value<BF16>((uint16_t)(bw[j] >> 16)), u[k + 2 * j + 1], v);
                    }
                }
                for (; k < ad.r; k++) v = fmaf(half_value<BF16>(b[k]), u[k], v);
                s = fmaf(ad.scale[id], v, s);
            }
            P.y[tok * P.ldy + row] = half_bits<BF16>(s);
        }
        __syncthreads();  // the sums may be written again
    }
    if (threadIdx.x == 0 && flag) {
        *(volatile int*)P.fail = 1;
        __threadfence_system();
    }
}

template <bool BF16, int BITS, int NT>
int decode_tokens(const PackedView& w, const AdapterArgs& ad, DecodeArgs p, cudaStream_t st) {
    // as many row tiles at a time as the two slots and the sums hold
    const int tile_bytes = dec_chunk(NT) * w.max_bits * 128, sum_bytes = DEC_GROUPS * dec_sums(NT) * 4;
    p.tiles = (int)ceil_div(w.tiles, sm_count());
    const int most = std::max(1, std::min(DEC_RING / (2 * tile_bytes), DEC_SUMS / sum_bytes));
    p.pass_tiles = (int)ceil_div(p.tiles, ceil_div(p.tiles, most));
    size_t smem = (size_t)p.pass_tiles * (2 * tile_bytes + sum_bytes);
    p.table_staged = w.units * 16 <= DEC_TABLE;
    if (p.table_staged) smem += (size_t)w.units * 16;
    p.grid_staged = smem + (size_t)p.tiles * w.groups * 64 <= DEC_SMEM;
    if (p.grid_staged) smem += (size_t)p.tiles * w.groups * 64;
    auto kern = packed_decode_kernel<BF16, BITS, NT>;
    static std::atomic<uint64_t> done{0};
    if (int rc = allow_smem(kern, DEC_SMEM, done, "packed_decode_kernel shared memory")) return rc;
    return launch_after(true, kern, dim3((unsigned)ceil_div(w.tiles, p.tiles)), dim3(DEC_THREADS), smem, st, "packed_decode_kernel launch",
                            w, ad, p);
}

template <bool BF16, int BITS>
int decode_width(const PackedView& w, const AdapterArgs& ad, const DecodeArgs& p, int nt, cudaStream_t st) {
    if (nt == 1) return decode_tokens<BF16, BITS, 1>(w, ad, p, st);
    return nt == 2 ? decode_tokens<BF16, BITS, 2>(w, ad, p, st) : decode_tokens<BF16, BITS, 4>(w, ad, p, st);
}

int token_tiles(int t) { return t <= 8 ? 1 : t <= 16 ? 2 : 4; }

template <bool BF16>
int decode(const PackedView& w, const void* x, int64_t ldx, int t, const AdapterArgs& ad, void* y, int64_t ldy, void* u,
           void* workspace, cudaStream_t st) {
    const int nt = token_tiles(t);
    uint2* xf = static_cast<uint2*>(workspace);
    DecodeArgs p{};
    p.xf = xf;
    float* u32 = reinterpret_cast<float*>(static_cast<char*>(workspace) + align_up((size_t)w.units * 4 * nt * 32 * sizeof(uint2)));
    p.u32 = u32;
    p.y = static_cast<uint16_t*>(y);
    p.ldy = ldy;
    p.t = t;
    p.fail = device_fail_word();
    if (!p.fail) return set_error(CDCLQ_ERR_CUDA, "projection_forward: no mapped host memory (is there a CUDA device?)");
    const int frag_blocks = (int)ceil_div((int64_t)w.units * 4 * nt * 32, 256);
    int cut = 1;
    while (cut < 8 && cut * 2048 < w.d_in) cut *= 2;
    const int dot_blocks = ad.n > 0 ? (int)ceil_div((int64_t)t * ad.r * cut, 8) : 0;
    CDCLQ_LAUNCH((packed_tokens_kernel<BF16>), frag_blocks + dot_blocks, 256, 0, st, w, static_cast<const uint16_t*>(x), ldx, t, nt, xf,
                 frag_blocks, cut, ad, u32, static_cast<uint16_t*>(u));
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_error(e, "packed_tokens_kernel launch");
    switch (w.bits) {
        case 2: return decode_width<BF16, 2>(w, ad, p, nt, st);
        case 3: return decode_width<BF16, 3>(w, ad, p, nt, st);
        case 4: return decode_width<BF16, 4>(w, ad, p, nt, st);
        case 8: return decode_width<BF16, 8>(w, ad, p, nt, st);
        default: return decode_width<BF16, 0>(w, ad, p, nt, st);
    }
}

}  // namespace

size_t packed_decode_workspace(const PackedView& w, int t, int rank) {
    return align_up((size_t)w.units * 4 * token_tiles(t) * 32 * sizeof(uint2)) + align_up((size_t)t * rank * sizeof(float));
}

int launch_packed_decode(const PackedView& w, bool bf16, const void* x, int64_t ldx, int t, const AdapterArgs& ad, void* y,
                         int64_t ldy, void* u, void* workspace, cudaStream_t st) {
    return bf16 ? decode<true>(w, x, ldx, t, ad, y, ldy, u, workspace, st) : decode<false>(w, x, ldx, t, ad, y, ldy, u, workspace, st);
}

}  // namespace cdclq

using namespace cdclq;

static int plan_layer(size_t d_out, size_t d_in, size_t group, const uint8_t* gbits, cdclq_packed_layer* w,
                      std::vector<PackedUnit>* unit, std::vector<int>* column) {
    if (!gbits || !w) return set_error(CDCLQ_ERR_ARG, "packed layer: null pointer");
    if (!d_out || !d_in) return set_error(CDCLQ_ERR_ARG, "packed layer: d_out and d_in must be > 0");
    if (d_out > 0x7ffffff0 || d_in > (1u << 24)) return set_error(CDCLQ_ERR_ARG, "packed layer: too large");
    const size_t g = group && group < d_in ? group : d_in;
    if ((d_in + g - 1) / g > 65535) return set_error(CDCLQ_ERR_ARG, "packed layer: more than 65535 column groups");
    uint64_t units = 0, words = 0;
    int most = 0, least = 0;
    if (!plan_units(d_in, g, gbits, unit, column, &units, &words, &most, &least))
        return set_error(CDCLQ_ERR_CONFIG, "packed layer: group widths must be in 2..=8 bits");
    w->d_out = d_out, w->d_in = d_in, w->group = g, w->groups = (d_in + g - 1) / g;
    w->units = units, w->tile_words = words, w->max_bits = (uint32_t)most;
    w->bits = most == least ? (uint32_t)most : 0;
    return 0;
}

extern "C" size_t cdclq_packed_layer_bytes(size_t d_out, size_t d_in, size_t group, const uint8_t* gbits) {
    cdclq_packed_layer w{};
    if (plan_layer(d_out, d_in, group, gbits, &w, nullptr, nullptr)) return 0;
    return sections(w.d_out, w.d_in, w.groups, w.units, w.tile_words).total;
}

static int build_layer(const uint8_t* qweight, const void* scales_f16, const uint8_t* qzeros, const int32_t* perm, size_t d_out,
                       size_t d_in, size_t group, const uint8_t* gbits, void* layout, size_t layout_bytes, cdclq_packed_layer* out,
                       void* stream) {
    if (!qweight || !scales_f16 || !qzeros || !perm || !layout || !out) return set_error(CDCLQ_ERR_ARG, "packed layer: null pointer");
    cdclq_packed_layer w{};
    std::vector<PackedUnit> unit;
    std::vector<int> column;
    int rc = plan_layer(d_out, d_in, group, gbits, &w, &unit, &column);
    if (rc) return rc;
    const Sections s = sections(w.d_out, w.d_in, w.groups, w.units, w.tile_words);
    if (layout_bytes < s.total || (reinterpret_cast<uintptr_t>(layout) & 255))
        return set_error(CDCLQ_ERR_ARG, "packed layer: the layout buffer is too small or not on 256 bytes");
    w.layout = layout;
    const PackedView v = packed_view(w);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const size_t ng = w.groups, g = w.group;
    // bit of a row's stream at which each group starts, and the unit of each word
    std::vector<uint64_t> group_bit(ng);
    uint64_t bit = 0;
    for (size_t i = 0; i < ng; i++) {
        group_bit[i] = bit;
        bit += (uint64_t)gbits[i] * std::min<size_t>(g, d_in - i * g);
    }
    std::vector<int> unit_of;
    for (size_t i = 0; i < unit.size(); i++) unit_of.insert(unit_of.end(), unit[i].bits, (int)i);
    const int64_t row_bytes = (int64_t)((bit + 7) / 8);
    // temporary: group starts, unit of each word, widths, permutation check, verdict
    const size_t o1 = align_up(ng * 8), o2 = o1 + align_up(unit_of.size() * 4), o3 = o2 + align_up(ng), o4 = o3 + align_up(d_in * 4);
    char* tmp = nullptr;
    CDCLQ_CUDA_TRY(cudaMallocAsync((void**)&tmp, o4 + 256, st));
    int bad = 0;
    cudaError_t e = cudaMemcpyAsync(tmp, group_bit.data(), ng * 8, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) e = cudaMemcpyAsync(tmp + o1, unit_of.data(), unit_of.size() * 4, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) e = cudaMemcpyAsync(tmp + o2, gbits, ng, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) e = cudaMemsetAsync(const_cast<uint32_t*>(v.place), 0, (d_in + 3) / 4 * 4 * sizeof(uint32_t), st);
    if (e == cudaSuccess) e = cudaMemsetAsync(tmp + o3, 0, o4 - o3 + 256, st);
    if (e == cudaSuccess) e = cudaMemcpyAsync(const_cast<PackedUnit*>(v.unit), unit.data(), unit.size() * sizeof(PackedUnit), cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) e = cudaMemcpyAsync(const_cast<int*>(v.column), column.data(), column.size() * 4, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) {
        int* verdict = reinterpret_cast<int*>(tmp + o4);
        const unsigned most = sm_count() * 16;
        const int64_t words = (int64_t)v.tiles * v.tile_words * 32, cells = (int64_t)v.tiles * v.groups * 16;
        CDCLQ_LAUNCH(packed_layout_kernel, (unsigned)std::min<int64_t>(most, ceil_div(words, 256)), 256, 0, st, qweight, row_bytes, v.d_out,
                     (int)g, reinterpret_cast<const uint64_t*>(tmp), v.unit, v.column, v.tiles, v.tile_words,
                     reinterpret_cast<const int*>(tmp + o1), const_cast<uint32_t*>(v.codes));
        CDCLQ_LAUNCH(packed_grid_kernel, (unsigned)std::min<int64_t>(most, ceil_div(cells, 256)), 256, 0, st,
                     static_cast<const uint16_t*>(scales_f16), qzeros, reinterpret_cast<const uint8_t*>(tmp + o2), v.d_out, v.groups,
                     v.tiles, const_cast<uint32_t*>(v.grid), verdict);
        CDCLQ_LAUNCH(packed_columns_kernel, (unsigned)std::min<int64_t>(most, ceil_div(v.units * 64, 256)), 256, 0, st, perm, v.units * 64,
                     v.d_in, const_cast<int*>(v.column), const_cast<uint32_t*>(v.place),
                     reinterpret_cast<int*>(tmp + o3), verdict);
        e = cudaGetLastError();
        if (e == cudaSuccess) e = cudaMemcpyAsync(&bad, verdict, sizeof(int), cudaMemcpyDeviceToHost, st);
    }
    cudaError_t f = cudaStreamSynchronize(st);
    cudaFreeAsync(tmp, st);
    if (e == cudaSuccess) e = f;
    if (e != cudaSuccess) return cuda_error(e, "packed layer layout");
    if (bad == 1) return set_error(CDCLQ_ERR_ARG, "packed layer: perm is not a permutation of the columns");
    if (bad == 2) return set_error(CDCLQ_ERR_ARG, "packed layer: a zero point is above the largest code of its group");
    *out = w;
    return 0;
}

extern "C" int cdclq_packed_layer_build(const uint8_t* qweight, const void* scales_f16, const uint8_t* qzeros, const int32_t* perm,
                                        size_t d_out, size_t d_in, size_t group, const uint8_t* gbits, void* layout,
                                        size_t layout_bytes, cdclq_packed_layer* out, void* stream) {
    try {
        return build_layer(qweight, scales_f16, qzeros, perm, d_out, d_in, group, gbits, layout, layout_bytes, out, stream);
    } catch (const std::exception& e) {  // host memory
        return set_error(CDCLQ_ERR_ARG, std::string("packed layer: ") + e.what());
    }
}

// packed.cu - the packed format (src/quant.rs:106-151) laid out for products with activations: the layout itself, its
// expansion to a 16-bit matrix, and the product with a few tokens.
#include <algorithm>
#include <exception>
#include <vector>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "half_gemm.h"
#include "packed.h"

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
    s.place = at, at += align_up(d_in * sizeof(int));
    s.grid = at, at += align_up(tiles * groups * 16 * sizeof(uint32_t));
    s.codes = at, at += align_up(tiles * tile_words * 32 * sizeof(uint32_t));
    s.total = at;
    return s;
}

// The units of a layer; false when the groups' widths are not 2..8.
bool plan_units(size_t d_in, size_t g, const uint8_t* gbits, std::vector<PackedUnit>* unit, std::vector<int>* column,
                uint64_t* units, uint64_t* tile_words, int* max_bits) {
    const size_t ng = (d_in + g - 1) / g;
    uint64_t n = 0, words = 0;
    int most = 0;
    for (size_t i = 0; i < ng;) {
        const int bits = gbits[i];
        if (bits < 2 || bits > 8) return false;
        most = std::max(most, bits);
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

// Code of k-step `ks`, column pair `pair` (0..3: see PackedUnit's lanes), member `odd`, from a lane's words `stride` apart.
template <typename Words>
__device__ __forceinline__ uint32_t code_at(Words w, int stride, int bits, int ks, int pair, int odd) {
    uint32_t code = 0;
    int shift = 0;
#pragma unroll
    for (int p = 0; p < 3; p++) {
        const int pb = plane_bits(bits, p);
        if (pb == 0) break;
        const int slot = ks * 4 + pair;                  // of the unit's 16 pairs
        const int per = pb == 4 ? 4 : pb == 2 ? 8 : 16;  // pairs in a word of the plane
        const uint32_t v = w[(slot / per) * stride];
        code |= ((v >> (pb * (slot % per) + 16 * odd)) & ((1u << pb) - 1u)) << shift;
        w += pb * stride;
        shift += pb;
    }
    return code;
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
__global__ void __launch_bounds__(256) packed_columns_kernel(const int* __restrict__ perm, int places, int d_in, int* column, int* place,
                                                             int* seen, int* bad) {
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < places; i += gridDim.x * blockDim.x) {
        const int j = column[i];
        if (j < 0) continue;
        const int c = perm[j];
        if (c < 0 || c >= d_in || atomicAdd(&seen[c], 1)) {
            *bad = 1;
            column[i] = -1;
            continue;
        }
        column[i] = c;
        place[c] = i;
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

template <bool BF16>
__device__ __forceinline__ uint16_t half_bits(float v) {
    return BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}
template <bool BF16>
__device__ __forceinline__ float half_value(uint16_t v) {
    return BF16 ? __uint_as_float((uint32_t)v << 16) : __half2float(__ushort_as_half(v));
}

// A row tile's 16 rows in the original column order: its codes are staged in shared memory (their places are a permutation),
// a thread takes two columns so that a warp writes 128 bytes along a row.
template <bool BF16>
__global__ void __launch_bounds__(512) packed_expand_kernel(const PackedView W, int staged, uint16_t* __restrict__ out, int64_t ldw,
                                                            int pairs_wide) {
    extern __shared__ uint32_t words[];
    const int tile = blockIdx.x;
    const uint32_t* codes = W.codes + (int64_t)tile * W.tile_words * 32;
    if (staged) {
        for (int i = threadIdx.x * 4; i < W.tile_words * 32; i += blockDim.x * 4)
            *reinterpret_cast<uint4*>(words + i) = *reinterpret_cast<const uint4*>(codes + i);
        __syncthreads();
    }
    const uint32_t* grid = W.grid + (int64_t)tile * W.groups * 16;
    const int rows = min(16, W.d_out - tile * 16);
    const int c_step = gridDim.y * blockDim.x * 2;
    for (int c = (blockIdx.y * blockDim.x + threadIdx.x) * 2; c < W.d_in; c += c_step) {
        const int n = min(2, W.d_in - c);
        uint32_t res[16];
#pragma unroll
        for (int r = 0; r < 16; r++) res[r] = 0;
        for (int e = 0; e < n; e++) {
            const int p = W.place[c + e];
            const PackedUnit u = W.unit[p >> 6];
            const int ks = (p >> 4) & 3, k = p & 15;
            const uint32_t* gs = grid + (int64_t)u.group[ks] * 16;
            const int first = (int)u.word * 32 + ((k & 7) >> 1);
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int at = first + (r & 7) * 4, pair = (k >> 3) * 2 + (r >> 3);
                const uint32_t q = staged ? code_at(words + at, 32, u.bits, ks, pair, k & 1) : code_at(codes + at, 32, u.bits, ks, pair, k & 1);
                const uint32_t sz = gs[r];
                const float v = __fmul_rn(__half2float(__ushort_as_half((uint16_t)sz)), (float)((int)q - (int)(sz >> 16)));
                res[r] |= (uint32_t)half_bits<BF16>(v) << (16 * e);
            }
        }
        uint16_t* dst = out + (int64_t)tile * 16 * ldw + c;
#pragma unroll
        for (int r = 0; r < 16; r++) {
            if (r >= rows) break;
            if (pairs_wide && n == 2) {
                *reinterpret_cast<uint32_t*>(dst + r * ldw) = res[r];
            } else {
                dst[r * ldw] = (uint16_t)res[r];
                if (n == 2) dst[r * ldw + 1] = (uint16_t)(res[r] >> 16);
            }
        }
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
    v.unit = reinterpret_cast<const PackedUnit*>(base + s.unit);
    v.column = reinterpret_cast<const int*>(base + s.column);
    v.place = reinterpret_cast<const int*>(base + s.place);
    v.grid = reinterpret_cast<const uint32_t*>(base + s.grid);
    v.codes = reinterpret_cast<const uint32_t*>(base + s.codes);
    return v;
}

int launch_packed_expand(const PackedView& w, bool bf16, void* out, int64_t ldw, cudaStream_t st) {
    const size_t bytes = (size_t)w.tile_words * 32 * 4;
    const int staged = bytes <= 200 * 1024;
    auto kern = bf16 ? packed_expand_kernel<true> : packed_expand_kernel<false>;
    if (staged) CDCLQ_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
    const int pairs_wide = ldw % 2 == 0 && (reinterpret_cast<uintptr_t>(out) & 3) == 0;
    // few row tiles: their columns over several CTAs
    const int chunks = (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(sm_count() * 2, w.tiles), ceil_div(w.d_in, 1024)));
    CDCLQ_LAUNCH(kern, dim3(w.tiles, chunks), 512, staged ? bytes : 0, st, w, staged, static_cast<uint16_t*>(out), ldw, pairs_wide);
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : cuda_error(e, "packed_expand_kernel launch");
}

// ---------------------------------------------------------------------------------------------------------------------
// The product with a few tokens.

namespace {

constexpr int DEC_WARPS = 8;

// First launch: x in the tensor instruction's order (its columns gathered through the permutation, padding zero), and
// u_t = A_i x_t, one warp for each (token, rank).
template <bool BF16>
__global__ void __launch_bounds__(256) packed_tokens_kernel(const PackedView W, const uint16_t* __restrict__ x, int64_t ldx, int t,
                                                            int token_tiles, uint2* __restrict__ xf, int frag_blocks,
                                                            const AdapterArgs ad, float* __restrict__ u32, uint16_t* __restrict__ u16) {
    if ((int)blockIdx.x < frag_blocks) {
        const int total = W.units * 4 * token_tiles * 32;
        const int i = blockIdx.x * 256 + threadIdx.x;
        if (i >= total) return;
        const int lane = i & 31, nt = (i >> 5) % token_tiles, step = (i >> 5) / token_tiles;
        const int tok = nt * 8 + lane / 4;
        uint32_t v[4];
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int c = W.column[step * 16 + (lane & 3) * 2 + (q & 1) + (q >> 1) * 8];
            v[q] = (tok < t && c >= 0) ? x[tok * ldx + c] : 0;
        }
        xf[i] = make_uint2(v[0] | v[1] << 16, v[2] | v[3] << 16);
        return;
    }
    const int w = (blockIdx.x - frag_blocks) * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (w >= t * ad.r) return;
    const int tok = w / ad.r, r = w - tok * ad.r, id = ad.index[tok];
    float s = 0.0f;
    if (id >= 0 && id < ad.n) {
        const uint16_t* a = static_cast<const uint16_t*>(ad.a) + ((int64_t)id * ad.r + r) * ad.lda;
        const uint16_t* xr = x + tok * ldx;
        float p[8] = {};
        int c = lane * 8;
        for (; c + 8 <= W.d_in; c += 256) {
            const uint4 av = *reinterpret_cast<const uint4*>(a + c), xv = *reinterpret_cast<const uint4*>(xr + c);
            const uint32_t aw[4] = {av.x, av.y, av.z, av.w}, xw[4] = {xv.x, xv.y, xv.z, xv.w};
#pragma unroll
            for (int q = 0; q < 4; q++) {
                p[2 * q] = fmaf(half_value<BF16>((uint16_t)aw[q]), half_value<BF16>((uint16_t)xw[q]), p[2 * q]);
                p[2 * q + 1] = fmaf(half_value<BF16>((uint16_t)(aw[q] >> 16)), half_value<BF16>((uint16_t)(xw[q] >> 16)), p[2 * q + 1]);
            }
        }
        for (; c < W.d_in; c++) p[0] = fmaf(half_value<BF16>(a[c]), half_value<BF16>(xr[c]), p[0]);  // one lane's last columns
        s = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    }
    if (lane == 0) {
        u32[w] = s;
        if (u16) u16[w] = half_bits<BF16>(s);
    }
}

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint2 b) {
    if constexpr (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
}

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

// The code minus zero point pairs of one k-step for the tensor instruction: rows l / 4 (even pairs) and l / 4 + 8.
// zero[]: the rows' zero points as pairs, with the offset of minus_zero; for 8 bits in bf16, which holds whole numbers to
// 256 only, the two nibbles are brought in one by one.
template <bool BF16, int BITS>
__device__ __forceinline__ void decode_step(const uint32_t (&w)[BITS], int ks, const uint32_t (&zero)[2], uint32_t (&a)[4]) {
#pragma unroll
    for (int p = 0; p < 4; p++) {
        const int slot = ks * 4 + p;
        if constexpr (BITS == 8 && BF16) {
            const uint32_t lo = (w[slot / 4] >> (4 * (slot % 4))) & 0x000f000fu, hi = (w[4 + slot / 4] >> (4 * (slot % 4))) & 0x000f000fu;
            const uint32_t h = hi | 0x45004500u;           // 2048 + 16 hi
            const uint32_t base = 0x45004500u;             // 2048
            __nv_bfloat162 high = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&h), *reinterpret_cast<const __nv_bfloat162*>(&base));
            const uint32_t l = lo | 0x43004300u, lbase = 0x43004300u;
            __nv_bfloat162 low = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&l), *reinterpret_cast<const __nv_bfloat162*>(&lbase));
            __nv_bfloat162 z = *reinterpret_cast<const __nv_bfloat162*>(&zero[p & 1]);  // the zero point itself
            __nv_bfloat162 r = __hadd2(__hsub2(high, z), low);
            a[p] = *reinterpret_cast<uint32_t*>(&r);
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
            a[p] = minus_zero<BF16>(q, zero[p & 1]);
        }
    }
}

template <bool BF16, int BITS, int NT>
__device__ __forceinline__ void decode_unit(const PackedView& W, const PackedUnit& u, const uint32_t* __restrict__ codes,
                                            const uint32_t* __restrict__ grid, const uint2* __restrict__ xf, int lane,
                                            float (&acc)[NT][4]) {
    uint32_t w[BITS];
#pragma unroll
    for (int i = 0; i < BITS; i++) w[i] = codes[(u.word + i) * 32 + lane];
    float part[NT][4];
    uint32_t zero[2];
    float scale[2];
#pragma unroll
    for (int ks = 0; ks < 4; ks++) {
        if (ks == 0 || u.group[ks] != u.group[ks - 1]) {
            const uint32_t* g = grid + (int64_t)u.group[ks] * 16 + lane / 4;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t sz = g[h * 8];
                scale[h] = __half2float(__ushort_as_half((uint16_t)sz));
                const float offset = BF16 ? (BITS == 8 ? 0.0f : 128.0f) : 1024.0f;
                zero[h] = pair_of<BF16>((float)(sz >> 16) + offset);
            }
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) part[n][i] = 0.0f;
        }
        uint32_t a[4];
        decode_step<BF16, BITS>(w, ks, zero, a);
#pragma unroll
        for (int n = 0; n < NT; n++) mma16816<BF16>(part[n], a, xf[(ks * NT + n) * 32 + lane]);
        if (ks == 3 || u.group[ks + 1] != u.group[ks]) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) acc[n][i] = fmaf(scale[i >> 1], part[n][i], acc[n][i]);
        }
    }
}

// Second launch: a CTA for each 16 rows, its warps over the units.  The scale of a (row, group) multiplies the group's f32
// sum, so the codes minus their zero points enter the tensor instruction exactly and no weight is rounded.
// Bound by the codes' bytes; mma.sync because M = 16 rows and a few tokens leave tcgen05's 128 rows empty.
template <bool BF16, int NT>
__global__ void __launch_bounds__(DEC_WARPS * 32) packed_decode_kernel(const PackedView W, const uint2* __restrict__ xf, int t,
                                                                       const AdapterArgs ad, const float* __restrict__ u32,
                                                                       uint16_t* __restrict__ y, int64_t ldy) {
    __shared__ float sums[DEC_WARPS][16][NT * 8 + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tile = blockIdx.x;
    const uint32_t* codes = W.codes + (int64_t)tile * W.tile_words * 32;
    const uint32_t* grid = W.grid + (int64_t)tile * W.groups * 16;
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[n][i] = 0.0f;
    for (int ui = warp; ui < W.units; ui += DEC_WARPS) {
        const PackedUnit u = W.unit[ui];
        const uint2* xu = xf + (int64_t)ui * 4 * NT * 32;
        switch (u.bits) {
            case 2: decode_unit<BF16, 2, NT>(W, u, codes, grid, xu, lane, acc); break;
            case 3: decode_unit<BF16, 3, NT>(W, u, codes, grid, xu, lane, acc); break;
            case 4: decode_unit<BF16, 4, NT>(W, u, codes, grid, xu, lane, acc); break;
            case 5: decode_unit<BF16, 5, NT>(W, u, codes, grid, xu, lane, acc); break;
            case 6: decode_unit<BF16, 6, NT>(W, u, codes, grid, xu, lane, acc); break;
            case 7: decode_unit<BF16, 7, NT>(W, u, codes, grid, xu, lane, acc); break;
            default: decode_unit<BF16, 8, NT>(W, u, codes, grid, xu, lane, acc); break;
        }
    }
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) sums[warp][lane / 4 + (i >> 1) * 8][n * 8 + (lane & 3) * 2 + (i & 1)] = acc[n][i];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * t; i += DEC_WARPS * 32) {
        const int r = i & 15, tok = i >> 4, row = tile * 16 + r;
        if (row >= W.d_out) continue;
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < DEC_WARPS; w++) s += sums[w][r][tok];
        const int id = ad.n > 0 ? ad.index[tok] : -1;
        if (id >= 0 && id < ad.n) {
            const uint16_t* b = static_cast<const uint16_t*>(ad.b) + ((int64_t)id * W.d_out + row) * ad.ldb;
            float v = 0.0f;
            for (int k = 0; k < ad.r; k++) v = fmaf(half_value<BF16>(b[k]), u32[tok * ad.r + k], v);
            s = fmaf(ad.scale[id], v, s);
        }
        y[tok * ldy + row] = half_bits<BF16>(s);
    }
}

}  // namespace

static int token_tiles(int t) { return t <= 8 ? 1 : t <= 16 ? 2 : 4; }

size_t packed_decode_workspace(const PackedView& w, int t, int rank) {
    return align_up((size_t)w.units * 4 * token_tiles(t) * 32 * sizeof(uint2)) + align_up((size_t)t * rank * sizeof(float));
}

template <bool BF16>
static int decode(const PackedView& w, const void* x, int64_t ldx, int t, const AdapterArgs& ad, void* y, int64_t ldy, void* u,
                  void* workspace, cudaStream_t st) {
    const int nt = token_tiles(t);
    uint2* xf = static_cast<uint2*>(workspace);
    float* u32 = reinterpret_cast<float*>(static_cast<char*>(workspace) + align_up((size_t)w.units * 4 * nt * 32 * sizeof(uint2)));
    const int frag_blocks = (int)ceil_div((int64_t)w.units * 4 * nt * 32, 256);
    const int dot_blocks = ad.n > 0 ? (int)ceil_div((int64_t)t * ad.r, 8) : 0;
    CDCLQ_LAUNCH((packed_tokens_kernel<BF16>), frag_blocks + dot_blocks, 256, 0, st, w, static_cast<const uint16_t*>(x), ldx, t, nt, xf,
                 frag_blocks, ad, u32, static_cast<uint16_t*>(u));
    uint16_t* out = static_cast<uint16_t*>(y);
    if (nt == 1)
        CDCLQ_LAUNCH((packed_decode_kernel<BF16, 1>), w.tiles, DEC_WARPS * 32, 0, st, w, xf, t, ad, u32, out, ldy);
    else if (nt == 2)
        CDCLQ_LAUNCH((packed_decode_kernel<BF16, 2>), w.tiles, DEC_WARPS * 32, 0, st, w, xf, t, ad, u32, out, ldy);
    else
        CDCLQ_LAUNCH((packed_decode_kernel<BF16, 4>), w.tiles, DEC_WARPS * 32, 0, st, w, xf, t, ad, u32, out, ldy);
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : cuda_error(e, "packed_decode_kernel launch");
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
    if (!d_out || !d_in || !group) return set_error(CDCLQ_ERR_ARG, "packed layer: d_out, d_in and the group size must be > 0");
    if (d_out > 0x7ffffff0 || d_in > (1u << 24)) return set_error(CDCLQ_ERR_ARG, "packed layer: too large");
    const size_t g = group < d_in ? group : d_in;
    if ((d_in + g - 1) / g > 65535) return set_error(CDCLQ_ERR_ARG, "packed layer: more than 65535 column groups");
    uint64_t units = 0, words = 0;
    int most = 0;
    if (!plan_units(d_in, g, gbits, unit, column, &units, &words, &most))
        return set_error(CDCLQ_ERR_CONFIG, "packed layer: group widths must be in 2..=8 bits");
    w->d_out = d_out, w->d_in = d_in, w->group = g, w->groups = (d_in + g - 1) / g;
    w->units = units, w->tile_words = words, w->max_bits = (uint32_t)most;
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
                     v.d_in, const_cast<int*>(v.column), const_cast<int*>(v.place), reinterpret_cast<int*>(tmp + o3), verdict);
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

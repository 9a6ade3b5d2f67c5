// half_gemm.cu - plans and launches the half-precision tensor-core product: tensor maps, tile width, K splits.
#include <algorithm>
#include <atomic>
#include <mutex>

#include "half_gemm_launch.cuh"

namespace cdclq {

using namespace hg;

int sm_count() {
    static std::atomic<int> known[64];  // of each device
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) != cudaSuccess) {
        cudaGetLastError();
        return sms;
    }
    if (dev < 64 && known[dev].load(std::memory_order_relaxed)) return known[dev].load(std::memory_order_relaxed);
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) cudaGetLastError();
    if (dev < 64) known[dev].store(sms, std::memory_order_relaxed);
    return sms;
}

// A word of mapped host memory for each device: the host reads it without a synchronisation.
constexpr int FAIL_DEVICES = 64;
static int* fail_word_host(int device) {
    static int* words = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        if (cudaHostAlloc(&p, FAIL_DEVICES * sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable) == cudaSuccess) {
            words = static_cast<int*>(p);
            std::fill(words, words + FAIL_DEVICES, 0);
        } else {
            cudaGetLastError();
        }
    });
    return words && device >= 0 && device < FAIL_DEVICES ? words + device : nullptr;
}

// Unified addressing: the words have the same addresses on every device.
int* device_fail_word() {
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess) cudaGetLastError();
    return fail_word_host(dev);
}

int check_fail_word(const char* what) {
    int* h = device_fail_word();
    if (!h) return set_error(CDCLQ_ERR_CUDA, std::string(what) + ": no mapped host memory (is there a CUDA device?)");
    if (*(volatile int*)h && __atomic_exchange_n(h, 0, __ATOMIC_RELAXED))
        return set_error(CDCLQ_ERR_CUDA, std::string(what) + ": a pipeline wait of an earlier launch on this device timed out (its outputs "
                                                             "are incomplete); this call has not run");
    return 0;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_tiled() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
        else
            cudaGetLastError();
    });
    return fn;
}

// Map of a 16-bit operand with boxes of 64 columns x box_rows rows (of one matrix of a batch when batched).
static int encode(CUtensorMap* map, const HalfOperand& o, bool bf16, bool batched, int box_rows) {
    EncodeTiledFn enc = encode_tiled();
    if (!enc) return set_error(CDCLQ_ERR_CUDA, "half product: cuTensorMapEncodeTiled is unavailable");
    if ((reinterpret_cast<uintptr_t>(o.p) & 15) || (o.ld & 7) || (o.step & 7) || o.rows <= 0 || o.cols <= 0 || o.ld < o.cols)
        return set_error(CDCLQ_ERR_ARG, "half product: operands need rows that start on 16 bytes");
    cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)o.batch};
    cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)(o.step ? o.step : o.ld * o.rows) * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, batched ? 3 : 2,
                     const_cast<void*>(o.p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(CDCLQ_ERR_CUDA, "half product: tensor map encoding failed");
    return 0;
}

static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The plan of least estimated time, in clocks, from what was measured on products of 2048..8191 rows: what a K block of 64
// costs a tile (512 clocks of MMAs for 256 x 256; its operands' way through L2 for the narrower ones), and what an item costs
// beside (filling the pipeline; a tile of 512 is not taken out of tensor memory while the next one's MMAs run at full rate).
// Splitting K adds the f32 sums' way out and back, and a launch.
HalfPlan plan_half_gemm(HalfForm form, int64_t m, int64_t n, int64_t k) {
    const bool store = form != HALF_STATS && form != HALF_GRAD;
    const int64_t sms = sm_count(), nkb = ceil_div(k, KB);
    HalfPlan p{1, 64, 1, 0};
    static const struct { int cg, bn, block, item; } shapes[] = {
        {2, 512, 1060, 6000}, {2, 256, 630, 3000}, {2, 128, 450, 3000}, {1, 128, 560, 2500}, {1, 64, 430, 2000}};
    double best = 1e300;
    for (const auto& s : shapes) {
        if ((s.bn == 64 && !store) || (s.bn == 512 && form == HALF_STATS)) continue;
        if (s.cg == 2 && m <= BM) continue;  // the second CTA's rows would be empty
        const int64_t tiles = ceil_div(m, s.cg * BM) * ceil_div(n, s.bn), slots = sms / s.cg;
        const int64_t most = store ? std::max<int64_t>(1, std::min(slots / tiles, nkb / 8)) : 1;
        for (int64_t want = 1; want <= most; want++) {
            const int64_t per = ceil_div(nkb, want), splits = ceil_div(nkb, per);
            if (splits != want) continue;
            double cost = (double)ceil_div(tiles * splits, slots) * ((double)per * s.block + s.item);
            if (splits > 1) cost += 6000.0 + (splits + 1.0) * m * n * 4.0 / 2000.0;
            if (cost < best) {
                best = cost;
                p.cg = s.cg, p.bn = s.bn, p.splits = (int)splits;
            }
        }
    }
    if (p.splits > 1) p.partial_bytes = (size_t)p.splits * m * (ceil_div(n, 4) * 4) * sizeof(float);
    return p;
}

int64_t half_stats_parts(const HalfPlan& plan, int64_t n) { return STATS_PARTS * ceil_div(n, plan.bn); }

RowLists row_lists(const HalfPlan& plan, const int* index, int64_t m, int64_t adapters, void* out) {
    RowLists l;
    l.index = index;
    l.m = (int)m, l.adapters = (int)adapters;
    l.rows = plan.cg * BM;
    l.tiles = (int)ceil_div(m, l.rows);
    l.out = static_cast<uint32_t*>(out);
    return l;
}
size_t row_lists_bytes(const HalfPlan& plan, int64_t m) {
    return (size_t)ceil_div(m, plan.cg * BM) * row_list_words(plan.cg * BM) * sizeof(uint32_t);
}

// out = alpha * (f32in + partial[0] + partial[1] + ...), splits in order; also or instead as f32.
template <bool BF16>
__global__ void __launch_bounds__(256) half_gemm_reduce_kernel(const float* __restrict__ partial, int splits, int64_t m, int64_t n,
                                                               int64_t ldp, const float* f32in, float* f32out, int64_t ldf,
                                                               const float* alpha, uint16_t* out, int64_t ldo) {
    const float a = alpha ? *alpha : 1.0f;
    const int64_t total = m * ldp, stride = m * ldp;
    for (int64_t i = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) * 4; i < total; i += (int64_t)gridDim.x * blockDim.x * 4) {
        const int64_t row = i / ldp;
        const int col = (int)(i - row * ldp);
        float4 s = make_float4(0, 0, 0, 0);
        if (f32in) {
            const float* src = f32in + row * ldf + col;
            s.x = src[0];
            if (col + 1 < n) s.y = src[1];
            if (col + 2 < n) s.z = src[2];
            if (col + 3 < n) s.w = src[3];
        }
        for (int k = 0; k < splits; k++) {
            const float4 v = *reinterpret_cast<const float4*>(partial + k * stride + i);
            s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
        }
        const float r[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int q = 0; q < 4; q++) {
            if (col + q >= n) break;
            if (f32out) f32out[row * ldf + col + q] = r[q];
            if (out) out[row * ldo + col + q] = hg::pack1<BF16>(r[q] * a);
        }
    }
}

int launch_half_gemm(const HalfGemm& g, const HalfPlan& plan, cudaStream_t st) {
    if (g.m <= 0 || g.n <= 0) return 0;
    const bool a_mn = g.form == HALF_TN;
    const bool b_mn = g.form == HALF_NN || g.form == HALF_TN || g.form == HALF_NN_EXTEND;
    const bool extend = (g.form == HALF_NT_EXTEND || g.form == HALF_NN_EXTEND) && g.lists;
    if (g.m > (int64_t)MOST_SIZE || g.n > (int64_t)MOST_SIZE || g.k > (int64_t)MOST_SIZE) return set_error(CDCLQ_ERR_ARG, "half product: too large");
    Maps maps{};
    int rc;
    // Where one CTA has all rows, copies bring no others; what the tile's other rows come to is never stored.  (2 tokens x 50292
    // words of 2048, bf16: 65 us with copies of 128 rows, 48 us so.)
    const int a_rows = !a_mn && plan.cg == 1 && g.m <= BM ? (int)ceil_div(g.m, 8) * 8 : BM;
    if ((rc = encode(&maps.a, g.a, g.bf16, false, a_mn ? KB : a_rows))) return rc;
    if ((rc = encode(&maps.b, g.b, g.bf16, false, b_mn ? KB : std::min(plan.bn, 256) / plan.cg))) return rc;
    if (extend && (rc = encode(&maps.u, g.u, g.bf16, false, a_rows))) return rc;
    if (extend && (rc = encode(&maps.x, g.x, g.bf16, true, b_mn ? KB : std::min(plan.bn, 256) / plan.cg))) return rc;
    Params p{};
    p.m = (int)g.m;
    p.n = (int)g.n;
    p.nkb = (int)ceil_div(g.k, KB);
    p.tiles_m = (int)ceil_div(g.m, plan.cg * BM);
    p.tiles_n = (int)ceil_div(g.n, plan.bn);
    if ((int64_t)p.tiles_m * p.tiles_n * plan.splits > 0x7fffffff) return set_error(CDCLQ_ERR_ARG, "half product: too many tiles");
    p.ntiles = p.tiles_m * p.tiles_n;
    p.splits = plan.splits;
    p.stage_bytes = (plan.cg * a_rows + plan.bn) * KB * 2;
    p.kb_per_split = (int)ceil_div(p.nkb, plan.splits);
    p.lists = extend ? g.lists : nullptr;
    p.rank = extend ? (int)g.u.cols : 0;
    if (extend) p.far = g.far;
    p.target = g.target;
    p.col0 = g.col0;
    p.vocab = g.vocab;
    p.stats = g.stats;
    p.label_logit = g.label_logit;
    p.lse = g.lse;
    p.dloss = g.dloss;
    p.gain = g.gain;
    p.fail = device_fail_word();
    if (!p.fail) return set_error(CDCLQ_ERR_CUDA, "half product: no mapped host memory (is there a CUDA device?)");
    if (plan.splits > 1) {
        p.f32out = g.partial;
        p.ldf = ceil_div(g.n, 4) * 4;
        p.split_stride = g.m * p.ldf;
    } else {
        p.out = g.out;
        p.ldo = g.ldo;
        p.out_vec = g.out && (reinterpret_cast<uintptr_t>(g.out) & 15) == 0 && g.ldo % 8 == 0;
        p.f32out = g.f32out;
        p.f32in = g.f32in;
        p.ldf = g.ldf;
        p.alpha = g.alpha;
    }
    rc = g.bf16 ? launch_form<true>(g.form, plan.cg, plan.bn, maps, p, st) : launch_form<false>(g.form, plan.cg, plan.bn, maps, p, st);
    if (rc || plan.splits == 1) return rc;
    const int64_t groups = ceil_div(g.m * p.ldf, 4 * 256);
    const unsigned grid = (unsigned)std::min<int64_t>(groups, (int64_t)sm_count() * 8);
    auto kern = g.bf16 ? half_gemm_reduce_kernel<true> : half_gemm_reduce_kernel<false>;
    CDCLQ_LAUNCH(kern, grid, 256, 0, st, g.partial, plan.splits, g.m, g.n, p.ldf, g.f32in, g.f32out, g.ldf, g.alpha,
                 static_cast<uint16_t*>(g.out), g.ldo);
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : cuda_error(e, "half_gemm_reduce_kernel launch");
}

}  // namespace cdclq

using namespace cdclq;

extern "C" int cdclq_operator_status(void) { return check_fail_word("operator"); }

extern "C" int* cdclq_operator_word(int device) { return fail_word_host(device); }

namespace cdclq {
__global__ void __launch_bounds__(256) align_rows_kernel(const uint16_t* __restrict__ src, int64_t rows, int64_t cols, int64_t lds,
                                                         uint16_t* __restrict__ dst, int64_t ldd) {
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < rows * ldd; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i / ldd, c = i - r * ldd;
        dst[i] = c < cols ? src[r * lds + c] : (uint16_t)0;
    }
}
}  // namespace cdclq

extern "C" int cdclq_align_rows_device(const void* src, size_t rows, size_t cols, size_t lds, void* dst, size_t ldd, void* stream) {
    if (!rows || !cols) return 0;
    if (!src || !dst || lds < cols || ldd < cols) return set_error(CDCLQ_ERR_ARG, "align_rows: null pointer, or rows overlap");
    if (int rc = check_fail_word("align_rows")) return rc;
    const int64_t blocks = ceil_div((int64_t)rows * (int64_t)ldd, 256);
    CDCLQ_LAUNCH(align_rows_kernel, (unsigned)std::min<int64_t>(blocks, sm_count() * 16), 256, 0, static_cast<cudaStream_t>(stream),
                 static_cast<const uint16_t*>(src), (int64_t)rows, (int64_t)cols, (int64_t)lds, static_cast<uint16_t*>(dst),
                 (int64_t)ldd);
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : cuda_error(e, "align_rows_kernel launch");
}

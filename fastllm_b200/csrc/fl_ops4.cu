// Operators on rows of 4-bit numbers (include/fastllm_b200.h, "operators on device memory"): argument checks and launches behind the C ABI.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <mutex>

#include "../../include/fastllm_b200.h"
#include "failed_word.hpp"
#include "linear4.cuh"
#include "op_launch.cuh"
#include "ops.hpp"

namespace fl {

constexpr int64_t kMaxCols4 = (int64_t)1 << 20, kMaxNumbers4 = (int64_t)1 << 39;         // (grids of threads of four numbers each, 2^31 - 1 blocks)

static int64_t blocks4(int64_t cols) { return (cols + kR4Block - 1) / kR4Block; }
static int64_t groups4(int64_t cols) { return 2 * ((blocks4(cols) + 7) / 8); }              // k blocks of 256 values are whole
static size_t up256(size_t n) { return (n + 255) / 256 * 256; }
// rows that scales in tiles of `tile` rows have room for, in whole 128 rows a tile
static int64_t slots4(int64_t rows, int tile) { return (rows + tile - 1) / tile * ((tile + 127) / 128 * 128); }

// threads of `per` pieces a row
static dim3 pieces_grid(int64_t rows, int64_t per) { return dim3((unsigned)((rows * per + kR4Threads - 1) / kR4Threads)); }
static bool rows_on_16(const void* x, int64_t rows, int64_t ld, size_t size) { return aligned(x, 16) && (rows == 1 || ld * size % 16 == 0); }

// f(T{}) with the element type of a float dtype
template <typename F>
static void by_type(int dtype, F f) {
    if (dtype == FL_DTYPE_F32) f(float{});
    else if (dtype == FL_DTYPE_BF16) f(__nv_bfloat16{});
    else f(__half{});
}

static void quantize4(LaunchCtx& lc, const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, const Rows4Out& o) {
    by_type(dtype, [&](auto t) {
        using T = decltype(t);
        const int64_t per = (o.tile > 0 ? o.groups * 4 : o.blocks) * kR4Lanes<T>;              // (tiles hold scales of whole k blocks)
        launch_op(lc, "quantize4", (uint64_t)rows * (cols * sizeof(T) + o.blocks * 17), rows_on_16(x, rows, ldx, sizeof(T)) ? quantize4_kernel<T, true> : quantize4_kernel<T, false>,
                  pieces_grid(rows, per), kR4Threads, 0, 1, false, static_cast<const T*>(x), (long long)ldx, (long long)rows, (int)cols, (int)per, o);
    });
}

template <typename T, bool kVec>
static void (*glu4_form(int act))(const T*, long long, long long, int, int, float, Rows4Out) {
    if (act == FL_ACT_SILU) return glu4_kernel<T, kGlu4Silu, kVec>;
    if (act == FL_ACT_GELU_TANH) return glu4_kernel<T, kGlu4GeluTanh, kVec>;
    if (act == FL_ACT_RELU) return glu4_kernel<T, kGlu4Relu, kVec>;
    return glu4_kernel<T, kGlu4SwishClamp, kVec>;
}
static void glu4(LaunchCtx& lc, const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, int act, float limit, const Rows4Out& o) {
    by_type(dtype, [&](auto t) {
        using T = decltype(t);
        const bool vec = rows_on_16(x, rows, ldx, sizeof(T)) && cols * sizeof(T) % 16 == 0;
        const int64_t per = o.blocks * kR4Lanes<T>;
        launch_op(lc, "glu4", (uint64_t)rows * (2 * cols * sizeof(T) + o.blocks * 17), vec ? glu4_form<T, true>(act) : glu4_form<T, false>(act), pieces_grid(rows, per), kR4Threads, 0, 1, false,
                  static_cast<const T*>(x), (long long)ldx, (long long)rows, (int)cols, (int)per, limit, o);
    });
}

static size_t weight4_bytes(int64_t n, int64_t k) { return (size_t)(slots4(n, 128) * groups4(k) * 4); }
static void arrange4(LaunchCtx& lc, const uint8_t* scale, int64_t lds, int64_t rows, int64_t k, int tile, uint8_t* tiles) {
    const int64_t slots = slots4(rows, tile), groups = groups4(k);
    launch_op(lc, "arrange4", (uint64_t)(2 * slots * groups * 4), arrange4_kernel, dim3((unsigned)(slots / 128), (unsigned)((groups + kArrange - 1) / kArrange)), 128, 0, 1, false, scale,
              (long long)lds, (long long)rows, (int)blocks4(k), tiles, tile, (int)groups, (tile + 127) / 128);
}

static bool token_fits4(int64_t rows, int64_t n, int64_t k) { return rows <= kL4TokenRows && rows * rows * n * blocks4(k) <= kL4TokenWork && rows * blocks4(k) <= kL4TokenBlocks; }
struct Linear4Room { size_t scale = 0, all = 0; int64_t slots = 0; };
// (ops.py keeps the same rule)
static Linear4Room linear4_room(int64_t rows, int64_t k, bool given) {
    Linear4Room r;
    if (rows <= kL4SelfRows) return r;                          // brought to the tensor cores inside the product's own launch
    r.scale = given ? 0 : up256((size_t)rows * blocks4(k) * 16);
    // the scales lie in tiles of as many rows as a product takes, each padded to 128: beyond 128 rows 64 to 224, which is twice the rows at most and 256
    r.slots = rows <= 128 ? (rows + 127) / 128 * 128 : (2 * rows + 127) / 128 * 128 + 256;
    r.all = r.scale + (size_t)r.slots * groups4(k) * 4;
    return r;
}

// How a product of more than kL4FewRows rows goes over the pairs of SMs: the tile width whose waves cost least.  A k block takes 60 + 1.1 bn ns where its operands come from L2
// (bn = 128, 160, 192, 208 and 224: 193, 228, 282, 257 to 290 and 287 to 307), and a tile no less than its results take, 1200 + 7 bn.  It ranks widths and does not foretell a call: first
// loads and last results are not in it, nor operands that come from memory (300 and 777 x 4096 x 28672 15 and 30 us by the rule, with the rounding's launch 26 and 45 measured; 3000 x 8192 x
// 8192 61 by the rule, 71 alone).
constexpr int kL4FewRows = 128;
static L4Pair pair_plan4(int64_t rows, int64_t n, int64_t k, int clusters) {
    L4Pair best{};
    double cost = -1;
    for (int bn = kL4PairMaxRows; bn >= kL4PairMinRows; bn -= 16) {
        L4Pair p{};
        p.bn = bn;
        p.nk = (int)(groups4(k) / 2);
        p.mt = (int)((n + 255) / 256);
        p.nt = (int)((rows + bn - 1) / bn);
        // weights come from memory once for as many activation tiles as stay in half of L2 (4096 x 3584 x 37888, 4, 8, 16 and 20 tiles: 230, 221, 215 and 208 us)
        p.raster = (int)std::max<int64_t>(8, std::min<int64_t>(p.nt, ((int64_t)64 << 20) / (bn * blocks4(k) * 17)));
        p.stages = (int)std::min<uint32_t>(kL4PairMaxStages, kL4PairRing / l4_pair_stage(bn));
        p.slots = std::min(l4_pair_slots(bn), p.stages);
        const double waves = (double)(((long long)p.mt * p.nt + clusters - 1) / clusters);
        const double c = waves * std::max(p.nk * (60 + 1.1 * bn), 1200.0 + 7.0 * bn);
        if (cost < 0 || c < cost) { cost = c; best = p; }
    }
    return best;
}

// What the operators keep for the process: a page-locked word that a kernel sets when a wait inside it ran out, told of once.
static FailedWord g_op4_failed;
static int g_pair_clusters = 0;                 // pairs of SMs that can be resident at once
bool products4_failed() { return g_op4_failed.take(); }

// Blocks that share a 128-row weight tile: one per SM at most, four k blocks each at least, and only where a block is spared twelve: the cluster's barriers and the exchange take as
// long (S = 1, 2 and 4: 16 x 4096 x 4096 8.8, 8.9 and 8.1 us, 64 x 4096 x 4096 9.9, 9.7 and 8.7, 32 x 14336 x 4096 20.5, 14.6 and 11.9, 8 x 1024 x 4096 5.0, 6.7 and 6.5; that is 16, 56 and 4 k blocks, and
// no number between them was measured).
static int few_slices4(int64_t tiles, int nk) {
    int S = 8;
    while (S > 1 && (S * tiles > kNumSMs || nk < 4 * S || nk - nk / S < 12)) S /= 2;
    return S;
}
template <int BN>
static void launch_few4(LaunchCtx& lc, uint64_t bytes, const uint8_t* x, int64_t ldx, const uint8_t* w, int64_t ldw, const Linear4Args& g) {
    const int tiles = (g.n + 127) / 128, S = few_slices4(tiles, g.groups / 2);
    const CUtensorMap tw = make_tmap_i8(w, g.n, g.blocks * 16, ldw, 128), tx = make_tmap_i8(x, g.rows, g.blocks * 16, ldx, BN);
    launch_op(lc, "linear4", bytes, linear4_few_kernel<BN>, dim3((unsigned)(tiles * S)), L4Few<BN>::kThreads, L4Few<BN>::kSmem, S, true, tw, tx, g, S);
}
template <typename T, bool kVec>
static void launch_self4(LaunchCtx& lc, uint64_t bytes, const void* x, int64_t ldx, int64_t k, int64_t lds, const uint8_t* w, int64_t ldw, const Linear4Args& g) {
    const int tiles = (g.n + 127) / 128, S = few_slices4(tiles, g.groups / 2);
    const CUtensorMap tw = make_tmap_i8(w, g.n, g.blocks * 16, ldw, 128);
    launch_op(lc, "linear4", bytes, linear4_self_kernel<T, kVec>, dim3((unsigned)(tiles * S)), L4Self::kThreads, L4Self::kSmem, S, false, tw, g, static_cast<const T*>(x), (long long)ldx, (int)k,
              (long long)lds, S);
}
static void launch_pair4(LaunchCtx& lc, uint64_t bytes, const uint8_t* x, int64_t ldx, const uint8_t* w, int64_t ldw, const Linear4Args& g, const L4Pair& p) {
    const int bn = p.bn, atoms = l4_pair_atoms(bn);
    const CUtensorMap tx = make_tmap_i8(x, g.rows, g.blocks * 16, ldx, bn / 2), tw = make_tmap_i8(w, g.n, g.blocks * 16, ldw, 128);
    const CUtensorMap tws = make_tmap_scales(g.ws, (int64_t)((g.n + 127) / 128) * g.groups, 2), txs = make_tmap_scales(g.xs, (int64_t)p.nt * g.groups * atoms, 2 * atoms);
    const long long clusters = std::min<long long>(g_pair_clusters, (long long)p.mt * p.nt);
    auto go = [&](auto kern) { launch_op(lc, "linear4", bytes, kern, dim3((unsigned)(2 * clusters)), kL4PairThreads, kL4PairSmem, 1, true, tw, tx, tws, txs, g, p); };
    atoms == 1 ? go(linear4_pair_kernel<1>) : go(linear4_pair_kernel<2>);
}

template <typename T, int R, bool kVec>
static void launch_token4(LaunchCtx& lc, uint64_t bytes, const void* x, int64_t ldx, int64_t k, const uint8_t* w, int64_t ldw, const Linear4Args& g) {
    const int per = kL4TokenThreads / 32;
    launch_op(lc, "linear4", bytes, linear4_token_kernel<T, R, kVec>, dim3((unsigned)std::min<int64_t>(((int64_t)g.n + per - 1) / per, 4 * kNumSMs)), kL4TokenThreads, (size_t)R * g.blocks * 36, 1,
              false, g, static_cast<const T*>(x), (long long)ldx, (int)k, w, (long long)ldw);
}

// x in 4 bits: lds its scales' row stride
static void run_linear4(LaunchCtx& lc, const void* x, int x_dtype, int64_t ldx, const uint8_t* x_scale, int64_t lds, const uint8_t* w, int64_t ldw, const uint8_t* w_tiles, const float* bias,
                        int64_t rows, int64_t n, int64_t k, void* y, int y_dtype, int64_t ldy, void* workspace, int* failed) {
    const bool given = x_dtype == FL_DTYPE_MX4, many = rows > kL4FewRows;
    FL_CHECK(!many || g_pair_clusters >= 1, FL_ERR_UNSUPPORTED, "linear4: no two SMs of this device form a pair");
    const Linear4Room room = linear4_room(rows, k, given);
    uint8_t *to = static_cast<uint8_t*>(workspace), *xs = to + room.scale;
    const int blocks = (int)blocks4(k), groups = (int)groups4(k);
    if (n == 1) ldw = 16 * blocks;
    const uint64_t bytes = (uint64_t)(n + rows) * blocks * 17 + rows * n * dtype_size(y_dtype);
    if (!given && token_fits4(rows, n, k)) {
        const Linear4Args a{(int)rows, (int)n, blocks, nullptr, w_tiles, groups, bias, y, ldy, y_dtype, failed, false};
        by_type(x_dtype, [&](auto t) {
            using T = decltype(t);
            const bool vec = rows_on_16(x, rows, ldx, sizeof(T));
            auto go = [&](auto one, auto two) { rows == 1 ? one(lc, bytes, x, ldx, k, w, ldw, a) : two(lc, bytes, x, ldx, k, w, ldw, a); };
            if (vec) go(launch_token4<T, 1, true>, launch_token4<T, 2, true>);
            else go(launch_token4<T, 1, false>, launch_token4<T, 2, false>);
        });
        return;
    }
    if (rows <= kL4SelfRows) {
        const Linear4Args a{(int)rows, (int)n, blocks, x_scale, w_tiles, groups, bias, y, ldy, y_dtype, failed, false};
        if (given) launch_self4<uint8_t, true>(lc, bytes, x, ldx, k, lds, w, ldw, a);
        else by_type(x_dtype, [&](auto t) {
            using T = decltype(t);
            rows_on_16(x, rows, ldx, sizeof(T)) ? launch_self4<T, true>(lc, bytes, x, ldx, k, 0, w, ldw, a) : launch_self4<T, false>(lc, bytes, x, ldx, k, 0, w, ldw, a);
        });
        return;
    }
    const L4Pair p = many ? pair_plan4(rows, n, k, g_pair_clusters) : L4Pair{};
    const int tile = many ? p.bn : 128;
    FL_CHECK(slots4(rows, tile) <= room.slots, FL_ERR_STATE, "linear4: the scales do not fit their workspace");
    const uint8_t* q = to;
    int64_t ldq = 16 * blocks;
    if (given) {
        arrange4(lc, x_scale, lds, rows, k, tile, xs);
        q = static_cast<const uint8_t*>(x);
        if (rows > 1) ldq = ldx;
    } else {
        quantize4(lc, x, x_dtype, rows, k, ldx, Rows4Out{to, ldq, xs, 0, blocks, tile, groups});
    }
    const Linear4Args a{(int)rows, (int)n, blocks, xs, w_tiles, groups, bias, y, ldy, y_dtype, failed, y_dtype != FL_DTYPE_F32 && rows_on_16(y, rows, ldy, 2)};
    if (many) launch_pair4(lc, bytes, q, ldq, w, ldw, a, p);
    else if (rows <= 32) launch_few4<32>(lc, bytes, q, ldq, w, ldw, a);
    else if (rows <= 64) launch_few4<64>(lc, bytes, q, ldq, w, ldw, a);
    else launch_few4<128>(lc, bytes, q, ldq, w, ldw, a);
}

template <typename T>
static void self_attr4() {
    for (auto kern : {linear4_self_kernel<T, false>, linear4_self_kernel<T, true>}) FL_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L4Self::kSmem));
}
template <int BN>
static void few_attr4() {
    FL_CUDA(cudaFuncSetAttribute(linear4_few_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L4Few<BN>::kSmem));
}
// One-time set-up on the bound device, by the first call that launches an operator.  It also loads the kernels, so that this call may be one inside a graph capture.
static void set_up() {
    static std::atomic<bool> done{false};
    static std::mutex one;
    if (done.load(std::memory_order_acquire)) return;
    std::lock_guard<std::mutex> lock(one);
    if (done.load(std::memory_order_relaxed)) return;
    RelaxedCapture relaxed;
    for (int dtype : {FL_DTYPE_F32, FL_DTYPE_BF16, FL_DTYPE_F16})
        by_type(dtype, [](auto t) {
            using T = decltype(t);
            load_kernels(quantize4_kernel<T, false>, quantize4_kernel<T, true>);
            load_kernels(dequantize4_kernel<T, false>, dequantize4_kernel<T, true>);
            self_attr4<T>();
            load_kernels(linear4_token_kernel<T, 1, false>, linear4_token_kernel<T, 1, true>, linear4_token_kernel<T, 2, false>, linear4_token_kernel<T, 2, true>);
            for (int act : {FL_ACT_SILU, FL_ACT_GELU_TANH, FL_ACT_RELU, FL_ACT_SWISH_CLAMP}) load_kernels(glu4_form<T, false>(act), glu4_form<T, true>(act));
        });
    load_kernels(arrange4_kernel);
    FL_CUDA(cudaFuncSetAttribute(linear4_self_kernel<uint8_t, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L4Self::kSmem));
    few_attr4<32>(); few_attr4<64>(); few_attr4<128>();
    for (auto kern : {linear4_pair_kernel<1>, linear4_pair_kernel<2>})
        FL_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kL4PairSmem));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(kNumSMs); cfg.blockDim = dim3(kL4PairThreads); cfg.dynamicSmemBytes = kL4PairSmem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 2; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = 1;
    int pairs = 0;
    FL_CUDA(cudaOccupancyMaxActiveClusters(&pairs, linear4_pair_kernel<2>, &cfg));
    g_pair_clusters = std::min(pairs, kNumSMs / 2);
    int* p = nullptr;
    FL_CUDA(cudaMallocHost(&p, sizeof(int)));
    *p = 0;
    g_op4_failed.word = p;
    done.store(true, std::memory_order_release);
}

static void check_rows4(const char* what, const void* q, int64_t ldq, const void* scale, int64_t lds, int64_t rows, int64_t cols) {
    FL_CHECK(rows <= 1 || (ldq >= 16 * blocks4(cols) && lds >= blocks4(cols)), FL_ERR_INVALID, std::string(what) + ": a row stride of the 4-bit rows or their scales is smaller than the row");
    FL_CHECK(aligned(q, 16) && (rows <= 1 || ldq % 16 == 0), FL_ERR_INVALID, std::string(what) + ": 4-bit rows start on 16-byte borders (pointer and row stride)");
}

}  // namespace fl

using namespace fl;

extern "C" {

FL_EXPORT int fl_quantize4(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, uint8_t* q, int64_t ldq, uint8_t* scale, int64_t lds, void* stream) {
    FL_API_BEGIN
    FL_CHECK(is_float(dtype), FL_ERR_INVALID, "quantize4: rows of f32, bf16 or f16");
    FL_CHECK(rows >= 0 && rows <= kMaxRows && cols >= 1 && cols <= kMaxCols4, FL_ERR_INVALID, "quantize4: rows from 0 to 2^30, columns from 1 to 2^20");
    FL_CHECK(rows <= kMaxNumbers4 / cols, FL_ERR_INVALID, "quantize4: more than 2^39 numbers");
    FL_CHECK(rows <= 1 || ldx >= cols, FL_ERR_INVALID, "quantize4: the row stride is smaller than the row");
    if (rows == 0) return FL_OK;
    FL_CHECK(x && q && scale, FL_ERR_INVALID, "NULL argument");
    FL_CHECK(aligned(x, dtype_size(dtype)), FL_ERR_INVALID, "quantize4: a pointer is not aligned to its type");
    check_rows4("quantize4", q, ldq, scale, lds, rows, cols);
    DeviceScope dev;
    set_up();
    LaunchCtx lc = op_ctx(stream);
    quantize4(lc, x, dtype, rows, cols, ldx, Rows4Out{q, ldq, scale, lds, (int)blocks4(cols), 0, 0});
    FL_API_END
}

FL_EXPORT int fl_dequantize4(const uint8_t* q, int64_t ldq, const uint8_t* scale, int64_t lds, int64_t rows, int64_t cols, void* y, int dtype, int64_t ldy, void* stream) {
    FL_API_BEGIN
    FL_CHECK(is_float(dtype), FL_ERR_INVALID, "dequantize4: results are f32, bf16 or f16");
    FL_CHECK(rows >= 0 && rows <= kMaxRows && cols >= 1 && cols <= kMaxCols4, FL_ERR_INVALID, "dequantize4: rows from 0 to 2^30, columns from 1 to 2^20");
    FL_CHECK(rows <= kMaxNumbers4 / cols, FL_ERR_INVALID, "dequantize4: more than 2^39 numbers");
    FL_CHECK(rows <= 1 || ldy >= cols, FL_ERR_INVALID, "dequantize4: the row stride is smaller than the row");
    if (rows == 0) return FL_OK;
    FL_CHECK(q && scale && y, FL_ERR_INVALID, "NULL argument");
    FL_CHECK(aligned(y, dtype_size(dtype)), FL_ERR_INVALID, "dequantize4: a pointer is not aligned to its type");
    check_rows4("dequantize4", q, ldq, scale, lds, rows, cols);
    DeviceScope dev;
    set_up();
    LaunchCtx lc = op_ctx(stream);
    by_type(dtype, [&](auto t) {
        using T = decltype(t);
        constexpr int V = 16 / sizeof(T);
        const bool shift = !rows_on_16(y, rows, ldy, sizeof(T));
        const int64_t per = (cols + (shift ? V - 1 : 0) + V - 1) / V;                          // (from the last border before the row on)
        const int threads = (int)std::min<int64_t>(256, (per + 63) / 64 * 32);                 // two pieces each
        launch_op(lc, "dequantize4", (uint64_t)rows * (cols * sizeof(T) + blocks4(cols) * 17), shift ? dequantize4_kernel<T, true> : dequantize4_kernel<T, false>,
                  dim3((unsigned)rows, (unsigned)((per + 2 * threads - 1) / (2 * threads))), threads, 0, 1, false, q, (long long)ldq, scale, (long long)lds, (int)cols, (int)(4 * blocks4(cols)),
                  static_cast<T*>(y), (long long)ldy);
    });
    FL_API_END
}

FL_EXPORT int fl_glu4(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, int act, float limit, uint8_t* q, int64_t ldq, uint8_t* scale, int64_t lds, void* stream) {
    FL_API_BEGIN
    FL_CHECK(is_float(dtype), FL_ERR_INVALID, "glu4: rows of f32, bf16 or f16");
    FL_CHECK(act == FL_ACT_SILU || act == FL_ACT_GELU_TANH || act == FL_ACT_RELU || act == FL_ACT_SWISH_CLAMP, FL_ERR_INVALID, "glu4: the activation is silu, gelu_tanh, relu or swish_clamp");
    FL_CHECK(act != FL_ACT_SWISH_CLAMP || (limit > 0 && std::isfinite(limit)), FL_ERR_INVALID, "glu4: the limit is a positive number");
    FL_CHECK(rows >= 0 && rows <= kMaxRows && cols >= 1 && cols <= kMaxCols4, FL_ERR_INVALID, "glu4: rows from 0 to 2^30, columns from 1 to 2^20");
    FL_CHECK(rows <= kMaxNumbers4 / cols, FL_ERR_INVALID, "glu4: more than 2^39 numbers");
    FL_CHECK(rows <= 1 || ldx >= 2 * cols, FL_ERR_INVALID, "glu4: the row stride is smaller than the row");
    if (rows == 0) return FL_OK;
    FL_CHECK(x && q && scale, FL_ERR_INVALID, "NULL argument");
    FL_CHECK(aligned(x, dtype_size(dtype)), FL_ERR_INVALID, "glu4: a pointer is not aligned to its type");
    check_rows4("glu4", q, ldq, scale, lds, rows, cols);
    DeviceScope dev;
    set_up();
    LaunchCtx lc = op_ctx(stream);
    glu4(lc, x, dtype, rows, cols, ldx, act, limit, Rows4Out{q, ldq, scale, lds, (int)blocks4(cols), 0, 0});
    FL_API_END
}

FL_EXPORT int fl_weight4_bytes(int64_t n, int64_t k, size_t* bytes) {
    FL_API_BEGIN
    FL_CHECK(bytes, FL_ERR_INVALID, "NULL argument");
    FL_CHECK(n >= 1 && n <= kMaxRows && k >= 1 && k <= kMaxCols4, FL_ERR_INVALID, "weight4: n from 1 to 2^30, k from 1 to 2^20");
    *bytes = weight4_bytes(n, k);
    FL_API_END
}

FL_EXPORT int fl_weight4(const uint8_t* scale, int64_t lds, int64_t n, int64_t k, void* tiles, void* stream) {
    FL_API_BEGIN
    FL_CHECK(n >= 1 && n <= kMaxRows && k >= 1 && k <= kMaxCols4, FL_ERR_INVALID, "weight4: n from 1 to 2^30, k from 1 to 2^20");
    FL_CHECK(n == 1 || lds >= blocks4(k), FL_ERR_INVALID, "weight4: the row stride is smaller than the row");
    FL_CHECK(scale && tiles, FL_ERR_INVALID, "NULL argument");
    FL_CHECK(aligned(tiles, 16), FL_ERR_INVALID, "weight4: the result starts on a 16-byte border");
    DeviceScope dev;
    set_up();
    LaunchCtx lc = op_ctx(stream);
    arrange4(lc, scale, lds, n, k, 128, static_cast<uint8_t*>(tiles));
    FL_API_END
}

FL_EXPORT int fl_linear4_workspace(int64_t rows, int64_t k, int x_dtype, size_t* bytes) {
    FL_API_BEGIN
    FL_CHECK(bytes, FL_ERR_INVALID, "NULL argument");
    FL_CHECK(is_float(x_dtype) || x_dtype == FL_DTYPE_MX4, FL_ERR_INVALID, "linear4: activations are f32, bf16, f16 or 4-bit rows");
    FL_CHECK(rows >= 0 && rows <= kMaxRows && k >= 1 && k <= kMaxCols4, FL_ERR_INVALID, "linear4: rows from 0 to 2^30, k from 1 to 2^20");
    *bytes = linear4_room(rows, k, x_dtype == FL_DTYPE_MX4).all;
    FL_API_END
}

FL_EXPORT int fl_linear4(const void* x, int x_dtype, int64_t ldx, const uint8_t* x_scale, int64_t lds, const uint8_t* w, int64_t ldw, const void* w_tiles, const float* bias, int64_t rows,
                         int64_t n, int64_t k, void* y, int y_dtype, int64_t ldy, void* workspace, size_t workspace_bytes, void* stream) {
    FL_API_BEGIN
    const bool given = x_dtype == FL_DTYPE_MX4;
    FL_CHECK(is_float(x_dtype) || given, FL_ERR_INVALID, "linear4: activations are f32, bf16, f16 or 4-bit rows");
    FL_CHECK(is_float(y_dtype), FL_ERR_INVALID, "linear4: results are f32, bf16 or f16");
    FL_CHECK(rows >= 0 && rows <= kMaxRows && n >= 1 && n <= kMaxRows && k >= 1 && k <= kMaxCols4, FL_ERR_INVALID, "linear4: rows from 0 to 2^30, n from 1 to 2^30, k from 1 to 2^20");
    FL_CHECK((rows <= 1 || (ldx >= (given ? 16 * blocks4(k) : k) && ldy >= n)) && (n == 1 || ldw >= 16 * blocks4(k)), FL_ERR_INVALID, "linear4: a row stride is smaller than the row");
    if (rows == 0) return FL_OK;
    FL_CHECK(x && w && w_tiles && y, FL_ERR_INVALID, "NULL argument");
    FL_CHECK(given == (x_scale != nullptr), FL_ERR_INVALID, "linear4: x_scale comes with activations of 4 bits, and only with them");
    FL_CHECK(aligned(w, 16) && (n == 1 || ldw % 16 == 0), FL_ERR_INVALID, "linear4: the weight's rows start on 16-byte borders (pointer and row stride)");
    FL_CHECK(aligned(w_tiles, 16), FL_ERR_INVALID, "linear4: the weight's scales start on a 16-byte border");
    if (given) check_rows4("linear4", x, ldx, x_scale, lds, rows, k);
    FL_CHECK((given || aligned(x, dtype_size(x_dtype))) && aligned(y, dtype_size(y_dtype)) && aligned(bias, 4), FL_ERR_INVALID, "linear4: a pointer is not aligned to its type");
    FL_CHECK(rows <= ((int64_t)1 << 40) / n && n <= kMaxNumbers4 / k && rows <= kMaxNumbers4 / k, FL_ERR_INVALID, "linear4: more than 2^40 results, or an operand of more than 2^39 numbers");
    const Linear4Room room = linear4_room(rows, k, given);
    FL_CHECK(room.all == 0 || (workspace && aligned(workspace, 256) && workspace_bytes >= room.all), FL_ERR_INVALID,
             "linear4: the workspace is smaller than fl_linear4_workspace asks for, or not on a 256-byte border");
    DeviceScope dev;
    set_up();
    LaunchCtx lc = op_ctx(stream);
    FL_CHECK(!products4_failed(), FL_ERR_CUDA, "a wait inside an operator's kernel ran out: a product since the last check is not valid");
    run_linear4(lc, x, x_dtype, ldx, x_scale, lds, w, ldw, static_cast<const uint8_t*>(w_tiles), bias, rows, n, k, y, y_dtype, ldy, workspace, g_op4_failed.word);
    FL_API_END
}

}  // extern "C"

// Operators on device memory: argument checks and launches behind the C ABI (include/fastllm_b200.h, "operators on device memory").
#include <atomic>
#include <cmath>
#include <mutex>

#include "../../include/fastllm_b200.h"
#include "bert_model.cuh"
#include "failed_word.hpp"
#include "linear8.cuh"
#include "logprobs.cuh"
#include "ops.hpp"

namespace fl {

// The bound device for the length of a call; the caller's own is put back.
struct DeviceScope {
    int before = -1, now;
    DeviceScope() : now(bound_device()) {
        FL_CUDA(cudaGetDevice(&before));
        if (before != now) FL_CUDA(cudaSetDevice(now));
    }
    ~DeviceScope() { if (before >= 0 && before != now) cudaSetDevice(before); }
};

static LaunchCtx op_ctx(void* stream) {
    LaunchCtx lc;
    lc.stream = static_cast<cudaStream_t>(stream);
    lc.pdl = false;
    if (g_prof.on) {                        // (no events inside a caller's capture)
        cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
        FL_CUDA(cudaStreamIsCapturing(lc.stream, &st));
        lc.capturing = st != cudaStreamCaptureStatusNone;
    }
    return lc;
}
static size_t dtype_size(int dtype) { return dtype == FL_DTYPE_F32 ? 4 : dtype == FL_DTYPE_I8 ? 1 : 2; }
static bool is_float(int dtype) { return dtype == FL_DTYPE_F32 || dtype == FL_DTYPE_BF16 || dtype == FL_DTYPE_F16; }
static bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

constexpr int64_t kMaxRows = (int64_t)1 << 30;
constexpr int64_t kLinear8MaxK = 131071;        // 128 * 128 * k stays below 2^31

static size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// How a product of more than kL8FewRows rows goes over the pairs of SMs: the tile width whose waves cost least, by what a k block takes (see
// linear8_pair_kernel).  Cutting the tiles of a last wave along K was measured and lost everywhere (1531 x 14336 x 4096 68 -> 78 us, 777 x 4096 x 32000 86 ->
// 96): the parts' way through the workspace takes longer than the idle pairs would.
constexpr int kL8FewRows = 128;
static L8Pair pair_plan8(int64_t rows, int64_t n, int64_t k, int clusters) {
    L8Pair best{};
    double cost = -1;
    for (int bn = 512; bn >= 64; bn -= bn > 256 ? 64 : 32) {
        L8Pair p{};
        p.bn = bn;
        p.nk = (int)((k + kL8BK - 1) / kL8BK);
        p.mt = (int)((n + 255) / 256);
        p.nt = (int)((rows + bn - 1) / bn);
        p.stages = (int)std::min<uint32_t>(kL8PairMaxStages, kL8PairRing / (kL8WBytes + (uint32_t)bn * (kL8BK / 2)));
        const double block = std::max(1.38 * bn, (16384.0 + 64.0 * bn) / 90.0), tail = bn > 256 ? 13.0 * bn : 0.0;      // ns; results that no product hides
        const double waves = (double)(((long long)p.mt * p.nt + clusters - 1) / clusters);
        const double c = waves * (p.nk * block + tail);
        if (cost < 0 || c < cost) { cost = c; best = p; }
    }
    return best;
}

// A call's workspace: rounded rows and their scales (none for activations that are 8-bit already)
struct L8Room { size_t scale = 0, all = 0; };
static bool token_fits(int64_t rows, int64_t k);
static L8Room linear8_room(int64_t rows, int64_t k, bool given) {
    L8Room r;
    if (given || token_fits(rows, k)) return r;
    r.scale = up256((size_t)rows * padded8(k));
    r.all = r.scale + (size_t)rows * 4;
    return r;
}

// Launch of an operator's kernel in clusters of `cluster` blocks; pdl: it may start under the kernel before it, which this call launched too
// (never under a caller's).
template <typename... KArgs, typename... Args>
static void launch_op(LaunchCtx& lc, const char* tag, uint64_t bytes, void (*kern)(KArgs...), dim3 grid, int threads, size_t smem, int cluster, bool pdl, Args&&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = lc.stream;
    cudaLaunchAttribute attr[2];
    const bool prof = g_prof.on && !lc.capturing;
    if (pdl && !prof) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = cluster; attr[cfg.numAttrs].val.clusterDim.y = 1; attr[cfg.numAttrs++].val.clusterDim.z = 1;
    }
    cfg.attrs = attr;
    ProfEntry pe;
    if (prof) {
        pe.tag = tag;
        pe.bytes = bytes;
        FL_CUDA(cudaEventCreate(&pe.e0));
        FL_CUDA(cudaEventCreate(&pe.e1));
        FL_CUDA(cudaEventRecord(pe.e0, lc.stream));
    }
    FL_CUDA(cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...));
    if (prof) {
        FL_CUDA(cudaEventRecord(pe.e1, lc.stream));
        g_prof.entries.push_back(pe);
    }
    if (lc.capturing) lc.captured++;
    else g_launches.fetch_add(1, std::memory_order_relaxed);
}

// What the operators keep for the process: one page-locked word that a kernel sets when a wait inside it ran out; the next product or fl_operators_check
// tells of it, once.
static FailedWord g_op_failed;
static int g_pair_clusters = 0;                 // pairs of SMs that can be resident at once

template <int BN>
static void few_attr() {
    FL_CUDA(cudaFuncSetAttribute(linear8_few_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L8Few<BN>::kSmem));
}
// Unsafe calls for the length of a scope: set-up does not belong to a graph that the caller's thread may be capturing.
struct RelaxedCapture {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    RelaxedCapture() { FL_CUDA(cudaThreadExchangeStreamCaptureMode(&mode)); }
    ~RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
};
template <typename... Kernels>
static void load_kernels(Kernels... kernels) {
    cudaFuncAttributes at;
    for (cudaError_t e : {cudaFuncGetAttributes(&at, kernels)...}) FL_CUDA(e);
}
template <typename T>
static void load_kernels_of() {
    load_kernels(quantize_rows_kernel<T, 0, 256>, quantize_rows_kernel<T, 2, 128>, quantize_rows_kernel<T, 2, 256>, quantize_rows_kernel<T, 4, 256>,
                 quantize_rows_kernel<T, 8, 256>, quantize_rows_kernel<T, -1, 256>, logprobs_kernel<T, true, 128>, logprobs_kernel<T, false, 128>);
    FL_CUDA(cudaFuncSetAttribute(logprobs_kernel<T, true, 256>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    FL_CUDA(cudaFuncSetAttribute(logprobs_kernel<T, false, 256>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    load_kernels(linear8_token_kernel<T, 1>, linear8_token_kernel<T, 2>);
}
// One-time set-up on the bound device, by the first call that launches an operator.  It also loads the kernels, so that this call may be one inside a graph capture.
static void set_up() {
    static std::atomic<bool> done{false};
    static std::mutex one;
    if (done.load(std::memory_order_acquire)) return;
    std::lock_guard<std::mutex> lock(one);
    if (done.load(std::memory_order_relaxed)) return;
    RelaxedCapture relaxed;
    load_kernels_of<float>(); load_kernels_of<__nv_bfloat16>(); load_kernels_of<__half>();
    few_attr<16>(); few_attr<32>(); few_attr<64>(); few_attr<128>();
    FL_CUDA(cudaFuncSetAttribute(linear8_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kL8PairSmem));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(kNumSMs); cfg.blockDim = dim3(kL8PairThreads); cfg.dynamicSmemBytes = kL8PairSmem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 2; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = 1;
    int k = 0;
    FL_CUDA(cudaOccupancyMaxActiveClusters(&k, linear8_pair_kernel, &cfg));
    g_pair_clusters = std::min(k, kNumSMs / 2);
    int* p = nullptr;
    FL_CUDA(cudaMallocHost(&p, sizeof(int)));
    *p = 0;
    g_op_failed.word = p;
    done.store(true, std::memory_order_release);
}
static void check_op_failed() {
    FL_CHECK(!g_op_failed.take(), FL_ERR_CUDA, "a wait inside an operator's kernel ran out: a product since the last check is not valid");
}

template <typename T>
static void quantize_rows_t(LaunchCtx& lc, const void* x, int64_t rows, int64_t cols, int64_t ldx, int8_t* q, int64_t ldq, int64_t cols_q, float* scale) {
    constexpr int V = 16 / sizeof(T);
    const uint64_t bytes = rows * cols * (sizeof(T) + 1);
    auto go = [&](auto kern, int threads) {
        launch_op(lc, "quantize_rows", bytes, kern, dim3((unsigned)rows), threads, 0, 1, false, static_cast<const T*>(x), (long long)ldx, (int)cols, q, (long long)ldq,
                  (int)cols_q, scale);
    };
    const bool vec = aligned(x, 16) && aligned(q, V) && (rows == 1 || (ldx % V == 0 && ldq % V == 0));
    const int64_t vecs = (cols_q + V - 1) / V;
    if (!vec) go(quantize_rows_kernel<T, 0, 256>, 256);
    else if (vecs <= 2 * 128) go(quantize_rows_kernel<T, 2, 128>, 128);
    else if (vecs <= 2 * 256) go(quantize_rows_kernel<T, 2, 256>, 256);
    else if (vecs <= 4 * 256) go(quantize_rows_kernel<T, 4, 256>, 256);
    else if (vecs <= 8 * 256) go(quantize_rows_kernel<T, 8, 256>, 256);
    else go(quantize_rows_kernel<T, -1, 256>, 256);
}
static void quantize_rows(LaunchCtx& lc, const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, int8_t* q, int64_t ldq, int64_t cols_q, float* scale) {
    if (dtype == FL_DTYPE_F32) quantize_rows_t<float>(lc, x, rows, cols, ldx, q, ldq, cols_q, scale);
    else if (dtype == FL_DTYPE_BF16) quantize_rows_t<__nv_bfloat16>(lc, x, rows, cols, ldx, q, ldq, cols_q, scale);
    else quantize_rows_t<__half>(lc, x, rows, cols, ldx, q, ldq, cols_q, scale);
}

// Blocks that share a 128-row weight tile: one per SM at most, eight k blocks each at least, and only where a block is spared 24 k blocks: the cluster's
// barriers and the exchange take as long (8 rows, S = 1 and 2: 14336 x 4096 13.2 and 16.1 us, 5632 x 2048 7.3 and 8.5, 9472 x 14336 29.7 and 27.6; 4096 x
// 4096, S = 1, 4 and 8: 9.9, 9.0 and 9.4).
static int few_slices(int64_t tiles, int nk) {
    int S = 8;
    while (S > 1 && (S * tiles > kNumSMs || nk < 8 * S || nk - nk / S < 24)) S /= 2;
    return S;
}
// whether a product's rows are rounded inside its own launch (ops.py keeps the same rule, for the workspace)
static bool token_fits(int64_t rows, int64_t k) { return rows <= kL8TokenRows && rows * rows * k <= kL8TokenValues; }
template <typename T>
static void launch_token(LaunchCtx& lc, uint64_t bytes, const void* x, int64_t ldx, const int8_t* w, int64_t ldw, const Linear8Args& g) {
    const bool vec = aligned(x, 16) && (g.rows == 1 || ldx * sizeof(T) % 16 == 0);
    const int per = kL8TokenThreads / 32;
    const dim3 grid((unsigned)std::min<int64_t>(((int64_t)g.n + per - 1) / per, 4 * kNumSMs));
    const size_t smem = (size_t)g.rows * padded8(g.k);
    auto go = [&](auto kern) { launch_op(lc, "linear8", bytes, kern, grid, kL8TokenThreads, smem, 1, false, g, static_cast<const T*>(x), (long long)ldx, vec, w, (long long)ldw); };
    if (g.rows == 1) go(linear8_token_kernel<T, 1>);
    else go(linear8_token_kernel<T, 2>);
}
template <int BN>
static void launch_few(LaunchCtx& lc, uint64_t bytes, const int8_t* x, int64_t ldx, const int8_t* w, int64_t ldw, const Linear8Args& g, bool pdl) {
    const int tiles = (g.n + 127) / 128, S = few_slices(tiles, (g.k + kL8BK - 1) / kL8BK);
    const CUtensorMap tw = make_tmap_i8(w, g.n, g.k, ldw, 128), tx = make_tmap_i8(x, g.rows, g.k, ldx, BN);
    launch_op(lc, "linear8", bytes, linear8_few_kernel<BN>, dim3((unsigned)(tiles * S)), L8Few<BN>::kThreads, L8Few<BN>::kSmem, S, pdl, tw, tx, g, S);
}
static void launch_pair(LaunchCtx& lc, uint64_t bytes, const int8_t* x, int64_t ldx, const int8_t* w, int64_t ldw, const Linear8Args& g, bool pdl) {
    FL_CHECK(g_pair_clusters >= 1, FL_ERR_UNSUPPORTED, "linear8: no two SMs of this device form a pair");
    const L8Pair p = pair_plan8(g.rows, g.n, g.k, g_pair_clusters);
    const CUtensorMap tx = make_tmap_i8(x, g.rows, g.k, ldx, p.bn / (p.bn > 256 ? 4 : 2)), tw = make_tmap_i8(w, g.n, g.k, ldw, 128);
    const long long clusters = std::min<long long>(g_pair_clusters, (long long)p.mt * p.nt);
    launch_op(lc, "linear8", bytes, linear8_pair_kernel, dim3((unsigned)(2 * clusters)), kL8PairThreads, kL8PairSmem, 1, pdl, tw, tx, g, p);
}

static void run_linear8(LaunchCtx& lc, const void* x, int x_dtype, int64_t ldx, const float* x_scale, const int8_t* w, int64_t ldw, const float* w_scale, const float* bias,
                        int64_t rows, int64_t n, int64_t k, void* y, int y_dtype, int64_t ldy, void* workspace, int* failed) {
    const bool given = x_dtype == FL_DTYPE_I8;
    const int8_t* q = static_cast<const int8_t*>(x);
    int64_t ldq = rows == 1 ? padded8(k) : ldx;
    Linear8Args g{(int)rows, (int)n, (int)k, x_scale, w_scale, bias, y, ldy, y_dtype, failed};
    if (n == 1) ldw = padded8(k);
    const uint64_t bytes = (uint64_t)n * k + (uint64_t)rows * (k + n * dtype_size(y_dtype));
    if (!given && token_fits(rows, k)) {
        if (x_dtype == FL_DTYPE_F32) launch_token<float>(lc, bytes, x, ldx, w, ldw, g);
        else if (x_dtype == FL_DTYPE_BF16) launch_token<__nv_bfloat16>(lc, bytes, x, ldx, w, ldw, g);
        else launch_token<__half>(lc, bytes, x, ldx, w, ldw, g);
        return;
    }
    if (!given) {
        int8_t* to = static_cast<int8_t*>(workspace);
        float* s = reinterpret_cast<float*>(to + linear8_room(rows, k, false).scale);
        quantize_rows(lc, x, x_dtype, rows, k, ldx, to, padded8(k), padded8(k), s);
        q = to; ldq = padded8(k); g.xs = s;
    }
    if (rows > kL8FewRows) launch_pair(lc, bytes, q, ldq, w, ldw, g, !given);
    else if (rows <= 16) launch_few<16>(lc, bytes, q, ldq, w, ldw, g, !given);
    else if (rows <= 32) launch_few<32>(lc, bytes, q, ldq, w, ldw, g, !given);
    else if (rows <= 64) launch_few<64>(lc, bytes, q, ldq, w, ldw, g, !given);
    else launch_few<128>(lc, bytes, q, ldq, w, ldw, g, !given);
}

// Blocks per row: three per SM over the rows, of the four that run at once, with 16 chunks each at least (200 x 152064 f32, 1, 2 and 3 blocks a row: 30, 21.5 and
// 27.9 us; 100 x 152064, 2, 4 and 6: 16.2, 13.2 and 16.9; 64 x 152064 and twenty alternatives, 4, 6 and 7: 14.1, 13.8 and 14.7).  At most six, since larger clusters find a
// place on fewer SMs (37 x 128256 bf16, 6 and 8: 5.9 and 6.4, with five alternatives 8.5 and 9.4), except where all have an SM each: 16 then, or eight
// with alternatives, whose lists the first block joins (3 x 152064 f32, 6, 8 and 16: 4.7, 4.2 and 3.6, with twenty 8.1, 8.0 and 9.9).  A cluster of 16 is not
// portable to every chip, but B200 has it.  Small blocks where there are more rows than SMs hold large ones (256 and 128
// threads, five alternatives: 1000 x 32003 f16 20.8 and 18.2 us, 777 x 32000 f32 23.8 and 22.3, 4000 x 5000 f32 46 and 26, but 400 x 32000 f32 13.5 and 16.3).
template <typename T>
static void run_logprobs(LaunchCtx& lc, const LogprobArgs& a) {
    const int chunks = (a.vocab + 2 * LpRow<T>::N - 1 + LpRow<T>::kChunk - 1) / LpRow<T>::kChunk;
    const int most = a.rows > kNumSMs / kLpMaxCluster ? 6 : a.top > 0 ? kLpMaxCluster / 2 : kLpMaxCluster;
    const int C = std::max(1, std::min({most, 3 * kNumSMs / a.rows, chunks / 16})), per = (chunks + C - 1) / C;
    const uint64_t bytes = (uint64_t)a.rows * a.vocab * sizeof(T);
    const dim3 grid((unsigned)((long long)a.rows * C));
    const size_t smem = a.top > 0 ? (size_t)per * 4 : 0;
    auto go = [&](auto kern, int threads) { launch_op(lc, "logprobs", bytes, kern, grid, threads, smem, C, false, a, C, per); };
    if (a.rows <= 4 * kNumSMs) {
        a.top > 0 ? go(logprobs_kernel<T, true, 256>, 256) : go(logprobs_kernel<T, false, 256>, 256);
    } else {
        a.top > 0 ? go(logprobs_kernel<T, true, 128>, 128) : go(logprobs_kernel<T, false, 128>, 128);
    }
}
template <typename T>
static void run_logprobs(LaunchCtx& lc, LogprobArgs a, double temperature) {
    a.inv_t = (float)(1.0 / temperature);
    a.c = (float)(1.4426950408889634 / temperature);
    run_logprobs<T>(lc, a);
}
static void check_temperature(double temperature) {
    const float inv_t = (float)(1.0 / temperature), c = (float)(1.4426950408889634 / temperature);
    FL_CHECK(temperature > 0 && std::isfinite(temperature) && std::isfinite(c) && inv_t > 0, FL_ERR_INVALID, "logprobs: the temperature is a positive number");
}

size_t linear8_workspace(int64_t rows, int64_t k) { return linear8_room(rows, k, false).all; }
void op_quantize_rows(LaunchCtx& lc, const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, int8_t* q, int64_t ldq, float* scale) {
    set_up();
    quantize_rows(lc, x, dtype, rows, cols, ldx, q, ldq, ldq, scale);
}
void op_linear8(LaunchCtx& lc, const float* x, const int8_t* w, const float* w_scale, int64_t rows, int64_t n, int64_t k, float* y, void* workspace, size_t workspace_bytes, int* failed) {
    FL_CHECK(workspace_bytes >= linear8_workspace(rows, k), FL_ERR_INVALID, "linear8: the workspace is smaller than the product needs");
    set_up();
    run_linear8(lc, x, FL_DTYPE_F32, k, nullptr, w, padded8(k), w_scale, nullptr, rows, n, k, y, FL_DTYPE_F32, n, workspace, failed);
}
void op_logprobs(LaunchCtx& lc, const float* logits, int64_t rows, int64_t vocab, const int32_t* tokens, int64_t given, double temperature, int top, float* logprob,
                 float* logsumexp, float* entropy, int32_t* top_ids, float* top_logprobs) {
    FL_CHECK(vocab <= kLpMaxVocab, FL_ERR_UNSUPPORTED, "logprobs: a vocabulary of at most 2^20");
    FL_CHECK(top >= 0 && top <= kLpMaxTop && top <= vocab, FL_ERR_INVALID, "logprobs: from 0 to 32 alternatives, and no more than the vocabulary has");
    check_temperature(temperature);
    set_up();
    run_logprobs<float>(lc, LogprobArgs{logits, vocab, (int)rows, (int)vocab, 1.f, 1.f, tokens, (int)given, 0, top, given ? logprob : nullptr, logsumexp, entropy, top_ids,
                                        top_logprobs}, temperature);
}

}  // namespace fl

using namespace fl;

extern "C" {

FL_EXPORT int fl_quantize_rows(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, int8_t* q, int64_t ldq, float* scale, void* stream) {
    FL_API_BEGIN
    FL_CHECK(is_float(dtype), FL_ERR_INVALID, "quantize_rows: rows of f32, bf16 or f16");
    FL_CHECK(rows >= 0 && rows <= kMaxRows && cols >= 1 && cols <= kLinear8MaxK, FL_ERR_INVALID, "quantize_rows: rows from 0 to 2^30, columns from 1 to 131071");
    FL_CHECK(rows <= 1 || (ldx >= cols && ldq >= cols), FL_ERR_INVALID, "quantize_rows: a row stride is smaller than the row");
    if (rows == 0) return FL_OK;
    FL_CHECK(x && q && scale, FL_ERR_INVALID, "NULL argument");
    FL_CHECK(aligned(x, dtype_size(dtype)) && aligned(scale, 4), FL_ERR_INVALID, "quantize_rows: a pointer is not aligned to its type");
    DeviceScope dev;
    set_up();
    LaunchCtx lc = op_ctx(stream);
    quantize_rows(lc, x, dtype, rows, cols, ldx, q, ldq, cols, scale);
    FL_API_END
}

FL_EXPORT int fl_linear8_workspace(int64_t rows, int64_t k, int x_dtype, size_t* bytes) {
    FL_API_BEGIN
    FL_CHECK(bytes, FL_ERR_INVALID, "NULL argument");
    FL_CHECK(is_float(x_dtype) || x_dtype == FL_DTYPE_I8, FL_ERR_INVALID, "linear8: activations are f32, bf16, f16 or i8");
    FL_CHECK(rows >= 0 && rows <= kMaxRows && k >= 1 && k <= kLinear8MaxK, FL_ERR_INVALID, "linear8: rows from 0 to 2^30, k from 1 to 131071");
    *bytes = linear8_room(rows, k, x_dtype == FL_DTYPE_I8).all;
    FL_API_END
}

FL_EXPORT int fl_linear8(const void* x, int x_dtype, int64_t ldx, const float* x_scale, const int8_t* w, int64_t ldw, const float* w_scale, const float* bias,
                         int64_t rows, int64_t n, int64_t k, void* y, int y_dtype, int64_t ldy, void* workspace, size_t workspace_bytes, void* stream) {
    FL_API_BEGIN
    const bool given = x_dtype == FL_DTYPE_I8;
    FL_CHECK(is_float(x_dtype) || given, FL_ERR_INVALID, "linear8: activations are f32, bf16, f16 or i8");
    FL_CHECK(is_float(y_dtype), FL_ERR_INVALID, "linear8: results are f32, bf16 or f16");
    FL_CHECK(rows >= 0 && rows <= kMaxRows && n >= 1 && n <= kMaxRows && k >= 1 && k <= kLinear8MaxK, FL_ERR_INVALID,
             "linear8: rows from 0 to 2^30, n from 1 to 2^30, k from 1 to 131071");
    FL_CHECK((rows <= 1 || (ldx >= k && ldy >= n)) && (n == 1 || ldw >= k), FL_ERR_INVALID, "linear8: a row stride is smaller than the row");
    if (rows == 0) return FL_OK;
    FL_CHECK(x && w && w_scale && y, FL_ERR_INVALID, "NULL argument");
    FL_CHECK(given == (x_scale != nullptr), FL_ERR_INVALID, "linear8: x_scale comes with activations of 8 bits, and only with them");
    FL_CHECK(aligned(w, 16) && (n == 1 || ldw % 16 == 0), FL_ERR_INVALID, "linear8: the weight's rows start on 16-byte borders (pointer and row stride)");
    FL_CHECK(!given || (aligned(x, 16) && (rows == 1 || ldx % 16 == 0)), FL_ERR_INVALID, "linear8: 8-bit activation rows start on 16-byte borders (pointer and row stride)");
    FL_CHECK(aligned(x, dtype_size(x_dtype)) && aligned(y, dtype_size(y_dtype)) && aligned(w_scale, 4) && aligned(x_scale, 4) && aligned(bias, 4), FL_ERR_INVALID,
             "linear8: a pointer is not aligned to its type");
    FL_CHECK(rows <= ((int64_t)1 << 40) / n, FL_ERR_INVALID, "linear8: more than 2^40 results");
    const L8Room room = linear8_room(rows, k, given);
    FL_CHECK(room.all == 0 || (workspace && aligned(workspace, 256) && workspace_bytes >= room.all), FL_ERR_INVALID,
             "linear8: the workspace is smaller than fl_linear8_workspace asks for, or not on a 256-byte border");
    DeviceScope dev;
    set_up();
    LaunchCtx lc = op_ctx(stream);
    check_op_failed();
    run_linear8(lc, x, x_dtype, ldx, x_scale, w, ldw, w_scale, bias, rows, n, k, y, y_dtype, ldy, workspace, g_op_failed.word);
    FL_API_END
}

FL_EXPORT int fl_logprobs(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t ld, const void* tokens, int token_bytes, int64_t given,
                          double temperature, int top, float* logprob, float* logsumexp, float* entropy, int32_t* top_ids, float* top_logprobs, void* stream) {
    FL_API_BEGIN
    FL_CHECK(is_float(dtype), FL_ERR_INVALID, "logprobs: logits are f32, bf16 or f16");
    FL_CHECK(rows >= 0 && rows <= kMaxRows && vocab >= 1 && vocab <= kLpMaxVocab, FL_ERR_INVALID, "logprobs: rows from 0 to 2^30, a vocabulary from 1 to 2^20");
    FL_CHECK(rows <= 1 || ld >= vocab, FL_ERR_INVALID, "logprobs: the row stride is smaller than the vocabulary");
    FL_CHECK(given >= 0 && given <= kLpMaxVocab && (given == 0 || token_bytes == 4 || token_bytes == 8), FL_ERR_INVALID, "logprobs: given tokens are 32- or 64-bit integers");
    FL_CHECK(top >= 0 && top <= kLpMaxTop && top <= vocab, FL_ERR_INVALID, "logprobs: from 0 to 32 alternatives, and no more than the vocabulary has");
    check_temperature(temperature);
    if (rows == 0) return FL_OK;
    FL_CHECK(logits && (given == 0 || (tokens && logprob)) && (top == 0 || (top_ids && top_logprobs)), FL_ERR_INVALID, "NULL argument");
    FL_CHECK(aligned(logits, dtype_size(dtype)) && (given == 0 || aligned(tokens, token_bytes)) && aligned(logprob, 4) && aligned(logsumexp, 4) && aligned(entropy, 4) &&
                 aligned(top_ids, 4) && aligned(top_logprobs, 4), FL_ERR_INVALID, "logprobs: a pointer is not aligned to its type");
    DeviceScope dev;
    set_up();
    LaunchCtx lc = op_ctx(stream);
    const LogprobArgs a{logits, ld, (int)rows, (int)vocab, 1.f, 1.f, tokens, (int)given, token_bytes == 8, top, given ? logprob : nullptr, logsumexp, entropy, top_ids, top_logprobs};
    if (dtype == FL_DTYPE_F32) run_logprobs<float>(lc, a, temperature);
    else if (dtype == FL_DTYPE_BF16) run_logprobs<__nv_bfloat16>(lc, a, temperature);
    else run_logprobs<__half>(lc, a, temperature);
    FL_API_END
}

FL_EXPORT int fl_operators_check(void) {
    FL_API_BEGIN
    check_op_failed();
    FL_API_END
}

}  // extern "C"

// Matrix product of 4-bit rows with a scale per 32 values (rows4.cuh):
//   y[r, n] = sum_k x[r, k] w[n, k] (+ b[n]),   x, w the values that the rows stand for, sums in f32, one rounding to the result's type.
// tcgen05.mma.kind::mxf4: 64 values of K per instruction, products of two e2m1 and two powers of two, accumulators in f32.  As in linear8.cuh the weights are the 128- or
// 256-row operand: a lane of the accumulators is a weight row.  A k block is 256 values, 128 bytes of a row, and eight scales of it.
//
// Scales reach the products through tensor memory.  Of 128 rows and a group of four blocks (128 values) they are 512 bytes, [32 lanes][4 runs of 32 rows][4 blocks], which
// tcgen05.cp puts into four columns, the same in all four lane quarters; a product names the columns and which half of their words it takes.  scale4_at is that order in
// memory, so a k block's scales of a tile are one run of 1024 bytes per 128 rows.
#pragma once
#include "op_tiles.cuh"
#include "rows4.cuh"

namespace fl {

struct Linear4Args {
    int rows, n, blocks;                                    // blocks of 32 values of a row
    const uint8_t *xs, *ws;                                 // scales in the order of scale4_at, xs in tiles of the product's rows, ws of 128
    int groups;                                             // of four blocks in them (even)
    const float* bias;                                      // [n] or null
    void* y; long long ldy; int y_dtype;                    // fl_dtype
    int* failed;                                            // set when a wait ran out
    bool wide;                                              // 16-bit results whose rows start on 16-byte borders
};

constexpr int kL4Row = 128;                                 // bytes of a row in a k block: one swizzle row
constexpr uint32_t kL4WBytes = 128 * kL4Row;                // a box of 128 weight rows
constexpr uint32_t kL4Scales = 1024;                        // scales of 128 rows in a k block

// Instruction descriptor, kind::mxf4: scale ids of B and A at 4 and 29, both e2m1 (bits 7-9 = 1, 10-11 = 1), K-major, N>>3 at 17, scales are powers of two (bit 23), M>>7 at 27.
__host__ __device__ constexpr uint32_t umma_idesc_mx4(int M, int N, int half) {
    return ((uint32_t)(2 * half) << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 7) << 27) | ((uint32_t)(2 * half) << 29);
}
// [32 lanes][16 bytes] without a swizzle: 8 x 16 bytes in a row, 128 bytes to the next
__device__ __forceinline__ uint64_t umma_smem_desc_scales(const void* p) {
    return (uint64_t)((smem_u32(p) & 0x3FFFF) >> 4) | ((uint64_t)8 << 32) | ((uint64_t)1 << 46);
}
// Issued by the lane that `lead` marks, in whole warps (see uniform_warp).  One election for all of a k block's instructions: an election each made the issuing warp's
// way through a k block, 690 clocks with all its waits, longer than the products.
__device__ __forceinline__ uint32_t elect_lead() {
    uint32_t e;
    asm volatile(
        "{\n"
        ".reg .pred e;\n"
        "elect.sync _|e, 0xFFFFFFFF;\n"
        "selp.u32 %0, 1, 0, e;\n"
        "}\n"
        : "=r"(e));
    return e;
}
// The four products of a k block: 32 bytes of every operand row each, groups of four scales in columns sa (weights) and sb, sa + 4 and sb + step, two scales of a group at
// a time (id0, id1)
template <int kCtas>
__device__ __forceinline__ void umma_mx4_block(uint32_t lead, uint32_t acc, uint64_t a, uint64_t b, uint32_t id0, uint32_t id1, uint32_t sa, uint32_t sb, uint32_t step, uint32_t accumulate) {
#define FL_MX4_BLOCK(ctas)                                                                                                    \
    asm volatile(                                                                                                             \
        "{\n"                                                                                                                 \
        ".reg .pred p, e, t;\n"                                                                                               \
        ".reg .b64 x, y;\n"                                                                                                   \
        ".reg .b32 u, v;\n"                                                                                                   \
        "setp.ne.b32 e, %8, 0;\n"                                                                                             \
        "setp.ne.b32 p, %7, 0;\n"                                                                                             \
        "setp.eq.b32 t, 0, 0;\n"                                                                                              \
        "@e tcgen05.mma.cta_group::" ctas ".kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n"          \
        "add.s64 x, %1, 2; add.s64 y, %2, 2;\n"                                                                               \
        "@e tcgen05.mma.cta_group::" ctas ".kind::mxf4.block_scale.scale_vec::2X [%0], x, y, %4, [%5], [%6], t;\n"            \
        "add.s64 x, %1, 4; add.s64 y, %2, 4; add.u32 u, %5, 4; add.u32 v, %6, %9;\n"                                          \
        "@e tcgen05.mma.cta_group::" ctas ".kind::mxf4.block_scale.scale_vec::2X [%0], x, y, %3, [u], [v], t;\n"              \
        "add.s64 x, %1, 6; add.s64 y, %2, 6;\n"                                                                               \
        "@e tcgen05.mma.cta_group::" ctas ".kind::mxf4.block_scale.scale_vec::2X [%0], x, y, %4, [u], [v], t;\n"              \
        "}\n" ::"r"(acc),                                                                                                     \
        "l"(a), "l"(b), "r"(id0), "r"(id1), "r"(sa), "r"(sb), "r"(accumulate), "r"(lead), "r"(step)                           \
        : "memory")
    if constexpr (kCtas == 1) FL_MX4_BLOCK("1");
    else FL_MX4_BLOCK("2");
#undef FL_MX4_BLOCK
}
// two groups' scales of 128 rows, 512 bytes each, into columns tmem and tmem + step; copies are ordered before the products behind them
template <int kCtas>
__device__ __forceinline__ void tmem_scales(uint32_t lead, uint32_t tmem, uint32_t step, uint64_t desc, uint32_t desc_step) {
#define FL_SCALES(ctas)                                                                   \
    asm volatile(                                                                         \
        "{\n"                                                                             \
        ".reg .pred e;\n"                                                                 \
        ".reg .b64 d;\n"                                                                  \
        ".reg .b32 c;\n"                                                                  \
        "setp.ne.b32 e, %2, 0;\n"                                                         \
        "@e tcgen05.cp.cta_group::" ctas ".32x128b.warpx4 [%0], %1;\n"                    \
        "add.s64 d, %1, %4; add.u32 c, %0, %3;\n"                                         \
        "@e tcgen05.cp.cta_group::" ctas ".32x128b.warpx4 [c], d;\n"                      \
        "}\n" ::"r"(tmem),                                                                \
        "l"(desc), "r"(lead), "r"(step), "l"((uint64_t)desc_step)                         \
        : "memory")
    if constexpr (kCtas == 1) FL_SCALES("1");
    else FL_SCALES("2");
#undef FL_SCALES
}
__device__ __forceinline__ void umma_commit_lead(uint32_t lead, uint64_t* bar) {
    asm volatile("{\n.reg .pred e;\nsetp.ne.b32 e, %1, 0;\n@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar)), "r"(lead) : "memory");
}
// arrives on the barrier of both CTAs
__device__ __forceinline__ void umma_commit_pair_lead(uint32_t lead, uint64_t* bar) {
    asm volatile(
        "{\n.reg .pred e;\nsetp.ne.b32 e, %1, 0;\n@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %2;\n}\n" ::"r"(smem_u32(bar)),
        "r"(lead), "h"((uint16_t)3)
        : "memory");
}
// Results of one weight row n (a lane each) and 16 activation rows from r on
__device__ __forceinline__ void l4_store16(const Linear4Args& g, int r, int n, int rows, float bn, const uint32_t (&sum)[16]) {
    float v[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = g.bias != nullptr ? __uint_as_float(sum[j]) + bn : __uint_as_float(sum[j]);
    write16(g.y, g.ldy, g.y_dtype, r, n, n < g.n ? rows : 0, v);
}

// ---- few rows -----------------------------------------------------------------------------------------------------------------------
// As linear8_few_kernel: the weights are nearly all the traffic, BN activation rows the other operand; a cluster of S blocks cuts K of one tile, and its blocks add up
// each other's parts in order through shared memory.  What bounds it: HBM behind 5 us of launch, rounding, first weights and last results (37 x 3584 x 152064 to f32 54 us, 5.6
// TB/s of the measured 6.56; 64 x 4096 x 28672 15.6, 64 x 4096 x 4096 8.7).  Two blocks per SM hold 68 KB of weights on their way each.
template <int BN> struct L4Few {
    static constexpr uint32_t kX = BN * kL4Row, kSW = kL4WBytes + kX, kStage = kSW + 2 * kL4Scales;     // weights | activations | their scales
    static constexpr int kPerSm = 2;                                                   // blocks that an SM holds
    static constexpr uint32_t kRing = 108 * 1024;
    static constexpr int kStages = kRing / kStage < 8 ? kRing / kStage : 8;
    static constexpr size_t kSmem = (size_t)kStages * kStage + 1024;
    static constexpr int kThreads = 192;
    static constexpr uint32_t kCols = BN + 16 * kStages, kTmem = kCols <= 64 ? 64 : (kCols <= 128 ? 128 : 256);      // every stage has its own columns for scales
    static_assert(kStages * kStage >= (uint32_t)BN * 512, "the parts of a tile fit the ring");
    static_assert(kCols <= 256, "two blocks share an SM's tensor memory");
};

// The accumulators of a block's part of K (all warps call it; those from 2 on are the epilogue's): written, or added up in the cluster.
template <int BN>
__device__ __forceinline__ void l4_few_finish(const Linear4Args& g, const int S, int s, int n0, uint32_t tmem, uint8_t* ring, bool ok) {
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const int row = (warp & 3) * 32 + lane;                                            // accumulator row = weight row of the tile
    const uint32_t at = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const int n = n0 + row;
    const float bn = warp >= 2 && g.bias != nullptr && n < g.n ? g.bias[n] : 0.f;
    if (S == 1) {
        if (warp >= 2 && ok) {
#pragma unroll 1
            for (int c = 0; c < BN && c < g.rows; c += 16) {
                uint32_t v[16];
                tmem_ld16(at + (uint32_t)c, v);
                l4_store16(g, c, n, min(g.rows - c, 16), bn, v);
            }
        }
        return;
    }
    const int per = BN / S;                                                            // columns that one block of the cluster adds up and writes
    __syncwarp();
    cluster_sync_all();                                                                // every block's products are done: the rings are free
    if (warp >= 2) {
        const uint32_t base = smem_u32(ring) + (uint32_t)(s * per * 128 + row) * 4;
#pragma unroll 1
        for (int c = 0; c < BN && c < g.rows; c += 16) {
            uint32_t v[16];
            tmem_ld16(at + (uint32_t)c, v);
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int owner = (c + j) / per;
                asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(mapa_u32(base + (uint32_t)((c + j) - owner * per) * 512, owner)), "r"(v[j]) : "memory");
            }
        }
    }
    __syncwarp();
    cluster_sync_all();
    if (warp >= 2 && ok) {
        const float* part = reinterpret_cast<const float*>(ring) + row;
#pragma unroll 1
        for (int c = 0; c < per && s * per + c < g.rows; c += 16) {
            const int r = s * per + c, cnt = min(min(per - c, 16), g.rows - r);
            float v[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = 0.f;
            for (int t = 0; t < S; ++t) {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (j < cnt) v[j] += part[(t * per + c + j) * 128];
            }
            if (g.bias != nullptr) {
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] += bn;
            }
            write16(g.y, g.ldy, g.y_dtype, r, n, n < g.n ? cnt : 0, v);
        }
    }
}

template <int BN>
__global__ void __launch_bounds__(L4Few<BN>::kThreads, L4Few<BN>::kPerSm)
linear4_few_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const Linear4Args g, const int S) {
    using L = L4Few<BN>;
    constexpr int kStages = L::kStages;
    extern __shared__ uint8_t gsm_raw[];
    uint8_t* gsm = gsm_raw + ((1024u - (smem_u32(gsm_raw) & 1023u)) & 1023u);          // (the same offset in all blocks of a cluster)
    __shared__ __align__(8) uint64_t full[kStages], empty[kStages], done;
    __shared__ uint32_t tmem_base_s;
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const int s = S == 1 ? 0 : (int)cluster_rank();
    const int tile = blockIdx.x / S, n0 = tile * 128;
    const int nk = g.groups / 2, kb0 = (int)((long long)s * nk / S), kb1 = (int)((long long)(s + 1) * nk / S);

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        mbar_init(&done, 1);
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc(&tmem_base_s, L::kTmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;
    bool ok = true;

    if (warp == 0) {
        if (lane == 0) {
            auto weights = [&](int kb, int st) {
                mbar_expect_tx(&full[st], L::kStage);
                tma_load_2d(gsm + st * L::kStage, &tmW, kb * kL4Row, n0, &full[st]);
                bulk_g2s(gsm + st * L::kStage + L::kSW, g.ws + ((long long)tile * nk + kb) * kL4Scales, kL4Scales, &full[st]);
            };
            auto rows = [&](int kb, int st) {
                tma_load_2d(gsm + st * L::kStage + kL4WBytes, &tmX, kb * kL4Row, 0, &full[st]);
                bulk_g2s(gsm + st * L::kStage + L::kSW + kL4Scales, g.xs + (long long)kb * kL4Scales, kL4Scales, &full[st]);
            };
            // the weights do not depend on the kernel that rounds the rows: a ring-full of them is requested ahead of the wait
            const int pre = min(kb1, kb0 + kStages);
            for (int kb = kb0; kb < pre; ++kb) weights(kb, kb - kb0);
            pdl_wait();
            asm volatile("fence.proxy.async;" ::: "memory");                           // the rows were written through the generic proxy
            for (int kb = kb0; kb < pre; ++kb) rows(kb, kb - kb0);
            int st = 0;
            uint32_t ph = 0;
            for (int kb = pre; kb < kb1; ++kb) {
                if (!(ok = mbar_wait_bounded(&empty[st], ph, kMbarTries))) break;
                weights(kb, st);
                rows(kb, st);
                if (++st == kStages) { st = 0; ph ^= 1; }
            }
        }
    } else if (warp == 1) {
        const uint64_t base = umma_smem_desc_sw128(gsm), scales = umma_smem_desc_scales(gsm + L::kSW);
        const uint32_t lead = elect_lead();
        int st = 0;
        uint32_t ph = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (ok) ok = mbar_wait_bounded(&full[st], ph, kMbarTries);
            __syncwarp();
            const uint64_t at = (uint64_t)(st * (L::kStage >> 4)), a = base + at, b = a + (kL4WBytes >> 4);
            const uint32_t sa = tmem + BN + 16 * st, sb = sa + 8;                      // (free: what was filled from this stage before has been used up)
            tmem_scales<1>(lead, sa, 4, scales + at, 512 >> 4);
            tmem_scales<1>(lead, sb, 4, scales + at + (kL4Scales >> 4), 512 >> 4);
            umma_mx4_block<1>(lead, tmem, a, b, umma_idesc_mx4(128, BN, 0), umma_idesc_mx4(128, BN, 1), sa, sb, 4, kb > kb0 ? 1u : 0u);
            umma_commit_lead(lead, &empty[st]);
            if (++st == kStages) { st = 0; ph ^= 1; }
        }
        umma_commit_lead(lead, &done);
    }
    if (warp >= 2) {
        pdl_wait();                                                                    // (no block ends before the kernel that rounds the rows has)
        ok = __all_sync(0xFFFFFFFFu, mbar_wait_bounded(&done, 0, kMbarTries));
        tc_fence_after();
    }
    l4_few_finish<BN>(g, S, s, n0, tmem, gsm, ok);
    if (!ok) op_give_up(g.failed);
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, L::kTmem);
    }
}

// ---- up to 16 rows, brought to 4 bits on the way ---------------------------------------------------------------------------------------
// The warps of the epilogue round a k block of all rows (a block of 32 a thread) while its weights are on their way, straight into the ring; rows that are in 4 bits already they
// bring there with their scales.  Every block of threads does that anew, from L2; what it saves is a launch, and the wait for it between the first weights and the first product.  What bounds it:
// HBM for one row of a large matrix (1 x 3584 x 152064 52 us, 5.6 TB/s), the rounding, done anew for every weight tile, for more rows of one, the way from launch to last result for
// small ones.  The rule looks at the rows alone, so that a call of up to 16 is one launch without a workspace (9 us of the host's time, of two launches 15), and where that does not count it is the
// slower form from three rows on: here 4, 8 and 16 rows, and 17 with the rounding in a launch of its own, take 60, 63, 66 and 53 us on the device; of 4096 x 28672 16.5, 17.2, 18.1 and
// 16.0, of 4096 x 4096 7.5, 7.7, 8.1 and 7.5.
constexpr int kL4SelfRows = 16;
struct L4Self {
    static constexpr int kRows = kL4SelfRows;
    static constexpr uint32_t kX = kRows * kL4Row, kSW = kL4WBytes + kX, kStage = kSW + 2 * kL4Scales;
    static constexpr int kPerSm = 2, kStages = 5, kThreads = 192, kRounders = 128;
    static constexpr size_t kSmem = (size_t)kStages * kStage + 1024;
    static constexpr uint32_t kTmem = 128;
    static_assert(kRows + 16 * kStages <= (int)kTmem && kStages * kStage >= kRows * 512u, "accumulators and every stage's scales; the parts of a tile fit the ring");
};

// T: the rows' type; uint8_t: 4-bit rows (ldx in bytes) with their scales g.xs [rows][lds]
template <typename T, bool kVec>
__global__ void __launch_bounds__(L4Self::kThreads, L4Self::kPerSm)
linear4_self_kernel(const __grid_constant__ CUtensorMap tmW, const Linear4Args g, const T* __restrict__ x, const long long ldx, const int k, const long long lds, const int S) {
    using L = L4Self;
    constexpr bool kGiven = std::is_same_v<T, uint8_t>;
    constexpr int kStages = L::kStages, BN = L::kRows, kPieces = BN * 8 * kR4Lanes<T> / L::kRounders;      // pieces of 64 bytes (16 of 4-bit rows) a thread and k block
    extern __shared__ uint8_t gsm_raw[];
    uint8_t* gsm = gsm_raw + ((1024u - (smem_u32(gsm_raw) & 1023u)) & 1023u);          // (the same offset in all blocks of a cluster)
    __shared__ __align__(8) uint64_t full[kStages], empty[kStages], done;
    __shared__ uint32_t tmem_base_s;
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const int s = S == 1 ? 0 : (int)cluster_rank();
    const int tile = blockIdx.x / S, n0 = tile * 128;
    const int nk = g.groups / 2, kb0 = (int)((long long)s * nk / S), kb1 = (int)((long long)(s + 1) * nk / S);

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) { mbar_init(&full[i], 1 + L::kRounders / 32); mbar_init(&empty[i], 1); }
        mbar_init(&done, 1);
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc(&tmem_base_s, L::kTmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;
    bool ok = true;

    if (warp == 0) {
        if (lane == 0) {
            int st = 0;
            uint32_t ph = 1;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!(ok = mbar_wait_bounded(&empty[st], ph, kMbarTries))) break;
                mbar_expect_tx(&full[st], kL4WBytes + kL4Scales);
                tma_load_2d(gsm + st * L::kStage, &tmW, kb * kL4Row, n0, &full[st]);
                bulk_g2s(gsm + st * L::kStage + L::kSW, g.ws + ((long long)tile * nk + kb) * kL4Scales, kL4Scales, &full[st]);
                if (++st == kStages) { st = 0; ph ^= 1; }
            }
        }
    } else if (warp == 1) {
        const uint64_t base = umma_smem_desc_sw128(gsm), scales = umma_smem_desc_scales(gsm + L::kSW);
        const uint32_t lead = elect_lead();
        int st = 0;
        uint32_t ph = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (ok) ok = mbar_wait_bounded(&full[st], ph, kMbarTries);
            __syncwarp();
            const uint64_t at = (uint64_t)(st * (L::kStage >> 4)), a = base + at, b = a + (kL4WBytes >> 4);
            const uint32_t sa = tmem + BN + 16 * st, sb = sa + 8;
            tmem_scales<1>(lead, sa, 4, scales + at, 512 >> 4);
            tmem_scales<1>(lead, sb, 4, scales + at + (kL4Scales >> 4), 512 >> 4);
            umma_mx4_block<1>(lead, tmem, a, b, umma_idesc_mx4(128, BN, 0), umma_idesc_mx4(128, BN, 1), sa, sb, 4, kb > kb0 ? 1u : 0u);
            umma_commit_lead(lead, &empty[st]);
            if (++st == kStages) { st = 0; ph ^= 1; }
        }
        umma_commit_lead(lead, &done);
    } else {
        const int t = threadIdx.x - 64;
        // piece i of a thread: row and place among a k block's pieces of that row
        auto row_of = [&](int i) { return (t + L::kRounders * i) / (8 * kR4Lanes<T>); };
        auto place_of = [&](int i) { return (t + L::kRounders * i) % (8 * kR4Lanes<T>); };
        constexpr int kWords = kGiven ? 5 : 16;
        uint32_t even[kPieces][kWords], odd[kPieces][kWords];   // two k blocks ahead: their way from L2 takes longer than a k block's weights
        auto fetch = [&](int kb, uint32_t (&to)[kPieces][kWords]) {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
#pragma unroll
                for (int j = 0; j < kWords; ++j) to[i][j] = 0u;
                if (kb >= kb1 || row_of(i) >= g.rows) continue;
                if constexpr (kGiven) {
                    const int b = kb * 8 + place_of(i);
                    if (b < g.blocks) {
                        const uint4 q = __ldg(reinterpret_cast<const uint4*>(x + row_of(i) * ldx) + b);
                        to[i][0] = q.x; to[i][1] = q.y; to[i][2] = q.z; to[i][3] = q.w;
                        to[i][4] = __ldg(g.xs + row_of(i) * lds + b);
                    }
                } else {
                    load64<T, kVec>(x + row_of(i) * ldx, kb * 256 + place_of(i) * kR4Own<T>, k, to[i]);
                }
            }
        };
        int st = 0;
        uint32_t ph = 1;
        auto round = [&](int kb, uint32_t (&from)[kPieces][kWords]) {
            uint32_t codes[kPieces][kR4Own<T> / 8], byte[kPieces];
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                if constexpr (kGiven) {
#pragma unroll
                    for (int h = 0; h < 4; ++h) codes[i][h] = from[i][h];
                    byte[i] = from[i][4];
                } else {
                    byte[i] = scale4(block_max<T>(most_of<T>(from[i])));
                    const float up = up4(byte[i]);
#pragma unroll
                    for (int h = 0; h < kR4Own<T> / 8; ++h) {
                        float v[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = byte[i] == 255u ? 0.f : number_of<T>(from[i], 8 * h + j) * up;
                        codes[i][h] = e2m1x8(v);
                    }
                }
            }
            fetch(kb + 2, from);
            if (ok) ok = __all_sync(0xFFFFFFFFu, mbar_wait_bounded(&empty[st], ph, kMbarTries));
            uint8_t *to = gsm + st * L::kStage + kL4WBytes, *sc = gsm + st * L::kStage + L::kSW + kL4Scales;
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int r = row_of(i), b = place_of(i) / kR4Lanes<T>;                // the 16 bytes of block b lie at b ^ (r mod 8) of the row's 128 (the operands' swizzle)
                uint8_t* at = to + r * kL4Row + ((b ^ (r & 7)) * 16);
                if constexpr (kR4Lanes<T> == 1) *reinterpret_cast<uint4*>(at) = make_uint4(codes[i][0], codes[i][1], codes[i][2], codes[i][3]);
                else *reinterpret_cast<uint2*>(at + 8 * (place_of(i) & 1)) = make_uint2(codes[i][0], codes[i][1]);
                if (place_of(i) % kR4Lanes<T> == 0) sc[b / 4 * 512 + r * 16 + b % 4] = (uint8_t)byte[i];
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");               // written through the generic proxy, read by the products
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[st]);
            if (++st == kStages) { st = 0; ph ^= 1; }
        };
        fetch(kb0, even);
        fetch(kb0 + 1, odd);
        for (int kb = kb0; kb < kb1; kb += 2) {
            round(kb, even);
            if (kb + 1 < kb1) round(kb + 1, odd);
        }
        if (ok) ok = __all_sync(0xFFFFFFFFu, mbar_wait_bounded(&done, 0, kMbarTries));
        tc_fence_after();
    }
    l4_few_finish<BN>(g, S, s, n0, tmem, gsm, ok);
    if (!ok) op_give_up(g.failed);
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, L::kTmem);
    }
}

// ---- a token or two -----------------------------------------------------------------------------------------------------------------
// One or two rows, rounded inside the product's own launch: a warp per weight row, a block of 32 weights a lane and load.  2 e2m1 is a whole number of 8 bits, so a block's
// products are summed exactly, four to an instruction, and its two scales are applied to the sum.  Every block of threads rounds the rows into its shared memory (from L2) while its
// first weights are on their way.  What bounds it: trips to memory for small matrices (2048 x 2048 3.2 us, on the tensor cores 6.0; 4096 x 4096 6.3 and 7.8), the look-ups that make
// e2m1 whole numbers for larger ones (28672 x 4096 23 and 13.6 us), which go the other way.  The rule's border is the first of these two sizes; where they cross above it was not
// measured (4096 x 4097, on the tensor cores, takes 7.4 us where 4096 x 4096 takes 6.4).
constexpr int kL4TokenRows = 2, kL4TokenBlocks = 1024, kL4TokenWork = 1 << 19, kL4TokenThreads = 256, kL4TokenAhead = 2;      // rows; most blocks of 32 of the rows, and over all products;
                                                                                                                                // loads on their way a lane

// codes of four columns in the low half (and what is above it), doubled, as four whole numbers of 8 bits
__device__ __forceinline__ uint32_t e2m1_doubled(uint32_t w) {
    const uint32_t at = w & 0x7777u, up = __byte_perm(0x03020100u, 0x0C080604u, at), down = __byte_perm(0xFDFEFF00u, 0xF4F8FAFCu, at);
    uint32_t neg;                                               // bytes of the codes' signs (which __byte_perm's selector does not ask for)
    asm("prmt.b32 %0, %1, %2, 0x9D8C;" : "=r"(neg) : "r"(w), "r"(w << 4));
    return (up & ~neg) | (down & neg);
}

// the smaller and the larger of two, NaN where one of them is
__device__ __forceinline__ void in_order(float a, float b, float& lo, float& hi) {
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(lo) : "f"(a), "f"(b));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(hi) : "f"(a), "f"(b));
}

template <typename T, int R, bool kVec>
__global__ void __launch_bounds__(kL4TokenThreads) linear4_token_kernel(const Linear4Args g, const T* __restrict__ x, const long long ldx, const int k, const uint8_t* __restrict__ w,
                                                                        const long long ldw) {
    constexpr int U = kL4TokenAhead, kWarps = kL4TokenThreads / 32;
    extern __shared__ uint4 sx[];                               // [R][2 halves of a block][blocks] whole numbers, then [R][blocks] scales / 4
    float* sscale = reinterpret_cast<float*>(sx + 2 * R * g.blocks);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, blocks = g.blocks;
    const int steps = (blocks + 32 * U - 1) / (32 * U), stride = gridDim.x * kWarps;
    struct Part { uint4 q; uint32_t s; };
    // a step: U blocks a lane of one weight row
    auto fetch = [&](int n, int step, Part (&to)[U]) {
        const uint4* row = reinterpret_cast<const uint4*>(w + (long long)n * ldw);
        const uint8_t* scales = g.ws + scale4_at(n, 0, 128, g.groups);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int b = (step * U + u) * 32 + lane;
            to[u] = Part{make_uint4(0, 0, 0, 0), 0};
            if (b < blocks) {
                to[u].q = ldg_stream(row + b);
                to[u].s = __ldg(scales + (long long)(b / 4) * 512 + b % 4);
            }
        }
    };
    int n = blockIdx.x * kWarps + warp, step = 0;
    Part now[U], next[U];
    if (n < g.n) fetch(n, 0, now);

    for (int r = 0; r < R; ++r) {
        const int per = blocks * kR4Lanes<T>;
        for (int p0 = 0; p0 < per; p0 += kL4TokenThreads) {     // (whole warps: two threads of a block of 32-bit numbers meet)
            const int piece = p0 + threadIdx.x, b = piece / kR4Lanes<T>;
            uint32_t v[16] = {};
            if (piece < per) load64<T, kVec>(x + r * ldx, piece * kR4Own<T>, k, v);
            const uint32_t s = scale4(block_max<T>(most_of<T>(v)));
            if (piece >= per) continue;
            const float up = up4(s);
            uint32_t out[8];
#pragma unroll
            for (int i = 0; i < kR4Own<T> / 8; ++i) {
                float f[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = s == 255u ? 0.f : number_of<T>(v, 8 * i + j) * up;
                const uint32_t c = e2m1x8(f);
                out[2 * i] = e2m1_doubled(c);
                out[2 * i + 1] = e2m1_doubled(c >> 16);
            }
            uint4* to = sx + 2 * r * blocks + b;
            if constexpr (kR4Lanes<T> == 1) {
                to[0] = make_uint4(out[0], out[1], out[2], out[3]);
                to[blocks] = make_uint4(out[4], out[5], out[6], out[7]);
            } else {
                to[(piece & 1) * blocks] = make_uint4(out[0], out[1], out[2], out[3]);
            }
            if (piece % kR4Lanes<T> == 0) sscale[r * blocks + b] = 0.25f * down4(s);
        }
    }
    __syncthreads();

    float sum[R] = {};
    while (n < g.n) {
        const bool last = step + 1 == steps;
        const int n1 = last ? n + stride : n, step1 = last ? 0 : step + 1;
        if (n1 < g.n) fetch(n1, step1, next);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int b = (step * U + u) * 32 + lane;
            if (b >= blocks) break;
            const uint32_t q[4] = {now[u].q.x, now[u].q.y, now[u].q.z, now[u].q.w};
            int dot[R] = {};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t m[4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    m[2 * i] = e2m1_doubled(q[2 * h + i]);
                    m[2 * i + 1] = e2m1_doubled(q[2 * h + i] >> 16);
                }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const uint4 a = sx[(2 * r + h) * blocks + b];
                    dot[r] = __dp4a((int)m[0], (int)a.x, dot[r]);
                    dot[r] = __dp4a((int)m[1], (int)a.y, dot[r]);
                    dot[r] = __dp4a((int)m[2], (int)a.z, dot[r]);
                    dot[r] = __dp4a((int)m[3], (int)a.w, dot[r]);
                }
            }
            const float d = down4(now[u].s);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                // times the smaller scale first, which is exact: the two scales' own product may be below f32's range, or above it beside a sum of zero
                float lo, hi;
                in_order(d, sscale[r * blocks + b], lo, hi);
                sum[r] = fmaf((float)dot[r] * lo, hi, sum[r]);
            }
        }
        if (last) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float v = warp_sum(sum[r]);
                sum[r] = 0.f;
                if (lane != r) continue;                        // (each row's result by a lane of its own)
                if (g.bias != nullptr) v += __ldg(g.bias + n);
                const long long at = (long long)r * g.ldy + n;
                if (g.y_dtype == 0) reinterpret_cast<float*>(g.y)[at] = v;
                else if (g.y_dtype == 1) reinterpret_cast<__nv_bfloat16*>(g.y)[at] = from_f32<__nv_bfloat16>(v);
                else reinterpret_cast<__half*>(g.y)[at] = from_f32<__half>(v);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) now[u] = next[u];
        n = n1;
        step = step1;
    }
}

// ---- many rows ----------------------------------------------------------------------------------------------------------------------
// As linear8_pair_kernel: pairs of SMs on tiles of 256 weight rows x bn activation rows, each with its 128 weight rows and half of the activation tile, and the scales
// of its weight rows and of all the tile's activation rows.  What bounds it: the tensor cores and what feeds them (4096 x 3584 x 37888 204 us, 5.5 Pop/s and 75 % of the tensor
// cores' cycles; 3000 x 8192 x 8192 71 us, 5.7 Pop/s), in long runs the power limit (256 us at 1.35 GHz); below some 800 rows the first loads, which wait for the rounding, and the last
// results (300 x 4096 x 28672 26 us with the rounding's launch, 12.5 at the copy rate; the shares were not measured apart).  bn is at most 224: two accumulators and the scales of two k blocks fill tensor memory.  (Tiles of 256 to 416 rows
// as two products, without a second accumulator, move a quarter less through L2, but nothing hides their results: 4096 x 3584 x 37888 251 us with 416 rows, 221 with 208.)
constexpr int kL4PairEpi = 16, kL4PairThreads = 64 + 32 * kL4PairEpi, kL4PairMaxStages = 8, kL4PairMinRows = 64, kL4PairMaxRows = 224;
constexpr uint32_t kL4PairRing = 200 * 1024, kL4PairOut = 16 * 256;            // the ring; 16 rows of 128 results on their way out, for each four warps
constexpr size_t kL4PairSmem = kL4PairRing + kL4PairEpi / 4 * kL4PairOut + 1024;

struct L4Pair {
    int bn;                     // activation rows of a tile, a multiple of 16
    int nk, mt, nt;             // k blocks; weight and activation tiles
    int raster;                 // activation tiles that share a weight tile before the walk moves on
    int stages, slots;          // of the ring; k blocks whose scales tensor memory holds
};
inline int l4_pair_atoms(int bn) { return (bn + 127) / 128; }
// bytes of a stage: weights | half of the activations | scales of the weights | of the activations
inline uint32_t l4_pair_stage(int bn) { return kL4WBytes + (uint32_t)bn * (kL4Row / 2) + kL4Scales * (uint32_t)(1 + l4_pair_atoms(bn)); }
// k blocks whose scales find a place in tensor memory beside two accumulators
inline int l4_pair_slots(int bn) { return (512 - 2 * bn) / (8 + 8 * l4_pair_atoms(bn)); }

__device__ __forceinline__ void expect_tx_lead(uint32_t lead, uint32_t bar, uint32_t bytes) {
    asm volatile("{\n.reg .pred e;\nsetp.ne.b32 e, %2, 0;\n@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n}\n" ::"r"(bar), "r"(bytes), "r"(lead) : "memory");
}
// completes on a barrier of the pair's first CTA (mbar: its shared::cluster address)
__device__ __forceinline__ void tma_load_2d_pair_lead(uint32_t lead, uint32_t dst, const CUtensorMap* tmap, int c0, int c1, uint32_t mbar) {
    asm volatile(
        "{\n.reg .pred e;\nsetp.ne.b32 e, %5, 0;\n"
        "@e cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n}\n" ::"r"(dst),
        "l"(tmap), "r"(c0), "r"(c1), "r"(mbar), "r"(lead)
        : "memory");
}
// 16 rows of the results of 128 weight rows from n0 on, by four warps through their shared memory: whole lines of a row at a time.  A warp alone writes 64 bytes of a row with
// an instruction (4096 x 3584 x 37888 without this 224 us, with it 218).
__device__ __forceinline__ void l4_store_wide(const Linear4Args& g, int r, int n0, int rows, float bn, const uint32_t (&sum)[16], uint8_t* out, int barrier) {
    const int lane = threadIdx.x & 31, q = (threadIdx.x >> 5) & 3;
    unsigned short* to = reinterpret_cast<unsigned short*>(out) + q * 32 + lane;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const float v = g.bias != nullptr ? __uint_as_float(sum[j]) + bn : __uint_as_float(sum[j]);
        to[j * 128] = g.y_dtype == 1 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
    }
    asm volatile("bar.sync %0, 128;" ::"r"(barrier) : "memory");
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int j = 4 * q + 2 * i + (lane >> 4);
        if (j < rows) *reinterpret_cast<uint4*>(reinterpret_cast<unsigned short*>(g.y) + (long long)(r + j) * g.ldy + n0 + (lane & 15) * 8) = *reinterpret_cast<const uint4*>(out + j * 256 + (lane & 15) * 16);
    }
    asm volatile("bar.sync %0, 128;" ::"r"(barrier) : "memory");
}

// kAtoms: l4_pair_atoms of a tile's rows
template <int kAtoms>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kL4PairThreads, 1)
linear4_pair_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmWS, const __grid_constant__ CUtensorMap tmXS,
                    const Linear4Args g, const L4Pair p) {
    extern __shared__ uint8_t gsm_raw[];
    uint8_t* gsm = gsm_raw + ((1024u - (smem_u32(gsm_raw) & 1023u)) & 1023u);          // (the same offset in both CTAs)
    __shared__ __align__(8) uint64_t full[kL4PairMaxStages], empty[kL4PairMaxStages], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_base_s;
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int cl = blockIdx.x >> 1, G = gridDim.x >> 1, nk = p.nk, T = p.mt * p.nt, bn = p.bn;
    const uint32_t x_bytes = (uint32_t)bn * (kL4Row / 2), stage = kL4WBytes + x_bytes + kL4Scales * (uint32_t)(1 + kAtoms);

    if (threadIdx.x == 0) {
        for (int i = 0; i < p.stages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], 2 * kL4PairEpi); }
        mbar_fence_init();
        tma_prefetch_desc(&tmX);
        tma_prefetch_desc(&tmW);
        tma_prefetch_desc(&tmXS);
        tma_prefetch_desc(&tmWS);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_s;
    auto place = [&](int tile, int& n, int& rt) {
        const int per = p.raster * p.mt, first = tile / per * p.raster, local = tile % per, cnt = min(p.raster, p.nt - first);
        rt = first + local % cnt;
        n = local / cnt * 256 + (int)rank * 128;
    };
    bool ok = true;

    if (warp == 0) {
        const uint32_t lead = elect_lead();
        pdl_wait();
        asm volatile("fence.proxy.async;" ::: "memory");
        int st = 0;
        uint32_t ph = 1;
        const int w_last = (g.n + 127) / 128 - 1;                                              // scales exist for tiles that hold a row
        for (int tile = cl; ok && tile < T; tile += G) {
            int n0, rt;
            place(tile, n0, rt);
            const int r0 = rt * bn + (int)rank * (bn >> 1);
            const int ws0 = min(n0 / 128, w_last) * nk * 2, xs0 = rt * nk * 2 * kAtoms;
            for (int kb = 0; kb < nk; ++kb) {
                if (!(ok = mbar_wait_bounded(&empty[st], ph, kMbarTries))) break;
                const uint32_t bar = mapa_u32(smem_u32(&full[st]), 0), sa = smem_u32(gsm) + st * stage, ss = sa + kL4WBytes + x_bytes;
                if (rank == 0) expect_tx_lead(lead, smem_u32(&full[st]), 2 * stage);                           // both CTAs' loads complete on the first one's barrier
                tma_load_2d_pair_lead(lead, sa, &tmW, kb * kL4Row, n0, bar);
                tma_load_2d_pair_lead(lead, sa + kL4WBytes, &tmX, kb * kL4Row, r0, bar);
                tma_load_2d_pair_lead(lead, ss, &tmWS, 0, ws0 + 2 * kb, bar);
                tma_load_2d_pair_lead(lead, ss + kL4Scales, &tmXS, 0, xs0 + 2 * kAtoms * kb, bar);
                if (++st == p.stages) { st = 0; ph ^= 1; }
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t id0 = umma_idesc_mx4(256, bn, 0), id1 = umma_idesc_mx4(256, bn, 1);
            constexpr uint32_t kCols = 8 + 8 * kAtoms;
            const uint32_t scale0 = tmem_base + 2 * bn, lead = elect_lead();
            const uint64_t base = umma_smem_desc_sw128(gsm), scales = umma_smem_desc_scales(gsm + kL4WBytes + x_bytes);
            const bool look_back = p.slots < p.stages;
            int st = 0, back = 0, slot = 0, free = p.slots;                            // back: the stage of p.slots k blocks ago
            uint32_t ph = 0, back_ph = 0, seg = 0;
            // Both waits of a k block are looked at while the products before it are issued: a look takes 160 clocks even where there is nothing to wait for.
            bool here = false, unused = false;
            auto wait = [&](uint64_t* bar, uint32_t parity) {
                if (ok) ok = pair_wait(bar, parity);
                __syncwarp();
                tc_fence_after();
            };
            for (int tile = cl; tile < T; tile += G, ++seg) {
                const uint32_t as = seg & 1, tacc = tmem_base + as * bn;
                wait(&acc_empty[as], ((seg >> 1) & 1) ^ 1);
                for (int kb = 0; kb < nk; ++kb) {
                    // (no fence behind these two: what they wait for are copies into shared memory and this thread's own products)
                    if (!here && ok) ok = mbar_wait_bounded(&full[st], ph, kMbarTries);
                    const int st0 = st;
                    if (++st == p.stages) { st = 0; ph ^= 1; }
                    if (look_back && free == 0) {                                      // the columns for scales are free when the products that took them last are done
                        if (!unused && ok) ok = mbar_wait_bounded(&empty[back], back_ph, kMbarTries);
                        if (++back == p.stages) { back = 0; back_ph ^= 1; }
                        unused = mbar_test(&empty[back], back_ph);
                    } else {
                        --free;
                    }
                    here = mbar_test(&full[st], ph);
                    __syncwarp();
                    const uint64_t at = (uint64_t)(st0 * (stage >> 4)), a = base + at, b = a + (kL4WBytes >> 4), sd = scales + at;
                    const uint32_t sa = scale0 + slot * kCols, sb = sa + 8, more = kb > 0 ? 1u : 0u;
                    if (++slot == p.slots) slot = 0;
                    // columns: weights' groups 0 and 1, then for each group the atoms of the activation rows
                    tmem_scales<2>(lead, sa, 4, sd, 512 >> 4);
#pragma unroll
                    for (int i = 0; i < kAtoms; ++i) tmem_scales<2>(lead, sb + 8 * i, 4, sd + (kL4Scales >> 4) * (1 + i), 512 >> 4);
                    umma_mx4_block<2>(lead, tacc, a, b, id0, id1, sa, sb, 4 * kAtoms, more);
                    umma_commit_pair_lead(lead, &empty[st0]);
                }
                umma_commit_pair_lead(lead, &acc_full[as]);
            }
        }
    } else {
        const int q = warp & 3, cs = (warp - 2) >> 2;                                  // TMEM lane quarter (hardware rule); every fourth run of 16 columns
        uint32_t seg = 0;
        pdl_wait();                                                                    // (no block ends before the kernel that rounds the rows has)
        for (int tile = cl; tile < T; tile += G, ++seg) {
            int n0, rt;
            place(tile, n0, rt);
            const int n = n0 + q * 32 + lane;
            const float bias = g.bias != nullptr && n < g.n ? __ldg(g.bias + n) : 0.f;
            const uint32_t as = seg & 1;
            const int r0 = rt * bn, last_col = min(bn, g.rows - r0);
            if (ok) ok = __all_sync(0xFFFFFFFFu, pair_wait(&acc_full[as], (seg >> 1) & 1));
            tc_fence_after();
            const uint32_t at = tmem_base + as * bn + ((uint32_t)(q * 32) << 16);
#pragma unroll 1
            for (int c = cs * 16; c < last_col; c += 64) {
                uint32_t v[16];
                tmem_ld16(at + (uint32_t)c, v);
                const int rows = ok ? min(last_col - c, 16) : 0;                       // (the warps that store together go on together, whoever gave up)
                if (g.wide && n0 + 128 <= g.n) l4_store_wide(g, r0 + c, n0, rows, bias, v, gsm + kL4PairRing + cs * kL4PairOut, 1 + cs);
                else l4_store16(g, r0 + c, n, rows, bias, v);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(mapa_u32(smem_u32(&acc_empty[as]), 0));
        }
    }
    if (!ok) op_give_up(g.failed);
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();          // the other CTA's products read this one's shared memory, its epilogue arrives on this one's barriers
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
    }
}

}  // namespace fl

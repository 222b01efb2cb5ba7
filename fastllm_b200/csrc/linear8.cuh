// Matrix product in 8-bit integers with a scale per token and per channel:
//   y[r, n] = (sum_k q[r, k] w[n, k]) s[r] t[n] + b[n],   q, w whole numbers of 8 bits, the sum exact in 32-bit integers,
// and the rounding of activations to such rows.  Products run on tcgen05.mma.kind::i8 with the weights as the 128- or 256-row operand throughout: a lane of the
// accumulators is a weight row, so the 32 lanes of a warp write 32 neighbours of a result row whatever its alignment, and a row count is cut
// into tiles of any multiple of 32.  Scales are applied to the finished sum in f32: the sum rounded once (2^-24), two products, the bias, then
// one rounding to the result's type.
#pragma once
#include "gemm_pair.cuh"
#include "op_tiles.cuh"

namespace fl {

// One row's rounding rule: q = 127 x / a to the nearest whole number, halves to the even one, of the exact quotient (a = max |x|).
// x * (127 / a) in f32 is off by at most 127 * 2^-23 = 1.5e-5, so only quotients that lie within 1e-4 of a half need the exact sign of
// 254 x - (2 low + 1) a.  (Rows of bf16 hold x = a / 2 once in a thousand: in 64 bits that sign took half of the kernel's time.)
struct RowScale {
    float a, mul, up;       // max |x|; 127 / a (0: all q are 0); 1, or a power of two that keeps 127 / (a up) finite in the smallest rows
    float scale;            // a / 127; NaN for a row with a NaN or an infinity
    __device__ explicit RowScale(uint32_t max_bits) {
        a = __uint_as_float(max_bits);
        const bool bad = max_bits >= 0x7F800000u;
        up = a < 1e-30f ? 0x1p96f : 1.f;
        mul = bad || a == 0.f ? 0.f : 127.f / (a * up);
        scale = bad ? __uint_as_float(0x7FFFFFFFu) : a / 127.f;
    }
    // The sign of 254 x - (2 low + 1) a, a 512th of it so that the largest rows stay in range, without a rounding that matters: the product's own is `lo`, and
    // next to a half the difference is exact (x is a 254th of a at least there: 18 bits are left).
    static __device__ __forceinline__ uint32_t exact(float x, float mul, float a) {
        const float low = floorf(x * mul), m = 2.f * low + 1.f, part = a * (1.f / 512.f), hi = m * part, lo = fmaf(m, part, -hi);
        const float over = fmaf(254.f / 512.f, x, -hi) - lo;
        const int l = (int)low;
        return (uint32_t)(over > 0.f ? l + 1 : (over < 0.f ? l : l + (l & 1)));
    }
    // four values, packed.  1.5 * 2^23 leaves the nearest whole number in the sum's low bits.
    __device__ __forceinline__ uint32_t four(float x0, float x1, float x2, float x3) const {
        constexpr float kBig = 12582912.f;
        if (mul == 0.f) return 0u;                                  // (the same for the whole row)
        const float x[4] = {x0, x1, x2, x3};
        float far = up != 1.f ? 1.f : 0.f;
        uint32_t b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float t = fmaf(x[i], mul, kBig);
            b[i] = __float_as_uint(t);
            far = fmaxf(far, fabsf(fmaf(x[i], mul, kBig - t)));
        }
        if (far > 0.4999f) {
#pragma unroll
            for (int i = 0; i < 4; ++i) b[i] = exact(x[i] * up, mul, a * up);
        }
        return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
};
// A block per row; columns [cols, cols_q) of q are filled with zeros.  kVecs > 0: the row starts on 16-byte borders on both sides (8 for q) and has at
// most kThreads * kVecs vectors of 16 bytes, which stay in registers between the maximum and the rounding; -1: such a row of any length, read
// again for the rounding, from L2 or nearer (1531 x 14336 15.9 us with eight vectors a thread in registers, 19.0 so; 8192 x 8192 f16 34.6, 5.8 TB/s); 0: any row.
template <typename T, int kVecs, int kThreads>
__global__ void __launch_bounds__(kThreads, kVecs == 8 ? 4 : 1536 / kThreads) quantize_rows_kernel(const T* __restrict__ x, long long ldx, int cols, int8_t* __restrict__ q, long long ldq,
                                                                                  int cols_q, float* __restrict__ scale) {
    constexpr int V = 16 / sizeof(T), kHeld = kVecs > 0 ? kVecs : 1;
    __shared__ uint32_t part[kThreads / 32];
    const T* xr = x + (long long)blockIdx.x * ldx;
    int8_t* qr = q + (long long)blockIdx.x * ldq;
    pdl_launch_dependents();
    auto load = [&](int at) {                                   // V values from column `at` on, zeros past the end
        uint4 h = make_uint4(0, 0, 0, 0);
        if (at + V <= cols) {
            h = *reinterpret_cast<const uint4*>(xr + at);
        } else if (at < cols) {
            T* e = reinterpret_cast<T*>(&h);
            for (int j = 0; j < V; ++j)
                if (at + j < cols) e[j] = xr[at + j];
        }
        return h;
    };
    auto most = [](uint32_t m, const uint4& h) {                // the larger magnitude, of two at once where they are 16-bit: their bits are in the order of their sizes
        if constexpr (sizeof(T) == 4)
            return max(max(m, max(h.x & 0x7FFFFFFFu, h.y & 0x7FFFFFFFu)), max(h.z & 0x7FFFFFFFu, h.w & 0x7FFFFFFFu));
        else
            return __vmaxu2(m, __vmaxu2(__vmaxu2(h.x & 0x7FFF7FFFu, h.y & 0x7FFF7FFFu), __vmaxu2(h.z & 0x7FFF7FFFu, h.w & 0x7FFF7FFFu)));
    };
    uint32_t m = 0;
    uint4 held[kHeld];
    if constexpr (kVecs > 0) {
#pragma unroll
        for (int u = 0; u < kVecs; ++u) held[u] = load((threadIdx.x + kThreads * u) * V);
#pragma unroll
        for (int u = 0; u < kVecs; ++u) m = most(m, held[u]);
    } else if constexpr (kVecs < 0) {
        int at = threadIdx.x * V;
        for (; at + (3 * kThreads + 1) * V <= cols; at += 4 * kThreads * V) {
            uint4 h[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) h[u] = *reinterpret_cast<const uint4*>(xr + at + u * kThreads * V);
#pragma unroll
            for (int u = 0; u < 4; ++u) m = most(m, h[u]);
        }
        for (; at < cols; at += kThreads * V) m = most(m, load(at));
    } else {
        for (int i = threadIdx.x; i < cols; i += kThreads) m = max(m, abs_bits(to_f32(xr[i])));
    }
    if constexpr (kVecs != 0 && sizeof(T) == 2) {
        const uint16_t h = (uint16_t)max(m & 0xFFFFu, m >> 16);
        m = abs_bits(to_f32(*reinterpret_cast<const T*>(&h)));
    }
    m = __reduce_max_sync(0xFFFFFFFFu, m);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) m = max(m, part[i]);
    const RowScale rs(m);
    auto put = [&](int at, const uint4& h) {
        const T* e = reinterpret_cast<const T*>(&h);
        uint32_t w[V / 4];
#pragma unroll
        for (int i = 0; i < V / 4; ++i) w[i] = rs.four(to_f32(e[4 * i]), to_f32(e[4 * i + 1]), to_f32(e[4 * i + 2]), to_f32(e[4 * i + 3]));
        if (at + V <= cols_q) {
            if constexpr (V == 8) *reinterpret_cast<uint2*>(qr + at) = make_uint2(w[0], w[1]);
            else *reinterpret_cast<uint32_t*>(qr + at) = w[0];
        } else {
            for (int j = 0; at + j < cols_q; ++j) qr[at + j] = (int8_t)(w[j / 4] >> (8 * (j % 4)));
        }
    };
    if constexpr (kVecs > 0) {
#pragma unroll
        for (int u = 0; u < kVecs; ++u) {
            const int at = (threadIdx.x + kThreads * u) * V;
            if (at < cols_q) put(at, held[u]);
        }
    } else if constexpr (kVecs < 0) {
#pragma unroll 2
        for (int at = threadIdx.x * V; at < cols_q; at += kThreads * V) put(at, load(at));
    } else {
        for (int i = threadIdx.x; i < cols_q; i += kThreads) qr[i] = i < cols ? (int8_t)rs.four(to_f32(xr[i]), 0.f, 0.f, 0.f) : (int8_t)0;
    }
    if (threadIdx.x == 0) scale[blockIdx.x] = rs.scale;
}

struct Linear8Args {
    int rows, n, k;
    const float* xs;                                        // [rows]
    const float* ws;                                        // [n]
    const float* bias;                                      // [n] or null
    void* y; long long ldy; int y_dtype;                    // fl_dtype
    int* failed;                                            // set when a wait ran out
};

constexpr int kL8BK = 128;                                  // 128 values = 128 bytes = one swizzle row
constexpr uint32_t kL8WBytes = 128 * kL8BK;                 // a box of 128 weight rows

// Instruction descriptor, kind::i8: D = s32 (bits 4-5 = 2), A = B = signed (bits 7-9 = 1, 10-12 = 1), both K-major, N>>3 at 17, M>>4 at 24.
__host__ __device__ constexpr uint32_t umma_idesc_i8(int M, int N) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// whole warps, one elected lane issues (see uniform_warp)
__device__ __forceinline__ void umma_i8_warp(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p, e;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "elect.sync _|e, 0xFFFFFFFF;\n"
        "@e tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_i8_pair_warp(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p, e;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "elect.sync _|e, 0xFFFFFFFF;\n"
        "@e tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void l8_store16(const Linear8Args& g, int r, int n, const float* xs, float wsn, float bn, const uint32_t (&sum)[16]) {
    float v[16];
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
        const float4 x = *reinterpret_cast<const float4*>(xs + j);
        v[j] = (float)(int)sum[j] * x.x * wsn;
        v[j + 1] = (float)(int)sum[j + 1] * x.y * wsn;
        v[j + 2] = (float)(int)sum[j + 2] * x.z * wsn;
        v[j + 3] = (float)(int)sum[j + 3] * x.w * wsn;
    }
    if (g.bias != nullptr) {
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] += bn;
    }
    write16(g.y, g.ldy, g.y_dtype, r, n, n < g.n ? min(g.rows - r, 16) : 0, v);
}
// ---- few rows -----------------------------------------------------------------------------------------------------------------------
// The weights are nearly all the traffic, BN activation rows the other operand; a cluster of S blocks cuts K of one tile, and its blocks add up each
// other's parts through shared memory: whole numbers, so the order does not matter, and no workspace.  What bounds it: HBM behind 4 to 6 us of
// launch, first weights and last results (64 x 4096 x 28672 25.3 us, 4.8 TB/s; 37 x 3584 x 152064 to f32 96.6, 5.9 TB/s of the measured 6.55; 64 x 4096 x 4096 10.1).
// Two blocks per SM hold 96 KB of weights on their way each: one writes its results while the other's arrive.
// Tiles of 64 weight rows instead, to even out the last wave, were slower nearly everywhere (64 x 4096 x 28672 23.9 -> 27.5 us, 37 x 3584 x 152064 95.8 -> 106.6,
// 16 x 4096 x 28672 23.3 -> 22.1): each needs its copy of the activations.
template <int BN> struct L8Few {
    static constexpr uint32_t kX = BN * kL8BK, kStage = kL8WBytes + kX;
    static constexpr int kPerSm = 2;                                                   // blocks that an SM holds
    static constexpr uint32_t kRing = 108 * 1024;
    static constexpr int kStages = kRing / kStage < 8 ? kRing / kStage : 8;
    static constexpr size_t kSmem = (size_t)kStages * kStage + 1024;
    static constexpr int kThreads = 192;
    static constexpr uint32_t kTmem = BN < 32 ? 32 : BN;
    static_assert(kStages * kStage >= (uint32_t)BN * 512, "the parts of a tile fit the ring");
};

// The accumulators of a block's part of K (all warps call it; those from 2 on are the epilogue's): written, or added up in the cluster.  xs: the tile's row
// scales, the calling warp's copy.
template <int BN>
__device__ __forceinline__ void l8_few_finish(const Linear8Args& g, const int S, int s, int n0, uint32_t tmem, uint8_t* ring, const float* xs, bool ok) {
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const int row = (warp & 3) * 32 + lane;                                            // accumulator row = weight row of the tile
    const uint32_t at = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const int n = n0 + row;
    const float wsn = warp >= 2 && n < g.n ? g.ws[n] : 0.f, bn = warp >= 2 && g.bias != nullptr && n < g.n ? g.bias[n] : 0.f;
    if (S == 1) {
        if (warp >= 2 && ok) {
#pragma unroll 1
            for (int c = 0; c < BN && c < g.rows; c += 16) {
                uint32_t v[16];
                tmem_ld16(at + (uint32_t)c, v);
                l8_store16(g, c, n, xs + c, wsn, bn, v);
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
        const int* part = reinterpret_cast<const int*>(ring) + row;
#pragma unroll 1
        for (int c = 0; c < per && s * per + c < g.rows; c += 16) {
            const int r = s * per + c, cnt = min(min(per - c, 16), g.rows - r);
            int sum[16];
            float v[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) sum[j] = 0;
            for (int t = 0; t < S; ++t) {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (j < cnt) sum[j] += part[(t * per + c + j) * 128];
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                v[j] = j < cnt ? (float)sum[j] * xs[s * per + c + j] * wsn : 0.f;
                if (g.bias != nullptr) v[j] += bn;
            }
            write16(g.y, g.ldy, g.y_dtype, r, n, n < g.n ? cnt : 0, v);
        }
    }
}

template <int BN>
__global__ void __launch_bounds__(L8Few<BN>::kThreads, L8Few<BN>::kPerSm)
linear8_few_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const Linear8Args g, const int S) {
    using L = L8Few<BN>;
    constexpr int kStages = L::kStages;
    extern __shared__ uint8_t gsm_raw[];
    uint8_t* gsm = gsm_raw + ((1024u - (smem_u32(gsm_raw) & 1023u)) & 1023u);          // (the same offset in all blocks of a cluster)
    __shared__ __align__(8) uint64_t full[kStages], empty[kStages], done;
    __shared__ __align__(16) float xs[4][BN];                                          // the rows' scales, a copy for each epilogue warp
    __shared__ uint32_t tmem_base_s;
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const int s = S == 1 ? 0 : (int)cluster_rank();
    const int n0 = blockIdx.x / S * 128;
    const int nk = (g.k + kL8BK - 1) / kL8BK, kb0 = (int)((long long)s * nk / S), kb1 = (int)((long long)(s + 1) * nk / S);

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
                tma_load_2d(gsm + st * L::kStage, &tmW, kb * kL8BK, n0, &full[st]);
            };
            auto rows = [&](int kb, int st) { tma_load_2d(gsm + st * L::kStage + kL8WBytes, &tmX, kb * kL8BK, 0, &full[st]); };
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
        constexpr uint32_t idesc = umma_idesc_i8(128, BN);
        const uint64_t base = umma_smem_desc_sw128(gsm);
        int st = 0;
        uint32_t ph = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (ok) ok = mbar_wait_bounded(&full[st], ph, kMbarTries);
            __syncwarp();
            tc_fence_after();
            const uint64_t a = base + (uint64_t)(st * (L::kStage >> 4)), b = a + (kL8WBytes >> 4);
#pragma unroll
            for (int q = 0; q < 4; ++q) umma_i8_warp(tmem, a + 2 * q, b + 2 * q, idesc, ((kb - kb0) | q) ? 1u : 0u);
            umma_commit_warp(&empty[st]);
            if (++st == kStages) { st = 0; ph ^= 1; }
        }
        umma_commit_warp(&done);
    }
    if (warp >= 2) {
        pdl_wait();
        for (int i = lane; i < BN; i += 32) xs[warp - 2][i] = i < g.rows ? g.xs[i] : 0.f;
        __syncwarp();
        ok = __all_sync(0xFFFFFFFFu, mbar_wait_bounded(&done, 0, kMbarTries));
        tc_fence_after();
    }
    l8_few_finish<BN>(g, S, s, n0, tmem, gsm, xs[max(warp - 2, 0)], ok);
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
// One or two rows, rounded inside the product's own launch: a warp per weight row, 16 bytes a lane and load, four products of 8 bits per instruction.  Every
// block rounds the rows into its shared memory (from L2) while its first weights are on their way.  What bounds it: HBM for large matrices (1 x 3584 x 152064
// 81 us, 6.7 TB/s), launch and two trips to memory for small ones (1 x 4096 x 4096 6.2 us, with the tensor cores 9.8; 2048 x 2048 3.6 and 7.5).  The
// products cost 7 us a row at 4096 x 28672, so from three rows on the tensor cores are faster (1, 2 and 4 rows 21.1, 22.7 and 43.9 us, there
// 23.0, 23.5 and 24.0), and so they are for two long rows, whose rounding every block repeats (2 x 4096 x 4096 8.6 and 10.0, 2 x 8192 x 8192 18.4 and 17.7,
// 2 x 14336 x 4096 20.2 and 16.4; 1 x 14336 x 4096 15.7 and 16.4).
constexpr int kL8TokenRows = 2, kL8TokenValues = 16384, kL8TokenThreads = 256, kL8TokenAhead = 4;      // rows; most rows^2 k; loads on their way a lane

template <typename T, int R>
__global__ void __launch_bounds__(kL8TokenThreads) linear8_token_kernel(const Linear8Args g, const T* __restrict__ x, const long long ldx, const bool vec, const int8_t* __restrict__ w,
                                                                        const long long ldw) {
    constexpr int V = 16 / sizeof(T), U = kL8TokenAhead, kWarps = kL8TokenThreads / 32;
    extern __shared__ uint4 sx[];                               // [R][pieces of 16 values], zeros past the end
    __shared__ uint32_t most[kWarps][R];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int pieces = (g.k + 15) / 16, whole = g.k / 16, steps = (pieces + 32 * U - 1) / (32 * U), stride = gridDim.x * kWarps;
    // a step: U pieces a lane of one weight row; pieces past the row's end are zeros, the one that holds it is read value by value
    auto fetch = [&](int n, int step, uint4 (&to)[U]) {
        const int8_t* row = w + (long long)n * ldw;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (step * U + u) * 32 + lane;
            to[u] = make_uint4(0, 0, 0, 0);
            if (i < whole) {
                to[u] = ldg_stream(reinterpret_cast<const uint4*>(row) + i);
            } else if (i < pieces) {
                uint32_t b[4] = {0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (i * 16 + j < g.k) b[j / 4] |= (uint32_t)(uint8_t)row[i * 16 + j] << (8 * (j % 4));
                to[u] = make_uint4(b[0], b[1], b[2], b[3]);
            }
        }
    };
    int n = blockIdx.x * kWarps + warp, step = 0;
    uint4 now[U], next[U];
    if (n < g.n) fetch(n, 0, now);

    // all rows' loads of a round are on their way together
    auto load = [&](int r, int at) {                            // V values of row r from column `at` on, zeros past the end
        uint4 h = make_uint4(0, 0, 0, 0);
        const T* xr = x + r * ldx;
        if (vec && at + V <= g.k) {
            h = __ldg(reinterpret_cast<const uint4*>(xr + at));
        } else {
            T* e = reinterpret_cast<T*>(&h);
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (at + j < g.k) e[j] = xr[at + j];
        }
        return h;
    };
    uint32_t m[R] = {};
#pragma unroll 2
    for (int i = threadIdx.x * V; i < g.k; i += kL8TokenThreads * V) {
        uint4 h[R];
#pragma unroll
        for (int r = 0; r < R; ++r)
            h[r] = load(r, i);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const T* e = reinterpret_cast<const T*>(&h[r]);
#pragma unroll
            for (int j = 0; j < V; ++j) m[r] = max(m[r], abs_bits(to_f32(e[j])));
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = __reduce_max_sync(0xFFFFFFFFu, m[r]);
        if (lane == 0) most[warp][r] = m[r];
    }
    __syncthreads();
    float scale[R];
    {
        float mul[R], a[R], up[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            uint32_t all = 0;
#pragma unroll
            for (int i = 0; i < kWarps; ++i) all = max(all, most[i][r]);
            const RowScale rs(all);
            scale[r] = rs.scale; mul[r] = rs.mul; a[r] = rs.a; up[r] = rs.up;
        }
#pragma unroll 2
        for (int i = threadIdx.x * V; i < pieces * 16; i += kL8TokenThreads * V) {
            uint4 h[R];
#pragma unroll
            for (int r = 0; r < R; ++r)
                h[r] = load(r, i);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                RowScale rs(0);
                rs.mul = mul[r]; rs.a = a[r]; rs.up = up[r];
                const T* e = reinterpret_cast<const T*>(&h[r]);
                uint32_t* to = reinterpret_cast<uint32_t*>(sx + r * pieces) + i / 4;
#pragma unroll
                for (int j = 0; j < V; j += 4) to[j / 4] = rs.four(to_f32(e[j]), to_f32(e[j + 1]), to_f32(e[j + 2]), to_f32(e[j + 3]));
            }
        }
    }
    __syncthreads();

    int sum[R] = {};
    while (n < g.n) {
        const bool last = step + 1 == steps;
        const int n1 = last ? n + stride : n, step1 = last ? 0 : step + 1;
        if (n1 < g.n) fetch(n1, step1, next);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (step * U + u) * 32 + lane;
            if (i >= pieces) break;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const uint4 q = sx[r * pieces + i];
                sum[r] = __dp4a((int)now[u].x, (int)q.x, sum[r]);
                sum[r] = __dp4a((int)now[u].y, (int)q.y, sum[r]);
                sum[r] = __dp4a((int)now[u].z, (int)q.z, sum[r]);
                sum[r] = __dp4a((int)now[u].w, (int)q.w, sum[r]);
            }
        }
        if (last) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int all = __reduce_add_sync(0xFFFFFFFFu, sum[r]);
                sum[r] = 0;
                if (lane != r) continue;                        // (each row's result by a lane of its own)
                float v = (float)all * scale[r] * __ldg(g.ws + n);
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
// Pairs of SMs on tiles of 256 weight rows x bn activation rows (tcgen05.mma.cta_group::2): each holds its 128 weight rows and half of the activation
// tile, 16 KB + 64 bn bytes per k block of 128.  What bounds it: below bn = 256 the operands' way from L2, about 90 bytes a nanosecond and SM (a k block took 268
// ns at bn = 128, 294 at 160), from there on the tensor cores at the clock that the power limit leaves them (348 at 256, 705 at 512: 1.38 bn; 4096 x 3584 x
// 37888 433 us or 2.57 Pop/s in a row, 355 and 3.1 once).  So tiles are as wide as the row count and whole waves allow, up to 512: two products of bn / 2
// then, in the two halves of the accumulators, which tiles of up to 256 use in turn (1531 x 14336 x 4096, bn = 192 and 384: 73 and 65 us).
constexpr int kL8PairEpi = 16, kL8PairThreads = 64 + 32 * kL8PairEpi, kL8PairMaxStages = 8;
constexpr uint32_t kL8PairRing = 200 * 1024;
constexpr size_t kL8PairSmem = kL8PairRing + 1024;

struct L8Pair {
    int bn;                     // activation rows of a tile: a multiple of 32, above 256 of 64
    int nk, mt, nt;             // k blocks; weight and activation tiles
    int stages;
};

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kL8PairThreads, 1)
linear8_pair_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const Linear8Args g, const L8Pair p) {
    extern __shared__ uint8_t gsm_raw[];
    uint8_t* gsm = gsm_raw + ((1024u - (smem_u32(gsm_raw) & 1023u)) & 1023u);          // (the same offset in both CTAs)
    __shared__ __align__(8) uint64_t full[kL8PairMaxStages], empty[kL8PairMaxStages], acc_full[2], acc_empty[2];
    __shared__ __align__(16) float xs[kL8PairEpi][64];                                 // the scales of the rows that an epilogue warp writes
    __shared__ uint32_t tmem_base_s;
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int cl = blockIdx.x >> 1, G = gridDim.x >> 1, nk = p.nk, T = p.mt * p.nt, bn = p.bn;
    const int parts = bn > 256 ? 2 : 1, pn = bn / parts;                               // products of a tile, their activation rows
    const uint32_t stage = kL8WBytes + (uint32_t)bn * (kL8BK / 2);

    if (threadIdx.x == 0) {
        for (int i = 0; i < p.stages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], 2 * kL8PairEpi); }
        mbar_fence_init();
        tma_prefetch_desc(&tmX);
        tma_prefetch_desc(&tmW);
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
    // 8 activation tiles share a weight tile before the walk moves on (see kGemmRasterRows)
    auto place = [&](int tile, int& n, int& r) {
        constexpr int RM = kGemmRasterRows / 2;
        const int per = RM * p.mt, first = tile / per * RM, local = tile % per, cnt = min(RM, p.nt - first);
        r = (first + local % cnt) * bn;
        n = local / cnt * 256 + (int)rank * 128;
    };
    bool ok = true;

    if (warp == 0) {
        if (lane == 0) {
            pdl_wait();
            asm volatile("fence.proxy.async;" ::: "memory");
            int st = 0;
            uint32_t ph = 1;
            for (int tile = cl; ok && tile < T; tile += G) {
                int n0, r0;
                place(tile, n0, r0);
                r0 += (int)rank * (pn >> 1);
                for (int kb = 0; kb < nk; ++kb) {
                    if (!(ok = pair_wait(&empty[st], ph))) break;
                    if (rank == 0) mbar_expect_tx(&full[st], 2 * stage);               // both CTAs' loads complete on the first one's barrier
                    const uint32_t bar = mapa_u32(smem_u32(&full[st]), 0), sa = smem_u32(gsm) + st * stage;
                    tma_load_2d_pair(sa, &tmW, kb * kL8BK, n0, bar);
                    tma_load_2d_pair(sa + kL8WBytes, &tmX, kb * kL8BK, r0, bar);
                    if (parts == 2) tma_load_2d_pair(sa + kL8WBytes + (uint32_t)pn * (kL8BK / 2), &tmX, kb * kL8BK, r0 + pn, bar);
                    if (++st == p.stages) { st = 0; ph ^= 1; }
                }
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t idesc = umma_idesc_i8(256, pn), second = ((uint32_t)pn * (kL8BK / 2)) >> 4;
            const uint64_t base = umma_smem_desc_sw128(gsm);
            int st = 0;
            uint32_t ph = 0, seg = 0;
            auto wait = [&](uint64_t* bar, uint32_t parity) {
                if (ok) ok = pair_wait(bar, parity);
                __syncwarp();
                tc_fence_after();
            };
            for (int tile = cl; tile < T; tile += G, ++seg) {
                const uint32_t as = parts == 2 ? 0 : seg & 1, uses = parts == 2 ? seg : seg >> 1, tacc = tmem_base + as * 256;
                wait(&acc_empty[as], (uses & 1) ^ 1);
                if (parts == 2) wait(&acc_empty[1], (uses & 1) ^ 1);
                for (int kb = 0; kb < nk; ++kb) {
                    wait(&full[st], ph);
                    const uint64_t a = base + (uint64_t)(st * (stage >> 4)), b = a + (kL8WBytes >> 4);
#pragma unroll
                    for (int q = 0; q < 4; ++q) umma_i8_pair_warp(tacc, a + 2 * q, b + 2 * q, idesc, (kb | q) ? 1u : 0u);
                    if (parts == 2) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) umma_i8_pair_warp(tacc + 256, a + 2 * q, b + second + 2 * q, idesc, (kb | q) ? 1u : 0u);
                    }
                    umma_commit_pair_warp(&empty[st]);
                    if (++st == p.stages) { st = 0; ph ^= 1; }
                }
                umma_commit_pair_warp(&acc_full[as]);
                if (parts == 2) umma_commit_pair_warp(&acc_full[1]);
            }
        }
    } else {
        const int q = warp & 3, cs = (warp - 2) >> 2;                                  // TMEM lane quarter (hardware rule); every fourth run of 16 columns
        uint32_t seg = 0;
        pdl_wait();                                                                    // (the rows' scales)
        for (int tile = cl; tile < T; tile += G, ++seg) {
            int n0, r0;
            place(tile, n0, r0);
            const int n = n0 + q * 32 + lane;
            const float wsn = n < g.n ? __ldg(g.ws + n) : 0.f, bias = g.bias != nullptr && n < g.n ? __ldg(g.bias + n) : 0.f;
            for (int h = 0; h < parts; ++h, r0 += pn) {
                const uint32_t as = parts == 2 ? (uint32_t)h : seg & 1, uses = parts == 2 ? seg : seg >> 1;
                float* own = xs[warp - 2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {                                          // run i of 16 columns: (cs + 4 i) 16 on; on its way while the products are
                    const int r = r0 + (cs + 4 * (2 * i + (lane >> 4))) * 16 + (lane & 15);
                    own[32 * i + lane] = r < g.rows ? __ldg(g.xs + r) : 0.f;
                }
                __syncwarp();
                if (ok) ok = __all_sync(0xFFFFFFFFu, pair_wait(&acc_full[as], uses & 1));
                tc_fence_after();
                const uint32_t at = tmem_base + as * 256 + ((uint32_t)(q * 32) << 16);
                const int last_col = min(pn, g.rows - r0);
#pragma unroll 1
                for (int c = cs * 16; ok && c < last_col; c += 64) {
                    uint32_t v[16];
                    tmem_ld16(at + (uint32_t)c, v);
                    l8_store16(g, r0 + c, n, own + (c >> 6) * 16, wsn, bias, v);
                }
                tc_fence_before();
                __syncwarp();                                                          // (and everyone is done with the scales)
                if (lane == 0) mbar_arrive_cluster(mapa_u32(smem_u32(&acc_empty[as]), 0));
            }
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

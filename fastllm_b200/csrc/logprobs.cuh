// Log probabilities over a vocabulary: z = x / T, logZ = log sum exp z, lp(t) = z_t - logZ, H = logZ - sum p z, and the largest logits with
// theirs, the lowest index first among equals.
//
// One pass over the logits.  A thread keeps a reference r near its running maximum and adds up e = 2^(c x - r) and e (c x - r), c = log2(e) / T; sums with
// different references are brought to the largest one and joined.  The reference moves when a maximum is 2^16 above it, so the exponentials
// stay far from overflow and the loop is nearly free of rescaling.  A row belongs to a cluster of C blocks (C = 1 when there are many rows), whose results
// meet in the first block's shared memory: no workspace, no atomics, the same bits every time.
// What bounds it: HBM for 32-bit rows (1000 x 152064 91 us, 6.7 TB/s), the exponentials for 16-bit ones (2048 x 152064 bf16 99 us, 6.3 TB/s: one per logit is
// 77 % of what the special-function units do, 5.6 instructions per logit half of the issue slots), latency for few (1 x 32000: 2.8 us, 5.3 with five
// alternatives): trips to memory one after the other.  So the given token is looked up while the row is read (1000 cycles when waited for), and chunks at the
// row's ends are asked for before the batches between them, not behind them.
//
// Alternatives: the row lies in chunks of 512 bytes (one load of a warp), whose maxima are kept.  A block's threads form 64 groups; the K-th largest of the groups'
// maxima is a lower bound for the block's K-th largest logit, since K groups hold one at least as large.  Only chunks that reach the bound are read again (from
// L2), only logits that reach it are ranked: 5 of 5, 24 of 20 or 44 of 32 where the order is random.  (Groups of one thread bring those to 21 and 34,
// but the bound is found in K steps over what a warp holds, 31 cycles each with two values a lane.)  Where fewer than K logits are above -infinity, all of them
// are ranked and the lowest indices fill up.  Where equal logits leave more than the tables hold, the K best chunks by (maximum, lower index) are
// taken instead: a logit outside them is behind K others, one per chunk; then K rounds pick one each.
#pragma once
#include "linear8.cuh"

namespace fl {

constexpr int kLpMaxTop = 32;
constexpr int kLpMaxVocab = 1 << 20;
constexpr int kLpMaxCluster = 16;
constexpr int kLpGroups = 64;                       // of a block's threads
// Where the loop over a row holds.  A distance c x - r is off by half a step of r, 4 up to 2^27: up to there sums stay far from overflow and lose a few bits at
// most.  So references begin at -2^27, and what lies below (masks: -infinity or any large negative number) does not move them; they begin kLpNothing above
// what -infinity is raised to (kLow) where that is higher, so that it counts 2^-256, which is 0.  Rows whose maximum is not that far above kLow or lies more than
// 2^27 from 0, and temperatures at which c kLow would overflow, are summed once more.
constexpr float kLpFarAt = 0x1p27f, kLpNothing = 256.f;
constexpr uint32_t kLpFinite = 0x00800000u;         // ordered_bits of the lowest finite value: the next above -infinity's
constexpr int kLpList = 96, kLpCand = 256;          // chunks that are read again, logits that are ranked

struct LogprobArgs {
    const void* x; long long ld;                // [rows, vocab]
    int rows, vocab;
    float inv_t, c;                             // 1 / T, log2(e) / T
    const void* tokens; int given, wide;        // [rows, given] int32, or int64 (wide)
    int top;
    float *logprob, *logsumexp, *entropy;       // [rows, given], [rows], [rows]; null = not wanted
    int* top_ids; float* top_logprobs;          // [rows, top]
};

// larger for the larger logit, and for the lower index among equal ones (-0 equals 0); NaN is not asked for
__device__ __forceinline__ uint32_t ordered_bits(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);
    return (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t o) { return __uint_as_float((o >> 31) ? o & 0x7FFFFFFFu : ~o); }
__device__ __forceinline__ unsigned long long order_key(uint32_t ordered, int i) { return (unsigned long long)ordered << 32 | (uint32_t)~i; }

__device__ __forceinline__ float ex2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// two f32 at once
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// 16 bytes of logits.  kLow: what lies below is raised to it before the sums, so that e (c x - r) is 0 and not 0 times infinity (NaN stays NaN)
template <typename T> struct LpVec;
template <> struct LpVec<float> {
    static constexpr int N = 4;
    static constexpr float kLow = -1e30f;
    static constexpr uint32_t kNone = 0xFF800000u;              // -infinity, in every place of a word
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
    static __device__ __forceinline__ float last(uint32_t m) { return __uint_as_float(m); }
    static __device__ __forceinline__ float raise(uint32_t w) {
        float r;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(w)), "f"(kLow));
        return r;
    }
    template <typename F> static __device__ __forceinline__ void pairs(const uint4& v, F&& f) {
        f(raise(v.x), raise(v.y));
        f(raise(v.z), raise(v.w));
    }
    static __device__ __forceinline__ float at(const uint4& v, int j) { return __uint_as_float(j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w); }
};
template <> struct LpVec<__nv_bfloat16> {
    static constexpr int N = 8;
    static constexpr float kLow = -1e30f;
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static constexpr uint32_t kNone = 0xFF80FF80u;
    static __device__ __forceinline__ float last(uint32_t m) { return fmaxf(bf16lo(m), bf16hi(m)); }
    template <typename F> static __device__ __forceinline__ void pairs(const uint4& v, F&& f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w = i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
            asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(w) : "r"(w), "r"(0xF14AF14Au));     // (-1.0002e30)
            f(bf16lo(w), bf16hi(w));
        }
    }
    static __device__ __forceinline__ float at(const uint4& v, int j) {
        const uint32_t w = j < 2 ? v.x : j < 4 ? v.y : j < 6 ? v.z : v.w;
        return (j & 1) ? bf16hi(w) : bf16lo(w);
    }
};
template <> struct LpVec<__half> {
    static constexpr int N = 8;
    static constexpr float kLow = -65504.f;
    static __device__ __forceinline__ float2 two(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static constexpr uint32_t kNone = 0xFC00FC00u;
    static __device__ __forceinline__ float last(uint32_t m) {
        const float2 p = two(m);
        return fmaxf(p.x, p.y);
    }
    template <typename F> static __device__ __forceinline__ void pairs(const uint4& v, F&& f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w = i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
            asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(w) : "r"(w), "r"(0xFBFFFBFFu));      // (-65504)
            const float2 p = two(w);
            f(p.x, p.y);
        }
    }
    static __device__ __forceinline__ float at(const uint4& v, int j) {
        const float2 p = two(j < 2 ? v.x : j < 4 ? v.y : j < 6 ? v.z : v.w);
        return (j & 1) ? p.y : p.x;
    }
};

// the maximum of a vector, of two values in a word where they are 16-bit; last(): of the word
template <typename T> __device__ __forceinline__ uint32_t lp_max(const uint4& v) {
    using L = LpVec<T>;
    return L::max2(L::max2(v.x, v.y), L::max2(v.z, v.w));
}

// A row in chunks of 32 vectors of 16 bytes, from the last 16-byte border at or before its start on; chunks that reach over an end are read value by value.
template <typename T> struct LpRow {
    static constexpr int N = LpVec<T>::N, kChunk = 32 * N;
    const T* x;
    int vocab, skip, chunks;                    // values between that border and the row; chunks of the row
    __device__ LpRow(const LogprobArgs& a, int row) : x(reinterpret_cast<const T*>(a.x) + (long long)row * a.ld), vocab(a.vocab) {
        skip = (int)(reinterpret_cast<uintptr_t>(x) & 15) / (int)sizeof(T);
        chunks = (skip + vocab + kChunk - 1) / kChunk;
    }
    __device__ __forceinline__ int first(int chunk, int lane) const { return chunk * kChunk + lane * N - skip; }        // index of the lane's first value
    // chunks [whole(), whole_end()) lie inside the row
    __device__ __forceinline__ int whole() const { return skip > 0; }
    __device__ __forceinline__ int whole_end() const { return (skip + vocab) / kChunk; }
    __device__ __forceinline__ const uint4* at(int chunk, int lane) const { return reinterpret_cast<const uint4*>(x - skip) + ((long long)chunk * 32 + lane); }
    // -infinity outside the row
    __device__ __forceinline__ uint4 load(int chunk, int lane) const {
        const int i0 = first(chunk, lane);
        if (i0 >= 0 && i0 + N <= vocab) return ldg_stream(reinterpret_cast<const uint4*>(x + i0));
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = LpVec<T>::kNone;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (i0 + j < 0 || i0 + j >= vocab) continue;
            if constexpr (sizeof(T) == 4) {
                w[j] = __float_as_uint(x[i0 + j]);
            } else {
                const uint32_t h = reinterpret_cast<const uint16_t*>(x)[i0 + j];
                w[j / 2] = (j & 1) ? (w[j / 2] & 0xFFFFu) | h << 16 : (w[j / 2] & 0xFFFF0000u) | h;
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

struct __align__(16) LpPart { float m, r, s, t; };     // largest x; reference; sum of e; sum of e (c x - r)
// the warp's largest value; NaN is passed over
__device__ __forceinline__ float lp_warp_max(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xFFFFFFFF;" : "=f"(r) : "f"(v));
    return r;
}
// those of the lanes (of each 2 WIDTH of them) as one, about the largest reference
template <int WIDTH>
__device__ __forceinline__ LpPart lp_join_warp(LpPart p) {
    const float r = lp_warp_max(p.r), f = ex2(p.r - r);
    p.m = lp_warp_max(p.m);
    p.t = (p.t + p.s * (p.r - r)) * f;
    p.s *= f;
#pragma unroll
    for (int o = WIDTH; o > 0; o >>= 1) {
        p.s += __shfl_xor_sync(0xFFFFFFFFu, p.s, o);
        p.t += __shfl_xor_sync(0xFFFFFFFFu, p.t, o);
    }
    p.r = r;
    return p;
}
// n of them, 16 at most, in shared memory (whole warps)
__device__ __forceinline__ LpPart lp_join(const LpPart* part, int n, int lane) {
    LpPart p = part[min(lane & 15, n - 1)];
    if ((lane & 15) >= n) p.s = p.t = 0.f;
    return lp_join_warp<8>(p);
}
// how many of the keys lie before `key`; n a multiple of 8 (zeros fill it up)
__device__ __forceinline__ int lp_place(const unsigned long long* keys, int n, unsigned long long key) {
    int before = 0;
    for (int j = 0; j < n; j += 8) {
        ulonglong2 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const ulonglong2*>(keys + j + 2 * i);
#pragma unroll
        for (int i = 0; i < 4; ++i) before += (v[i].x > key) + (v[i].y > key);
    }
    return before;
}

__device__ __forceinline__ int cluster_id() {
    int r;
    asm("mov.u32 %0, %clusterid.x;" : "=r"(r));
    return r;
}

// TOP: with alternatives.  A cluster of C blocks per row, `per` chunks each.  A batch is on its way while the one before is added up (16-bit rows with alternatives
// of one batch at a time, whose registers let two more blocks onto an SM: 1000 x 32003 f16 18.2 -> 19.2 us, 2048 x 32000 bf16 32.4 -> 34.4, 1300 x 32000 24.5 -> 21.9).
// Four large blocks to an SM (64 registers a thread instead of 66: 500 x 128256 f32 with five alternatives 59 -> 44 us); for small ones the compiler keeps to 64
// by itself (asked for it: 1000 x 32003 f16 17.7 -> 18.0).
template <typename T, bool TOP, int kThreads>
__global__ void __launch_bounds__(kThreads, kThreads == 256 ? 4 : 0) logprobs_kernel(const LogprobArgs a, const int C, const int per) {
    constexpr int kWarps = kThreads / 32, U = 4;
    extern __shared__ float chunk_max[];                        // TOP: maxima of this block's chunks
    __shared__ LpPart part[kWarps], parts[kLpMaxCluster];
    __shared__ float sup[TOP ? kThreads : 1];
    __shared__ __align__(16) unsigned long long cand[TOP ? kLpCand : 1], best[TOP ? kLpMaxCluster * kLpMaxTop : 1];
    __shared__ unsigned long long round_best[TOP ? kWarps : 1];
    __shared__ int list[TOP ? kLpList : 1];
    __shared__ int n_list, n_cand;
    __shared__ float bound;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = C == 1 ? 0 : (int)cluster_rank(), row = C == 1 ? (int)blockIdx.x : cluster_id();
    const LpRow<T> x(a, row);
    const int ch0 = min(rank * per, x.chunks), ch1 = min(ch0 + per, x.chunks);
    const float c = a.c, nan = __uint_as_float(0x7FFFFFFFu);
    if (C > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");      // (that the first block has started, before anyone writes to it)
    if (tid == 0) { n_list = 0; n_cand = 0; }
    const int K = a.top;
    unsigned long long* mine_best = best + rank * K;            // (in the first block's table, this block's place)
    if (TOP) {
        for (int i = tid; i < kLpCand; i += kThreads) cand[i] = 0;
        if (tid < K) mine_best[tid] = 0;
    }

    // the given tokens, on their way while the row is read (as they lie: a conversion here would wait for them)
    const int turn = kThreads - 1 - tid;                        // (the last warp's, so that they do not wait for the alternatives, nor these for them)
    const bool mine = rank == 0 && turn < a.given;
    int2 token_bits{-1, -1};
    if (mine) {
        const long long at = (long long)row * a.given + turn;
        if (a.wide) token_bits = reinterpret_cast<const int2*>(a.tokens)[at];
        else token_bits.x = reinterpret_cast<const int*>(a.tokens)[at];
    }
    auto token_of = [&](int2 bits) { return a.wide ? (long long)bits.y << 32 | (uint32_t)bits.x : (long long)bits.x; };

    LpPart p{-INFINITY, fmaxf(-kLpFarAt, fmaf(LpVec<T>::kLow, c, kLpNothing)), 0.f, 0.f};
    uint64_t s2 = pack2(0.f, 0.f), t2 = s2;
    const uint64_t c2 = pack2(c, c);
    // U vectors of a lane, one of each of U chunks; at(u): the u-th chunk's place in chunk_max, or -1
    auto absorb = [&](const uint4 (&v)[U], auto&& at) {
        uint32_t w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = lp_max<T>(v[u]);
        if constexpr (TOP) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float m = lp_warp_max(LpVec<T>::last(w[u]));
                if (lane == 0 && at(u) >= 0) chunk_max[at(u)] = m;
            }
        }
#pragma unroll
        for (int u = 1; u < U; ++u) w[0] = LpVec<T>::max2(w[0], w[u]);
        const float m = LpVec<T>::last(w[0]);
        p.m = fmaxf(p.m, m);
        if (m * c > p.r + 16.f) {
            const float r = m * c, f = ex2(p.r - r);
            float sa, sb, ta, tb;
            unpack2(s2, sa, sb);
            unpack2(t2, ta, tb);
            s2 = pack2(sa * f, sb * f);
            t2 = pack2((ta + sa * (p.r - r)) * f, (tb + sb * (p.r - r)) * f);
            p.r = r;
        }
        const uint64_t r2 = pack2(-p.r, -p.r);
#pragma unroll
        for (int u = 0; u < U; ++u)
            LpVec<T>::pairs(v[u], [&](float va, float vb) {
                const uint64_t d = fma2(pack2(va, vb), c2, r2);
                float da, db;
                unpack2(d, da, db);
                const uint64_t e = pack2(ex2(da), ex2(db));
                s2 = add2(s2, e);
                t2 = fma2(e, d, t2);
            });
    };
    // batches of U chunks a warp that lie inside the row, without a look at its ends, and the chunks in front of them and behind
    const int first = max(ch0, x.whole()), batches = max(0, min(ch1, x.whole_end()) - first) / (kWarps * U);
    const int head = min(first, ch1) - ch0, rest = ch1 - ch0 - batches * kWarps * U;       // chunks in front of the batches; all that are in none
    auto rest_place = [&](int j, int u) {
        const int k = j + u * kWarps;
        return k >= rest ? -1 : k < head ? k : k + batches * kWarps * U;
    };
    auto fetch_rest = [&](uint4 (&v)[U], int j) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            v[u] = make_uint4(LpVec<T>::kNone, LpVec<T>::kNone, LpVec<T>::kNone, LpVec<T>::kNone);
            if (rest_place(j, u) >= 0) v[u] = x.load(ch0 + rest_place(j, u), lane);
        }
    };
    int j_rest = warp;
    {
        const uint4* q = x.at(first + warp, lane);
        auto fetch = [&](uint4 (&v)[U]) {
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = ldg_stream(q + u * kWarps * 32);
            q += U * kWarps * 32;
        };
        uint4 v[U], w[U];
        int ch = first + warp - ch0;
        auto place = [&](int u) { return ch + u * kWarps; };
        if (j_rest < rest) fetch_rest(w, j_rest);
        if (batches > 0) fetch(v);
        if (j_rest < rest) absorb(w, [&](int u) { return rest_place(warp, u); });
        for (int i = 0; i < batches; i += 2) {
            if (i + 1 < batches) fetch(w);
            absorb(v, place);
            ch += U * kWarps;
            if (i + 1 >= batches) break;
            if (i + 2 < batches) fetch(v);
            absorb(w, place);
            ch += U * kWarps;
        }
    }
    for (j_rest += U * kWarps; j_rest < rest; j_rest += U * kWarps) {
        uint4 v[U];
        fetch_rest(v, j_rest);
        absorb(v, [&](int u) { return rest_place(j_rest, u); });
    }
    // the given tokens' logits (again not converted yet)
    T token_x{};
    if (mine) {
        const long long t = token_of(token_bits);
        if (t >= 0 && t < a.vocab) token_x = x.x[t];
    }
    {
        float sa, sb, ta, tb;
        unpack2(s2, sa, sb);
        unpack2(t2, ta, tb);
        p.s = sa + sb;
        p.t = ta + tb;
    }
    if (TOP) sup[tid] = p.m;
    p = lp_join_warp<16>(p);
    if (lane == 0) part[warp] = p;
    __syncthreads();

    // ---- this block's K best logits, largest first ----
    if (TOP) {
        const int n = ch1 - ch0;
        if (warp == 0) {                                        // the K-th largest group maximum: K times the largest, which its lane drops; a lane's number in
            float f0 = -INFINITY, f1 = -INFINITY;               // the lowest bits keeps them apart
#pragma unroll
            for (int i = 0; i < kThreads; i += kLpGroups) {
                f0 = fmaxf(f0, sup[i + lane]);
                f1 = fmaxf(f1, sup[i + 32 + lane]);
            }
            uint32_t v = ordered_bits(fmaxf(f0, f1)) & ~31u | lane, next = ordered_bits(fminf(f0, f1)) & ~31u | lane, least = 0;
            for (int k = 0; k < K; ++k) {
                least = __reduce_max_sync(0xFFFFFFFFu, v);
                if (v == least) { v = next; next = 0; }
            }
            if (lane == 0) bound = from_ordered(max(least & ~31u, kLpFinite));
        }
        __syncthreads();
        const float least = bound;
        for (int i = tid; i < n; i += kThreads)
            if (chunk_max[i] >= least) {
                const int at = atomicAdd(&n_list, 1);
                if (at < kLpList) list[at] = ch0 + i;
            }
        __syncthreads();
        bool fits = n_list <= kLpList;
        if (fits) {
            for (int i = warp; i < n_list; i += 4 * kWarps) {
                uint4 v[4];
                uint32_t hits = 0;                              // (N values of a vector, 4 vectors: 32 bits at most; -infinity, outside the row too, is none)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    v[u] = make_uint4(LpVec<T>::kNone, LpVec<T>::kNone, LpVec<T>::kNone, LpVec<T>::kNone);
                    if (i + u * kWarps < n_list) v[u] = x.load(list[i + u * kWarps], lane);
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int j = 0; j < LpVec<T>::N; ++j) hits |= (uint32_t)(LpVec<T>::at(v[u], j) >= least) << (u * LpVec<T>::N + j);
                int at = hits != 0 ? atomicAdd(&n_cand, __popc(hits)) : 0;
                for (; hits != 0; hits &= hits - 1, ++at) {
                    const int b = __ffs(hits) - 1, u = b / LpVec<T>::N, j = b % LpVec<T>::N;
                    const uint4 low = (u & 1) ? v[1] : v[0], high = (u & 1) ? v[3] : v[2];
                    if (at < kLpCand) cand[at] = order_key(ordered_bits(LpVec<T>::at((u & 2) ? high : low, j)), x.first(list[i + u * kWarps], lane) + j);
                }
            }
            __syncthreads();
            fits = n_cand <= kLpCand;
        }
        if (fits) {
            const int held = n_cand, even = (held + 7) / 8 * 8;         // (zeros behind them)
            for (int i = tid; i < held; i += kThreads) {
                const int at = lp_place(cand, even, cand[i]);
                if (at < K) mine_best[at] = cand[i];
            }
            // fewer than K logits above -infinity: its lowest indices, all of which lie in the block's first K values
            if (held < K && warp == 0) {
                const int i = max(x.first(ch0, 0), 0) + lane;
                const bool out = lane < K && i < min(x.first(ch1, 0), a.vocab) && to_f32(x.x[i]) == -INFINITY;
                const int at = held + __popc(__ballot_sync(0xFFFFFFFFu, out) & ((1u << lane) - 1));
                if (out && at < K) mine_best[at] = order_key(kLpFinite - 1, i);
            }
        } else {
            // the K-th best chunk by (maximum, lower index), then K rounds over the chunks up to it
            __shared__ unsigned long long chunk_bound;
            __syncthreads();                                    // (everyone has seen that the tables did not do)
            if (warp == 0) {
                unsigned long long lo = 0, hi = ~0ull;          // K chunks reach lo (or all do), fewer reach hi
                while (hi - lo > 1) {
                    const unsigned long long mid = lo + (hi - lo) / 2;
                    int k = 0;
                    for (int i = lane; i < n; i += 32) k += order_key(ordered_bits(chunk_max[i]), i) >= mid;
                    k = __reduce_add_sync(0xFFFFFFFFu, k);
                    if (k >= K) lo = mid; else hi = mid;
                    if (k == K) break;
                }
                if (lane == 0) { chunk_bound = lo; n_list = 0; }
            }
            __syncthreads();
            for (int i = tid; i < n; i += kThreads)
                if (order_key(ordered_bits(chunk_max[i]), i) >= chunk_bound) list[atomicAdd(&n_list, 1)] = ch0 + i;       // (K of them at most: keys are distinct)
            __syncthreads();
            const int chunks = n_list;
            unsigned long long last = ~0ull;
            for (int k = 0; k < K; ++k) {
                unsigned long long b = 0;
                for (int i = warp; i < chunks; i += kWarps) {
                    const uint4 v = x.load(list[i], lane);
                    const int i0 = x.first(list[i], lane);
#pragma unroll
                    for (int j = 0; j < LpVec<T>::N; ++j) {
                        const unsigned long long key = order_key(ordered_bits(LpVec<T>::at(v, j)), i0 + j);
                        if (i0 + j >= 0 && i0 + j < a.vocab && key < last && key > b) b = key;
                    }
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const unsigned long long q = __shfl_xor_sync(0xFFFFFFFFu, b, o);
                    b = q > b ? q : b;
                }
                if (lane == 0) round_best[warp] = b;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < kWarps; ++i) b = round_best[i] > b ? round_best[i] : b;
                __syncthreads();
                if (tid == 0) mine_best[k] = b;
                last = b;
                if (b == 0) break;
            }
        }
        __syncthreads();
    }

    // ---- the cluster's results meet in its first block ----
    if (C > 1) {
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (rank != 0) {
            p = lp_join(part, kWarps, lane);
            if (TOP && tid < K)
                asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(mapa_u32(smem_u32(mine_best + tid), 0)), "l"(mine_best[tid]) : "memory");
            if (tid == 0) {
                const uint32_t to = mapa_u32(smem_u32(&parts[rank]), 0);
                asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(p.m), "f"(p.r), "f"(p.s), "f"(p.t) : "memory");
            }
            __syncwarp();
            asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
            return;
        }
        if (warp == 0) {
            p = lp_join(part, kWarps, lane);
            if (lane == 0) parts[0] = p;
        }
        __syncwarp();
        cluster_sync_all();
        p = lp_join(parts, C, lane);
    } else {
        p = lp_join(part, kWarps, lane);
    }

    // ---- the row's numbers, the same in all threads ----
    // a row that the loop's references do not hold for (see kLpFarAt): summed once more, about the maximum itself
    const bool far = p.m > -INFINITY && p.m < INFINITY && (fabsf(p.m) * c > kLpFarAt || (p.m - LpVec<T>::kLow) * c < kLpNothing || LpVec<T>::kLow * c < -1e38f);
    const bool none = p.m == -INFINITY && p.s == p.s;
    // (v - m) / T - s; a finite logit can lie further from a large maximum than f32 reaches: half of both then (at T <= 1 the quotient is past it anyway)
    const float part_of = p.m > 1e30f && a.inv_t < 1.f ? 0.5f : 1.f, inv = part_of < 1.f ? 2.f * a.inv_t : a.inv_t;
    auto from_max = [&](float v, float s) { return fmaf(fmaf(v, part_of, -part_of * p.m), inv, -s); };
    float log_s, entropy;                                       // log of the sum about the maximum
    bool bad;
    if (far) {
        __syncthreads();                                        // (part is written again below: with one block per row a warp may still read it)
        float s = 0.f, t = 0.f;
        for (int i = tid; i < a.vocab; i += kThreads) {
            const float d = from_max(to_f32(x.x[i]), 0.f), e = expf(d);
            s += e;
            if (e > 0.f) t += e * d;
        }
        s = warp_sum(s);
        t = warp_sum(t);
        if (lane == 0) part[warp] = LpPart{0.f, 0.f, s, t};
        __syncthreads();
        s = t = 0.f;
        for (int i = 0; i < kWarps; ++i) { s += part[i].s; t += part[i].t; }
        bad = !(s <= 3.4e38f);
        log_s = logf(s);
        entropy = log_s - t / s;
    } else {
        constexpr float ln2 = 0.693147180559945309f;
        bad = !(p.s <= 3.4e38f);
        const float l = log2f(p.s);
        log_s = ln2 * (l + fmaf(-p.m, c, p.r));
        entropy = ln2 * (l - p.t / p.s);
    }
    const float log_z = fmaf(p.m, a.inv_t, log_s);
    auto lp = [&](float v) { return bad ? nan : (none || v == -INFINITY ? -INFINITY : from_max(v, log_s)); };
    if (tid == kThreads / 2) {
        if (a.logsumexp) a.logsumexp[row] = bad ? nan : (none ? -INFINITY : log_z);
        if (a.entropy) a.entropy[row] = bad ? nan : (none ? 0.f : entropy);
    }
    for (int j = turn; j < a.given; j += kThreads) {
        const long long at = (long long)row * a.given + j;
        if (j >= kThreads) {
            if (a.wide) token_bits = reinterpret_cast<const int2*>(a.tokens)[at];
            else token_bits.x = reinterpret_cast<const int*>(a.tokens)[at];
        }
        const long long t = token_of(token_bits);
        if (j >= kThreads && t >= 0 && t < a.vocab) token_x = x.x[t];
        a.logprob[at] = t < 0 ? 0.f : (t >= a.vocab ? nan : lp(to_f32(token_x)));
    }
    if (TOP) {
        const int all = C * K, even = (all + 7) / 8 * 8;
        if (C > 1) {
            if (tid < even - all) best[all + tid] = 0;
            __syncthreads();
        }
        for (int i = tid; i < all; i += kThreads) {
            const unsigned long long key = best[i];
            if (key == 0) continue;
            const int place = C == 1 ? i : lp_place(best, even, key);
            if (place < K) {
                const long long to = (long long)row * K + place;
                a.top_ids[to] = bad ? -1 : (int)~(uint32_t)key;
                a.top_logprobs[to] = lp(from_ordered((uint32_t)(key >> 32)));
            }
        }
        if (bad && tid < a.top) {                               // (keys of NaN are no order)
            a.top_ids[(long long)row * a.top + tid] = -1;
            a.top_logprobs[(long long)row * a.top + tid] = nan;
        }
    }
}

}  // namespace fl

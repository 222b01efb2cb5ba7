// Log probabilities over a vocabulary: z = x / T, logZ = log sum exp z, lp(t) = z_t - logZ, H = logZ - sum p z, and the largest logits with
// theirs, the lowest index first among equals.
#pragma once
#include "linear8.cuh"

namespace fl {

constexpr int kLpMaxTop = 32;
constexpr int kLpMaxVocab = 1 << 20;

struct LogprobArgs {
    const void* x; long long ld;                // [rows, vocab]
    int rows, vocab;
    float inv_t;
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
__device__ __forceinline__ unsigned long long order_key(float v, int i) { return (unsigned long long)ordered_bits(v) << 32 | (uint32_t)~i; }

// A block per row: one walk for the maximum, one for the sums, one per alternative.
template <typename T>
__global__ void __launch_bounds__(256) logprobs_kernel(const LogprobArgs a) {
    __shared__ float red[3][8];
    __shared__ unsigned long long best[8];
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T* x = reinterpret_cast<const T*>(a.x) + (long long)row * a.ld;
    auto z = [&](int i) { return to_f32(x[i]) * a.inv_t; };
    float m = -INFINITY;
    for (int i = tid; i < a.vocab; i += 256) m = fmaxf(m, z(i));
    m = warp_max(m);
    if (lane == 0) red[0][warp] = m;
    __syncthreads();
    for (int i = 0; i < 8; ++i) m = fmaxf(m, red[0][i]);
    const float ref = m == -INFINITY ? 0.f : m;
    float s = 0.f, t = 0.f;
    for (int i = tid; i < a.vocab; i += 256) {
        const float d = z(i) - ref, e = expf(d);
        s += e;
        if (e > 0.f) t += e * d;
    }
    s = warp_sum(s);
    t = warp_sum(t);
    if (lane == 0) { red[1][warp] = s; red[2][warp] = t; }
    __syncthreads();
    s = t = 0.f;
    for (int i = 0; i < 8; ++i) { s += red[1][i]; t += red[2][i]; }
    const bool none = m == -INFINITY && s == 0.f, bad = !(s == s) || m == INFINITY;
    const float nan = __uint_as_float(0x7FFFFFFFu);
    const float log_s = logf(s);
    const float log_z = bad ? nan : (none ? -INFINITY : ref + log_s);
    auto lp = [&](float zi) { return bad ? nan : (none || zi == -INFINITY ? -INFINITY : (zi - ref) - log_s); };
    if (tid == 0) {
        if (a.logsumexp) a.logsumexp[row] = log_z;
        if (a.entropy) a.entropy[row] = bad ? nan : (none ? 0.f : log_s - t / s);
    }
    if (a.logprob)
        for (int j = tid; j < a.given; j += 256) {
            const long long at = (long long)row * a.given + j;
            const long long k = a.wide ? reinterpret_cast<const long long*>(a.tokens)[at] : reinterpret_cast<const int*>(a.tokens)[at];
            a.logprob[at] = k < 0 ? 0.f : (k >= a.vocab ? nan : lp(z((int)k)));
        }
    unsigned long long last = ~0ull;
    for (int k = 0; k < a.top; ++k) {
        unsigned long long b = 0;
        for (int i = tid; i < a.vocab && !bad; i += 256) {
            const unsigned long long key = order_key(to_f32(x[i]), i);
            if (key < last && key > b) b = key;
        }
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long other = __shfl_xor_sync(0xFFFFFFFFu, b, o);
            b = other > b ? other : b;
        }
        if (lane == 0) best[warp] = b;
        __syncthreads();
        for (int i = 0; i < 8; ++i) b = best[i] > b ? best[i] : b;
        __syncthreads();
        last = b;
        if (tid == 0) {
            const int id = bad ? -1 : (int)~(uint32_t)b;
            a.top_ids[(long long)row * a.top + k] = id;
            a.top_logprobs[(long long)row * a.top + k] = bad ? nan : lp(z(id));
        }
    }
}

}  // namespace fl

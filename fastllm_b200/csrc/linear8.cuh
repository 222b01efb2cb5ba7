// Matrix product in 8-bit integers with a scale per token and per channel:
//   y[r, n] = (sum_k q[r, k] w[n, k]) s[r] t[n] + b[n],   q, w whole numbers of 8 bits, the sum exact in 32-bit integers,
// and the rounding of activations to such rows.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace fl {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// One row's rounding rule: q = 127 x / a to the nearest whole number, halves to the even one, of the exact quotient (a = max |x|).
// x * (127 / a) in f32 is off by at most 127 * 2^-23 = 1.5e-5, so only quotients that lie within 1e-4 of a half need the exact sign of
// 254 x - (2 low + 1) a, which 64 bits hold without rounding.
struct RowScale {
    float a, mul, up;       // max |x| times `up`; 127 / a; a power of two that keeps 127 / a finite for the smallest rows
    float scale;            // a / 127; NaN for a row with a NaN or an infinity
    __device__ explicit RowScale(uint32_t max_bits) {
        const float most = __uint_as_float(max_bits);
        const bool bad = max_bits >= 0x7F800000u;
        up = most < 1e-30f ? 0x1p96f : 1.f;
        a = most * up;
        mul = bad || most == 0.f ? 0.f : 127.f / a;
        scale = bad ? __uint_as_float(0x7FFFFFFFu) : most / 127.f;
    }
    __device__ int operator()(float x) const {
        if (mul == 0.f) return 0;
        x *= up;
        const float v = x * mul, n = rintf(v);
        if (fabsf(v - n) < 0.4999f) return (int)n;
        const float low = floorf(v);
        const double over = fma(254.0, (double)x, -(2.0 * (double)low + 1.0) * (double)a);
        const int l = (int)low;
        return over > 0.0 ? l + 1 : (over < 0.0 ? l : l + (l & 1));
    }
};
// larger for every NaN than for an infinity, and for that than for any number
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// A block per row; columns [cols, cols_q) of q are filled with zeros.
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* __restrict__ x, long long ldx, int cols, int8_t* __restrict__ q, long long ldq, int cols_q,
                                                            float* __restrict__ scale) {
    __shared__ uint32_t part[8];
    const T* xr = x + (long long)blockIdx.x * ldx;
    int8_t* qr = q + (long long)blockIdx.x * ldq;
    uint32_t m = 0;
    for (int i = threadIdx.x; i < cols; i += 256) m = max(m, abs_bits(to_f32(xr[i])));
    m = __reduce_max_sync(0xFFFFFFFFu, m);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
    for (int i = 0; i < 8; ++i) m = max(m, part[i]);
    const RowScale rs(m);
    for (int i = threadIdx.x; i < cols_q; i += 256) qr[i] = i < cols ? (int8_t)rs(to_f32(xr[i])) : (int8_t)0;
    if (threadIdx.x == 0) scale[blockIdx.x] = rs.scale;
}

struct Linear8Args {
    const int8_t* xq; long long ldq; const float* xs;       // [rows, k], [rows]
    const int8_t* w; long long ldw; const float* ws;        // [n, k], [n]
    const float* bias;                                      // [n] or null
    void* y; long long ldy;
    int rows, n, k;
};

// 64 x 64 outputs per block, four products of 8 bits per instruction
template <typename T>
__global__ void __launch_bounds__(256) linear8_kernel(const Linear8Args g) {
    __shared__ int sx[64][17], sw[64][17];
    const int n0 = blockIdx.x * 64, r0 = blockIdx.y * 64;
    const int tn = threadIdx.x & 15, tr = threadIdx.x >> 4;
    int acc[4][4] = {};
    auto word = [&](const int8_t* row, int k) {             // four values from column k on, zeros past the end
        uint32_t v = 0;
        for (int j = 0; j < 4; ++j)
            if (k + j < g.k) v |= (uint32_t)(uint8_t)row[k + j] << (8 * j);
        return (int)v;
    };
    for (int k0 = 0; k0 < g.k; k0 += 64) {
        for (int i = threadIdx.x; i < 64 * 16; i += 256) {
            const int row = i >> 4, c = i & 15;
            sx[row][c] = r0 + row < g.rows ? word(g.xq + (long long)(r0 + row) * g.ldq, k0 + 4 * c) : 0;
            sw[row][c] = n0 + row < g.n ? word(g.w + (long long)(n0 + row) * g.ldw, k0 + 4 * c) : 0;
        }
        __syncthreads();
        for (int c = 0; c < 16; ++c)
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(sx[tr + 16 * i][c], sw[tn + 16 * j][c], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int r = r0 + tr + 16 * i, n = n0 + tn + 16 * j;
            if (r >= g.rows || n >= g.n) continue;
            float v = (float)acc[i][j] * g.xs[r] * g.ws[n];
            if (g.bias) v += g.bias[n];
            reinterpret_cast<T*>(g.y)[(long long)r * g.ldy + n] = from_f32<T>(v);
        }
}

}  // namespace fl

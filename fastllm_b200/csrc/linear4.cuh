// Matrix product of 4-bit rows with a scale per 32 values (rows4.cuh):
//   y[r, n] = sum_k x[r, k] w[n, k] (+ b[n]),   x, w the values that the rows stand for, sums in f32, one rounding to the result's type.
#pragma once
#include "rows4.cuh"

namespace fl {

struct Linear4Args {
    int rows, n, blocks;                                        // blocks of 32 values of a row
    const uint8_t* x; long long ldx;                            // bytes
    const uint8_t* xs; int x_tile;                              // scales as the tensor cores take them, in tiles of so many rows
    const uint8_t* w; long long ldw;
    const uint8_t* ws;                                          // in tiles of 128 rows
    int groups;                                                 // of four blocks, as the scales' layout counts them
    const float* bias;                                          // [n] or null
    void* y; long long ldy; int y_dtype;                        // fl_dtype
};

// 32 x 32 results of a block, a block of 32 values at a time through shared memory
__global__ void __launch_bounds__(256) linear4_plain_kernel(const Linear4Args a) {
    __shared__ float xv[32][33], wv[32][33];
    const int r0 = blockIdx.y * 32, n0 = blockIdx.x * 32, col = threadIdx.x & 31, row = threadIdx.x >> 5;
    float sum[4] = {};
    for (int b = 0; b < a.blocks; ++b) {
        const int i = threadIdx.x / 8, part = threadIdx.x & 7;         // a row's four columns
        auto fill = [&](const uint8_t* q, long long ld, const uint8_t* scales, int tile, int at, int rows, float (&to)[32][33]) {
            float s = 0.f;
            uint32_t w = 0;
            if (at < rows) {
                s = down4(scales[scale4_at(at, b / 4, tile, a.groups) + b % 4]);
                w = reinterpret_cast<const uint16_t*>(q + at * ld + b * 16)[part];
            }
            float v[8];
            from_e2m1x8(w, v);
#pragma unroll
            for (int j = 0; j < 4; ++j) to[i][part * 4 + j] = v[j] * s;
        };
        fill(a.x, a.ldx, a.xs, a.x_tile, r0 + i, a.rows, xv);
        fill(a.w, a.ldw, a.ws, 128, n0 + i, a.n, wv);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            const float w = wv[col][j];
#pragma unroll
            for (int c = 0; c < 4; ++c) sum[c] = fmaf(xv[row + 8 * c][j], w, sum[c]);
        }
        __syncthreads();
    }
    const int n = n0 + col;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const int r = r0 + row + 8 * c;
        if (r >= a.rows || n >= a.n) continue;
        const float v = a.bias != nullptr ? sum[c] + a.bias[n] : sum[c];
        const long long at = (long long)r * a.ldy + n;
        if (a.y_dtype == 0) reinterpret_cast<float*>(a.y)[at] = v;
        else if (a.y_dtype == 1) reinterpret_cast<__nv_bfloat16*>(a.y)[at] = from_f32<__nv_bfloat16>(v);
        else reinterpret_cast<__half*>(a.y)[at] = from_f32<__half>(v);
    }
}

}  // namespace fl

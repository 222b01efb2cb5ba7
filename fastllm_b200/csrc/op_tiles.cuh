// What the products of the operators on device memory share: weights are the 128- or 256-row operand, a lane of the accumulators is a weight row.
#pragma once
#include "gemm_pair.cuh"
#include "op_values.cuh"

namespace fl {

// Results of one weight row n (a lane each) and 16 activation rows r, r + 1, ..: for a fixed row the 32
// lanes write 32 neighbours.  (16-bit results in twos, after an exchange between neighbouring lanes, took as long or longer: 64 x 152064 20 -> 26 us.)
__device__ __forceinline__ void write16(void* y, long long ldy, int y_dtype, int r, int n, int rows, const float (&v)[16]) {
    if (y_dtype == 0) {
        float* o = reinterpret_cast<float*>(y) + (long long)r * ldy + n;
        if (rows == 16) {
#pragma unroll
            for (int j = 0; j < 16; ++j) { *o = v[j]; o += ldy; }
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                if (j < rows) *o = v[j];
                o += ldy;
            }
        }
        return;
    }
    uint16_t* o = reinterpret_cast<uint16_t*>(y) + (long long)r * ldy + n;
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
        uint32_t w;
        if (y_dtype == 1) {
            w = pack_bf16x2(v[j], v[j + 1]);
        } else {
            const __half2 h = __floats2half2_rn(v[j], v[j + 1]);
            w = *reinterpret_cast<const uint32_t*>(&h);
        }
        if (j < rows) o[0] = (uint16_t)w;
        if (j + 1 < rows) o[ldy] = (uint16_t)(w >> 16);
        o += 2 * ldy;
    }
}
// A wait ran out: report it and leave the copies in flight time to land; the block goes on to its end.
__device__ __forceinline__ void op_give_up(int* failed) {
    if ((threadIdx.x & 31) == 0) *failed = 1;
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
}

}  // namespace fl

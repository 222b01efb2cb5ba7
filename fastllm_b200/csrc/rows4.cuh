// Rows of 4-bit numbers with a scale per 32 neighbours (OCP Microscaling, MXFP4): value = e2m1 * 2^(s - 127), e2m1 one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 and
// their negatives, s a byte (255: NaN); the even column lies in the low half of a byte.  Rounding to such rows, the way back, and gated activations that end in them.
#pragma once
#include <type_traits>

#include "op_values.cuh"

namespace fl {

constexpr int kR4Block = 32;                                    // values that share a scale
constexpr int kR4Threads = 128;

// Where rounded rows go.  tile = 0: scales [rows][lds].  tile > 0: as the tensor cores take them (linear4.cuh), in tiles of that many rows.
struct Rows4Out {
    uint8_t* q; long long ldq;                                  // on 16-byte borders
    uint8_t* scale; long long lds;
    int blocks;                                                 // of a row
    int tile, groups;                                           // groups of four blocks that a row has in a tile (even)
};

// Byte offset of the four scales of row r's blocks 4 g .. 4 g + 3 in the layout of the tensor cores: [tile][group][128 rows][32 lanes][4][4 blocks], the rows
// 32 i + lane of 128 at [lane][i].
__host__ __device__ inline long long scale4_at(long long r, int g, int tile, int groups) {
    const int atoms = (tile + 127) / 128, in = (int)(r % tile);
    return ((r / tile * groups + g) * atoms + in / 128) * 512 + in % 32 * 16 + in % 128 / 32 * 4;
}

// byte of a block whose largest magnitude has these bits, and 2^-(s - 127) to bring its values to e2m1's range
__device__ __forceinline__ uint32_t scale4(uint32_t max_bits) { return max_bits >= 0x7F800000u ? 255u : (uint32_t)max((int)(max_bits >> 23) - 2, 0); }
__device__ __forceinline__ float up4(uint32_t s) { return s == 255u ? 0.f : __uint_as_float((254u - s) << 23); }
__device__ __forceinline__ float down4(uint32_t s) { return __uint_as_float(s == 0u ? 0x00400000u : (s == 255u ? 0x7FFFFFFFu : s << 23)); }

// number j of words of T, the bits of one, and words of V numbers
template <typename T> __device__ __forceinline__ float number_of(const uint32_t* w, int j);
template <> __device__ __forceinline__ float number_of<float>(const uint32_t* w, int j) { return __uint_as_float(w[j]); }
template <> __device__ __forceinline__ float number_of<__nv_bfloat16>(const uint32_t* w, int j) { return j & 1 ? bf16hi(w[j / 2]) : bf16lo(w[j / 2]); }
template <> __device__ __forceinline__ float number_of<__half>(const uint32_t* w, int j) { return __half2float(__ushort_as_half((unsigned short)(w[j / 2] >> (16 * (j & 1))))); }
__device__ __forceinline__ uint32_t bits_of(float v) { return __float_as_uint(v); }
__device__ __forceinline__ uint32_t bits_of(__nv_bfloat16 v) { return __bfloat16_as_ushort(v); }
__device__ __forceinline__ uint32_t bits_of(__half v) { return __half_as_ushort(v); }

// To the nearest e2m1, halves to the even mantissa, beyond 6 to 6, of a c >= 0 (c = 1 or folded into the sums): numbers up to 2 lie half a step apart, up to 4 a whole, then two, so the
// code is the least of 2 a, a + 2 and a / 2 + 4, each rounded to a whole number, and 7; 2^23 leaves a whole number in a sum's low bits.  (cvt.e2m1x2 did 5 numbers a
// clock and SM: 28672 x 4096 bf16 took 75 us.)
constexpr float kE2m1Big = 8388608.f;
__device__ __forceinline__ float e2m1_sum(float a, float c) {
    return fminf(fminf(fmaf(a, 2.f * c, kE2m1Big), fmaf(a, c, kE2m1Big + 2.f)), fminf(fmaf(a, 0.5f * c, kE2m1Big + 4.f), kE2m1Big + 7.f));
}
// Codes of eight columns, the first in the low bits, from such sums and what has the numbers' signs in its top bits
__device__ __forceinline__ uint32_t e2m1x8(const float (&sum)[8], const uint32_t (&sign)[8]) {
    uint32_t w = 0;
#pragma unroll
    for (int j = 7; j >= 0; --j) w = __funnelshift_l(sign[j], w, 1) * 8u + __float_as_uint(sum[j]);
    constexpr uint32_t kBits = 0x4B000000u;                     // of 2^23
    return w - kBits * 0x11111111u;
}
// the same of eight bf16 numbers times a power of two, two at a time: bf16's sums with 128 round to whole numbers
__device__ __forceinline__ uint32_t e2m1x8_bf16(const uint32_t* in, uint32_t up2) {
    auto bf = [](uint32_t v) { return __halves2bfloat162(__ushort_as_bfloat16((unsigned short)v), __ushort_as_bfloat16((unsigned short)(v >> 16))); };
    auto sum = [&](uint32_t v) {                                // 128 + code in both halves
        const __nv_bfloat162 a = __hmul2(bf(v & 0x7FFF7FFFu), bf(up2));
        const __nv_bfloat162 t = __hmin2(__hmin2(__hfma2(a, bf(0x40004000u), bf(0x43004300u)), __hadd2(a, bf(0x43024302u))),
                                         __hmin2(__hfma2(a, bf(0x3F003F00u), bf(0x43044304u)), bf(0x43074307u)));
        return (uint32_t)__bfloat16_as_ushort(__low2bfloat16(t)) | (uint32_t)__bfloat16_as_ushort(__high2bfloat16(t)) << 16;
    };
    auto four = [&](uint32_t v0, uint32_t v1) {                 // four codes in the low half
        const uint32_t sign = ((v0 >> 12) & 0x00080008u) | ((v1 >> 4) & 0x08000800u);
        const uint32_t c = sum(v1) * 256u + (sum(v0) + sign - 0x43004300u * 257u);     // codes of columns 0, 2, 1, 3 in the low halves of the bytes
        return c | (c >> 12);
    };
    return __byte_perm(four(in[0], in[1]), four(in[2], in[3]), 0x5410);
}
__device__ __forceinline__ void from_e2m1x8(uint32_t w, float (&v)[8]) {
    uint32_t h[4];
    asm("{\n"
        ".reg .b8 a, b, c, d;\n"
        "mov.b32 {a, b, c, d}, %4;\n"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n"
        "}\n"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = number_of<__half>(h, 2 * i);
        v[2 * i + 1] = number_of<__half>(h, 2 * i + 1);
    }
}

// 16 kWords / 4 bytes from column `at` on, zeros past the row's end.  Rows may start anywhere: `off` bytes behind a 16-byte border, the same for the whole row; vectors
// that hold a part of the row are then shifted together.
template <typename T, int kWords>
__device__ __forceinline__ void load_row(const T* row, int at, int cols, uint32_t (&w)[kWords]) {
    constexpr int V = kWords * 4 / sizeof(T);
    const T* p = row + at;
    const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(p) & 15u;
    if (at + V <= cols) {
        if (off == 0) {
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i) {
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i);
                w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
            }
        } else {
            uint32_t h[kWords + 4];
            const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) - off);
#pragma unroll
            for (int i = 0; i <= kWords / 4; ++i) {
                const uint4 v = __ldg(q + i);
                h[4 * i] = v.x; h[4 * i + 1] = v.y; h[4 * i + 2] = v.z; h[4 * i + 3] = v.w;
            }
            if (off & 8) {
#pragma unroll
                for (int i = 0; i < kWords + 2; ++i) h[i] = h[i + 2];
            }
            if (off & 4) {
#pragma unroll
                for (int i = 0; i < kWords + 1; ++i) h[i] = h[i + 1];
            }
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = (off & 2) ? __funnelshift_r(h[i], h[i + 1], 16) : h[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0u;
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (at + j < cols) w[j * kWords / V] |= bits_of(p[j]) << (32 / (V / kWords) * (j % (V / kWords)));
    }
}
// A thread takes a block: which one, of all rows' blocks (`per` a row) in order
struct At4 {
    long long r;
    int block;
    bool here;
    __device__ At4(long long rows, int per) {
        const unsigned long long id = (unsigned long long)blockIdx.x * kR4Threads + threadIdx.x, all = (unsigned long long)rows * per;
        here = id < all;
        if (all <= 0xFFFFFFFFull) {
            const uint32_t q = (uint32_t)id / (uint32_t)per;
            r = q;
            block = (int)((uint32_t)id - q * (uint32_t)per);
        } else {
            r = (long long)(id / per);
            block = (int)(id - (unsigned long long)r * per);
        }
    }
};
__device__ __forceinline__ void put4(const Rows4Out& o, long long r, int block, const uint32_t (&codes)[4], uint32_t s) {
    if (block < o.blocks) *reinterpret_cast<uint4*>(o.q + r * o.ldq + block * 16) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
    uint8_t* to = o.tile == 0 ? o.scale + r * o.lds + block : o.scale + scale4_at(r, block / 4, o.tile, o.groups) + block % 4;
    *to = (uint8_t)s;
}
// 32 values from column `at` on, zeros past the row's end.  kVec: rows start on 16-byte borders.
template <typename T, bool kVec>
__device__ __forceinline__ void load32(const T* row, int at, int cols, uint32_t (&w)[8 * sizeof(T)]) {
    if (kVec && at + kR4Block <= cols) {
#pragma unroll
        for (int i = 0; i < (int)(2 * sizeof(T)); ++i) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + at) + i);
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t part[2 * sizeof(T)];
            load_row(row, at + 8 * i, cols, part);
#pragma unroll
            for (int j = 0; j < (int)(2 * sizeof(T)); ++j) w[2 * sizeof(T) * i + j] = part[j];
        }
    }
}
// bits, as of f32, of the largest magnitude among the words' numbers; those of 16 bits are in the order of their bits too
template <typename T, int kWords>
__device__ __forceinline__ uint32_t most_of(const uint32_t (&w)[kWords]) {
    uint32_t m = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < kWords; ++j) m = max(m, w[j] & 0x7FFFFFFFu);
        return m;
    } else {
#pragma unroll
        for (int j = 0; j < kWords; ++j) m = __vmaxu2(m, w[j] & 0x7FFF7FFFu);
        m = max(m & 0xFFFFu, m >> 16);
        return abs_bits(number_of<T>(&m, 0));
    }
}

// A thread per block: nothing passes between threads, and what a block costs once (its place, its scale) counts little beside its 32 numbers: with eight numbers a
// thread the instructions were the bound, 19 a number.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kR4Threads) quantize4_kernel(const T* __restrict__ x, long long ldx, long long rows, int cols, int per, const Rows4Out o) {
    pdl_launch_dependents();
    const At4 at(rows, per);
    if (!at.here) return;
    uint32_t w[8 * sizeof(T)], codes[4] = {};
    load32<T, kVec>(x + at.r * ldx, at.block * kR4Block, cols, w);
    const uint32_t s = scale4(most_of<T>(w));
    if (s != 255u) {
        if constexpr (std::is_same_v<T, __nv_bfloat16>) {
#pragma unroll
            for (int i = 0; i < 4; ++i) codes[i] = e2m1x8_bf16(w + 4 * i, (254u - s) * 0x00800080u);
        } else {
            const float up = up4(s);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float sum[8];
                uint32_t sign[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float v = number_of<T>(w, 8 * i + j);
                    sign[j] = __float_as_uint(v);
                    sum[j] = e2m1_sum(fabsf(v) * up, 1.f);      // (the product is exact, or far below the smallest border)
                }
                codes[i] = e2m1x8(sum, sign);
            }
        }
    }
    put4(o, at.r, at.block, codes, s);
}

// Eight numbers a thread (of 32 bits: four), which it writes at once.  kShift: rows of results may start anywhere, some numbers behind a 16-byte border; a thread then takes the
// columns between two borders, and its codes out of two words.
template <typename T, bool kShift>
__global__ void __launch_bounds__(kR4Threads) dequantize4_kernel(const uint8_t* __restrict__ q, long long ldq, const uint8_t* __restrict__ scale, long long lds, long long rows, int cols, int words,
                                                                 int per, T* __restrict__ y, long long ldy) {
    constexpr int V = 16 / sizeof(T);
    const At4 place(rows, per);
    if (!place.here) return;
    const uint32_t* qr = reinterpret_cast<const uint32_t*>(q + place.r * ldq);         // `words` of eight codes
    const uint8_t* sr = scale + place.r * lds;
    T* yr = y + place.r * ldy;
    int at = place.block * V;
    uint32_t w, s0, s1;
    if constexpr (kShift) {
        at -= (int)((reinterpret_cast<uintptr_t>(yr) & 15u) / sizeof(T));
        if (at >= cols) return;
        const int lo = at >> 3, hi = (at + V - 1) >> 3;
        const uint32_t w0 = lo >= 0 ? __ldg(qr + lo) : 0u, w1 = hi != lo && hi < words ? __ldg(qr + hi) : 0u;
        s0 = lo >= 0 ? __ldg(sr + (lo >> 2)) : 0u;
        s1 = hi >> 2 != lo >> 2 && hi < words ? __ldg(sr + (hi >> 2)) : s0;
        w = __funnelshift_r(w0, w1, 4 * (at & 7));
    } else {
        w = __ldg(qr + (at >> 3)) >> (4 * (at & 7));
        s0 = s1 = __ldg(sr + (at >> 5));
    }
    float v[8];
    from_e2m1x8(w, v);
    const float d0 = down4(s0), d1 = kShift ? down4(s1) : d0;
    const int own = 32 - (at & 31);                             // columns left in the first word's block
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] *= kShift && j >= own ? d1 : d0;
    if ((!kShift || at >= 0) && at + V <= cols) {
        uint32_t t[4] = {};
#pragma unroll
        for (int j = 0; j < V; ++j) t[j * 4 / V] |= bits_of(from_f32<T>(v[j])) << (V == 8 ? 16 * (j & 1) : 0);
        *reinterpret_cast<uint4*>(yr + at) = make_uint4(t[0], t[1], t[2], t[3]);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (at + j >= 0 && at + j < cols) yr[at + j] = from_f32<T>(v[j]);
    }
}

// Gated activations h = act(g) u
enum { kGlu4SwishClamp = 0, kGlu4GeluTanh = 1, kGlu4Relu = 3, kGlu4Silu = 4 };          // fl_ffn_act
template <int kAct>
__device__ __forceinline__ double glu4_exact(float limit, float gf, float uf) {
    const double g = gf, u = uf;
    if constexpr (kAct == kGlu4Silu) return g / (1.0 + exp(-g)) * u;
    if constexpr (kAct == kGlu4GeluTanh) return g / (1.0 + exp(-1.5957691216057308 * (g + 0.044715 * g * g * g))) * u;
    if constexpr (kAct == kGlu4Relu) return fmax(g, 0.0) * u;
    const double c = fmin(g, (double)limit);
    return c / (1.0 + exp(-1.702 * c)) * (fmin(fmax(u, -(double)limit), (double)limit) + 1.0);
}
// |h| in f32, with e = 2^t = e^-z, t held to 100.  t is off by |t| 2^-22 at most (a cubic's sum: four roundings), which moves h as far as e counts beside 1; ex2 and the
// reciprocal are off by 2^-22 and 2^-23, the sum and the products by 2^-24 each: h (2^-20 + max(t, 0) 2^-21) is more than all of it.  Where t is held h is too large.
template <int kAct>
__device__ __forceinline__ float glu4_near(float limit, float g, float u) {
    constexpr float kLog2e = 1.4426950408889634f;
    if constexpr (kAct == kGlu4Relu) return fabsf(fmaxf(g, 0.f)) * fabsf(u);
    float t, gate = g, up = u;
    if constexpr (kAct == kGlu4Silu) {
        t = -kLog2e * g;
    } else if constexpr (kAct == kGlu4GeluTanh) {
        constexpr float kC = -1.5957691216057308f * kLog2e;
        t = g * fmaf(kC * 0.044715f, g * g, kC);
    } else {
        gate = fminf(g, limit);
        up = fminf(fmaxf(u, -limit), limit) + 1.f;
        t = -1.702f * kLog2e * gate;
    }
    float e, r;
    asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(fminf(t, 100.f)));
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    return fabsf(gate * r) * fabsf(up);
}
// no less than max(t, 0) of gates up to `in`
template <int kAct>
__device__ __forceinline__ float glu4_far(float in) {
    if constexpr (kAct == kGlu4Relu) return 0.f;
    return fminf(100.f, kAct == kGlu4Silu ? 1.5f * in : kAct == kGlu4GeluTanh ? in * fmaf(0.11f * in, in, 2.4f) : 2.5f * in);
}
// A block in 64 bits, a number a lane, all of the warp: its scale's byte and its codes.
template <int kAct>
__device__ __forceinline__ uint32_t glu4_block_exact(float limit, float g, float u, bool here, uint32_t (&codes)[4]) {
    const int lane = threadIdx.x & 31;
    const double h = here ? glu4_exact<kAct>(limit, g, u) : 0.0, a = fabs(h);
    // truncated, so that the exponent is h's own; beyond f32: an infinity
    const uint32_t s = scale4(__reduce_max_sync(0xFFFFFFFFu, a >= 0x1p128 ? 0x7F800000u : __float_as_uint(__double2float_rz(a))));
    const double t = s == 255u ? 0.0 : a * __hiloint2double((int)(1023u + 127u - s) << 20, 0);
    const uint32_t c = t > 5.0 ? 7u : t >= 3.5 ? 6u : t > 2.5 ? 5u : t >= 1.75 ? 4u : t > 1.25 ? 3u : t >= 0.75 ? 2u : t > 0.25 ? 1u : 0u;
    const uint32_t w = (c | (h < 0.0 ? 8u : 0u)) << (4 * (lane & 7));
#pragma unroll
    for (int i = 0; i < 4; ++i) codes[i] = __reduce_or_sync(0xFFFFFFFFu, lane / 8 == i && s != 255u ? w : 0u);
    return s;
}

// Rounded once, of the exact h: computed in f32, and where numbers that far above and below do not round alike (one next to a border, a maximum next to a power of two) the
// block is taken in 64 bits by its warp.  All in 64 bits took 287 us at 4096 x 14336.
template <typename T, int kAct, bool kVec>
__global__ void __launch_bounds__(kR4Threads) glu4_kernel(const T* __restrict__ x, long long ldx, long long rows, int cols, int per, float limit, const Rows4Out o) {
    __shared__ float2 unsure[kR4Threads / 32][kR4Block];
    pdl_launch_dependents();
    const At4 at(rows, per);
    uint32_t gw[8 * sizeof(T)] = {}, uw[8 * sizeof(T)] = {}, codes[4] = {};
    if (at.here) {
        load32<T, kVec>(x + at.r * ldx, at.block * kR4Block, cols, gw);
        load32<T, kVec>(x + at.r * ldx + cols, at.block * kR4Block, cols, uw);
    }
    const uint32_t in_bits = max(most_of<T>(gw), most_of<T>(uw));
    uint32_t s = 255u;
    bool sure = true;
    if (in_bits < 0x7F800000u) {
        const float in = __uint_as_float(in_bits), off = kAct == kGlu4Relu ? 0x1p-22f : fmaf(glu4_far<kAct>(in), 0x1p-21f, 0x1p-20f);
        float h[kR4Block], most = 0.f;
#pragma unroll
        for (int j = 0; j < kR4Block; ++j) {
            h[j] = glu4_near<kAct>(limit, number_of<T>(gw, j), number_of<T>(uw, j));
            most = fmaxf(most, h[j]);
        }
        const float most_hi = most * (1.f + off), most_lo = most * (1.f - off);
        s = scale4(__float_as_uint(most_hi));
        // 64 bits too where f32 has fewer, and where a number whose exponent was held (below |g u| 2^-98) might count
        const float least = fmaxf(0x1p-100f, in * 0x1p-45f * (in * 0x1p-45f));
        sure = most == 0.f || (most_hi < INFINITY && most_hi >= least && s == scale4(__float_as_uint(most_lo)));
        if (sure && most != 0.f) {
            const float up = up4(s), hi = up * (1.f + off), lo = up * (1.f - off);
            uint32_t other = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float sum[8];
                uint32_t sign[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float v = number_of<T>(uw, 8 * i + j);
                    sign[j] = __float_as_uint(number_of<T>(gw, 8 * i + j)) ^ __float_as_uint(kAct == kGlu4SwishClamp ? fminf(fmaxf(v, -limit), limit) + 1.f : v);
                    sum[j] = e2m1_sum(h[8 * i + j], hi);
                    other |= __float_as_uint(sum[j]) ^ __float_as_uint(e2m1_sum(h[8 * i + j], lo));
                }
                codes[i] = e2m1x8(sum, sign);
            }
            sure = other == 0u;
        }
    }
    const int lane = threadIdx.x & 31;
    for (uint32_t left = __ballot_sync(0xFFFFFFFFu, !sure); left != 0u; left &= left - 1u) {
        const int who = __ffs((int)left) - 1;
        float2* mine = unsure[threadIdx.x / 32];
        if (lane == who) {
#pragma unroll
            for (int j = 0; j < kR4Block; ++j) mine[j] = make_float2(number_of<T>(gw, j), number_of<T>(uw, j));
        }
        __syncwarp();
        const int count = __shfl_sync(0xFFFFFFFFu, cols - at.block * kR4Block, who);
        uint32_t other[4];
        const uint32_t exact = glu4_block_exact<kAct>(limit, mine[lane].x, mine[lane].y, lane < count, other);
        if (lane == who) {
            s = exact;
#pragma unroll
            for (int i = 0; i < 4; ++i) codes[i] = other[i];
        }
        __syncwarp();
    }
    if (at.here) put4(o, at.r, at.block, codes, s);
}

// scales [n][lds] into the layout of the tensor cores (tiles of `tile` rows; zeros behind the last row and block): a thread per row and group
__global__ void arrange4_kernel(const uint8_t* __restrict__ scale, long long lds, long long rows, int blocks, uint8_t* __restrict__ tiles, int tile, int groups, long long slots) {
    const long long r = (long long)blockIdx.x * blockDim.x + threadIdx.x;       // counted in whole 128 rows of each tile
    const int g = blockIdx.y;
    pdl_launch_dependents();
    if (r >= slots) return;
    const int atoms = (tile + 127) / 128;
    const long long t = r / (atoms * 128), in = r % (atoms * 128), row = t * tile + in;
    uint32_t w = 0;
    if (in < tile && row < rows) {
        const uint8_t* from = scale + row * lds + 4 * g;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (4 * g + i < blocks) w |= (uint32_t)from[i] << (8 * i);
    }
    *reinterpret_cast<uint32_t*>(tiles + ((t * groups + g) * atoms + in / 128) * 512 + in % 32 * 16 + in % 128 / 32 * 4) = w;
}

}  // namespace fl

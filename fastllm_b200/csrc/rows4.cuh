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

__device__ __forceinline__ uint32_t down4_bf16(uint32_t s) { return s == 0u ? 0x0040u : (s == 255u ? 0x7FFFu : s << 7); }
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// number j of words of T, and the bits of one
template <typename T> __device__ __forceinline__ float number_of(const uint32_t* w, int j);
template <> __device__ __forceinline__ float number_of<float>(const uint32_t* w, int j) { return __uint_as_float(w[j]); }
template <> __device__ __forceinline__ float number_of<__nv_bfloat16>(const uint32_t* w, int j) { return j & 1 ? bf16hi(w[j / 2]) : bf16lo(w[j / 2]); }
template <> __device__ __forceinline__ float number_of<__half>(const uint32_t* w, int j) { return __half2float(__ushort_as_half((unsigned short)(w[j / 2] >> (16 * (j & 1))))); }
__device__ __forceinline__ uint32_t bits_of(float v) { return __float_as_uint(v); }
__device__ __forceinline__ uint32_t bits_of(__nv_bfloat16 v) { return __bfloat16_as_ushort(v); }
__device__ __forceinline__ uint32_t bits_of(__half v) { return __half_as_ushort(v); }

// to the nearest e2m1, halves to the even mantissa, beyond 6 to 6; eight columns, the first in the low bits
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8]) {
    uint32_t w;
    asm("{\n"
        ".reg .b8 a, b, c, d;\n"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
        "mov.b32 %0, {a, b, c, d};\n"
        "}\n"
        : "=r"(w)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return w;
}
// eight codes, the first in the low bits, as bf16 numbers: both bytes of a number by a look-up among eight, then the sign
__device__ __forceinline__ void from_e2m1x8(uint32_t w, uint32_t (&bf16)[4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i, w >>= 16) {
        const uint32_t at = w & 0x7777u, low = __byte_perm(0xC0800000u, 0xC0804000u, at), high = __byte_perm(0x3F3F3F00u, 0x40404040u, at);
        bf16[2 * i] = __byte_perm(low, high, 0x5140) | ((w << 12) & 0x8000u) | ((w << 24) & 0x80000000u);
        bf16[2 * i + 1] = __byte_perm(low, high, 0x7362) | ((w << 4) & 0x8000u) | ((w << 16) & 0x80000000u);
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
// A thread takes 64 bytes of a row: a block of 16-bit numbers, half a block of 32-bit ones.  Which one, of all rows' pieces (`per` a row) in order
struct At4 {
    long long r;
    int piece;
    bool here;
    __device__ At4(long long rows, int per) {
        const unsigned long long id = (unsigned long long)blockIdx.x * kR4Threads + threadIdx.x, all = (unsigned long long)rows * per;
        here = id < all;
        if (all <= 0xFFFFFFFFull) {
            const uint32_t q = (uint32_t)id / (uint32_t)per;
            r = q;
            piece = (int)((uint32_t)id - q * (uint32_t)per);
        } else {
            r = (long long)(id / per);
            piece = (int)(id - (unsigned long long)r * per);
        }
    }
};
template <typename T> constexpr int kR4Lanes = sizeof(T) == 4 ? 2 : 1;                 // threads of a block of 32
template <typename T> constexpr int kR4Own = kR4Block / kR4Lanes<T>;                   // numbers of a thread
template <typename T>
__device__ __forceinline__ void put4(const Rows4Out& o, long long r, int piece, const uint32_t (&codes)[kR4Own<T> / 8], uint32_t s) {
    const int block = piece / kR4Lanes<T>;
    uint8_t* q = o.q + r * o.ldq + piece * (kR4Own<T> / 2);
    if (block < o.blocks) {
        if constexpr (kR4Lanes<T> == 1) *reinterpret_cast<uint4*>(q) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
        else *reinterpret_cast<uint2*>(q) = make_uint2(codes[0], codes[1]);
    }
    uint8_t* to = o.tile == 0 ? o.scale + r * o.lds + block : o.scale + scale4_at(r, block / 4, o.tile, o.groups) + block % 4;
    if (piece % kR4Lanes<T> == 0) *to = (uint8_t)s;
}
// 64 bytes from column `at` on, zeros past the row's end.  kVec: rows start on 16-byte borders.
template <typename T, bool kVec>
__device__ __forceinline__ void load64(const T* row, int at, int cols, uint32_t (&w)[16]) {
    if (kVec && at + kR4Own<T> <= cols) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + at) + i);
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
    } else if (!kVec && at + kR4Own<T> <= cols) {
        load_row(row, at, cols, w);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t part[4];
            load_row(row, at + kR4Own<T> / 4 * i, cols, part);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[4 * i + j] = part[j];
        }
    }
}
// bits, as of f32, of the largest magnitude among the words' numbers; those of 16 bits are in the order of their bits too
template <typename T>
__device__ __forceinline__ uint32_t most_of(const uint32_t (&w)[16]) {
    uint32_t m = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 16; j += 2) m = __vimax3_u32(m, w[j] & 0x7FFFFFFFu, w[j + 1] & 0x7FFFFFFFu);
        return m;
    } else {
#pragma unroll
        for (int j = 0; j < 16; j += 2) m = __vimax3_u16x2(m, w[j] & 0x7FFF7FFFu, w[j + 1] & 0x7FFF7FFFu);
        m = max(m & 0xFFFFu, m >> 16);
        return abs_bits(number_of<T>(&m, 0));
    }
}
// the largest of a block's threads
template <typename T>
__device__ __forceinline__ uint32_t block_max(uint32_t m) { return kR4Lanes<T> == 1 ? m : max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1)); }

// What a block costs once, its place and its scale, counts little beside the 32 numbers of a thread: with eight a thread the instructions were the bound, 19 a number.  What
// bounds it: HBM (28672 x 4096 bf16 there and back 99 us, 6.0 TB/s; 16384 x 4000 f32 55, 5.4 TB/s).
template <typename T, bool kVec>
__global__ void __launch_bounds__(kR4Threads) quantize4_kernel(const T* __restrict__ x, long long ldx, long long rows, int cols, int per, const Rows4Out o) {
    pdl_launch_dependents();
    const At4 at(rows, per);
    uint32_t w[16] = {}, codes[kR4Own<T> / 8] = {};
    if (at.here) load64<T, kVec>(x + at.r * ldx, at.piece * kR4Own<T>, cols, w);
    const uint32_t s = scale4(block_max<T>(most_of<T>(w)));
    if (!at.here) return;
    if (s != 255u) {
        const float up = up4(s);
#pragma unroll
        for (int i = 0; i < kR4Own<T> / 8; ++i) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = number_of<T>(w, 8 * i + j) * up;        // exact, or far below the smallest border
            codes[i] = e2m1x8(v);
        }
    }
    put4<T>(o, at.r, at.piece, codes, s);
}

// Eight numbers a thread (of 32 bits: four), which it writes at once.  kShift: rows of results may start anywhere, some numbers behind a 16-byte border; a thread then takes the
// columns between two borders, and its codes out of two words.  grid (rows, threads' pieces of a row): a division for eight numbers cost a fifth of the time.  What bounds it: HBM's
// writes and the look-ups (28672 x 4096 bf16 54 us, 5.5 TB/s).
template <typename T, bool kShift>
__global__ void __launch_bounds__(256) dequantize4_kernel(const uint8_t* __restrict__ q, long long ldq, const uint8_t* __restrict__ scale, long long lds, int cols, int words,
                                                                 T* __restrict__ y, long long ldy) {
    constexpr int V = 16 / sizeof(T), U = 2;                    // pieces of a thread
    const long long r = blockIdx.x;
    const uint32_t* qr = reinterpret_cast<const uint32_t*>(q + r * ldq);               // `words` of eight codes
    const uint8_t* sr = scale + r * lds;
    T* yr = y + r * ldy;
    const int at0 = (blockIdx.y * U * blockDim.x + threadIdx.x) * V - (kShift ? (int)((reinterpret_cast<uintptr_t>(yr) & 15u) / sizeof(T)) : 0), step = blockDim.x * V;
    uint32_t w[U], s0[U], s1[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int at = at0 + i * step;
        w[i] = s0[i] = s1[i] = 0u;
        if (at >= cols) break;
        if constexpr (kShift) {
            const int lo = at >> 3, hi = (at + V - 1) >> 3;
            const uint32_t w0 = lo >= 0 ? __ldg(qr + lo) : 0u, w1 = hi != lo && hi < words ? __ldg(qr + hi) : 0u;
            s0[i] = lo >= 0 ? __ldg(sr + (lo >> 2)) : 0u;
            s1[i] = hi >> 2 != lo >> 2 && hi < words ? __ldg(sr + (hi >> 2)) : s0[i];
            w[i] = __funnelshift_r(w0, w1, 4 * (at & 7));
        } else {
            w[i] = __ldg(qr + (at >> 3)) >> (4 * (at & 7));
            s0[i] = __ldg(sr + (at >> 5));
        }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int at = at0 + i * step;
        if (at >= cols) break;
        uint32_t e2m1[4];
        from_e2m1x8(w[i], e2m1);
        const int own = 32 - (at & 31);                         // columns left in the first word's block
        uint32_t t[4] = {};
        if constexpr (std::is_same_v<T, __nv_bfloat16>) {       // powers of two and e2m1 are bf16 numbers, and so is every product in range
            const uint32_t d0 = down4_bf16(s0[i]), d1 = kShift ? down4_bf16(s1[i]) : d0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t d = (kShift && 2 * j >= own ? d1 : d0) | (kShift && 2 * j + 1 >= own ? d1 : d0) << 16;
                t[j] = mul_bf16x2(e2m1[j], d);
            }
        } else {
            const float d0 = down4(s0[i]), d1 = kShift ? down4(s1[i]) : d0;
#pragma unroll
            for (int j = 0; j < V; ++j)
                t[j * 4 / V] |= bits_of(from_f32<T>(number_of<__nv_bfloat16>(e2m1, j) * (kShift && j >= own ? d1 : d0))) << (V == 8 ? 16 * (j & 1) : 0);
        }
        if ((!kShift || at >= 0) && at + V <= cols) {
            *reinterpret_cast<uint4*>(yr + at) = make_uint4(t[0], t[1], t[2], t[3]);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (at + j >= 0 && at + j < cols) yr[at + j] = from_f32<T>(number_of<T>(t, j));
        }
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
// h in f32, with e = 2^t = e^-z.  t is off by |t| 2^-22 at most (a cubic's sum: four roundings), which moves h as far as e counts beside 1; ex2 and the reciprocal are
// off by 2^-22 and 2^-23, the sum and the products by 2^-24 each: h (2^-20 + max(t, 0) 2^-21) is more than all of it.  From t = 126 on h is 0, and has fewer bits from
// t = 100 on: there it is below |g u| 2^-99.
template <int kAct>
__device__ __forceinline__ float glu4_near(float limit, float g, float u) {
    constexpr float kLog2e = 1.4426950408889634f;
    if constexpr (kAct == kGlu4Relu) return fmaxf(g, 0.f) * u;
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
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    return gate * r * up;
}
// no less than max(t, 0) of gates up to `in`, where that is below 100
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
// block is taken in 64 bits by its warp.  What bounds it: HBM beside two special functions a number (4096 x 14336 bf16 silu 50 us, 5.3 TB/s; 2048 x 14336 f32 42, 6.0 TB/s; all
// in 64 bits 287).
template <typename T, int kAct, bool kVec>
__global__ void __launch_bounds__(kR4Threads) glu4_kernel(const T* __restrict__ x, long long ldx, long long rows, int cols, int per, float limit, const Rows4Out o) {
    constexpr int kOwn = kR4Own<T>;
    pdl_launch_dependents();
    const At4 at(rows, per);
    uint32_t codes[kOwn / 8] = {}, s, in_bits = 0;
    float h[kOwn], most = 0.f;
    {
        uint32_t gw[16] = {}, uw[16] = {};
        if (at.here) {
            load64<T, kVec>(x + at.r * ldx, at.piece * kOwn, cols, gw);
            load64<T, kVec>(x + at.r * ldx + cols, at.piece * kOwn, cols, uw);
        }
        in_bits = block_max<T>(max(most_of<T>(gw), most_of<T>(uw)));
#pragma unroll
        for (int j = 0; j < kOwn; ++j) {
            h[j] = glu4_near<kAct>(limit, number_of<T>(gw, j), number_of<T>(uw, j));
            most = fmaxf(most, fabsf(h[j]));
        }
    }
    most = __uint_as_float(block_max<T>(__float_as_uint(most)));
    const float in = __uint_as_float(in_bits), off = kAct == kGlu4Relu ? 0x1p-22f : fmaf(glu4_far<kAct>(in), 0x1p-21f, 0x1p-20f);
    const float most_hi = most * (1.f + off), most_lo = most * (1.f - off);
    s = scale4(__float_as_uint(most_hi));
    // not where f32 has fewer bits, nor where a number from t = 100 on might count
    const float least = fmaxf(0x1p-100f, in * 0x1p-45f * (in * 0x1p-45f));
    bool sure = most == 0.f ? kAct == kGlu4Relu || in == 0.f : most_hi < INFINITY && most_hi >= least && s == scale4(__float_as_uint(most_lo));
    if (sure && most != 0.f) {
        const float up = up4(s), hi = up * (1.f + off), lo = up * (1.f - off);
        uint32_t other = 0;
#pragma unroll
        for (int i = 0; i < kOwn / 8; ++i) {
            float a[8], b[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                a[j] = h[8 * i + j] * hi;
                b[j] = h[8 * i + j] * lo;
            }
            codes[i] = e2m1x8(a);
            other |= codes[i] ^ e2m1x8(b);
        }
        sure = other == 0u;
    }
    if (in_bits >= 0x7F800000u) {
        sure = true;
        s = 255u;
#pragma unroll
        for (int i = 0; i < kOwn / 8; ++i) codes[i] = 0u;
    }
    const int lane = threadIdx.x & 31;
    uint32_t left = __ballot_sync(0xFFFFFFFFu, !sure && at.here);
    if constexpr (kR4Lanes<T> == 2) left = (left | left >> 1) & 0x55555555u;           // a block by its first thread
    for (; left != 0u; left &= left - 1u) {
        const int who = __ffs((int)left) - 1;
        const long long r = __shfl_sync(0xFFFFFFFFu, at.r, who);
        const int col = __shfl_sync(0xFFFFFFFFu, at.piece, who) * kOwn + lane;
        const bool here = col < cols;
        const T* row = x + r * ldx + col;
        uint32_t exact[4];
        const uint32_t es = glu4_block_exact<kAct>(limit, here ? to_f32(row[0]) : 0.f, here ? to_f32(row[cols]) : 0.f, here, exact);
        if (lane / kR4Lanes<T> == who / kR4Lanes<T>) {
            s = es;
#pragma unroll
            for (int i = 0; i < kOwn / 8; ++i) codes[i] = kR4Lanes<T> == 2 && (lane & 1) ? exact[2 + i] : exact[i];
        }
    }
    if (at.here) put4<T>(o, at.r, at.piece, codes, s);
}

// Scales [rows][lds] into the layout of the tensor cores, in tiles of `tile` rows, zeros behind the last row and block.  A block of threads takes 128 rows (an atom of a tile) and
// kArrange groups: a thread reads 32 neighbours of its row, and whole atoms of 512 bytes are written.
constexpr int kArrange = 8;
__global__ void __launch_bounds__(128) arrange4_kernel(const uint8_t* __restrict__ scale, long long lds, long long rows, int blocks, uint8_t* __restrict__ tiles, int tile, int groups, int atoms) {
    __shared__ __align__(16) uint32_t part[kArrange][128];
    const int t = threadIdx.x, g0 = blockIdx.y * kArrange;
    const long long i = blockIdx.x / atoms;                     // the tile, and the atom's place in it
    const int atom = (int)(blockIdx.x - i * atoms), in = atom * 128 + t;
    const long long row = i * tile + in;
    pdl_launch_dependents();
    const uint8_t* from = scale + row * lds + 4 * g0;
    const bool here = in < tile && row < rows, words = (reinterpret_cast<uintptr_t>(from) & 3u) == 0;
#pragma unroll
    for (int g = 0; g < kArrange; ++g) {
        const int left = here ? blocks - 4 * (g0 + g) : 0;
        uint32_t w = 0;
        if (words && left >= 4) {
            w = __ldg(reinterpret_cast<const uint32_t*>(from) + g);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < left) w |= (uint32_t)from[4 * g + j] << (8 * j);
        }
        part[g][t % 32 * 4 + t / 32] = w;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kArrange / 4; ++j) {
        const int g = 4 * j + t / 32;
        if (g0 + g < groups) *reinterpret_cast<uint4*>(tiles + ((i * groups + g0 + g) * atoms + atom) * 512 + t % 32 * 16) = *reinterpret_cast<const uint4*>(&part[g][t % 32 * 4]);
    }
}

}  // namespace fl

// Rows of 4-bit numbers with a scale per 32 neighbours (OCP Microscaling, MXFP4): value = e2m1 * 2^(s - 127), e2m1 one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 and
// their negatives, s a byte (255: NaN); the even column lies in the low half of a byte.  Rounding to such rows, the way back, and gated activations that end in them.
#pragma once
#include "op_values.cuh"

namespace fl {

constexpr int kR4Block = 32;                                    // values that share a scale
constexpr int kR4Span = 256;                                    // columns of a warp: eight neighbours a lane, four lanes a block

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
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        v[2 * i] = f.x; v[2 * i + 1] = f.y;
    }
}

// eight values from column `at` of a row on, zeros past its end.  vec: they start on a 16-byte border.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int at, int cols, bool vec, float (&v)[8]) {
    if (vec && at + 8 <= cols) {
        uint4 h[sizeof(T) / 2];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) h[i] = __ldg(reinterpret_cast<const uint4*>(row + at) + i);
        const T* e = reinterpret_cast<const T*>(h);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = to_f32(e[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = at + j < cols ? to_f32(row[at + j]) : 0.f;
    }
}

// A warp's eight blocks: codes of this lane's eight columns, the byte of its block's scale (the same in its four lanes)
__device__ __forceinline__ void put4(const Rows4Out& o, long long r, int at, uint32_t codes, uint32_t s) {
    const int lane = threadIdx.x & 31, block = at / kR4Block;
    if (block < o.blocks) *reinterpret_cast<uint32_t*>(o.q + r * o.ldq + at / 2) = codes;
    if (o.tile == 0) {
        if (lane % 4 == 0 && block < o.blocks) o.scale[r * o.lds + block] = (uint8_t)s;
        return;
    }
    uint32_t w = s << (8 * (lane / 4 % 4));
    w |= __shfl_xor_sync(0xFFFFFFFFu, w, 4);
    w |= __shfl_xor_sync(0xFFFFFFFFu, w, 8);
    if (lane % 16 == 0 && block / 4 < o.groups) *reinterpret_cast<uint32_t*>(o.scale + scale4_at(r, block / 4, o.tile, o.groups)) = w;
}
__device__ __forceinline__ uint32_t quad_max(uint32_t m) {
    m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
    return max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
}

// grid (rows, spans of a row / warps of a block)
template <typename T>
__global__ void quantize4_kernel(const T* __restrict__ x, long long ldx, int cols, bool vec, const Rows4Out o) {
    const long long r = blockIdx.x;
    const int at = (blockIdx.y * blockDim.x + threadIdx.x) * 8;
    pdl_launch_dependents();
    float v[8];
    load8(x + r * ldx, at, cols, vec, v);
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, abs_bits(v[j]));
    const uint32_t s = scale4(quad_max(m));
    const float up = up4(s);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = s == 255u ? 0.f : v[j] * up;        // exact, or far below the smallest border
    put4(o, r, at, e2m1x8(v), s);
}

template <typename T>
__global__ void dequantize4_kernel(const uint8_t* __restrict__ q, long long ldq, const uint8_t* __restrict__ scale, long long lds, int cols, T* __restrict__ y, long long ldy,
                                   bool vec) {
    const long long r = blockIdx.x;
    const int at = (blockIdx.y * blockDim.x + threadIdx.x) * 8;
    if (at >= cols) return;
    float v[8];
    from_e2m1x8(__ldg(reinterpret_cast<const uint32_t*>(q + r * ldq + at / 2)), v);
    const float d = down4(__ldg(scale + r * lds + at / kR4Block));
    T t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = from_f32<T>(v[j] * d);
    T* to = y + r * ldy + at;
    if (vec && at + 8 <= cols) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(to)[i] = reinterpret_cast<const uint4*>(t)[i];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (at + j < cols) to[j] = t[j];
    }
}

// Gated activations h = act(g) u in 64 bits
enum { kGlu4SwishClamp = 0, kGlu4GeluTanh = 1, kGlu4Relu = 3, kGlu4Silu = 4 };          // fl_ffn_act
__device__ __forceinline__ double glu4_exact(int act, float limit, float gf, float uf) {
    const double g = gf, u = uf;
    if (act == kGlu4Silu) return g / (1.0 + exp(-g)) * u;
    if (act == kGlu4GeluTanh) return g / (1.0 + exp(-1.5957691216057308 * (g + 0.044715 * g * g * g))) * u;
    if (act == kGlu4Relu) return fmax(g, 0.0) * u;
    const double c = fmin(g, (double)limit);
    return c / (1.0 + exp(-1.702 * c)) * (fmin(fmax(u, -(double)limit), (double)limit) + 1.0);
}

template <typename T>
__global__ void glu4_kernel(const T* __restrict__ x, long long ldx, int cols, bool vec_gate, bool vec_up, int act, float limit, const Rows4Out o) {
    const long long r = blockIdx.x;
    const int at = (blockIdx.y * blockDim.x + threadIdx.x) * 8;
    pdl_launch_dependents();
    float g[8], u[8], v[8];
    load8(x + r * ldx, at, cols, vec_gate, g);
    load8(x + r * ldx + cols, at, cols, vec_up, u);
    uint32_t m = 0;
    double h[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        h[j] = at + j < cols ? glu4_exact(act, limit, g[j], u[j]) : 0.0;
        const bool bad = max(abs_bits(g[j]), abs_bits(u[j])) >= 0x7F800000u;
        // truncated, so that the exponent is h's own; beyond f32: an infinity
        m = max(m, bad ? 0x7FFFFFFFu : abs_bits(fabs(h[j]) >= 0x1p128 ? INFINITY : __double2float_rz(h[j])));
    }
    const uint32_t s = scale4(quad_max(m));
    const double up = s == 255u ? 0.0 : __hiloint2double((int)(1023u + 127u - s) << 20, 0);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const double t = s == 255u ? 0.0 : fabs(h[j]) * up;
        // the nearest e2m1 to t, which f32 then holds: its own rounding might cross a border
        const float e = t > 5.0 ? 6.f : t >= 3.5 ? 4.f : t > 2.5 ? 3.f : t >= 1.75 ? 2.f : t > 1.25 ? 1.5f : t >= 0.75 ? 1.f : t > 0.25 ? 0.5f : 0.f;
        v[j] = h[j] < 0.0 ? -e : e;
    }
    put4(o, r, at, e2m1x8(v), s);
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

// Microscaled 4-bit rows: the format, and its conversions on the device.
//
// A row of `cols` values is nb = ceil(cols/32) blocks.  Block b has sixteen
// bytes of codes (value i of the row in byte i/2, the even one in the low
// nibble; past cols the codes are 0) and one scale byte s that stands for
// 2^(s - 127), 255 for NaN.  A code is sign, two exponent bits, one mantissa
// bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6.  Codes of successive rows are 16*nb bytes
// apart, scales nb bytes rounded up to a whole dword.  This is what
// v_mfma_scale_f32_*_f8f6f4 takes: one lane holds one block and its scale.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace q4mi {

// ggml type ids of the rows that go in and come out
constexpr uint32_t kTypeF32 = 0, kTypeF16 = 1, kTypeBF16 = 30, kTypeMx4 = 39;

constexpr bool is_float_type(uint32_t t) {
    return t == kTypeF32 || t == kTypeF16 || t == kTypeBF16;
}
constexpr uint32_t type_bytes(uint32_t t) { return t == kTypeF32 ? 4u : 2u; }

__host__ __device__ inline uint32_t mx4_blocks(uint64_t cols) {
    return (uint32_t)((cols + 31) / 32);
}
__host__ __device__ inline uint32_t mx4_scale_row(uint32_t nb) { return (nb + 3u) & ~3u; }

__device__ inline float bits_f32(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ inline uint32_t f32_bits(float f) { return __builtin_bit_cast(uint32_t, f); }

// One value of a float row (t is uniform over the launch).
__device__ inline float load_as_f32(const void *p, uint32_t t, uint64_t i) {
    if (t == kTypeF32) return ((const float *)p)[i];
    const uint16_t h = ((const uint16_t *)p)[i];
    return t == kTypeF16 ? (float)__builtin_bit_cast(_Float16, h) : bits_f32((uint32_t)h << 16);
}

// Two floats as F16 or BF16, the first in the low half: to nearest, ties to
// even, NaN stays NaN.  One instruction each way and a choice between them, no
// branch: with a rounding by hand, which tests each element for NaN and for its
// type, 8192 rows x 16384 x 2048 took 231 us for 196, 16384 rows x 16384 x 1024
// 301 for 230.
__device__ inline uint32_t f32_to_16x2(float a, float b, uint32_t t) {
    typedef _Float16 half2 __attribute__((ext_vector_type(2)));
    typedef __bf16 brain2 __attribute__((ext_vector_type(2)));
    typedef float float2v __attribute__((ext_vector_type(2)));
    const float2v v = {a, b};
    const uint32_t h = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, half2));
    const uint32_t l = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, brain2));
    return t == kTypeF16 ? h : l;
}
__device__ inline uint16_t f32_to_16(float f, uint32_t t) {
    return (uint16_t)f32_to_16x2(f, 0.f, t);
}

__device__ inline void store_from_f32(void *p, uint32_t t, uint64_t i, float f) {
    if (t == kTypeF32)
        ((float *)p)[i] = f;
    else
        ((uint16_t *)p)[i] = f32_to_16(f, t);
}

// Scale byte of a block whose largest magnitude has the fp32 bits `top`
// (sign cleared): floor(log2(top)) - 2 with bias 127 is the exponent field
// minus 2, not below 0; 255 when the block holds an infinity or a NaN (whose
// bits are the largest as integers).
__device__ inline uint32_t mx4_scale_of(uint32_t top) {
    if (top >= 0x7f800000u) return 255u;
    const uint32_t f = top >> 23;
    return f > 2u ? f - 2u : 0u;
}

// Factor that takes the block's values to the codes' range: 2^(127 - s), a
// normal fp32 for every scale byte that mx4_scale_of gives; 0 for a block
// without finite values, whose codes are 0.
__device__ inline float mx4_factor(uint32_t s) {
    return s == 255u ? 0.f : bits_f32((254u - s) << 23);
}

// Two scaled values as codes, in byte `SEL` of `old`: to nearest, ties to the
// even code, at most 6 in magnitude.
template <int SEL>
__device__ inline uint32_t mx4_pack2(uint32_t old, float a, float b) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(old, a, b, 1.0f, SEL);
}

// Eight values of a block as one dword of codes.  A block without finite
// values multiplies by 0: an infinity or a NaN there would come out as NaN,
// so its codes are set.
__device__ inline uint32_t mx4_pack8(const float *v, uint32_t s) {
    const float f = mx4_factor(s);
    uint32_t q = 0;
    q = mx4_pack2<0>(q, v[0] * f, v[1] * f);
    q = mx4_pack2<1>(q, v[2] * f, v[3] * f);
    q = mx4_pack2<2>(q, v[4] * f, v[5] * f);
    q = mx4_pack2<3>(q, v[6] * f, v[7] * f);
    return s == 255u ? 0u : q;
}

// Vectors in memory at any address of their elements (global loads and stores
// take 16 bytes at any of them).
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4_a4 __attribute__((aligned(4)));
typedef u32x4 u32x4_a4 __attribute__((aligned(4)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
typedef u32x2 u32x2_a2 __attribute__((aligned(2)));

// Eight values of a float row from column c0 on (0 past cols).  row: index of
// the row's first element.
__device__ inline void load_row8(const void *x, uint32_t xt, uint64_t row, uint32_t c0,
                                 uint32_t cols, float *v) {
    const uint64_t at = row + c0;
    if (c0 + 8 <= cols) {
        if (xt == kTypeF32) {
            const f32x4 lo = *(const f32x4_a4 *)((const float *)x + at);
            const f32x4 hi = *(const f32x4_a4 *)((const float *)x + at + 4);
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = lo[i], v[4 + i] = hi[i];
        } else {
            const u32x4 w = *(const u32x4_a2 *)((const uint16_t *)x + at);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (xt == kTypeBF16) {
                    v[2 * i] = bits_f32(w[i] << 16);
                    v[2 * i + 1] = bits_f32(w[i] & 0xffff0000u);
                } else {
                    v[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)w[i]);
                    v[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] >> 16));
                }
            }
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; i++)
            v[i] = c0 + i < cols ? load_as_f32(x, xt, at + i) : 0.f;
    }
}

// Scale byte of a block of which 32 / N adjacent lanes hold N values each.
template <uint32_t N>
__device__ inline uint32_t mx4_block_scale(const float *v) {
    uint32_t top = 0;
#pragma unroll
    for (uint32_t i = 0; i < N; i++) top = max(top, f32_bits(v[i]) & 0x7fffffffu);
#pragma unroll
    for (uint32_t d = 1; d < 32 / N; d *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, d, 64));
    return mx4_scale_of(top);
}

// 2^(s - 127) as fp32 (a subnormal for s = 0), NaN for 255.
__device__ inline float mx4_scale_value(uint32_t s) {
    return bits_f32(s == 255u ? 0x7fc00000u : s ? s << 23 : 0x00400000u);
}

// Two codes (byte SEL of q) as fp32 values, before their scale.
typedef float mx4_f2 __attribute__((ext_vector_type(2)));
template <int SEL>
__device__ inline mx4_f2 mx4_unpack2(uint32_t q) {
    return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, SEL);
}

}  // namespace q4mi

// 8-bit floating point rows in blocks of 128: the format, and its conversions
// on the device.
//
// A row of `cols` values is nb = ceil(cols/128) blocks and 128 * nb bytes of
// e4m3 codes (sign, four exponent bits of bias 7, three mantissa bits; no
// infinity, 0x7f and 0xff are NaN, the largest is 448), 0 past cols.  A block
// has one fp32 scale: of 128 values of a row (activations, scales [rows][nb])
// or of 128 x 128 values (weights, scales [ceil(rows / 128)][nb]).
//
// The quantiser's scales are powers of two: the least 2^k >= 2^-120 with
// max|x| <= 448 * 2^k.  Then x / 2^k is exact, the codes are the nearest ones
// whatever the order of operations, and a real tie of two codes stays one (with
// max|x| / 448 it would fall either way with the scale's last bit).  A code
// loses no bits by that but at the small end, where it has 2^-9 steps.
#pragma once
#include "mx4.h"

namespace q4mi {

constexpr uint32_t kTypeF8 = 248;   // this library's own number: ggml has no such type

__host__ __device__ inline uint32_t f8_blocks(uint64_t cols) {
    return (uint32_t)((cols + 127) / 128);
}

// The block's scale as fp32 bits, from the fp32 bits of its largest magnitude
// (sign cleared); NaN when the block holds an infinity or a NaN (whose bits are
// the largest as integers).  448 = 1.75 * 2^8.
__device__ inline uint32_t f8_scale_of(uint32_t top) {
    const int32_t f = (int32_t)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    return top >= 0x7f800000u ? 0x7fc00000u : (uint32_t)max(f, 7) << 23;
}

// 1 / scale, exact; 0 for NaN.
__device__ inline float f8_factor(uint32_t s) {
    return s == 0x7fc00000u ? 0.f : bits_f32(0x7f000000u - s);
}

// Four scaled values (at most 448 in magnitude) as a dword of codes, to nearest,
// ties to the even code.
__device__ inline uint32_t f8_pack4(float a, float b, float c, float d) {
    int q = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, q, true);
}

// N values of a block as N / 4 dwords.  Without finite values the factor is 0,
// an infinity or a NaN times that would be NaN: the codes are set.
template <uint32_t N>
__device__ inline void f8_pack(const float *v, uint32_t s, uint32_t *q) {
    const float f = f8_factor(s);
#pragma unroll
    for (uint32_t i = 0; i < N; i += 4) {
        const uint32_t c = f8_pack4(v[i] * f, v[i + 1] * f, v[i + 2] * f, v[i + 3] * f);
        q[i / 4] = s == 0x7fc00000u ? 0u : c;
    }
}

template <uint32_t N>
__device__ inline uint32_t f8_top(const float *v) {
    uint32_t top = 0;
#pragma unroll
    for (uint32_t i = 0; i < N; i++) top = max(top, f32_bits(v[i]) & 0x7fffffffu);
    return top;
}

// The largest over an aligned group of 8 or 16 lanes, all of them active:
// swaps inside quads, then of a row's quads and halves by mirrors (after each
// step the lanes that a mirror pairs agree within their part).
template <int CTRL>
__device__ inline uint32_t f8_max_dpp(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true));
}
template <uint32_t LANES>
__device__ inline uint32_t f8_max_lanes(uint32_t v) {
    static_assert(LANES == 8 || LANES == 16, "part of a row of lanes");
    v = f8_max_dpp<0xB1>(v);            // lane ^ 1
    v = f8_max_dpp<0x4E>(v);            // lane ^ 2
    v = f8_max_dpp<0x141>(v);           // the other quad of eight
    if (LANES == 16) v = f8_max_dpp<0x140>(v);   // the other eight of sixteen
    return v;
}

typedef float f8_f2 __attribute__((ext_vector_type(2)));

// The four values of a dword of codes.
__device__ inline void f8_unpack4(uint32_t q, float *v) {
    const f8_f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, false);
    const f8_f2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, true);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
}

// Eight columns as they are in memory (B bytes a value), so that a lane's loads
// all go out before the first is converted.
template <uint32_t B>
struct Raw8 {
    u32x4 q[B / 2];
};
template <uint32_t B>
__device__ inline void load_raw8(const void *p, uint64_t row, uint32_t c0, uint32_t cols,
                                 Raw8<B> &r) {
    const uint8_t *at = (const uint8_t *)p + (row + c0) * B;
    if (c0 + 8 <= cols) {
#pragma unroll
        for (uint32_t i = 0; i < B / 2; i++) {
            if constexpr (B == 4)
                r.q[i] = *(const u32x4_a4 *)(at + 16 * i);
            else
                r.q[i] = *(const u32x4_a2 *)(at + 16 * i);
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < B / 2; i++) r.q[i] = (u32x4){0, 0, 0, 0};
        // columns past the last are 0
        if (c0 >= cols) return;
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            if (c0 + i >= cols) continue;
            if constexpr (B == 4)
                r.q[i / 4][i % 4] = ((const uint32_t *)at)[i];
            else
                r.q[0][i / 2] |= (uint32_t)((const uint16_t *)at)[i] << (16 * (i % 2));
        }
    }
}
template <uint32_t B>
__device__ inline void raw8_to_f32(const Raw8<B> &r, uint32_t t, float *v) {
    if constexpr (B == 4) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = bits_f32(r.q[i / 4][i % 4]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t h = i % 2 ? r.q[0][i / 2] >> 16 : r.q[0][i / 2] & 0xffffu;
            v[i] = t == kTypeF16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)h)
                                 : bits_f32(h << 16);
        }
    }
}

}  // namespace q4mi

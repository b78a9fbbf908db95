// Float rows to microscaled 4-bit rows and back (mx4.h has the format).
//
// Per block of 32 values: s = max(floor(log2(max |x|)) - 2, -127), codes
// RNE(x / 2^s) capped at 6.  The scale is a power of two, so x / 2^s is exact
// wherever a code other than 0 can come of it, and the codes depend on
// nothing but the 32 values.
#include "mx4.h"
#include "q4mi_internal.h"

using namespace q4mi;

// Four lanes a block, eight values a lane; a 256-thread workgroup takes 64
// successive blocks of the row-major block order.  VEC: rows are 16-byte
// aligned and whole, so a lane's values come in 16-byte loads.
template <bool VEC>
__global__ __launch_bounds__(256) void mx4_quant_k(const void *__restrict__ x, uint32_t xt,
                                                   uint64_t ld, const int32_t *__restrict__ ids,
                                                   uint64_t rows, uint32_t cols,
                                                   uint8_t *__restrict__ codes,
                                                   uint8_t *__restrict__ scales) {
    const uint32_t nb = mx4_blocks(cols), sld = mx4_scale_row(nb);
    const uint64_t base = (uint64_t)blockIdx.x * 64;
    const uint32_t off = (uint32_t)(base % nb) + (threadIdx.x >> 2);
    const uint64_t r = base / nb + off / nb;
    if (r >= rows) return;
    const uint32_t b = off % nb, sub = threadIdx.x & 3u;
    const uint64_t src = ids ? (uint64_t)(int64_t)ids[r] : r;
    const uint32_t c0 = b * 32 + sub * 8;
    float v[8];
    load_row8(x, xt, src * ld, c0, cols, VEC, v);
    uint32_t s;
    const uint32_t q = mx4_quant8(v, &s);
    *(uint32_t *)(codes + r * (16ull * nb) + b * 16u + sub * 4u) = q;
    if (sub == 0) {
        uint8_t *p = scales + r * sld;
        p[b] = (uint8_t)s;
        if (b == nb - 1)
            for (uint32_t i = nb; i < sld; i++) p[i] = 0;
    }
}

// The mirror: four lanes a block, eight values a lane.
template <bool VEC>
__global__ __launch_bounds__(256) void mx4_dequant_k(const uint8_t *__restrict__ codes,
                                                     const uint8_t *__restrict__ scales,
                                                     const int32_t *__restrict__ ids,
                                                     uint64_t rows, uint32_t cols,
                                                     void *__restrict__ y, uint32_t yt,
                                                     uint64_t ld) {
    const uint32_t nb = mx4_blocks(cols), sld = mx4_scale_row(nb);
    const uint64_t base = (uint64_t)blockIdx.x * 64;
    const uint32_t off = (uint32_t)(base % nb) + (threadIdx.x >> 2);
    const uint64_t r = base / nb + off / nb;
    if (r >= rows) return;
    const uint32_t b = off % nb, sub = threadIdx.x & 3u;
    const uint64_t src = ids ? (uint64_t)(int64_t)ids[r] : r;
    const uint32_t q = *(const uint32_t *)(codes + src * (16ull * nb) + b * 16u + sub * 4u);
    const float f = mx4_scale_value(scales[src * sld + b]);
    const mx4_f2 p0 = mx4_unpack2<0>(q), p1 = mx4_unpack2<1>(q), p2 = mx4_unpack2<2>(q),
                 p3 = mx4_unpack2<3>(q);
    const float v[8] = {p0.x * f, p0.y * f, p1.x * f, p1.y * f,
                        p2.x * f, p2.y * f, p3.x * f, p3.y * f};
    const uint32_t c0 = b * 32 + sub * 8;
    const uint64_t at = r * ld + c0;
    if (VEC && c0 + 8 <= cols) {
        if (yt == kTypeF32) {
            *(float4 *)((float *)y + at) = make_float4(v[0], v[1], v[2], v[3]);
            *(float4 *)((float *)y + at + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
                w[i] = f32_to_16(v[2 * i], yt) | (uint32_t)f32_to_16(v[2 * i + 1], yt) << 16;
            *(uint4 *)((uint16_t *)y + at) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; i++)
            if (c0 + i < cols) store_from_f32(y, yt, at + i, v[i]);
    }
}

namespace {

// What both directions ask of their arguments.
bool rows_ok(const char *who, const void *f, uint32_t type, uint64_t ld, uint64_t rows,
             uint64_t cols, const uint8_t *codes, const uint8_t *scales) {
    if (!f || !codes || !scales || !cols) {
        set_error("%s: bad arguments", who);
        return false;
    }
    if (!is_float_type(type)) {
        set_error("%s: type %u not covered (F32, F16, BF16)", who, type);
        return false;
    }
    if (cols > (1u << 30) || rows > (1ull << 32) || rows * mx4_blocks(cols) > (uint64_t)0x7fffffffu * 64) {
        set_error("%s: %llu x %llu too large", who, (unsigned long long)rows,
                  (unsigned long long)cols);
        return false;
    }
    if (ld < cols) {
        set_error("%s: row stride %llu below %llu columns", who, (unsigned long long)ld,
                  (unsigned long long)cols);
        return false;
    }
    if (((uintptr_t)f & (type_bytes(type) - 1)) || ((uintptr_t)codes & 15) ||
        ((uintptr_t)scales & 3)) {
        set_error("%s: float rows must be aligned to their type, codes to 16 bytes, scales to 4",
                  who);
        return false;
    }
    return true;
}

// Whether a lane's eight values can move 16 bytes at a time.
bool wide(const void *f, uint32_t type, uint64_t ld) {
    return !((uintptr_t)f & 15) && ld * type_bytes(type) % 16 == 0;
}

}  // namespace

extern "C" {

/* Bytes of the codes / scales of rows x cols values (see include/q4mi.h). */
uint64_t q4mi_mx4_code_bytes(uint64_t rows, uint64_t cols) {
    return rows * 16 * ((cols + 31) / 32);
}
uint64_t q4mi_mx4_scale_bytes(uint64_t rows, uint64_t cols) {
    return rows * ((((cols + 31) / 32) + 3) & ~3ull);
}

/* Float rows to microscaled 4-bit rows (see include/q4mi.h). */
bool q4mi_mx4_quant(const void *d_x, uint32_t x_type, uint64_t ld_x, const int32_t *d_ids,
                    uint64_t rows, uint64_t cols, uint8_t *d_codes, uint8_t *d_scales) {
    if (!rows_ok("q4mi_mx4_quant", d_x, x_type, ld_x, rows, cols, d_codes, d_scales)) return false;
    if (!rows) return true;
    const uint32_t grid = (uint32_t)((rows * mx4_blocks(cols) + 63) / 64);
    auto k = wide(d_x, x_type, ld_x) ? mx4_quant_k<true> : mx4_quant_k<false>;
    k<<<dim3(grid), dim3(256), 0, stream()>>>(d_x, x_type, ld_x, d_ids, rows, (uint32_t)cols,
                                              d_codes, d_scales);
    return launch_ok("mx4_quant_k");
}

/* Microscaled 4-bit rows to float rows (see include/q4mi.h). */
bool q4mi_mx4_dequant(const uint8_t *d_codes, const uint8_t *d_scales, const int32_t *d_ids,
                      uint64_t rows, uint64_t cols, void *d_y, uint32_t y_type, uint64_t ld_y) {
    if (!rows_ok("q4mi_mx4_dequant", d_y, y_type, ld_y, rows, cols, d_codes, d_scales))
        return false;
    if (!rows) return true;
    const uint32_t grid = (uint32_t)((rows * mx4_blocks(cols) + 63) / 64);
    auto k = wide(d_y, y_type, ld_y) ? mx4_dequant_k<true> : mx4_dequant_k<false>;
    k<<<dim3(grid), dim3(256), 0, stream()>>>(d_codes, d_scales, d_ids, rows, (uint32_t)cols, d_y,
                                              y_type, ld_y);
    return launch_ok("mx4_dequant_k");
}

}  // extern "C"

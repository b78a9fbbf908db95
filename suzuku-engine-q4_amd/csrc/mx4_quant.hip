// Float rows to microscaled 4-bit rows and back (mx4.h has the format).
//
// Per block of 32 values: s = max(floor(log2(max |x|)) - 2, -127), codes
// RNE(x / 2^s) capped at 6.  The scale is a power of two, so x / 2^s is exact
// wherever a code other than 0 can come of it, and the codes depend on
// nothing but the 32 values.
#include <algorithm>

#include "mx4.h"
#include "q4mi_internal.h"

using namespace q4mi;

// Place of a thread's block: `off` blocks past the first of the `each` (64 or
// 128) that the workgroup takes in the row-major order of all rows' blocks,
// off < each.  Workgroups
// with one blockIdx.y share a group of whole rows with fewer than 2^29 blocks,
// so that the divisions stay in 32 bits.
struct Place {
    uint64_t r;
    uint32_t b;
    __device__ Place(uint32_t each, uint64_t group, uint32_t off, uint32_t nb) {
        const uint32_t base = blockIdx.x * each, r0 = base / nb;
        b = base - r0 * nb + off;
        // a row of `each` blocks or more: at most one row further
        const uint32_t q = nb >= each ? (b >= nb ? 1u : 0u) : b / nb;
        b -= q * nb;
        const uint32_t in = r0 + q;
        r = in < group ? blockIdx.y * group + in : ~0ull;
    }
};

// N values a lane, 32 / N lanes a block: 32 bytes of input, eight fp32 or
// sixteen 16-bit values.
template <uint32_t N>
__global__ __launch_bounds__(256) void mx4_quant_k(const void *__restrict__ x, uint32_t xt,
                                                   uint64_t ld, const int32_t *__restrict__ ids,
                                                   uint64_t rows, uint64_t group, uint32_t cols,
                                                   uint8_t *__restrict__ codes,
                                                   uint8_t *__restrict__ scales) {
    constexpr uint32_t L = 32 / N;
    const uint32_t nb = mx4_blocks(cols), sld = mx4_scale_row(nb), sub = threadIdx.x % L;
    const Place p(256 / L, group, threadIdx.x / L, nb);
    if (p.r >= rows) return;
    const uint64_t src = ids ? (uint64_t)(int64_t)ids[p.r] : p.r;
    float v[N];
#pragma unroll
    for (uint32_t i = 0; i < N; i += 8)
        load_row8(x, xt, src * ld, p.b * 32 + sub * N + i, cols, v + i);
    const uint32_t s = mx4_block_scale<N>(v);
    uint32_t *c = (uint32_t *)(codes + p.r * (16ull * nb) + p.b * 16u + sub * (N / 2));
    if constexpr (N == 16)
        *(uint2 *)c = make_uint2(mx4_pack8(v, s), mx4_pack8(v + 8, s));
    else
        *c = mx4_pack8(v, s);
    if (sub == 0) {
        uint8_t *d = scales + p.r * sld;
        d[p.b] = (uint8_t)s;
        if (p.b == nb - 1)
            for (uint32_t i = nb; i < sld; i++) d[i] = 0;
    }
}

// The mirror, G values a lane (32 / G lanes a block), so that a lane's values
// are 16 bytes of output and a wave's one stretch: eight for 16-bit outputs,
// four for fp32.  Stored past the caches, whatever the size: alone that is the
// faster way from 2 MiB on (us through / past them, bf16: 16 MiB 5.8 / 4.7, 64
// MiB 14.5 / 11.4, 128 MiB 26.1 / 24.9, 256 MiB 67 / 47), while a quantiser that
// reads the values next has 64 and 128 MiB sooner through them (33 / 35 and
// 55 / 59 together; 16 MiB 15.5 / 15.2, 256 MiB 140 / 124).
template <uint32_t G>
__global__ __launch_bounds__(256) void mx4_dequant_k(const uint8_t *__restrict__ codes,
                                                     const uint8_t *__restrict__ scales,
                                                     const int32_t *__restrict__ ids,
                                                     uint64_t rows, uint64_t group,
                                                     uint32_t cols, void *__restrict__ y,
                                                     uint32_t yt, uint64_t ld) {
    constexpr uint32_t L = 32 / G, U = 8 / G;       // lanes a block; sets of blocks a workgroup
    const uint32_t nb = mx4_blocks(cols), sld = mx4_scale_row(nb), sub = threadIdx.x % L;
#pragma unroll
    for (uint32_t u = 0; u < U; u++) {
        const Place p(64, group, 256 / L * u + threadIdx.x / L, nb);
        if (p.r >= rows) continue;
        const uint64_t src = ids ? (uint64_t)(int64_t)ids[p.r] : p.r;
        const uint8_t *c = codes + src * (16ull * nb) + p.b * 16u + sub * (G / 2);
        const float f = mx4_scale_value(scales[src * sld + p.b]);
        const uint32_t c0 = p.b * 32 + sub * G;
        const uint64_t at = p.r * ld + c0;
        float v[G];
        const uint32_t q = G == 8 ? *(const uint32_t *)c : (uint32_t)*(const uint16_t *)c;
        const mx4_f2 p0 = mx4_unpack2<0>(q), p1 = mx4_unpack2<1>(q);
        v[0] = p0.x * f, v[1] = p0.y * f, v[2] = p1.x * f, v[3] = p1.y * f;
        if constexpr (G == 8) {
            const mx4_f2 p2 = mx4_unpack2<2>(q), p3 = mx4_unpack2<3>(q);
            v[4] = p2.x * f, v[5] = p2.y * f, v[6] = p3.x * f, v[7] = p3.y * f;
        }
        if (c0 + G <= cols) {
            if constexpr (G == 4) {
                __builtin_nontemporal_store((f32x4){v[0], v[1], v[2], v[3]},
                                            (f32x4_a4 *)((float *)y + at));
            } else {
                u32x4 w;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    w[i] = f32_to_16x2(v[2 * i], v[2 * i + 1], yt);
                __builtin_nontemporal_store(w, (u32x4_a2 *)((uint16_t *)y + at));
            }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < G; i++)
                if (c0 + i < cols) store_from_f32(y, yt, at + i, v[i]);
        }
    }
}

namespace {

// What both directions ask of their arguments.
bool rows_ok(const char *who, const void *f, uint32_t type, uint64_t ld, uint64_t rows,
             uint64_t cols, const uint8_t *codes, const uint8_t *scales) {
    if ((rows && (!f || !codes || !scales)) || !cols) {
        set_error("%s: bad arguments", who);
        return false;
    }
    if (!is_float_type(type)) {
        set_error("%s: type %u not covered (F32, F16, BF16)", who, type);
        return false;
    }
    if (cols > (1u << 30) || rows > (1ull << 32) || rows * mx4_blocks(cols) > (1ull << 45)) {
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

// `each` blocks a workgroup over groups of whole rows (see Place), of fewer
// than 2^29 blocks: a launch has fewer than 2^32 threads along x.
dim3 block_grid(uint32_t each, uint64_t rows, uint64_t cols, uint64_t *group) {
    const uint32_t nb = mx4_blocks(cols);
    *group = std::min<uint64_t>(rows, ((1u << 29) - each) / nb);
    return dim3((uint32_t)((*group * nb + each - 1) / each),
                (uint32_t)((rows + *group - 1) / *group));
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
    uint64_t group;
    const bool f32 = x_type == kTypeF32;
    const dim3 grid = block_grid(f32 ? 64 : 128, rows, cols, &group);
    auto k = f32 ? mx4_quant_k<8> : mx4_quant_k<16>;
    k<<<grid, dim3(256), 0, stream()>>>(d_x, x_type, ld_x, d_ids, rows, group, (uint32_t)cols,
                                        d_codes, d_scales);
    return launch_ok("mx4_quant_k");
}

/* Microscaled 4-bit rows to float rows (see include/q4mi.h). */
bool q4mi_mx4_dequant(const uint8_t *d_codes, const uint8_t *d_scales, const int32_t *d_ids,
                      uint64_t rows, uint64_t cols, void *d_y, uint32_t y_type, uint64_t ld_y) {
    if (!rows_ok("q4mi_mx4_dequant", d_y, y_type, ld_y, rows, cols, d_codes, d_scales))
        return false;
    if (!rows) return true;
    uint64_t group;
    const dim3 grid = block_grid(64, rows, cols, &group);
    auto k = y_type == kTypeF32 ? mx4_dequant_k<4> : mx4_dequant_k<8>;
    k<<<grid, dim3(256), 0, stream()>>>(d_codes, d_scales, d_ids, rows, group, (uint32_t)cols, d_y,
                                        y_type, ld_y);
    return launch_ok("mx4_dequant_k");
}

}  // extern "C"

// Products of 8-bit floating point rows in blocks of 128 (f8.h has the format):
//   y[t][r] = sum over blocks b of xs[t][b] * ws[r / 128][b] * sum_i w[r][128b+i] x[t][128b+i]
// A block is summed from zero by matrix instructions of sixteen weight rows and
// sixteen activation rows; its four sums a lane are then multiplied by both
// scales and added in fp32.  Weight rows are the first operand, so a lane's sums
// are four adjacent outputs of one activation row.
//
// The 8-bit matrix instructions add eight neighbouring products with only 14 bits
// below the largest of them (measured: a product 2^-14 of its neighbour is lost,
// one in another eight only at 2^-24), which leaves y 1.5e-5 off (2-norm).  Codes
// are exact in bf16, whose instruction adds in fp32 (1e-8 off) at half the rate.
#include <algorithm>

#include "f8.h"
#include "q4mi_internal.h"

using namespace q4mi;

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

struct F8Args {
    const uint8_t *w;               // weights: codes
    const float *ws;                // and scales
    const void *x;                  // activations: codes, or float rows
    const float *xs;                // scales of codes
    const int32_t *act, *bounds;    // packed rows: their activation rows, each expert's stretch
    const int32_t *eid;             // listed rows: their experts
    void *y;
    uint64_t w_rows, cols, w_stride, ws_stride, ldx, xrows, n, ldy;
    uint32_t n_expert, x_type, y_type, x_div;
};

// Four adjacent outputs, rounded once.
__device__ inline void store4(void *y, uint32_t yt, uint64_t at, v4f v) {
    if (yt == kTypeF32) {
        *(f32x4_a4 *)((float *)y + at) = (f32x4)v;
    } else {
        const u32x2 q = {f32_to_16x2(v[0], v[1], yt), f32_to_16x2(v[2], v[3], yt)};
        *(u32x2_a2 *)((uint16_t *)y + at) = q;
    }
}

__device__ inline v8i join(u32x4 a, u32x4 b) {
    const v8i r = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
    return r;
}

// Eight codes as bf16, exact.
__device__ inline v8b widen(uint32_t lo, uint32_t hi) {
    typedef __bf16 v2b __attribute__((ext_vector_type(2)));
    const v2b a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
    const v2b b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    const v2b c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
    const v2b d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    const v8b r = {a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
    return r;
}

// Sixteen rows against sixteen over one block, from zero.  Which of the block's
// values a lane holds is free as long as both sides agree: lane (row, g) has
// bytes 16g .. and 64 + 16g .. of its row, so that four lanes read 64 bytes.
__device__ inline v4f block_sums(v8i w, v8i x) {
    v4f d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 8; i += 2)
        d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(w[i], w[i + 1]), widen(x[i], x[i + 1]),
                                                    d, 0, 0, 0);
    return d;
}

// Activation rows p0 .. p0 + rows (<= 16) of expert weights w against weight
// rows 16 * tile ..: a wave, both sides straight from memory.
__device__ inline void plain_tile(const F8Args &a, const uint8_t *w, const float *ws,
                                  uint64_t tile, uint64_t p0, uint32_t rows) {
    const uint32_t lane = threadIdx.x & 63u, m = lane & 15u, g = lane >> 4;
    const uint32_t nb = f8_blocks(a.cols);
    const uint64_t p = p0 + min(m, rows - 1);
    int64_t xr = a.act ? (int64_t)a.act[p] : (int64_t)((uint32_t)p / a.x_div);
    if (xr >= (int64_t)a.xrows) xr = -1;
    const uint64_t xrow = (uint64_t)max(xr, (int64_t)0);
    const uint8_t *wp = w + min(tile * 16 + m, a.w_rows - 1) * (128ull * nb) + 16 * g;
    const float *wsp = ws + tile / 8 * nb;
    const uint8_t *xp = (const uint8_t *)a.x + xrow * (128ull * nb) + 16 * g;
    v4f acc = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t b = 0; b < nb; b++) {
        const v8i wq = join(*(const u32x4 *)(wp + 128ull * b), *(const u32x4 *)(wp + 128ull * b + 64));
        v8i xq;
        float s;
        if (a.x_type == kTypeF8) {
            xq = join(*(const u32x4 *)(xp + 128ull * b), *(const u32x4 *)(xp + 128ull * b + 64));
            s = a.xs[xrow * nb + b];
        } else {
            float v[32];
#pragma unroll
            for (uint32_t i = 0; i < 32; i += 8)
                load_row8(a.x, a.x_type, xrow * a.ldx, 128 * b + 64 * (i / 16) + 16 * g + i % 16,
                          (uint32_t)a.cols, v + i);
            uint32_t top = f8_top<32>(v), q[8];
            top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
            top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
            const uint32_t bits = f8_scale_of(top);
            f8_pack<32>(v, bits, q);
#pragma unroll
            for (int i = 0; i < 8; i++) xq[i] = (int)q[i];
            s = bits_f32(bits);
        }
        s *= wsp[b];
        const v4f d = block_sums(wq, xq);
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] = fmaf(d[i], s, acc[i]);
    }
    if (m >= rows || xr < 0) return;
    const uint64_t r = tile * 16 + 4 * g, at = p * a.ldy + r;
    if (r + 4 <= a.w_rows)
        store4(a.y, a.y_type, at, acc);
    else
        for (uint32_t k = 0; k < 4; k++)
            if (r + k < a.w_rows) store_from_f32(a.y, a.y_type, at + k, acc[k]);
}

}  // namespace

// Dense: grid (weight tiles / 4, sets of 16 activation rows).
__global__ __launch_bounds__(256) void f8_dense_k(F8Args a) {
    const uint64_t tile = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint64_t p0 = (uint64_t)blockIdx.y * 16;
    if (tile * 16 >= a.w_rows) return;
    plain_tile(a, a.w, a.ws, tile, p0, (uint32_t)min((uint64_t)16, a.n - p0));
}

// Listed rows: grid (weight tiles / 4, rows).
__global__ __launch_bounds__(256) void f8_sel_k(F8Args a) {
    const uint64_t tile = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int32_t e = a.eid[blockIdx.y];
    if (tile * 16 >= a.w_rows || e < 0 || (uint32_t)e >= a.n_expert) return;
    plain_tile(a, a.w + e * a.w_stride, (const float *)((const uint8_t *)a.ws + e * a.ws_stride),
               tile, blockIdx.y, 1);
}

// Packed rows: grid (weight tiles / 4, an upper bound of the experts' sets of 16).
__global__ __launch_bounds__(256) void f8_id_k(F8Args a) {
    const uint64_t tile = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (tile * 16 >= a.w_rows) return;
    const int64_t end = (int64_t)(a.act ? a.n : min(a.n, a.xrows));
    uint32_t set = blockIdx.y;
    for (uint32_t e = 0; e < a.n_expert; e++) {
        const int64_t lo = max(a.bounds[e], 0), hi = min((int64_t)a.bounds[e + 1], end);
        const uint32_t sets = hi > lo ? (uint32_t)((hi - lo + 15) / 16) : 0u;
        if (set < sets) {
            const int64_t p0 = lo + 16 * (int64_t)set;
            plain_tile(a, a.w + e * a.w_stride,
                       (const float *)((const uint8_t *)a.ws + e * a.ws_stride), tile,
                       (uint64_t)p0, (uint32_t)min((int64_t)16, hi - p0));
            return;
        }
        set -= sets;
    }
}

namespace {

// rows: whether the call has any; without, their pointers may be NULL.
bool mul_ok(const char *who, const F8Args &a, bool rows) {
    if (!a.w || !a.ws || (rows && (!a.x || !a.y)) || !a.w_rows || !a.cols) {
        set_error("%s: bad arguments", who);
        return false;
    }
    if (a.cols > (1u << 24) || a.w_rows > (1u << 30) || a.n > (1u << 30)) {
        set_error("%s: sizes not covered (cols <= 2^24, rows <= 2^30)", who);
        return false;
    }
    if (!is_float_type(a.y_type) || (a.x_type != kTypeF8 && !is_float_type(a.x_type))) {
        set_error("%s: types %u -> %u not covered (F32, F16, BF16; inputs also 248)", who,
                  a.x_type, a.y_type);
        return false;
    }
    if (a.x_type == kTypeF8 ? (rows && !a.xs) || ((uintptr_t)a.x & 15) || ((uintptr_t)a.xs & 3)
                            : a.xs || a.ldx < a.cols ||
                                  ((uintptr_t)a.x & (type_bytes(a.x_type) - 1))) {
        set_error("%s: 8-bit inputs need scales, codes aligned to 16 bytes and scales to 4; float "
                  "inputs no scales, their type's alignment and a row stride of at least cols",
                  who);
        return false;
    }
    if (((uintptr_t)a.w & 15) || ((uintptr_t)a.ws & 3) || a.w_stride % 16 || a.ws_stride % 4) {
        set_error("%s: weight codes must be 16-byte and scales 4-byte aligned", who);
        return false;
    }
    if (a.ldy < a.w_rows || ((uintptr_t)a.y & (type_bytes(a.y_type) - 1))) {
        set_error("%s: output stride below its row, or output not aligned to its type", who);
        return false;
    }
    return true;
}

constexpr uint64_t kFloatRows = 16;     // float rows that q4mi_f8_mul takes
constexpr uint32_t kIdExperts = 1024;

uint32_t tiles4(const F8Args &a) { return (uint32_t)((a.w_rows + 63) / 64); }

}  // namespace

extern "C" {

/* y = X . W^T (see include/q4mi.h). */
bool q4mi_f8_mul(const uint8_t *d_w, const float *d_ws, uint64_t w_rows, uint64_t cols,
                 const void *d_x, const float *d_xs, uint32_t x_type, uint64_t ld_x, uint64_t n,
                 void *d_y, uint32_t y_type, uint64_t ld_y) {
    F8Args a = {};
    a.w = d_w, a.ws = d_ws, a.w_rows = w_rows, a.cols = cols;
    a.x = d_x, a.xs = d_xs, a.x_type = x_type, a.ldx = ld_x, a.n = a.xrows = n, a.x_div = 1;
    a.y = d_y, a.y_type = y_type, a.ldy = ld_y;
    if (!mul_ok("q4mi_f8_mul", a, n > 0)) return false;
    if (x_type != kTypeF8 && n > kFloatRows) {
        set_error("q4mi_f8_mul: %llu float rows not covered (<= %llu; quantise them first)",
                  (unsigned long long)n, (unsigned long long)kFloatRows);
        return false;
    }
    if (!n) return true;
    if (n > 16 * 65535) {
        set_error("q4mi_f8_mul: too many tiles");
        return false;
    }
    f8_dense_k<<<dim3(tiles4(a), (uint32_t)((n + 15) / 16)), dim3(256), 0, stream()>>>(a);
    return launch_ok("f8_dense_k");
}

/* Every row through its own expert (see include/q4mi.h). */
bool q4mi_f8_mul_sel(const uint8_t *d_w, const float *d_ws, uint64_t w_rows, uint64_t cols,
                     uint64_t w_stride, uint64_t ws_stride, uint32_t n_expert, const void *d_x,
                     const float *d_xs, uint32_t x_type, uint64_t ld_x, uint32_t x_div,
                     const int32_t *d_eid, uint64_t n, void *d_y, uint32_t y_type, uint64_t ld_y) {
    F8Args a = {};
    a.w = d_w, a.ws = d_ws, a.w_rows = w_rows, a.cols = cols;
    a.w_stride = w_stride, a.ws_stride = ws_stride, a.n_expert = n_expert;
    a.x = d_x, a.xs = d_xs, a.x_type = x_type, a.ldx = ld_x, a.x_div = x_div, a.eid = d_eid;
    a.n = a.xrows = n, a.y = d_y, a.y_type = y_type, a.ldy = ld_y;
    if (!mul_ok("q4mi_f8_mul_sel", a, n > 0)) return false;
    if ((n && !d_eid) || !n_expert || !x_div || n > 65535) {
        set_error("q4mi_f8_mul_sel: needs a list, experts, x_div >= 1 and at most 65535 rows");
        return false;
    }
    if (!n) return true;
    f8_sel_k<<<dim3(tiles4(a), (uint32_t)n), dim3(256), 0, stream()>>>(a);
    return launch_ok("f8_sel_k");
}

/* Packed rows, each expert's in one stretch (see include/q4mi.h). */
bool q4mi_f8_mul_id(const uint8_t *d_w, const float *d_ws, uint64_t w_rows, uint64_t cols,
                    uint64_t w_stride, uint64_t ws_stride, uint32_t n_expert, const uint8_t *d_xq,
                    const float *d_xs, uint64_t xrows, const int32_t *d_act_row,
                    const int32_t *d_bounds, uint64_t total_rows, void *d_y, uint32_t y_type,
                    uint64_t ld_y) {
    F8Args a = {};
    a.w = d_w, a.ws = d_ws, a.w_rows = w_rows, a.cols = cols;
    a.w_stride = w_stride, a.ws_stride = ws_stride, a.n_expert = n_expert;
    a.x = d_xq, a.xs = d_xs, a.x_type = kTypeF8, a.xrows = xrows, a.act = d_act_row, a.x_div = 1;
    a.bounds = d_bounds, a.n = total_rows, a.y = d_y, a.y_type = y_type, a.ldy = ld_y;
    if (!mul_ok("q4mi_f8_mul_id", a, total_rows && xrows)) return false;
    if (!d_bounds || !n_expert || n_expert > kIdExperts) {
        set_error("q4mi_f8_mul_id: needs bounds of 1 to %u experts", kIdExperts);
        return false;
    }
    if (!total_rows || !xrows) return true;
    if (total_rows > 16 * 64000) {
        set_error("q4mi_f8_mul_id: too many tiles");
        return false;
    }
    f8_id_k<<<dim3(tiles4(a), (uint32_t)(total_rows / 16 + n_expert)), dim3(256), 0, stream()>>>(a);
    return launch_ok("f8_id_k");
}

}  // extern "C"

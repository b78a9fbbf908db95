// Products of microscaled 4-bit rows (mx4.h has the format):
//   y[t][r] = sum over blocks b of 2^(sw + sx - 254) * sum_i w[r][32b+i] x[t][32b+i]
// on v_mfma_scale_f32_16x16x128_f8f6f4, whose lane (row m, group g) takes one
// block of 32 codes and its scale byte, and which adds in fp32.
#include "mx4.h"
#include "q4mi_internal.h"

using namespace q4mi;

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

struct MulArgs {
    const uint8_t *w, *ws;          // weights: codes, scales
    const void *x;                  // activations: codes, or float rows
    const uint8_t *xs;              // scales of codes
    const int32_t *act, *bounds;    // packed rows: their activation rows, each expert's stretch
    const int32_t *eid;             // listed rows: their experts
    void *y;
    uint64_t w_rows, cols, w_stride, ws_stride, ldx, xrows, n, ldy;
    uint32_t n_expert, x_type, y_type, x_div;
};

__device__ inline v8i widen(uint4 q) {
    v8i a = {(int)q.x, (int)q.y, (int)q.z, (int)q.w, 0, 0, 0, 0};
    return a;
}

// Block kb of a float row as codes and scale.
__device__ inline uint4 quant_block(const void *x, uint32_t xt, uint64_t at, uint32_t left,
                                    uint32_t *s) {
    float v[32];
    uint32_t top = 0;
#pragma unroll
    for (uint32_t i = 0; i < 32; i++) {
        v[i] = i < left ? load_as_f32(x, xt, at + i) : 0.f;
        top = max(top, f32_bits(v[i]) & 0x7fffffffu);
    }
    *s = mx4_scale_of(top);
    return make_uint4(mx4_pack8(v, *s), mx4_pack8(v + 8, *s), mx4_pack8(v + 16, *s),
                      mx4_pack8(v + 24, *s));
}

// One wave: 16 weight rows from r0 against up to 16 activation rows; lane
// l holds activation row l % 16 (xr, or -1 for none) and output row yr.
__device__ inline void wave_tile(const MulArgs &a, const uint8_t *w, const uint8_t *ws,
                                 uint64_t r0, int64_t xr, int64_t yr) {
    const uint32_t lane = threadIdx.x & 63u, m = lane & 15u, g = lane >> 4;
    const uint32_t nb = mx4_blocks(a.cols), sld = mx4_scale_row(nb);
    const uint64_t wr = min(r0 + m, a.w_rows - 1);
    v4f acc = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t b0 = 0; b0 < nb; b0 += 4) {
        const uint32_t b = b0 + g;
        uint4 wq = make_uint4(0, 0, 0, 0), xq = wq;
        uint32_t wsc = 127, xsc = 127;
        if (b < nb) {
            wq = *(const uint4 *)(w + wr * (16ull * nb) + 16u * b);
            wsc = ws[wr * sld + b];
            if (xr >= 0) {
                if (a.x_type == kTypeMx4) {
                    xq = *(const uint4 *)((const uint8_t *)a.x + xr * (16ull * nb) + 16u * b);
                    xsc = a.xs[xr * (uint64_t)sld + b];
                } else {
                    const uint32_t left = (uint32_t)min((uint64_t)32, a.cols - 32ull * b);
                    xq = quant_block(a.x, a.x_type, xr * a.ldx + 32ull * b, left, &xsc);
                }
            }
        }
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(widen(wq), widen(xq), acc, 4, 4, 0,
                                                               (int)wsc, 0, (int)xsc);
    }
    if (yr < 0) return;
    for (uint32_t i = 0; i < 4; i++) {
        const uint64_t r = r0 + 4 * g + i;
        if (r < a.w_rows) store_from_f32(a.y, a.y_type, yr * a.ldy + r, acc[i]);
    }
}

// grid (16-row tiles / 4, 16-row tiles of activations)
__global__ __launch_bounds__(256) void mx4_dense_k(MulArgs a) {
    const uint64_t r0 = ((uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 16;
    if (r0 >= a.w_rows) return;
    const uint64_t t = (uint64_t)blockIdx.y * 16 + (threadIdx.x & 15u);
    const int64_t row = t < a.n ? (int64_t)t : -1;
    wave_tile(a, a.w, a.ws, r0, row, row);
}

// grid (16-row tiles / 4, rows)
__global__ __launch_bounds__(256) void mx4_sel_k(MulArgs a) {
    const uint64_t r0 = ((uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 16;
    if (r0 >= a.w_rows) return;
    const uint64_t p = blockIdx.y;
    const int32_t e = a.eid[p];
    if (e < 0 || (uint32_t)e >= a.n_expert) return;
    const bool me = (threadIdx.x & 15u) == 0;
    wave_tile(a, a.w + e * a.w_stride, a.ws + e * a.ws_stride, r0, me ? (int64_t)(p / a.x_div) : -1,
              me ? (int64_t)p : -1);
}

// grid (16-row tiles / 4, experts): every 16 packed rows of the expert
__global__ __launch_bounds__(256) void mx4_id_k(MulArgs a) {
    const uint64_t r0 = ((uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 16;
    if (r0 >= a.w_rows) return;
    const uint32_t e = blockIdx.y;
    const int64_t lo = max(a.bounds[e], 0), hi = min((int64_t)a.bounds[e + 1], (int64_t)a.n);
    for (int64_t p0 = lo; p0 < hi; p0 += 16) {
        const int64_t p = p0 + (threadIdx.x & 15u);
        int64_t xr = -1;
        if (p < hi) xr = a.act ? (int64_t)a.act[p] : p;
        if (xr >= (int64_t)a.xrows) xr = -1;
        wave_tile(a, a.w + e * a.w_stride, a.ws + e * a.ws_stride, r0, xr, xr < 0 ? -1 : p);
    }
}

bool mul_ok(const char *who, const MulArgs &a) {
    if (!a.w || !a.ws || !a.x || !a.y || !a.w_rows || !a.cols) {
        set_error("%s: bad arguments", who);
        return false;
    }
    if (a.cols > (1u << 24) || a.w_rows > (1u << 30) || a.n > (1u << 30)) {
        set_error("%s: sizes not covered (cols <= 2^24, rows <= 2^30)", who);
        return false;
    }
    if (!is_float_type(a.y_type) || (a.x_type != kTypeMx4 && !is_float_type(a.x_type))) {
        set_error("%s: types %u -> %u not covered (F32, F16, BF16; inputs also MXFP4)", who,
                  a.x_type, a.y_type);
        return false;
    }
    if (a.x_type == kTypeMx4 ? !a.xs || ((uintptr_t)a.x & 15) || ((uintptr_t)a.xs & 3)
                             : a.xs || a.ldx < a.cols ||
                                   ((uintptr_t)a.x & (type_bytes(a.x_type) - 1))) {
        set_error("%s: 4-bit inputs need scales, codes aligned to 16 bytes and scales to 4; float "
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

constexpr uint64_t kFloatRows = 8;   // float rows that q4mi_mx4_mul takes

}  // namespace

extern "C" {

/* y = X . W^T (see include/q4mi.h). */
bool q4mi_mx4_mul(const uint8_t *d_w, const uint8_t *d_ws, uint64_t w_rows, uint64_t cols,
                  const void *d_x, const uint8_t *d_xs, uint32_t x_type, uint64_t ld_x, uint64_t n,
                  void *d_y, uint32_t y_type, uint64_t ld_y) {
    MulArgs a = {};
    a.w = d_w, a.ws = d_ws, a.w_rows = w_rows, a.cols = cols;
    a.x = d_x, a.xs = d_xs, a.x_type = x_type, a.ldx = ld_x, a.n = a.xrows = n;
    a.y = d_y, a.y_type = y_type, a.ldy = ld_y;
    if (!mul_ok("q4mi_mx4_mul", a)) return false;
    if (x_type != kTypeMx4 && n > kFloatRows) {
        set_error("q4mi_mx4_mul: %llu float rows not covered (<= %llu; quantise them first)",
                  (unsigned long long)n, (unsigned long long)kFloatRows);
        return false;
    }
    if (!n) return true;
    mx4_dense_k<<<dim3((uint32_t)((w_rows + 63) / 64), (uint32_t)((n + 15) / 16)), dim3(256), 0,
                  stream()>>>(a);
    return launch_ok("mx4_dense_k");
}

/* Every row through its own expert (see include/q4mi.h). */
bool q4mi_mx4_mul_sel(const uint8_t *d_w, const uint8_t *d_ws, uint64_t w_rows, uint64_t cols,
                      uint64_t w_stride, uint64_t ws_stride, uint32_t n_expert, const void *d_x,
                      const uint8_t *d_xs, uint32_t x_type, uint64_t ld_x, uint32_t x_div,
                      const int32_t *d_eid, uint64_t n, void *d_y, uint32_t y_type, uint64_t ld_y) {
    MulArgs a = {};
    a.w = d_w, a.ws = d_ws, a.w_rows = w_rows, a.cols = cols;
    a.w_stride = w_stride, a.ws_stride = ws_stride, a.n_expert = n_expert;
    a.x = d_x, a.xs = d_xs, a.x_type = x_type, a.ldx = ld_x, a.x_div = x_div, a.eid = d_eid;
    a.n = n, a.y = d_y, a.y_type = y_type, a.ldy = ld_y;
    if (!mul_ok("q4mi_mx4_mul_sel", a)) return false;
    if (!d_eid || !n_expert || !x_div || n > 65535) {
        set_error("q4mi_mx4_mul_sel: needs a list, experts, x_div >= 1 and at most 65535 rows");
        return false;
    }
    if (!n) return true;
    mx4_sel_k<<<dim3((uint32_t)((w_rows + 63) / 64), (uint32_t)n), dim3(256), 0, stream()>>>(a);
    return launch_ok("mx4_sel_k");
}

/* Packed rows, each expert's in one stretch (see include/q4mi.h). */
bool q4mi_mx4_mul_id(const uint8_t *d_w, const uint8_t *d_ws, uint64_t w_rows, uint64_t cols,
                     uint64_t w_stride, uint64_t ws_stride, uint32_t n_expert, const uint8_t *d_xq,
                     const uint8_t *d_xs, uint64_t xrows, const int32_t *d_act_row,
                     const int32_t *d_bounds, uint64_t total_rows, void *d_y, uint32_t y_type,
                     uint64_t ld_y) {
    MulArgs a = {};
    a.w = d_w, a.ws = d_ws, a.w_rows = w_rows, a.cols = cols;
    a.w_stride = w_stride, a.ws_stride = ws_stride, a.n_expert = n_expert;
    a.x = d_xq, a.xs = d_xs, a.x_type = kTypeMx4, a.xrows = xrows, a.act = d_act_row;
    a.bounds = d_bounds, a.n = total_rows, a.y = d_y, a.y_type = y_type, a.ldy = ld_y;
    if (!mul_ok("q4mi_mx4_mul_id", a)) return false;
    if (!d_bounds || !n_expert || n_expert > 65535) {
        set_error("q4mi_mx4_mul_id: needs bounds of 1 to 65535 experts");
        return false;
    }
    if (!total_rows || !xrows) return true;
    mx4_id_k<<<dim3((uint32_t)((w_rows + 63) / 64), n_expert), dim3(256), 0, stream()>>>(a);
    return launch_ok("mx4_id_k");
}

}  // extern "C"

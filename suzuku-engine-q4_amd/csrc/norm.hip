// Root-mean-square norm of rows, with the residual's addition ahead of it and
// float and 8-bit outputs:
//   h = x + res, rounded to the residual's type (what the next layer reads is
//       what is normed); without residual and sum h = x
//   i = 1 / sqrt(sum h^2 / cols + eps), the sum in 64 bits, rounded to fp32
//   y = (h * i) * w in fp32
// The 64-bit sum (squares are exact, two instructions a value in a kernel that
// memory bounds) makes i the same for every order of the sum, but where it lies
// within 2^-52 of a border, and with it y and its 8-bit codes, bit for bit.
#include <algorithm>

#include "f8.h"
#include "q4mi_common.h"
#include "q4mi_internal.h"

using namespace q4mi;

namespace {

struct NormArgs {
    const void *x, *res, *w;
    void *sum, *y;
    uint8_t *codes;
    float *scales;
    uint64_t ldx, ldr, ldy, rows;
    uint32_t cols, lanes, x_type, r_type, w_type, y_type, q_type;
    float eps;
};

__device__ inline float round_to(float v, uint32_t t) {
    if (t == kTypeF32) return v;
    const uint32_t b = f32_to_16(v, t);
    return t == kTypeF16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)b) : bits_f32(b << 16);
}

// Eight values of a float row from column c0 on.
__device__ inline void store_row8(void *p, uint32_t t, uint64_t row, uint32_t c0, uint32_t cols,
                                  const float *v) {
    const uint64_t at = row + c0;
    if (c0 + 8 <= cols) {
        if (t == kTypeF32) {
            *(f32x4_a4 *)((float *)p + at) = (f32x4){v[0], v[1], v[2], v[3]};
            *(f32x4_a4 *)((float *)p + at + 4) = (f32x4){v[4], v[5], v[6], v[7]};
        } else {
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = f32_to_16x2(v[2 * i], v[2 * i + 1], t);
            *(u32x4_a2 *)((uint16_t *)p + at) = w;
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; i++)
            if (c0 + i < cols) store_from_f32(p, t, at + i, v[i]);
    }
}

// A lane's eight columns of x and of the residual.
template <uint32_t XB, uint32_t RB>
struct NormIn {
    Raw8<XB> x;
    Raw8<RB> r;
    __device__ void load(const NormArgs &a, uint64_t row, uint32_t c0) {
        load_raw8<XB>(a.x, row * a.ldx, c0, a.cols, x);
        if (a.res) load_raw8<RB>(a.res, row * a.ldr, c0, a.cols, r);
    }
    __device__ void h(const NormArgs &a, float *v) const {
        raw8_to_f32<XB>(x, a.x_type, v);
        if (a.res) {
            float u[8];
            raw8_to_f32<RB>(r, a.r_type, u);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] += u[i];
        }
        if (RB == 2 && (a.res || a.sum)) {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = round_to(v[i], a.r_type);
        }
    }
};

// Outputs of eight columns of row r from y; every lane of the wave is here.
__device__ inline void norm_out(const NormArgs &a, uint64_t r, uint32_t c0, const float *y) {
    if (a.y && c0 < a.cols) store_row8(a.y, a.y_type, r * a.ldy, c0, a.cols, y);
    if (!a.codes) return;
    if (a.q_type == kTypeF8) {
        // sixteen lanes a block of 128
        const uint32_t nb = f8_blocks(a.cols);
        const uint32_t s = f8_scale_of(f8_max_lanes<16>(f8_top<8>(y)));
        uint32_t q[2];
        f8_pack<8>(y, s, q);
        if (c0 >= 128 * nb) return;
        *(u32x2 *)(a.codes + r * (128ull * nb) + c0) = (u32x2){q[0], q[1]};
        if (c0 % 128 == 0) a.scales[r * nb + c0 / 128] = bits_f32(s);
    } else {
        // four lanes a group of 32
        float d;
        const uint2 q = q4mi_quant_team4(make_float4(y[0], y[1], y[2], y[3]),
                                         make_float4(y[4], y[5], y[6], y[7]), &d);
        if (c0 >= a.cols) return;
        *(u32x2 *)(a.codes + r * a.cols + c0) = (u32x2){q.x, q.y};
        if (c0 % 32 == 0) a.scales[r * (a.cols / 32) + c0 / 32] = d;
    }
}

}  // namespace

constexpr uint32_t kNormGridX = 1u << 20;   // fewer than 2^32 threads along x

// a.lanes lanes a row (64: four rows a workgroup, else the workgroup), I chunks of
// eight columns a lane in registers (lane l has chunks l, l + lanes, ..); I = 0: any
// length, h read again after the sum.  XB, RB: bytes of x's values and the
// residual's.
template <uint32_t I, uint32_t XB, uint32_t RB>
__global__ __launch_bounds__(I == 1 ? 256 : 1024) void rms_norm_k(NormArgs a) {
    const uint32_t L = a.lanes, nw = L / 64;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint64_t block = (uint64_t)blockIdx.y * kNormGridX + blockIdx.x;
    const uint64_t r = nw == 1 ? block * 4 + wave : block;
    if (r >= a.rows) return;    // whole waves; with more than one a row the whole workgroup
    const uint32_t l = nw == 1 ? threadIdx.x & 63u : threadIdx.x;
    float v[I ? I : 1][8], w[I ? I : 1][8];
    double sum = 0.;
    auto add = [&](const float *h) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 8; i++) sum = fma((double)h[i], (double)h[i], sum);
    };
    auto weights = [&](uint32_t c0, float *u) __attribute__((always_inline)) {
        if (a.w && c0 < a.cols) {
            load_row8(a.w, a.w_type, 0, c0, a.cols, u);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) u[i] = 1.f;
        }
    };
    NormIn<XB, RB> in[I ? I : 1];
    if constexpr (I > 0) {
#pragma unroll
        for (uint32_t i = 0; i < I; i++) in[i].load(a, r, 8 * (l + L * i));
#pragma unroll
        for (uint32_t i = 0; i < I; i++) weights(8 * (l + L * i), w[i]);
#pragma unroll
        for (uint32_t i = 0; i < I; i++) {
            in[i].h(a, v[i]);
            add(v[i]);
        }
    } else {
        for (uint32_t c0 = 8 * l; c0 < a.cols; c0 += 8 * L) {
            in[0].load(a, r, c0);
            in[0].h(a, v[0]);
            add(v[0]);
        }
    }
    sum = q4mi_rsum<64>(sum);       // the wave's total, in its last lane
    const uint64_t bits = __builtin_bit_cast(uint64_t, sum);
    sum = __builtin_bit_cast(
        double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(bits >> 32), 63) << 32 |
                    (uint32_t)__builtin_amdgcn_readlane((int)bits, 63));
    if (nw > 1) {
        __shared__ double part[16];
        if ((threadIdx.x & 63u) == 0) part[wave] = sum;
        __syncthreads();
        sum = 0.;
        for (uint32_t k = 0; k < nw; k += 4) {      // four reads at once; past nw is nothing
            double p[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) p[i] = part[k + i];
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) sum += k + i < nw ? p[i] : 0.;
        }
    }
    const float inv = (float)(1. / sqrt(sum / (double)a.cols + (double)a.eps));
    auto out = [&](uint32_t c0, float *h, const float *u) __attribute__((always_inline)) {
        if (a.sum && c0 < a.cols) store_row8(a.sum, a.r_type, r * a.ldr, c0, a.cols, h);
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = h[i] * inv * u[i];
        norm_out(a, r, c0, h);
    };
    if constexpr (I > 0) {
#pragma unroll
        for (uint32_t i = 0; i < I; i++)
            if (8 * L * i < a.cols) out(8 * (l + L * i), v[i], w[i]);
    } else {
        // whole waves to the end of the last block
        for (uint32_t c0 = 8 * l; c0 - 8 * (l & 63u) < a.cols; c0 += 8 * L) {
            in[0].load(a, r, c0);
            in[0].h(a, v[0]);
            weights(c0, w[0]);
            out(c0, v[0], w[0]);
        }
    }
}

namespace {

bool norm_ok(const NormArgs &a, uint64_t cols) {
    const char *who = "q4mi_rms_norm";
    if ((a.rows && (!a.x || (!a.y && !a.codes) || !a.codes != !a.scales)) || !cols) {
        set_error("%s: bad arguments (needs y, or codes with scales)", who);
        return false;
    }
    if (!is_float_type(a.x_type) || ((a.res || a.sum) && !is_float_type(a.r_type)) ||
        (a.w && !is_float_type(a.w_type)) || (a.y && !is_float_type(a.y_type))) {
        set_error("%s: types not covered (F32, F16, BF16)", who);
        return false;
    }
    if (a.codes && a.q_type != kTypeF8 && a.q_type != Q4MI_T_Q8_0) {
        set_error("%s: 8-bit type %u not covered (8, 248)", who, a.q_type);
        return false;
    }
    if (cols > (1u << 24) || a.rows >= (1ull << 30)) {
        set_error("%s: %llu x %llu too large", who, (unsigned long long)a.rows,
                  (unsigned long long)cols);
        return false;
    }
    if (a.codes && a.q_type == Q4MI_T_Q8_0 && cols % 32) {
        set_error("%s: groups of 32 need whole groups a row", who);
        return false;
    }
    if (!(a.eps >= 0.f) || a.eps > 3e38f) {
        set_error("%s: eps must be finite and not negative", who);
        return false;
    }
    if (a.ldx < cols || ((a.res || a.sum) && a.ldr < cols) || (a.y && a.ldy < cols)) {
        set_error("%s: row stride below its columns", who);
        return false;
    }
    auto off = [](const void *p, uint32_t t) { return ((uintptr_t)p & (type_bytes(t) - 1)) != 0; };
    if (off(a.x, a.x_type) || off(a.res, a.r_type) || off(a.sum, a.r_type) || off(a.w, a.w_type) ||
        off(a.y, a.y_type) || ((uintptr_t)a.codes & 15) || ((uintptr_t)a.scales & 3)) {
        set_error("%s: rows must be aligned to their type, codes to 16 bytes, scales to 4", who);
        return false;
    }
    return true;
}

// As many waves a row as its chunks need, I a lane: one up to 2048 columns, then two,
// as four waves' loads already cover memory's latency (bf16 with residual, 8 bits out,
// 33.5 M values, us: 8192 x 4096 47, 46 with one; 6990 x 4800 58, 90 with four a lane
// in 256; 4096 x 8192 49 and 59; 32768 x 1024 49, 70 with 256 lanes).  Memory bounds
// it: 4 to 5.5 TB/s.
template <uint32_t I>
bool norm_launch(NormArgs &a) {
    const uint32_t chunks = (a.cols + 7) / 8;
    const uint32_t waves = I ? (chunks + 64 * I - 1) / (64 * I) : 16;
    a.lanes = 64 * waves;
    const uint64_t per = a.lanes == 64 ? 4 : 1, blocks = (a.rows + per - 1) / per;
    const dim3 grid((uint32_t)std::min<uint64_t>(blocks, kNormGridX),
                    (uint32_t)((blocks + kNormGridX - 1) / kNormGridX));
    const bool x4 = a.x_type == kTypeF32, r4 = !(a.res || a.sum) || a.r_type == kTypeF32;
    auto k = x4 ? (r4 ? rms_norm_k<I, 4, 4> : rms_norm_k<I, 4, 2>)
                : (r4 ? rms_norm_k<I, 2, 4> : rms_norm_k<I, 2, 2>);
    k<<<grid, dim3(a.lanes * (uint32_t)per), 0, stream()>>>(a);
    return launch_ok("rms_norm_k");
}

}  // namespace

extern "C" {

/* Root-mean-square norm (see include/q4mi.h). */
bool q4mi_rms_norm(const void *d_x, uint32_t x_type, uint64_t ld_x, const void *d_res, void *d_sum,
                   uint32_t r_type, uint64_t ld_r, const void *d_w, uint32_t w_type, float eps,
                   uint64_t rows, uint64_t cols, void *d_y, uint32_t y_type, uint64_t ld_y,
                   uint32_t q_type, void *d_codes, float *d_scales) {
    NormArgs a = {d_x, d_res, d_w, d_sum, d_y, (uint8_t *)d_codes, d_scales, ld_x, ld_r, ld_y,
                  rows, (uint32_t)cols, 0, x_type, r_type, w_type, y_type, q_type, eps};
    if (!norm_ok(a, cols)) return false;
    if (!rows) return true;
    if (cols <= 2048) return norm_launch<1>(a);
    if (cols <= 16384) return norm_launch<2>(a);
    if (cols <= 32768) return norm_launch<4>(a);
    return norm_launch<0>(a);
}

}  // extern "C"

// Float rows to 8-bit floating point in blocks of 128 and back (f8.h has the
// format).
#include <algorithm>

#include "f8.h"
#include "q4mi_internal.h"

using namespace q4mi;

namespace {

// Place of block `i` among a group of whole rows with fewer than 2^28 blocks, in
// row-major order (32-bit divisions); workgroups with one blockIdx.y share a
// group.
struct F8Place {
    uint64_t r;
    uint32_t b;
    __device__ F8Place(uint32_t i, uint64_t group, uint64_t rows, uint32_t nb) {
        const uint32_t in = i / nb;
        b = i - in * nb;
        r = in < group ? blockIdx.y * group + in : rows;
    }
};

}  // namespace

// A scale for each 128 values of a row: N values a lane (32 bytes of input:
// eight fp32, sixteen 16-bit), 128 / N lanes a block.  Memory bounds it: 8192 x
// 8192 bf16 38 us, 5.3 TB/s.
template <uint32_t N>
__global__ __launch_bounds__(256) void f8_quant_k(const void *__restrict__ x, uint32_t xt,
                                                  uint64_t ld, const int32_t *__restrict__ ids,
                                                  uint64_t rows, uint64_t group, uint32_t cols,
                                                  uint8_t *__restrict__ codes,
                                                  float *__restrict__ scales) {
    constexpr uint32_t L = 128 / N;
    const uint32_t nb = f8_blocks(cols), sub = threadIdx.x % L;
    const F8Place p(blockIdx.x * (256 / L) + threadIdx.x / L, group, rows, nb);
    if (p.r >= rows) return;    // whole groups of L lanes
    const uint64_t src = ids ? (uint64_t)(int64_t)ids[p.r] : p.r;
    float v[N];
#pragma unroll
    for (uint32_t i = 0; i < N; i += 8)
        load_row8(x, xt, src * ld, p.b * 128 + sub * N + i, cols, v + i);
    const uint32_t s = f8_scale_of(f8_max_lanes<L>(f8_top<N>(v)));
    uint32_t q[N / 4];
    f8_pack<N>(v, s, q);
    uint8_t *c = codes + p.r * (128ull * nb) + p.b * 128u + sub * N;
    if constexpr (N == 16)
        *(u32x4 *)c = (u32x4){q[0], q[1], q[2], q[3]};
    else
        *(u32x2 *)c = (u32x2){q[0], q[1]};
    if (sub == 0) scales[p.r * nb + p.b] = bits_f32(s);
}

// A scale for each 128 x 128 values: one workgroup a block, sixteen lanes a
// row of it with eight values each, so sixteen rows a step and eight steps,
// whose values stay in registers until the block's largest is known.  XB: bytes of
// a value; all loads go out before the first is converted (16384 x 4096 bf16 37
// us, 5.4 TB/s; 52 us when each step's values were converted first).
template <uint32_t XB>
__global__ __launch_bounds__(256) void f8_quant_blocks_k(const void *__restrict__ x, uint32_t xt,
                                                         uint64_t ld,
                                                         const int32_t *__restrict__ ids,
                                                         uint64_t rows, uint64_t group,
                                                         uint32_t cols,
                                                         uint8_t *__restrict__ codes,
                                                         float *__restrict__ scales) {
    __shared__ uint32_t tops[4];
    const uint32_t nb = f8_blocks(cols), sub = threadIdx.x & 15u;
    const uint64_t rb = (rows + 127) / 128;
    const F8Place p(blockIdx.x, group, rb, nb);
    if (p.r >= rb) return;      // the whole workgroup
    Raw8<XB> raw[8];
    float v[8][8];
    uint32_t top = 0;
#pragma unroll
    for (uint32_t i = 0; i < 8; i++) {
        const uint64_t r = p.r * 128 + i * 16 + (threadIdx.x >> 4);
        const uint64_t src = ids && r < rows ? (uint64_t)(int64_t)ids[r] : r;
        // rows past the last have no values
        load_raw8<XB>(x, src * ld, p.b * 128 + sub * 8, r < rows ? cols : 0u, raw[i]);
    }
#pragma unroll
    for (uint32_t i = 0; i < 8; i++) {
        raw8_to_f32<XB>(raw[i], xt, v[i]);
        top = max(top, f8_top<8>(v[i]));
    }
    top = f8_max_lanes<16>(top);
    top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
    top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
    if ((threadIdx.x & 63u) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    const uint32_t s = f8_scale_of(max(max(tops[0], tops[1]), max(tops[2], tops[3])));
#pragma unroll
    for (uint32_t i = 0; i < 8; i++) {
        const uint64_t r = p.r * 128 + i * 16 + (threadIdx.x >> 4);
        if (r >= rows) continue;
        uint32_t q[2];
        f8_pack<8>(v[i], s, q);
        *(u32x2 *)(codes + r * (128ull * nb) + p.b * 128u + sub * 8) = (u32x2){q[0], q[1]};
    }
    if (threadIdx.x == 0) scales[p.r * nb + p.b] = bits_f32(s);
}

// The mirror, G values a lane, so that a lane's values are 16 bytes of output
// and a wave's one stretch: eight for 16-bit outputs, four for fp32.  AROUND: past
// the caches.
template <uint32_t G, bool AROUND>
__global__ __launch_bounds__(256) void f8_dequant_k(const uint8_t *__restrict__ codes,
                                                    const float *__restrict__ scales,
                                                    const int32_t *__restrict__ ids,
                                                    uint64_t rows, uint64_t group, uint32_t cols,
                                                    uint32_t shift, void *__restrict__ y,
                                                    uint32_t yt, uint64_t ld) {
    constexpr uint32_t L = 128 / G;
    const uint32_t nb = f8_blocks(cols), sub = threadIdx.x % L;
    const F8Place p(blockIdx.x * (256 / L) + threadIdx.x / L, group, rows, nb);
    if (p.r >= rows) return;
    const uint64_t src = ids ? (uint64_t)(int64_t)ids[p.r] : p.r;
    const uint32_t c0 = p.b * 128 + sub * G;
    const uint8_t *c = codes + src * (128ull * nb) + c0;
    const float f = scales[(src >> shift) * nb + p.b];
    float v[G];
    f8_unpack4(*(const uint32_t *)c, v);
    if constexpr (G == 8) f8_unpack4(*(const uint32_t *)(c + 4), v + 4);
#pragma unroll
    for (uint32_t i = 0; i < G; i++) v[i] *= f;
    const uint64_t at = p.r * ld + c0;
    if (c0 + G <= cols) {
        if constexpr (G == 4) {
            const f32x4 w = {v[0], v[1], v[2], v[3]};
            f32x4_a4 *q = (f32x4_a4 *)((float *)y + at);
            AROUND ? __builtin_nontemporal_store(w, q) : (void)(*q = w);
        } else {
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = f32_to_16x2(v[2 * i], v[2 * i + 1], yt);
            u32x4_a2 *q = (u32x4_a2 *)((uint16_t *)y + at);
            AROUND ? __builtin_nontemporal_store(w, q) : (void)(*q = w);
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < G; i++)
            if (c0 + i < cols) store_from_f32(y, yt, at + i, v[i]);
    }
}

namespace {

// What both directions ask of their arguments.
bool f8_rows_ok(const char *who, const void *f, uint32_t type, uint64_t ld, uint64_t rows,
                uint64_t cols, uint32_t block_rows, const uint8_t *codes, const float *scales) {
    if ((rows && (!f || !codes || !scales)) || !cols) {
        set_error("%s: bad arguments", who);
        return false;
    }
    if (!is_float_type(type)) {
        set_error("%s: type %u not covered (F32, F16, BF16)", who, type);
        return false;
    }
    if (block_rows != 1 && block_rows != 128) {
        set_error("%s: %u rows a scale not covered (1, 128)", who, block_rows);
        return false;
    }
    if (cols > (1u << 30) || rows > (1ull << 32) || rows * f8_blocks(cols) > (1ull << 40)) {
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

// `each` blocks a workgroup over groups of whole rows of fewer than 2^24 *
// `each` blocks, so that a launch has fewer than 2^32 threads along x and fewer
// than 2^28 blocks a group.
dim3 f8_grid(uint32_t each, uint64_t rows, uint64_t cols, uint64_t *group) {
    const uint32_t nb = f8_blocks(cols);
    *group = std::min<uint64_t>(rows, (((uint64_t)each << 24) - each) / nb);
    return dim3((uint32_t)((*group * nb + each - 1) / each),
                (uint32_t)((rows + *group - 1) / *group));
}

}  // namespace

extern "C" {

/* Bytes of the codes / scales of rows x cols values (see include/q4mi.h). */
uint64_t q4mi_f8_code_bytes(uint64_t rows, uint64_t cols) {
    return rows * 128 * ((cols + 127) / 128);
}
uint64_t q4mi_f8_scale_bytes(uint64_t rows, uint64_t cols, uint32_t block_rows) {
    return block_rows ? (rows + block_rows - 1) / block_rows * 4 * ((cols + 127) / 128) : 0;
}

/* Float rows to 8-bit floating point (see include/q4mi.h). */
bool q4mi_f8_quant(const void *d_x, uint32_t x_type, uint64_t ld_x, const int32_t *d_ids,
                   uint64_t rows, uint64_t cols, uint32_t block_rows, uint8_t *d_codes,
                   float *d_scales) {
    if (!f8_rows_ok("q4mi_f8_quant", d_x, x_type, ld_x, rows, cols, block_rows, d_codes, d_scales))
        return false;
    if (!rows) return true;
    uint64_t group;
    if (block_rows == 128) {
        const dim3 grid = f8_grid(1, (rows + 127) / 128, cols, &group);
        auto k = x_type == kTypeF32 ? f8_quant_blocks_k<4> : f8_quant_blocks_k<2>;
        k<<<grid, dim3(256), 0, stream()>>>(d_x, x_type, ld_x, d_ids, rows, group, (uint32_t)cols,
                                            d_codes, d_scales);
        return launch_ok("f8_quant_blocks_k");
    }
    const bool f32 = x_type == kTypeF32;
    const dim3 grid = f8_grid(f32 ? 16 : 32, rows, cols, &group);
    auto k = f32 ? f8_quant_k<8> : f8_quant_k<16>;
    k<<<grid, dim3(256), 0, stream()>>>(d_x, x_type, ld_x, d_ids, rows, group, (uint32_t)cols,
                                        d_codes, d_scales);
    return launch_ok("f8_quant_k");
}

/* 8-bit floating point to float rows (see include/q4mi.h). */
bool q4mi_f8_dequant(const uint8_t *d_codes, const float *d_scales, const int32_t *d_ids,
                     uint64_t rows, uint64_t cols, uint32_t block_rows, void *d_y, uint32_t y_type,
                     uint64_t ld_y) {
    if (!f8_rows_ok("q4mi_f8_dequant", d_y, y_type, ld_y, rows, cols, block_rows, d_codes,
                    d_scales))
        return false;
    if (!rows) return true;
    uint64_t group;
    const bool f32 = y_type == kTypeF32;
    const dim3 grid = f8_grid(f32 ? 8 : 16, rows, cols, &group);
    // Outputs larger than the eight L2s together would only take the place of what
    // else is read (16384 x 4096 bf16, quantised and back: 79 us through the caches,
    // 69.6 around them); but parts of lines cost more there.
    const bool large = rows * cols * type_bytes(y_type) > 32ull << 20 &&
                       ((uintptr_t)d_y | ld_y * type_bytes(y_type)) % 64 == 0;
    auto k = f32 ? (large ? f8_dequant_k<4, true> : f8_dequant_k<4, false>)
                 : (large ? f8_dequant_k<8, true> : f8_dequant_k<8, false>);
    k<<<grid, dim3(256), 0, stream()>>>(d_codes, d_scales, d_ids, rows, group, (uint32_t)cols,
                                        block_rows == 128 ? 7u : 0u, d_y, y_type, ld_y);
    return launch_ok("f8_dequant_k");
}

}  // extern "C"

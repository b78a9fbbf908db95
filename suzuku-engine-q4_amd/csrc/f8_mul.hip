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
    uint32_t ks, seg, blocks;       // waves a tile, blocks of K in LDS, workgroups
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

// ---------------------------------------------------------------- few rows
//
// Up to sixteen activation rows against all weight rows: bound by reading the
// weights once.  A wave takes 16 weight rows straight from memory into
// registers, a chunk of two blocks at a time (256 bytes a row, 4 KB): lane
// (m, g) has bytes 64s + 16g .. of row m (s = 0..3), so four lanes read 64
// adjacent bytes.  One chunk is multiplied while the next, also of the next
// tile, is in flight.  The activation rows sit in LDS as codes; float rows are
// quantised on the way there, once a workgroup.  ks waves share a tile along K
// and their sums are joined in LDS in wave order, so a short matrix still
// occupies the chip; a workgroup goes over several tiles, so a tall one pays the
// LDS fill once.
constexpr uint32_t kFewRows = 16, kFewWaves = 4;

// LDS strides of a row's codes and scales, seg blocks: 16 bytes more than a
// multiple of 128, so that the rows of a fragment start in different banks.
__host__ __device__ inline uint32_t few_code_ld(uint32_t seg) { return seg * 128u + 16u; }
__host__ __device__ inline uint32_t few_scale_ld(uint32_t seg) { return seg * 4u + 8u; }

// The activation rows of a workgroup: `rows` rows from p0 on, or those at the
// places that `list` (in LDS) names past p0.
struct FewRange {
    uint64_t p0;
    uint32_t rows, x_div;
    const uint32_t *list;
    __device__ uint64_t row(uint32_t t) const { return p0 + (list ? list[t] : t); }
    __device__ uint64_t x_row(uint32_t t) const {
        return x_div == 1 ? row(t) : (uint32_t)row(t) / x_div;
    }
};

// Blocks [b0, b0 + seg) of the rows into LDS; blocks from nb on get codes and
// scales of 0.
__device__ inline void few_stage(const F8Args &a, const FewRange &f, uint32_t b0, uint32_t seg,
                                 uint32_t nb, uint8_t *codes, uint8_t *scales) {
    constexpr uint32_t T = kFewWaves * 64;
    const uint32_t cld = few_code_ld(seg), sld = few_scale_ld(seg);
    if (a.x_type == kTypeF8) {
        const uint32_t lane = threadIdx.x & 63u;
#pragma unroll 2
        for (uint32_t t = threadIdx.x >> 6; t < f.rows; t += kFewWaves) {
            const uint64_t xr = f.x_row(t);
            const u32x4 *c = (const u32x4 *)((const uint8_t *)a.x + xr * (128ull * nb));
            const float *s = a.xs + xr * nb;
            for (uint32_t i = lane; i < seg * 8; i += 64)
                *(u32x4 *)(codes + t * cld + 16u * i) =
                    b0 + i / 8 < nb ? c[8 * b0 + i] : (u32x4){0, 0, 0, 0};
            for (uint32_t i = lane; i < seg; i += 64)
                *(float *)(scales + t * sld + 4u * i) = b0 + i < nb ? s[b0 + i] : 0.f;
        }
        return;
    }
    // sixteen lanes a block, eight values each
    for (uint32_t i = threadIdx.x; i < f.rows * seg * 16; i += T) {
        const uint32_t sub = i & 15u, q = i >> 4, t = q / seg, b = q - t * seg;
        uint32_t code[2] = {0, 0}, s = 0;
        if (b0 + b < nb) {
            float v[8];
            load_row8(a.x, a.x_type, f.x_row(t) * a.ldx, 128u * (b0 + b) + 8u * sub,
                      (uint32_t)a.cols, v);
            s = f8_scale_of(f8_max_lanes<16>(f8_top<8>(v)));
            f8_pack<8>(v, s, code);
        }
        *(u32x2 *)(codes + t * cld + 128u * b + 8u * sub) = (u32x2){code[0], code[1]};
        if (sub == 0) *(uint32_t *)(scales + t * sld + 4u * b) = s;
    }
}

// Weight tiles of 16 rows, of which workgroup `block` of a.blocks takes every
// a.blocks-th set.  FULL: nb is even.
template <bool FULL>
__device__ inline void few_rows(const F8Args &a, const uint8_t *w, const float *ws,
                                const FewRange &f, uint32_t block, uint8_t *lds) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t m = lane & 15u, g = lane >> 4;
    const uint32_t ks = a.ks, kw = wave & (ks - 1), sub = wave / ks, per = kFewWaves / ks;
    const uint32_t nb = f8_blocks(a.cols), last = (uint32_t)((a.w_rows + 15) / 16);
    const uint32_t seg = a.seg, nseg = (nb + seg - 1) / seg;
    const uint32_t cld = few_code_ld(seg), sld = few_scale_ld(seg);
    uint8_t *codes = lds, *scales = lds + f.rows * cld;
    v4f *red = (v4f *)(lds + (f.rows * (cld + sld) + 15) / 16 * 16);
    const uint32_t t = min(m, f.rows - 1), xc = t * cld + 16u * g, xsc = t * sld;
    const uint32_t rounds = (last + per * a.blocks - 1) / (per * a.blocks);
    auto tile_of = [&](uint32_t i) { return (i * a.blocks + block) * per + sub; };
    auto chunks = [&](uint32_t sg) { return (min(seg, nb - sg * seg) + 1) / 2; };
    struct Batch {
        u32x4 codes[4];
        float s[2];
    };
    // an address that no scalar load takes: those return out of order with LDS reads
    uint32_t zero = 0;
    asm volatile("" : "+v"(zero));
    // chunk c of segment sg of round i's weight tile
    auto load = [&](Batch &q, uint32_t i, uint32_t sg, uint32_t c) __attribute__((always_inline)) {
        const uint32_t tile = min(tile_of(i), last - 1);
        const uint64_t wr = min((uint64_t)tile * 16 + m, a.w_rows - 1);
        const uint32_t b = sg * seg + 2 * min(c, chunks(sg) - 1);
        const uint32_t b1 = FULL ? b + 1 : min(b + 1, nb - 1);
        const uint8_t *wp = w + wr * (128ull * nb) + 16 * g;
        const float *wsp = ws + (uint64_t)(tile >> 3) * nb + zero;
        q.codes[0] = *(const u32x4 *)(wp + 128u * b);
        q.codes[1] = *(const u32x4 *)(wp + 128u * b + 64);
        q.codes[2] = *(const u32x4 *)(wp + 128u * b1);
        q.codes[3] = *(const u32x4 *)(wp + 128u * b1 + 64);
        q.s[0] = wsp[b], q.s[1] = wsp[b1];
    };
    v4f acc = {0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](const Batch &q, uint32_t sg, uint32_t c) __attribute__((always_inline)) {
        if (c >= chunks(sg)) return;
        const f8_f2 xs = *(const f8_f2 *)(scales + xsc + 8u * c);
#pragma unroll
        for (uint32_t h = 0; h < 2; h++) {
            if (!FULL && h == 1 && sg * seg + 2 * c + 1 >= nb) break;
            const uint8_t *xp = codes + xc + 256u * c + 128u * h;
            const v4f d = block_sums(join(q.codes[2 * h], q.codes[2 * h + 1]),
                                     join(*(const u32x4 *)xp, *(const u32x4 *)(xp + 64)));
            const float s = q.s[h] * xs[h];
#pragma unroll
            for (int k = 0; k < 4; k++) acc[k] = fmaf(d[k], s, acc[k]);
        }
    };
    auto finish = [&](uint32_t i) __attribute__((always_inline)) {
        if (ks > 1) {
            if (i) __syncthreads();   // the last round's sums have been read
            red[wave * 64 + lane] = acc;
            __syncthreads();
            if (kw) return;
            for (uint32_t k = 1; k < ks; k++) acc += red[(wave + k) * 64 + lane];
        }
        const uint32_t tile = tile_of(i);
        if (tile >= last || m >= f.rows) return;
        const uint64_t r = (uint64_t)tile * 16 + 4 * g, at = f.row(m) * a.ldy + r;
        if (r + 4 <= a.w_rows)
            store4(a.y, a.y_type, at, acc);
        else
            for (uint32_t k = 0; k < 4; k++)
                if (r + k < a.w_rows) store_from_f32(a.y, a.y_type, at + k, acc[k]);
    };

    // Every wave goes through every segment of every round, so all meet the
    // barriers.
    Batch now, then;
    uint32_t i = 0, sg = 0, c = kw;
    load(now, 0, 0, kw);
    few_stage(a, f, 0, seg, nb, codes, scales);
    __syncthreads();
    for (;;) {
        uint32_t ni = i, nsg = sg, nc = c + ks;
        const bool done = nc >= chunks(sg);
        if (done) {
            nc = kw;
            if (++nsg == nseg) nsg = 0, ni++;
        }
        const bool more = ni < rounds;
        if (more) load(then, ni, nsg, nc);
        multiply(now, sg, c);
        if (ni != i) {
            finish(i);
            acc = (v4f){0.f, 0.f, 0.f, 0.f};
        }
        if (!more) break;
        if (done && nseg > 1) {
            __syncthreads();
            few_stage(a, f, nsg * seg, seg, nb, codes, scales);
            __syncthreads();
        }
        now = then, i = ni, sg = nsg, c = nc;
    }
}

// Dense: grid (blocks, sets of 16 activation rows).
template <bool FULL>
__global__ __launch_bounds__(64 * kFewWaves) void f8_few_k(F8Args a) {
    extern __shared__ __align__(16) uint8_t lds[];
    const uint64_t p0 = (uint64_t)blockIdx.y * kFewRows;
    const FewRange f = {p0, (uint32_t)min((uint64_t)kFewRows, a.n - p0), 1, nullptr};
    few_rows<FULL>(a, a.w, a.ws, f, blockIdx.x, lds);
}

// Rows through the experts that the list names; grid (blocks, rows).  GROUP:
// rows of one expert among 256 go together, sixteen at a time, so that its
// weights are read once: the first of them does the work, the others'
// workgroups end.
constexpr size_t kSelList = 4 * 8 + kFewRows * 4;
template <bool FULL, bool GROUP>
__global__ __launch_bounds__(64 * kFewWaves) void f8_sel_k(F8Args a) {
    extern __shared__ __align__(16) uint8_t lds[];
    uint64_t *same = (uint64_t *)lds;           // which of the 256 rows are of this expert
    uint32_t *list = (uint32_t *)(same + 4);
    const uint32_t p = blockIdx.y, p0 = p & ~255u, q = p0 + threadIdx.x;
    const int32_t e = a.eid[p];
    if (e < 0 || (uint32_t)e >= a.n_expert) return;
    const uint8_t *w = a.w + e * a.w_stride;
    const float *ws = (const float *)((const uint8_t *)a.ws + e * a.ws_stride);
    if constexpr (!GROUP) {
        const FewRange f = {p, 1, a.x_div, nullptr};
        few_rows<FULL>(a, w, ws, f, blockIdx.x, lds);
        return;
    }
    const uint64_t bits = __ballot(q < a.n && a.eid[q] == e);
    if ((threadIdx.x & 63u) == 0) same[threadIdx.x >> 6] = bits;
    __syncthreads();
    // how many of them lie before place i
    auto before = [&](uint32_t i) {
        uint32_t c = 0;
#pragma unroll
        for (uint32_t w = 0; w < 4; w++)
            c += i >= 64 * w + 64 ? (uint32_t)__popcll(same[w])
                 : i > 64 * w     ? (uint32_t)__popcll(same[w] & ((1ull << (i - 64 * w)) - 1))
                                  : 0u;
        return c;
    };
    const uint32_t rank = before(p - p0), rows = min(before(256) - rank, kFewRows);
    if (rank % kFewRows) return;
    FewRange f = {p, rows, a.x_div, nullptr};
    if (rows > 1) {
        const uint32_t mine = before(threadIdx.x) - rank;
        if ((same[threadIdx.x >> 6] >> (threadIdx.x & 63u) & 1u) && mine < rows)
            list[mine] = threadIdx.x;
        __syncthreads();
        f.p0 = p0, f.list = list;
    }
    few_rows<FULL>(a, w, ws, f, blockIdx.x, lds + kSelList);
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

// Dense: grid (weight tiles / 4, sets of 16 activation rows).
__global__ __launch_bounds__(256) void f8_dense_k(F8Args a) {
    const uint64_t tile = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint64_t p0 = (uint64_t)blockIdx.y * 16;
    if (tile * 16 >= a.w_rows) return;
    plain_tile(a, a.w, a.ws, tile, p0, (uint32_t)min((uint64_t)16, a.n - p0));
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

}  // namespace

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

// K segment of the few-rows kernels for `rows` activation rows a workgroup:
// whole rows where they fit in `room` bytes, else equal parts of whole chunks;
// returns the LDS bytes.
size_t few_fit(F8Args &a, uint32_t rows, size_t room) {
    const uint32_t nb = f8_blocks(a.cols);
    uint32_t parts = 1;
    size_t need;
    do {
        a.seg = ((nb + parts - 1) / parts + 1) / 2 * 2;
        need = (size_t)rows * (few_code_ld(a.seg) + few_scale_ld(a.seg));
        parts++;
    } while (need > room && a.seg > 2);
    return (need + 15) / 16 * 16 + (a.ks > 1 ? kFewWaves * 64 * sizeof(v4f) : 0);
}

// One set of `rows` (<= 16) activation rows a workgroup, `lists` of them, of
// which about `busy` have work.  As many workgroups as are resident at once, each
// with the same number of rounds.  Waves a tile: as many as there are chunks,
// while the whole launch has fewer than 8 waves a CU.
template <class F>
bool few_launch(F8Args &a, uint32_t rows, uint32_t lists, uint32_t busy, size_t extra, F pick,
                const char *name) {
    const uint64_t tiles = (a.w_rows + 15) / 16;
    const uint32_t chunks = (f8_blocks(a.cols) + 1) / 2;
    a.ks = 1;
    while (a.ks < kFewWaves && a.ks * 2 <= chunks && tiles * busy * a.ks < 8ull * cu_count())
        a.ks *= 2;
    const size_t lds = extra + few_fit(a, rows, 36 * 1024);
    const uint64_t sets = (tiles * a.ks + kFewWaves - 1) / kFewWaves;
    const uint64_t resident = std::max(1u, 4u * cu_count() / busy);
    const uint64_t rounds = (sets + resident - 1) / resident;
    a.blocks = (uint32_t)((sets + rounds - 1) / rounds);
    auto k = pick(f8_blocks(a.cols) % 2 == 0);
    k<<<dim3(a.blocks, lists), dim3(64 * kFewWaves), lds, stream()>>>(a);
    return launch_ok(name);
}
typedef void (*F8Kernel)(F8Args);
F8Kernel few_kernel(bool full) { return full ? f8_few_k<true> : f8_few_k<false>; }
F8Kernel sel_kernel(bool full) { return full ? f8_sel_k<true, false> : f8_sel_k<false, false>; }
F8Kernel sel_group_kernel(bool full) {
    return full ? f8_sel_k<true, true> : f8_sel_k<false, true>;
}

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
    if (n <= kFewRows)
        return few_launch(a, (uint32_t)n, 1, 1, 0, few_kernel, "f8_few_k");
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
    const uint32_t lists = (uint32_t)n;
    if (4 * n < n_expert) return few_launch(a, 1, lists, lists, 0, sel_kernel, "f8_sel_k");
    return few_launch(a, std::min(lists, kFewRows), lists,
                      std::min(lists, n_expert + lists / kFewRows), kSelList, sel_group_kernel,
                      "f8_sel_k");
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

// Products of 8-bit floating point rows in blocks of 128 (f8.h has the format):
//   y[t][r] = sum over blocks b of xs[t][b] * ws[r / 128][b] * sum_i w[r][128b+i] x[t][128b+i]
// A block is summed from zero by matrix instructions of sixteen weight rows and
// sixteen activation rows; its four sums a lane are then multiplied by both
// scales and added in fp32.  Weight rows are the first operand, so a lane's sums
// are four adjacent outputs of one activation row.
//
// The 8-bit matrix instructions add eight neighbouring products with only 14 bits
// below the largest of them (measured: a product 2^-14 of its neighbour is lost,
// one in another eight only at 2^-24): with large products that cancel nothing of
// the others is left.  Codes are exact in bf16, whose instruction adds in fp32 (y 1e-8
// off, 2-norm) at half the rate, so every sum here comes from that one.
#include <algorithm>

#include "f8.h"
#include "q4mi_internal.h"

using namespace q4mi;

namespace {

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
    uint32_t ks, waves, seg, blocks;    // waves a tile, a workgroup; blocks of K in LDS; workgroups
    uint32_t m_tiles;               // tiles along the activations
};

// Four adjacent outputs, rounded once; AROUND: past the caches.
template <bool AROUND>
__device__ inline void store4(void *y, uint32_t yt, uint64_t at, v4f v) {
    if (yt == kTypeF32) {
        f32x4_a4 *p = (f32x4_a4 *)((float *)y + at);
        AROUND ? __builtin_nontemporal_store((f32x4)v, p) : (void)(*p = (f32x4)v);
    } else {
        const u32x2 q = {f32_to_16x2(v[0], v[1], yt), f32_to_16x2(v[2], v[3], yt)};
        u32x2_a2 *p = (u32x2_a2 *)((uint16_t *)y + at);
        AROUND ? __builtin_nontemporal_store(q, p) : (void)(*p = q);
    }
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

// A lane's part of a block of sixteen rows.  Which of the block's values that is
// is free as long as both sides agree: lane (row, g) has bytes 16g .. and 64 +
// 16g .. of its row, so that four lanes read 64 bytes.
struct Frag {
    v8b v[4];
    __device__ Frag() {}
    __device__ Frag(u32x4 a, u32x4 b)
        : v{widen(a.x, a.y), widen(a.z, a.w), widen(b.x, b.y), widen(b.z, b.w)} {}
};

// Sixteen rows against sixteen over one block, from zero.
__device__ inline v4f block_sums(const Frag &w, const Frag &x) {
    v4f d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; i++)
        d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[i], x.v[i], d, 0, 0, 0);
    return d;
}

// acc += d * s, here: the compiler would rather keep every block's sums in
// registers and add them after the loop's last product.
__device__ inline void add_scaled(v4f &acc, v4f d, float s) {
#pragma unroll
    for (int i = 0; i < 4; i++) acc[i] = fmaf(d[i], s, acc[i]);
    asm volatile("" : "+v"(acc));
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
//
// Measured, codes to BF16: one row through 151936 x 2048 58 us (5.4 TB/s), 8192 x
// 8192 14.6 us (4.6 TB/s), 2560 x 2560 4.7 us (an empty launch: 2 us); sixteen rows
// 66.3, 17.4 and 5.8 us.  What bounds the middle ones is how much a CU can have on
// its way with loads to registers, 30 KB/us.
constexpr uint32_t kFewRows = 16, kFewWaves = 8;     // at most

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

// Blocks [b0, b0 + seg) of float rows (XB bytes a value) into LDS: sixteen lanes a
// block, eight values each, two blocks' loads on their way at once.
template <uint32_t XB>
__device__ inline void few_stage_floats(const F8Args &a, const FewRange &f, uint32_t b0,
                                        uint32_t seg, uint32_t nb, uint8_t *codes,
                                        uint8_t *scales) {
    const uint32_t cld = few_code_ld(seg), sld = few_scale_ld(seg);
    const uint32_t step = 64 * a.waves, end = f.rows * seg * 16, at = 8 * (threadIdx.x & 15u);
    for (uint32_t i = threadIdx.x; i < end; i += 2 * step) {
        Raw8<XB> raw[2];
        uint32_t t[2], b[2];
#pragma unroll
        for (uint32_t u = 0; u < 2; u++) {
            const uint32_t q = (i + u * step) >> 4;
            t[u] = q / seg, b[u] = q - t[u] * seg;
            // past the end and past K as columns past the last: zeros
            const bool in = i + u * step < end && b0 + b[u] < nb;
            load_raw8<XB>(a.x, f.x_row(in ? t[u] : 0) * a.ldx, 128u * (b0 + b[u]) + at,
                          in ? (uint32_t)a.cols : 0u, raw[u]);
        }
#pragma unroll
        for (uint32_t u = 0; u < 2; u++) {
            if (i + u * step >= end) break;
            float v[8];
            raw8_to_f32<XB>(raw[u], a.x_type, v);
            uint32_t code[2], s = f8_scale_of(f8_max_lanes<16>(f8_top<8>(v)));
            f8_pack<8>(v, s, code);
            if (b0 + b[u] >= nb) s = 0;
            *(u32x2 *)(codes + t[u] * cld + 128u * b[u] + at) = (u32x2){code[0], code[1]};
            if (at == 0) *(uint32_t *)(scales + t[u] * sld + 4u * b[u]) = s;
        }
    }
}

// Blocks [b0, b0 + seg) of the rows into LDS; blocks from nb on get codes and
// scales of 0.  Four loads a lane are on their way at once.
__device__ inline void few_stage(const F8Args &a, const FewRange &f, uint32_t b0, uint32_t seg,
                                 uint32_t nb, uint8_t *codes, uint8_t *scales) {
    const uint32_t cld = few_code_ld(seg), sld = few_scale_ld(seg);
    if (a.x_type == kTypeF8) {
        const uint32_t lane = threadIdx.x & 63u, here = min(seg, nb - b0);
        for (uint32_t t = threadIdx.x >> 6; t < f.rows; t += a.waves) {
            const uint64_t xr = f.x_row(t);
            const u32x4 *c = (const u32x4 *)((const uint8_t *)a.x + xr * (128ull * nb)) + 8 * b0;
            const float *s = a.xs + xr * nb + b0;
            for (uint32_t i = lane; i < seg; i += 64)
                *(float *)(scales + t * sld + 4u * i) = i < here ? s[i] : 0.f;
            for (uint32_t i = lane; i < seg * 8; i += 256) {
                u32x4 v[4];
#pragma unroll
                for (uint32_t u = 0; u < 4; u++)
                    v[u] = i + 64 * u < here * 8 ? c[i + 64 * u] : (u32x4){0, 0, 0, 0};
#pragma unroll
                for (uint32_t u = 0; u < 4; u++)
                    if (i + 64 * u < seg * 8) *(u32x4 *)(codes + t * cld + 16u * (i + 64 * u)) = v[u];
            }
        }
        return;
    }
    if (a.x_type == kTypeF32)
        few_stage_floats<4>(a, f, b0, seg, nb, codes, scales);
    else
        few_stage_floats<2>(a, f, b0, seg, nb, codes, scales);
}

// Weight tiles of 16 rows, of which workgroup `block` of a.blocks takes every
// a.blocks-th set.  FULL: nb is even.
template <bool FULL>
__device__ inline void few_rows(const F8Args &a, const uint8_t *w, const float *ws,
                                const FewRange &f, uint32_t block, uint8_t *lds) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t m = lane & 15u, g = lane >> 4;
    const uint32_t ks = a.ks, kw = wave & (ks - 1), sub = wave / ks, per = a.waves / ks;
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
            const v4f d = block_sums(
                Frag(q.codes[2 * h], q.codes[2 * h + 1]),
                Frag(*(const u32x4 *)xp, *(const u32x4 *)(xp + 64)));
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
            store4<false>(a.y, a.y_type, at, acc);
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
// rows of one expert among kSelRows go together, sixteen at a time, so that its
// weights are read once: the first of them does the work, the others'
// workgroups end.
constexpr uint32_t kSelRows = 256, kSelSets = kSelRows / 64;
constexpr size_t kSelList = kSelSets * 8 + kFewRows * 4;
template <bool FULL, bool GROUP>
__global__ __launch_bounds__(64 * kFewWaves) void f8_sel_k(F8Args a) {
    extern __shared__ __align__(16) uint8_t lds[];
    uint64_t *same = (uint64_t *)lds;           // which of the rows are of this expert
    uint32_t *list = (uint32_t *)(same + kSelSets);
    const uint32_t p = blockIdx.y, p0 = p & ~(kSelRows - 1), q = p0 + threadIdx.x;
    const int32_t e = a.eid[p];
    if (e < 0 || (uint32_t)e >= a.n_expert) return;
    const uint8_t *w = a.w + e * a.w_stride;
    const float *ws = (const float *)((const uint8_t *)a.ws + e * a.ws_stride);
    if constexpr (!GROUP) {
        const FewRange f = {p, 1, a.x_div, nullptr};
        few_rows<FULL>(a, w, ws, f, blockIdx.x, lds);
        return;
    }
    const uint64_t bits = __ballot(threadIdx.x < kSelRows && q < a.n && a.eid[q] == e);
    if ((threadIdx.x & 63u) == 0 && threadIdx.x < kSelRows) same[threadIdx.x >> 6] = bits;
    __syncthreads();
    // how many of them lie before place i
    auto before = [&](uint32_t i) {
        uint32_t c = 0;
#pragma unroll
        for (uint32_t w = 0; w < kSelSets; w++)
            c += i >= 64 * w + 64 ? (uint32_t)__popcll(same[w])
                 : i > 64 * w     ? (uint32_t)__popcll(same[w] & ((1ull << (i - 64 * w)) - 1))
                                  : 0u;
        return c;
    };
    const uint32_t rank = before(p - p0), rows = min(before(kSelRows) - rank, kFewRows);
    if (rank % kFewRows) return;
    FewRange f = {p, rows, a.x_div, nullptr};
    if (rows > 1) {
        const uint32_t mine = before(threadIdx.x) - rank;
        if (threadIdx.x < kSelRows && (same[threadIdx.x >> 6] >> (threadIdx.x & 63u) & 1u) && mine < rows)
            list[mine] = threadIdx.x;
        __syncthreads();
        f.p0 = p0, f.list = list;
    }
    few_rows<FULL>(a, w, ws, f, blockIdx.x, lds + kSelList);
}

// ------------------------------------------------------------ rows in tiles
//
// BM activation rows x BN weight rows a workgroup of WM x WN waves.  K goes in
// stages of one block: 128 bytes a row, a whole cache line, come by global -> LDS
// copies into a ring of S stages, spread over the products of S - 1 stages
// before.  The activations' scales come for eight stages at once, 32 bytes a row;
// a wave's weight rows share one scale a stage.  A wave holds all its weight
// fragments of a stage, and the next stage's as it is read, over its activation
// fragments one by one.
//
// Measured, codes to BF16: 8192 x 8192 x 8192 935 to 1000 us (1.1 to 1.18 PFLOP/s, by
// the card; a library's bf16 product 1.37), 2048 rows of that 239 to 262 us, 512 rows 78
// us, 32 rows 22 us (3.1 TB/s), 77 x 2560 x 2560 8.4 us.  The bf16 instruction and the
// widening ahead of it bound it: at 8192^3 the matrix units are busy 57 % of the time, and
// 134 M of the 237 M other vector instructions convert two codes each, every code in
// both waves that read it.
//
// LDS places: chunk c (16 bytes) of row r at c ^ ((r >> 1) & 7), dword d of a
// row's scales at d ^ ((r >> 3) & 7), so that a fragment's reads spread over all
// 64 banks; the copies fill LDS in lane order, so the lanes permute their source
// addresses instead.

__device__ inline uint32_t tile_swz(uint32_t row) { return (row >> 1) & 7u; }

// Lane i's 16 (4) bytes land at LDS address lds + 16 i (4 i); from a pointer, or
// from a uniform base and a 32-bit offset.  Inline asm, so that the compiler adds
// no wait before the next LDS read.  Nor does it see that
// a base is read: one that a vector instruction wrote (a spilled one read back)
// needs five wait states, which the move and the s_nop 3 are.
__device__ inline void copy16(const void *base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off),
                 "s"(base), "s"(lds)
                 : "memory", "m0");
}
__device__ inline void copy16(const void *g, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g),
                 "s"(lds)
                 : "memory", "m0");
}
__device__ inline void copy4(const void *g, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(g),
                 "s"(lds)
                 : "memory", "m0");
}
__device__ inline void copy4(const void *base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dword %0, %1" ::"v"(off),
                 "s"(base), "s"(lds)
                 : "memory", "m0");
}
// All but this wave's last `LEFT` memory operations have landed; then the
// workgroup meets.  Later operations of the compiler's make it wait for more.
template <int LEFT>
__device__ inline void landed_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
}

// LDS: S stages of codes, two windows (eight stages) of scales.
template <uint32_t BM, uint32_t BN, uint32_t S>
constexpr uint32_t tile_lds() { return (BM + BN) * S * 128 + BM * 2 * 32; }

// The row of the weights' scales that a wave reads whose weight rows begin at r0 +
// first: the last one where all of them are past the last row, as their codes are
// the last row's.
__host__ __device__ inline uint64_t tile_scale_row(uint64_t w_rows, uint64_t r0, uint32_t first) {
    return (r0 + first < w_rows ? r0 + first : w_rows - 1) / 128;
}

// Weight rows [r0, r0 + BN) of w against activation rows [p0, p0 + BM), of which
// those below phi exist; the row read for p is act[p] with GATHER, else p.  Rows
// past either end are read as the last one and not stored.  AROUND: outputs past the
// caches.
template <uint32_t BM, uint32_t BN, uint32_t WM, uint32_t WN, uint32_t S, bool GATHER, bool AROUND>
__device__ inline void tile(const F8Args &a, const uint8_t *w, const float *ws, uint64_t r0,
                            uint64_t p0, uint64_t phi, uint8_t *lds) {
    constexpr uint32_t NW = WM * WN;
    constexpr uint32_t FM = BM / (16 * WM), FN = BN / (16 * WN);
    constexpr uint32_t RA = BM / 8 / NW, RB = BN / 8 / NW;   // 8-row copies of each side a wave
    constexpr uint32_t kLeft = (S - 2) * (RA + RB);     // copies on their way past the next stage's
    static_assert(FM && FN && RA && RB && 16 * FN <= 128 && kLeft < 64, "tile and waves");
    static_assert(S - 2 + RA <= 8, "a window's scales land in time");
    constexpr uint32_t kX = BM * 128, kW = BN * 128, kWin = BM * 32;
    constexpr uint32_t kWeights = S * kX, kScales = S * (kX + kW);
    // opaque, or what follows from it would be kept from one tile to the next, spilled
    uint32_t tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const uint32_t lane = tid & 63u, l8 = lane >> 3;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t nb = f8_blocks(a.cols);
    const uint32_t base = (uint32_t)(uintptr_t)lds;     // LDS offset: low half of the address
    const uint32_t row_bytes = 128 * nb;

    // sources of this lane's part of every copy, without the place in K: offsets
    // from the tile's first row, or numbers of rows with GATHER
    const uint8_t *xc = (const uint8_t *)a.x;
    const float *xs = a.xs;
    if (!GATHER) xc += p0 * row_bytes, xs += p0 * nb;
    const uint32_t xlast = (uint32_t)min((uint64_t)BM, phi - p0) - 1;
    const uint32_t wlast = (uint32_t)min((uint64_t)BN, a.w_rows - r0) - 1;
    w += r0 * row_bytes;
    auto gathered = [&](uint32_t t) -> uint32_t {
        const int64_t r = a.act ? (int64_t)a.act[p0 + t] : (int64_t)(p0 + t);
        return r < 0 || r >= (int64_t)a.xrows ? 0u : (uint32_t)r;
    };
    const uint32_t c0 = 16 * ((lane & 7u) ^ (l8 >> 1));     // chunk of an even copy; ^ 64 of an odd
    uint32_t xo[RA], wo[RB];
#pragma unroll
    for (uint32_t j = 0; j < RA; j++) {
        const uint32_t c = wave * RA + j, t = min(c * 8 + l8, xlast);
        xo[j] = GATHER ? gathered(t) : t * row_bytes + (c0 ^ 64 * (c & 1u));
    }
#pragma unroll
    for (uint32_t j = 0; j < RB; j++) {
        const uint32_t c = wave * RB + j;
        wo[j] = min(c * 8 + l8, wlast) * row_bytes + (c0 ^ 64 * (c & 1u));
    }
    // copy q (of RA + RB) of this wave's of stage k; stages past the last as the last
    auto fetch = [&](uint32_t k, uint32_t q) __attribute__((always_inline)) {
        const uint32_t at = 128u * min(k, nb - 1), c = wave * RA + q;
        const uint32_t to = base + k % S * kX + c * 1024;
        if (q >= RA)
            copy16(w + at, wo[q - RA], base + kWeights + k % S * kW + (wave * RB + q - RA) * 1024);
        else if (GATHER)
            copy16(xc + at + (c0 ^ 64 * (c & 1u)) + (uint64_t)xo[q] * row_bytes, to);
        else
            copy16(xc + at, xo[q], to);
    };
    // Copy q (of RA; 8 rows each) of this wave's of window v's scales.
    auto fetch_scales = [&](uint32_t v, uint32_t q) __attribute__((always_inline)) {
        const uint32_t c = wave * RA + q, to = base + kScales + (v & 1u) * kWin + c * 256;
        const uint32_t d = min(8 * v + ((lane & 7u) ^ (c & 7u)), nb - 1);
        if (GATHER) {
            // not xo[q], nor choices that become it: an index puts the array into memory
            uint32_t r = 0;
#pragma unroll
            for (uint32_t j = 0; j < RA; j++) {
                uint32_t mask = q == j ? ~0u : 0u;
                asm("" : "+v"(mask));
                r |= xo[j] & mask;
            }
            copy4(xs + (uint64_t)r * nb + d, to);
        } else {
            copy4(xs, 4 * (min(c * 8 + l8, xlast) * nb + d), to);
        }
    };
    const uint32_t wm = wave / WN, wn = wave % WN, m = lane & 15u, g = lane >> 4;
    const uint32_t ra = wm * FM * 16 + m, rb = wn * FN * 16 + m;
    const uint32_t lo = 16 * (g ^ tile_swz(m)), hi = lo ^ 64;
    // read by scalar loads: one of the compiler's vector loads would wait for every copy
    typedef const float __attribute__((address_space(4))) *Constant;
    const Constant wsp =
        (Constant)(uintptr_t)(ws + tile_scale_row(a.w_rows, r0, wn * FN * 16) * nb);

    v4f acc[FN][FM];
#pragma unroll
    for (uint32_t j = 0; j < FN; j++)
#pragma unroll
        for (uint32_t i = 0; i < FM; i++) acc[j][i] = (v4f){0.f, 0.f, 0.f, 0.f};

#pragma unroll
    for (uint32_t q = 0; q < RA; q++) fetch_scales(0, q);
#pragma unroll
    for (uint32_t k = 0; k + 1 < S; k++)
#pragma unroll
        for (uint32_t q = 0; q < RA + RB; q++) fetch(k, q);
    landed_barrier<kLeft>();
    Frag wf[2][FN], xf[2];
    float sx[2], s = wsp[0];
    auto read_w = [&](uint32_t k, Frag *f, uint32_t j) __attribute__((always_inline)) {
        const uint8_t *p = lds + kWeights + k % S * kW + rb * 128 + j * 2048;
        f[j] = Frag(*(const u32x4 *)(p + lo), *(const u32x4 *)(p + hi));
    };
    auto read_x = [&](uint32_t k, uint32_t i) __attribute__((always_inline)) {
        const uint8_t *p = lds + k % S * kX + ra * 128 + i * 2048;
        xf[i & 1u] = Frag(*(const u32x4 *)(p + lo), *(const u32x4 *)(p + hi));
        const uint32_t d = 4 * ((k & 7u) ^ ((ra + 16 * i) >> 3 & 7u));
        sx[i & 1u] = *(const float *)(lds + kScales + (k >> 3 & 1u) * kWin + ra * 32 + i * 512 + d);
    };
#pragma unroll
    for (uint32_t j = 0; j < FN; j++) read_w(0, wf[0], j);
    read_x(0, 0);
    // A stage begins with its weights and its first activations in registers.  The
    // barrier that says that the next stage has landed and this one is read stands
    // before the last activations' products, which cover the next stage's first
    // reads.  Sums are added two products later, copies go out four an activation
    // fragment (8192 x 8192 x 8192, us: one to four products later 972, 959, 961, 957;
    // two, three, four, eight copies 960, 959, 938, 936).
    auto stage = [&](uint32_t k, Frag *now, Frag *next) __attribute__((always_inline)) {
        const float s_next = wsp[min(k + 1, nb - 1)];
        constexpr uint32_t kPairs = FM * FN, kLag = 2;
        constexpr uint32_t kFirst = FM > 1 ? FM - 1 : 1;
        constexpr uint32_t kNeed = (RA + RB + kFirst - 1) / kFirst, kEach = kNeed > 4 ? kNeed : 4;
        v4f d[kLag + 1];
        float ds[kLag + 1];
#pragma unroll
        for (uint32_t t = 0; t < kPairs + kLag; t++) {
            const uint32_t i = t / FN, j = t % FN;
            if (t < kPairs) {
                if (j == 0) {
                    if (i + 1 < FM) read_x(k, i + 1);
#pragma unroll
                    for (uint32_t q = kEach * i; q < min(kEach * (i + 1), RA + RB); q++)
                        fetch(k + S - 1, q);
                    if (i + 1 == FM) {
                        landed_barrier<kLeft>();
                        // a window's copies spread over the stages of the one before it
                        if ((k & 7u) < RA) fetch_scales((k >> 3) + 1, k & 7u);
#pragma unroll
                        for (uint32_t u = 0; u < FN; u++) read_w(k + 1, next, u);
                    }
                }
                d[t % (kLag + 1)] = block_sums(now[j], xf[i & 1u]);
                ds[t % (kLag + 1)] = sx[i & 1u];
                if (t + 1 == kPairs) read_x(k + 1, 0);
            }
            if (t >= kLag) {
                const uint32_t o = t - kLag;
                add_scaled(acc[o % FN][o / FN], d[o % (kLag + 1)], s * ds[o % (kLag + 1)]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        s = s_next;
    };
    for (uint32_t k = 0; k < nb; k += 2) {
        stage(k, wf[0], wf[1]);
        if (k + 1 < nb) stage(k + 1, wf[1], wf[0]);
    }

    // Sums of 16 activation rows at a time through LDS (the stages are read), so
    // that a wave stores whole stretches of an output row: lane (m, g) holds
    // weight rows 4g .. 4g + 3 of its fragments.
    constexpr uint32_t kRow = FN * 16 + 4, kLanes = FN * 4;   // floats a row, lanes that store one
    static_assert(NW * 16 * kRow * 4 <= tile_lds<BM, BN, S>(), "sums fit the stages");
    static_assert(kLanes <= 64, "a row's stores");
    landed_barrier<0>();
    float *sums = (float *)lds + wave * 16 * kRow;
    const uint64_t rw = r0 + wn * FN * 16 + lane % kLanes * 4;   // weight row of this lane's stores
    auto listed = [&](uint64_t p) {     // whether row p has an activation row
        return !GATHER || !a.act || (a.act[p] >= 0 && (int64_t)a.act[p] < (int64_t)a.xrows);
    };
#pragma unroll
    for (uint32_t i = 0; i < FM; i++) {
#pragma unroll
        for (uint32_t j = 0; j < FN; j++)
            *(v4f *)(sums + m * kRow + 16 * j + 4 * g) = acc[j][i];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const uint64_t p1 = p0 + (wm * FM + i) * 16;
#pragma unroll
        for (uint32_t u = 0; u < 16 * kLanes / 64; u++) {
            const uint32_t t = u * (64 / kLanes) + lane / kLanes;
            const v4f v = *(const v4f *)(sums + t * kRow + lane % kLanes * 4);
            const uint64_t at = (p1 + t) * a.ldy + rw;
            if (p1 + t >= phi || !listed(p1 + t)) continue;
            if (rw + 4 <= a.w_rows)
                store4<AROUND>(a.y, a.y_type, at, v);
            else
                for (uint32_t n = 0; n < 4; n++)
                    if (rw + n < a.w_rows) store_from_f32(a.y, a.y_type, at + n, v[n]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// Tiles of a dense product, `a.blocks` of them, a.m_tiles along the
// activations.  Workgroups go to the eight dies in turn, each with an L2 of its
// own: a die takes a contiguous run of tiles, in groups of kGroup activation
// tiles, so that its L2 holds what its tiles share (8192 x 8192 x 8192, us: groups of
// four 959, eight 965, sixteen 989).
constexpr uint32_t kGroup = 4;
template <uint32_t BM, uint32_t BN, uint32_t WM, uint32_t WN, uint32_t S, bool AROUND>
__global__ __launch_bounds__(64 * WM * WN, 2) void f8_tile_k(F8Args a) {
    extern __shared__ __align__(16) uint8_t lds[];
    const uint32_t die = blockIdx.x & 7u, i = blockIdx.x >> 3;
    const uint32_t q = a.blocks >> 3, rem = a.blocks & 7u;
    const uint32_t t = die * q + min(die, rem) + i;
    const uint32_t n_tiles = a.blocks / a.m_tiles;
    const uint32_t group = t / (kGroup * n_tiles), in = t - group * kGroup * n_tiles;
    const uint32_t gm = min(kGroup, a.m_tiles - group * kGroup);
    const uint32_t mt = group * kGroup + in % gm, nt = in / gm;
    tile<BM, BN, WM, WN, S, false, AROUND>(a, a.w, a.ws, (uint64_t)nt * BN, (uint64_t)mt * BM, a.n,
                                           lds);
}

// ------------------------------------------------------------- packed rows
//
// Persistent workgroups go over the experts' sets of up to ROWS rows x ROWS weight
// rows, each in the tile that its rows fill.  With 128, two a CU, so that one
// workgroup's first copies and last stores are covered by the other's stages.
// Every workgroup makes the lists of sets by
// itself, as prefix sums over the experts' stretches in LDS: no scratch in memory,
// no launch before.  It takes every a.blocks-th of them, the large ones first, so
// that all have as many of each size (512 experts of 1024 x 2048, 2048 tokens of
// ten picks: 284 us, 308 in the experts' order, with Zipf's popularities, 266 and
// 280 with equal ones; 3.9 and 4.2 TB/s).
constexpr uint32_t kIdExperts = 1024;
// LDS: each expert's last set of more than half of ROWS, of less, of up to a quarter
struct IdLists {
    uint32_t most[kIdExperts];
    uint16_t half[kIdExperts], few[kIdExperts];
};
// Sets of up to ROWS rows x ROWS weight rows: waves and workgroups a CU, the sizes
// of the sets that have tiles of their own, stages of each, the largest tile's LDS.
template <uint32_t ROWS>
struct IdSets {
    static constexpr uint32_t kWaves = 4;
    static constexpr uint32_t kCu = ROWS == 64 ? 1 : 2;
    static constexpr uint32_t kHalf = ROWS == 32 ? 0 : ROWS / 2, kFew = ROWS < 128 ? 0 : ROWS / 4;
    static constexpr uint32_t kAllS = ROWS < 128 ? 8 : 2;
    static constexpr uint32_t kHalfS = ROWS < 128 ? 8 : 2, kFewS = 3;
    static constexpr uint32_t kTiles =
        std::max({tile_lds<ROWS, ROWS, kAllS>(), tile_lds<kHalf, ROWS, kHalfS>(),
                  tile_lds<kFew, ROWS, kFewS>()});
    static constexpr size_t kLds = sizeof(IdLists) + kTiles;
    static_assert(kCu * kLds <= 160 * 1024, "workgroups a CU");
};

// The first of n ascending sums that is above i.
template <class T>
__device__ inline uint32_t owner(const T *ends, uint32_t n, uint32_t i) {
    uint32_t lo = 0, hi = n - 1;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if (ends[mid] > i)
            hi = mid;
        else
            lo = mid + 1;
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

template <uint32_t ROWS, bool AROUND>
__global__ __launch_bounds__(64 * IdSets<ROWS>::kWaves, 2) void f8_id_k(F8Args a) {
    extern __shared__ __align__(16) uint8_t lds[];
    typedef IdSets<ROWS> Sets;
    constexpr uint32_t kWaves = Sets::kWaves, kHalf = Sets::kHalf, kFew = Sets::kFew;
    IdLists &list = *(IdLists *)lds;
    uint8_t *work = lds + sizeof(IdLists);
    // without a row list, packed row p is activation row p: those past xrows do not exist
    const int64_t end = (int64_t)(a.act ? a.n : min(a.n, a.xrows));
    const uint32_t n = a.n_expert;
    auto stretch = [&](uint32_t e, int64_t *lo) __attribute__((always_inline)) -> int64_t {
        *lo = max(a.bounds[e], 0);
        return min((int64_t)a.bounds[e + 1], end) - *lo;
    };
    // sums of the experts' sets: of more than kHalf rows, and in one word the others
    constexpr uint32_t kEach = kIdExperts / (64 * kWaves);
    uint32_t most[kEach], less[kEach], m = 0, l = 0;
#pragma unroll
    for (uint32_t i = 0; i < kEach; i++) {
        const uint32_t e = threadIdx.x * kEach + i;
        int64_t lo, rows = e < n ? stretch(e, &lo) : 0;
        rows = max(rows, (int64_t)0);
        const uint32_t rest = (uint32_t)rows % ROWS;
        m += (uint32_t)(rows / ROWS) + (rest > kHalf ? 1u : 0u);
        l += rest == 0 || rest > kHalf ? 0u : rest > kFew ? 1u << 16 : 1u;
        most[i] = m, less[i] = l;
    }
    uint32_t *tmp = (uint32_t *)work, vm = m, vl = l;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
#pragma unroll
    for (uint32_t d = 1; d < 64; d *= 2) {
        const uint32_t om = __shfl_up(vm, d, 64), ol = __shfl_up(vl, d, 64);
        if (lane >= d) vm += om, vl += ol;
    }
    if (lane == 63) tmp[wave] = vm, tmp[kWaves + wave] = vl;
    __syncthreads();
    uint32_t all_m = 0, all_l = 0;
    vm -= m, vl -= l;
    for (uint32_t i = 0; i < kWaves; i++) {
        if (i < wave) vm += tmp[i], vl += tmp[kWaves + i];
        all_m += tmp[i], all_l += tmp[kWaves + i];
    }
#pragma unroll
    for (uint32_t i = 0; i < kEach; i++) {
        const uint32_t e = threadIdx.x * kEach + i;
        list.most[e] = vm + most[i];
        list.half[e] = (uint16_t)((vl + less[i]) >> 16);
        list.few[e] = (uint16_t)(vl + less[i]);
    }
    __syncthreads();
    const uint32_t slices = (uint32_t)((a.w_rows + ROWS - 1) / ROWS);
    const uint32_t n_most = __builtin_amdgcn_readfirstlane(all_m);
    const uint32_t n_less = __builtin_amdgcn_readfirstlane(all_l), n_half = n_less >> 16;
    const uint64_t items = ((uint64_t)n_most + n_half + (n_less & 0xffffu)) * slices;
    for (uint64_t i = blockIdx.x; i < items; i += a.blocks) {
        const uint32_t unit = (uint32_t)(i / slices), part = (uint32_t)(i - (uint64_t)unit * slices);
        uint32_t e;
        int64_t lo, all, skip;
        if (unit < n_most) {
            e = owner(list.most, n, unit);
            const uint32_t before = e ? list.most[e - 1] : 0u;
            all = stretch(e, &lo);
            skip = (int64_t)__builtin_amdgcn_readfirstlane(unit - before) * ROWS;
        } else {
            e = unit - n_most < n_half ? owner(list.half, n, unit - n_most)
                                       : owner(list.few, n, unit - n_most - n_half);
            all = stretch(e, &lo);
            skip = all / ROWS * ROWS;
        }
        if (skip < 0 || skip >= all) continue;      // never, with bounds that ascend
        const uint32_t rows = (uint32_t)min((int64_t)ROWS, all - skip);
        const uint8_t *w = a.w + e * a.w_stride;
        const float *ws = (const float *)((const uint8_t *)a.ws + e * a.ws_stride);
        const uint64_t r0 = (uint64_t)part * ROWS, p0 = (uint64_t)(lo + skip), phi = p0 + rows;
        if (rows > kHalf) {
            tile<ROWS, ROWS, 2, kWaves / 2, Sets::kAllS, true, AROUND>(a, w, ws, r0, p0, phi, work);
        } else if (rows > kFew) {
            if constexpr (kHalf > 0)
                tile<kHalf, ROWS, 2, kWaves / 2, Sets::kHalfS, true, AROUND>(a, w, ws, r0, p0, phi, work);
        } else {
            if constexpr (kFew > 0)
                tile<kFew, ROWS, 2, kWaves / 2, Sets::kFewS, true, AROUND>(a, w, ws, r0, p0, phi, work);
        }
        __syncthreads();    // the next item overwrites what slower waves may still read
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

// LDS for activation rows: two workgroups a CU with a list and the waves' sums; three
constexpr size_t kFewAll = 80 * 1024;
constexpr size_t kFewLds = kFewAll - kSelList - kFewWaves * 64 * sizeof(v4f) - 16;
constexpr size_t kFewFour = 48 * 1024;
inline uint64_t few_lds(uint32_t rows, uint32_t seg) {
    return (uint64_t)rows * (few_code_ld(seg) + few_scale_ld(seg));
}
// Blocks of K at a time of `rows` activation rows a workgroup: all where they fit,
// else equal parts of whole chunks.
uint32_t few_seg(uint64_t cols, uint32_t rows) {
    const uint32_t nb = f8_blocks(cols);
    uint32_t parts = 1, seg;
    do {
        seg = ((nb + parts - 1) / parts + 1) / 2 * 2;
        parts++;
    } while (few_lds(rows, seg) > kFewLds && seg > 2);
    return seg;
}

// One set of `rows` (<= 16) activation rows a workgroup, `lists` of them, of
// which about `busy` have work.
//
// Waves a tile: as many as there are chunks, up to eight, while the whole launch
// has fewer than 8 waves a CU.  Workgroups have eight waves where a tile has, or
// where the rows leave LDS for no more than two of them, which then share them;
// else four (one row, us, four / eight: 2048 x 8192 11.6 / 9.8, 4096 x 4096 8.2 /
// 7.4, 8192 x 8192 16.2 / 18.6, 12288 x 8192 22.0 / 28.2; sixteen rows, 8192 x 8192
// 30.5 / 24.8).
//
// Three workgroups of four waves (two of eight) a CU, all with the same number of
// rounds: more of them at once ask memory for too many places (151936 x 2048, one
// row: two 56.8, three 58.1, four 67.2, six 63.8 us; 100000 x 1024: 26.4, 23.8,
// 24.2, 24.1).
typedef void (*F8Kernel)(F8Args);
template <F8Kernel EVEN, F8Kernel ODD>     // blocks of K
bool few_launch(F8Args &a, uint32_t rows, uint32_t lists, uint32_t busy, size_t extra,
                const char *name) {
    const uint64_t tiles = (a.w_rows + 15) / 16, all = tiles * busy, cus = cu_count();
    const uint32_t nb = f8_blocks(a.cols), chunks = (nb + 1) / 2;
    a.seg = few_seg(a.cols, rows);
    a.ks = 1;
    while (a.ks < kFewWaves && a.ks * 2 <= chunks && all * a.ks < 8 * cus) a.ks *= 2;
    a.waves = a.ks == kFewWaves || few_lds(rows, a.seg) > kFewFour ? kFewWaves : kFewWaves / 2;
    const size_t lds = extra + (few_lds(rows, a.seg) + 15) / 16 * 16 +
                       (a.ks > 1 ? a.waves * 64 * sizeof(v4f) : 0);
    const uint64_t sets = (tiles * a.ks + a.waves - 1) / a.waves;
    const uint64_t resident = std::max<uint64_t>(1, (a.waves == kFewWaves ? 2 : 3) * cus / busy);
    const uint64_t rounds = (sets + resident - 1) / resident;
    a.blocks = (uint32_t)((sets + rounds - 1) / rounds);
    static DynLds st[2];
    const F8Kernel k = nb % 2 ? ODD : EVEN;
    if (!dyn_lds_ok((const void *)k, lds, kFewAll, st[nb % 2], name)) return false;
    k<<<dim3(a.blocks, lists), dim3(64 * a.waves), lds, stream()>>>(a);
    return launch_ok(name);
}

// Outputs of more than 128 MiB go around the caches where rows begin at whole 64
// bytes: half of the last cache, so that who reads them next finds little there
// (product, and with the quantiser that reads it, us, through / around: 8192 x 9216 x
// 1024 bf16 177 / 181 and 210 / 211; 4096 x 54656 x 128 196 / 161 and 331 / 320; packed, 128
// experts, 20480 x 2048 x 1024 fp32 170 / 153 and 204 / 196).  Smaller ones stay for the
// reader, though the product alone would be shorter around them (2048 x 8192 x 1024
// fp32 45 / 43 and 55 / 57; 4096 x 8192 x 1024 bf16 76 / 75 and 93 / 97).  Rows at odd
// addresses would write parts of lines (4266 x 54613 x 128 210 / 247).
bool around(const F8Args &a) {
    return a.n * a.w_rows * type_bytes(a.y_type) > 128ull << 20 &&
           ((uintptr_t)a.y | a.ldy * type_bytes(a.y_type)) % 64 == 0;
}

template <uint32_t BM, uint32_t BN, uint32_t WM, uint32_t WN, uint32_t S, bool AROUND = false>
bool tile_launch(F8Args &a) {
    static DynLds st;
    constexpr size_t lds = tile_lds<BM, BN, S>();
    auto k = f8_tile_k<BM, BN, WM, WN, S, AROUND>;
    if (!dyn_lds_ok((const void *)k, lds, lds, st, "f8_tile_k")) return false;
    const uint64_t m = (a.n + BM - 1) / BM, n = (a.w_rows + BN - 1) / BN;
    if (m * n >= (1ull << 32) / (64 * WM * WN)) {    // threads along x; no 288 GB hold more
        set_error("q4mi_f8_mul: too many tiles");
        return false;
    }
    a.m_tiles = (uint32_t)m, a.blocks = (uint32_t)(m * n);
    k<<<dim3(a.blocks), dim3(64 * WM * WN), lds, stream()>>>(a);
    return launch_ok("f8_tile_k");
}

// Which kernel a product takes.
//
// While all its tiles are resident at once, the smallest of them, with as deep a
// ring as LDS has room for, so that every CU has a part (8192 x 8192, us: 64 rows, 32 x
// 32 26, 64 x 64 37; 128 rows, 32 x 32 49, 64 x 64 37, 128 x 64 57; 256 rows, 64 x 64
// 73, 128 x 64 58, 128 x 128 77; 512 rows, 128 x 64 113, 128 x 128 78, 256 x 128 108;
// 1024 rows, 128 x 128 154, 256 x 128 117).
//
// More tiles: of up to 128 rows those that hold them all, two workgroups a CU, so
// that the weights come once (151936 x 2048, us: 32 rows, 32 x 128 63, 32 x 32 84; 64
// rows, 64 x 128 75, 64 x 64 120; 128 rows, 128 x 128 105, in one workgroup a CU 123);
// else 128 x 128 as well (8192 x 8192 x 128, 2048, 8192: 49, 259, 960 us; 256 x 128 in
// one workgroup a CU 55, 262, 952).
bool mul_pick(F8Args &a) {
    const uint64_t cus = cu_count();
    auto tiles = [&](uint64_t bm, uint64_t bn) {
        return ((a.n + bm - 1) / bm) * ((a.w_rows + bn - 1) / bn);
    };
    if (a.n <= kFewRows)
        return few_launch<f8_few_k<true>, f8_few_k<false>>(a, (uint32_t)a.n, 1, 1, 0, "f8_few_k");
    if (tiles(32, 32) <= 2 * cus) return tile_launch<32, 32, 2, 2, 8>(a);
    if (a.n <= 32) return tile_launch<32, 128, 2, 2, 3>(a);
    if (tiles(64, 64) <= cus) return tile_launch<64, 64, 2, 2, 8>(a);
    if (a.n <= 64) return tile_launch<64, 128, 2, 2, 3>(a);
    if (tiles(128, 64) <= cus) return tile_launch<128, 64, 2, 2, 6>(a);
    if (tiles(128, 128) <= cus) return tile_launch<128, 128, 2, 2, 4>(a);
    if (a.n > 128 && tiles(256, 128) <= cus) return tile_launch<256, 128, 4, 2, 3>(a);
    return around(a) ? tile_launch<128, 128, 2, 2, 2, true>(a) : tile_launch<128, 128, 2, 2, 2>(a);
}

template <uint32_t ROWS, bool AROUND>
bool id_launch(F8Args &a) {
    constexpr size_t lds = IdSets<ROWS>::kLds;
    a.blocks = IdSets<ROWS>::kCu * (uint32_t)cu_count();
    static DynLds st;
    auto k = f8_id_k<ROWS, AROUND>;
    if (!dyn_lds_ok((const void *)k, lds, lds, st, "f8_id_k")) return false;
    k<<<dim3(a.blocks), dim3(64 * IdSets<ROWS>::kWaves), lds, stream()>>>(a);
    return launch_ok("f8_id_k");
}
template <uint32_t ROWS>
bool id_stores(F8Args &a) {
    constexpr bool kLarge = ROWS >= 128;
    return kLarge && around(a) ? id_launch<ROWS, kLarge>(a) : id_launch<ROWS, false>(a);
}

// Small sets with deep rings where the chip has room for all at once: then a set's
// stages in a row are the time (8 experts of 1024 x 2048, 32 rows each, us: sets of
// 32 rows 11.8, 64 15.1, 128 21.5; one of 2048 x 2048, 256 rows: 64 14.5, 128 26; 8 of
// 2048 x 2048, 128 rows each: 64 36.8, 128 30.5).
bool id_pick(F8Args &a) {
    const uint64_t cus = cu_count();
    auto sets = [&](uint64_t rows) {    // at most
        return (a.n / rows + std::min<uint64_t>(a.n, a.n_expert)) * ((a.w_rows + rows - 1) / rows);
    };
    if (sets(32) <= 2 * cus) return id_stores<32>(a);
    if (sets(64) <= cus) return id_stores<64>(a);
    return id_stores<128>(a);
}

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
    return mul_pick(a);
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
    // Groups from more rows on than a wave's tile holds and there are experts, or from 64
    // on: before, two rows of one expert find its weights in a cache (1024 x 2048, picks
    // even, us, alone / in groups: 10 of 128 7.7 / 8.5, 16 of 8 8.4 / 9.0, 32 of 8 12.2 /
    // 10.8, 40 of 128 15.7 / 17.1, 128 of 64 42 / 33, 128 of 8 38 / 17.6).
    const uint32_t lists = (uint32_t)n;
    if (n <= kFewRows || (n < 64 && n <= n_expert))
        return few_launch<f8_sel_k<true, false>, f8_sel_k<false, false>>(a, 1, lists, lists, 0,
                                                                         "f8_sel_k");
    // sets with work, at most; any n_expert is taken
    const uint64_t sets = std::min<uint64_t>(lists, (uint64_t)n_expert + lists / kFewRows);
    return few_launch<f8_sel_k<true, true>, f8_sel_k<false, true>>(
        a, std::min(lists, kFewRows), lists, (uint32_t)sets, kSelList, "f8_sel_k");
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
    return id_pick(a);
}

#ifdef Q4MI_MEASURE
uint64_t q4mi_f8_tile_scale_row(uint64_t w_rows, uint64_t r0, uint32_t first) {
    return tile_scale_row(w_rows, r0, first);
}
bool q4mi_f8_around(void *d_y, uint32_t y_type, uint64_t ld_y, uint64_t n, uint64_t w_rows) {
    F8Args a = {};
    a.y = d_y, a.y_type = y_type, a.ldy = ld_y, a.n = n, a.w_rows = w_rows;
    return around(a);
}
#endif

}  // extern "C"

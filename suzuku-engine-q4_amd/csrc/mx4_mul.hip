// Products of microscaled 4-bit rows (mx4.h has the format):
//   y[t][r] = sum over blocks b of 2^(sw + sx - 254) * sum_i w[r][32b+i] x[t][32b+i]
// on v_mfma_scale_f32_16x16x128_f8f6f4 and _32x32x64_f8f6f4: a lane holds one
// row's block of 32 codes and its scale byte, the sums are fp32.  Weight rows
// are the first operand, so a lane's sums are four adjacent outputs of one
// activation row.
//
// Three kernels: few rows (weights straight to registers), rows in tiles (both
// sides through LDS) and packed rows (both of these, per expert).
#include <algorithm>
#include <type_traits>

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
    uint32_t ks, seg, blocks;       // waves a tile, blocks of K in LDS, workgroups
    uint32_t m_tiles;               // tiles along the activations
};

__device__ inline v8i widen(u32x4 q) {
    const v8i a = {(int)q.x, (int)q.y, (int)q.z, (int)q.w, 0, 0, 0, 0};
    return a;
}

// Four adjacent outputs, rounded once.  STREAM: past the caches.
template <bool STREAM = false>
__device__ inline void store4(void *y, uint32_t yt, uint64_t at, v4f v) {
    if (yt == kTypeF32) {
        f32x4_a4 *p = (f32x4_a4 *)((float *)y + at);
        if constexpr (STREAM)
            __builtin_nontemporal_store((f32x4)v, p);
        else
            *p = v;
    } else {
        const u32x2 q = {f32_to_16x2(v[0], v[1], yt), f32_to_16x2(v[2], v[3], yt)};
        u32x2_a2 *p = (u32x2_a2 *)((uint16_t *)y + at);
        if constexpr (STREAM)
            __builtin_nontemporal_store(q, p);
        else
            *p = q;
    }
}

// ---------------------------------------------------------------- few rows
//
// Up to 16 * MT activation rows against all weight rows: bound by reading the
// weights once.  A wave takes 16 weight rows straight from memory into
// registers; lane (m, g) of it holds row m's blocks 4s + g of a chunk of 16
// blocks (s = 0..3), so four lanes read 64 adjacent bytes and a chunk's 16
// scales are one 16-byte load, of which step s uses byte g of dword s.  PF
// chunks (4 KB each with 16 rows) are multiplied while PF more are in flight.
// The activation rows sit in LDS, as codes, in groups of 16 for one instruction
// each: float rows are quantised on the way there, once a workgroup.  ks waves
// share a tile along K and their sums are joined in LDS in wave order, so a
// short matrix still occupies the chip; a workgroup goes over several tiles, so
// a tall one pays the LDS fill once.  LM head 151936 x 2048, one row: 30 us,
// 5.6 TB/s with part of the weights in the last cache; from memory alone 4.4
// TB/s for 16 rows (a large copy: 4.8).

constexpr uint32_t kFewRows = 16;

// LDS strides of a row's codes and scales, seg blocks: 16 bytes more than a
// power of two, so that the rows of a fragment start in different banks.
__host__ __device__ inline uint32_t few_code_ld(uint32_t seg) { return seg * 16u + 16u; }
__host__ __device__ inline uint32_t few_scale_ld(uint32_t seg) { return seg + 16u; }

// The activation rows of a workgroup: `rows` packed rows from p0 on, or those
// at the places that `list` (in LDS) names past p0.
struct FewRange {
    uint64_t p0;
    uint32_t rows, x_div;
    const int32_t *act;      // their activation rows; NULL: p / x_div
    const uint32_t *list;
    __device__ uint64_t row(uint32_t t) const { return p0 + (list ? list[t] : t); }
    __device__ int64_t x_row(uint32_t t, uint64_t xrows) const {
        if (!act) return x_div == 1 ? (int64_t)row(t) : (int64_t)((uint32_t)row(t) / x_div);
        const int64_t r = act[row(t)];
        return r < (int64_t)xrows ? r : -1;
    }
};

// Blocks [b0, b0 + seg) of the rows into LDS; blocks from nb on get codes 0
// and scale 1.
template <uint32_t NW, bool FLOATS>
__device__ inline void few_stage(const MulArgs &a, const FewRange &f, uint32_t b0, uint32_t seg,
                                 uint32_t nb, uint32_t sld, uint8_t *codes, uint8_t *scales) {
    const uint32_t cld = few_code_ld(seg), scld = few_scale_ld(seg);
    if (!FLOATS || a.x_type == kTypeMx4) {
        const uint32_t lane = threadIdx.x & 63u;
#pragma unroll 2
        for (uint32_t t = threadIdx.x >> 6; t < f.rows; t += NW) {
            const uint64_t xr = (uint64_t)max(f.x_row(t, a.xrows), (int64_t)0);
            const u32x4 *c = (const u32x4 *)((const uint8_t *)a.x + xr * (16ull * nb));
            const uint32_t *s = (const uint32_t *)(a.xs + xr * sld);
            for (uint32_t b = lane; b < seg; b += 64)
                *(u32x4 *)(codes + t * cld + 16u * b) =
                    b0 + b < nb ? c[b0 + b] : (u32x4){0, 0, 0, 0};
            for (uint32_t d = lane; d < seg / 4; d += 64) {
                const int32_t left = (int32_t)(nb - (b0 + 4 * d));
                const uint32_t in = left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1;
                const uint32_t v = left > 0 ? s[b0 / 4 + d] : 0u;
                *(uint32_t *)(scales + t * scld + 4u * d) = (v & in) | (0x7f7f7f7fu & ~in);
            }
        }
        return;
    }
    for (uint32_t i = threadIdx.x; i < f.rows * seg * 4; i += NW * 64) {
        const uint32_t sub = i & 3u, q = i >> 2, t = q / seg, b = q - t * seg;
        uint32_t code = 0, s = 127;
        if (b0 + b < nb) {
            float v[8];
            load_row8(a.x, a.x_type, (uint64_t)f.x_row(t, a.xrows) * a.ldx,
                      32u * (b0 + b) + 8u * sub, (uint32_t)a.cols, v);
            s = mx4_block_scale<8>(v);
            code = mx4_pack8(v, s);
        }
        *(uint32_t *)(codes + t * cld + 16u * b + 4u * sub) = code;
        if (sub == 0) scales[t * scld + b] = (uint8_t)s;
    }
}

// FULL: rows are whole chunks of 16 blocks.  Weight tiles [first, last), of
// which workgroup `block` of `blocks` takes every blocks-th set.
template <bool FULL, uint32_t PF, uint32_t MT, uint32_t NW, bool FLOATS>
__device__ inline void few_rows(const MulArgs &a, const uint8_t *w, const uint8_t *ws,
                                const FewRange &f, uint32_t first, uint32_t last, uint32_t block,
                                uint32_t blocks, uint8_t *lds) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t m = lane & 15u, g = lane >> 4;
    const uint32_t ks = a.ks, kw = wave & (ks - 1), sub = wave / ks, per = NW / ks;
    const uint32_t nb = mx4_blocks(a.cols), sld = mx4_scale_row(nb);
    const uint32_t seg = a.seg, nseg = (nb + seg - 1) / seg;
    const uint32_t cld = few_code_ld(seg), scld = few_scale_ld(seg);
    uint8_t *codes = lds, *scales = lds + f.rows * cld;
    v4f *red = (v4f *)(scales + f.rows * scld);
    uint32_t xc[MT], xsc[MT];       // this lane's row of every group, in codes and scales
#pragma unroll
    for (uint32_t n = 0; n < MT; n++) {
        const uint32_t t = min(16 * n + m, f.rows - 1);
        xc[n] = t * cld + 16u * g, xsc[n] = t * scld;
    }
    const uint32_t rounds = (last - first + per * blocks - 1) / (per * blocks);
    auto tile_of = [&](uint32_t i) { return first + (i * blocks + block) * per + sub; };
    auto chunks = [&](uint32_t sg) { return (min(seg, nb - sg * seg) + 15) / 16; };
    struct Batch {
        u32x4 codes[PF][4], scales[PF];
    };
    // chunks c, c + ks, .. (PF of them) of segment sg of round i's weight tile
    auto load = [&](Batch &q, uint32_t i, uint32_t sg, uint32_t c0) __attribute__((always_inline)) {
        const uint32_t tile = min(tile_of(i), last - 1), most = chunks(sg) - 1;
        const uint64_t wr = min((uint64_t)tile * 16 + m, a.w_rows - 1);
        const uint8_t *wp = w + wr * (16ull * nb), *wsp = ws + wr * sld;
#pragma unroll
        for (uint32_t j = 0; j < PF; j++) {
            const uint32_t bc = sg * seg + 16 * min(c0 + j * ks, most);
#pragma unroll
            for (uint32_t s = 0; s < 4; s++) {
                uint32_t b = bc + 4 * s + g;
                if (!FULL) b = min(b, nb - 1);
                q.codes[j][s] = *(const u32x4 *)(wp + 16u * b);
                if (!FULL) q.scales[j][s] = ((const uint32_t *)wsp)[min(bc / 4 + s, sld / 4 - 1)];
            }
            if (FULL) q.scales[j] = *(const u32x4_a4 *)(wsp + bc);
        }
    };
    v4f acc[MT];
    auto multiply = [&](const Batch &q, uint32_t sg, uint32_t c0) __attribute__((always_inline)) {
        const uint32_t nch = chunks(sg);
#pragma unroll
        for (uint32_t j = 0; j < PF; j++) {
            const uint32_t c = c0 + j * ks;
            if (c >= nch) break;
            u32x4 xv[MT];
#pragma unroll
            for (uint32_t n = 0; n < MT; n++) xv[n] = *(const u32x4 *)(scales + xsc[n] + 16u * c);
#pragma unroll
            for (uint32_t s = 0; s < 4; s++) {
                uint32_t wb = q.scales[j][s] >> (8 * g);
                if (!FULL && sg * seg + 16 * c + 4 * s + g >= nb) wb = 127;
#pragma unroll
                for (uint32_t n = 0; n < MT; n++) {
                    const u32x4 xq = *(const u32x4 *)(codes + xc[n] + 256u * c + 64u * s);
                    acc[n] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                        widen(q.codes[j][s]), widen(xq), acc[n], 4, 4, 0, (int)wb, 0,
                        (int)(xv[n][s] >> (8 * g)));
                }
                if (MT > 1) __builtin_amdgcn_sched_barrier(0);   // registers: one step's reads
            }
        }
    };
    auto finish = [&](uint32_t i) __attribute__((always_inline)) {
        if (ks > 1) {
            if (i) __syncthreads();   // the last round's sums have been read
#pragma unroll
            for (uint32_t n = 0; n < MT; n++) red[(wave * MT + n) * 64 + lane] = acc[n];
            __syncthreads();
            if (kw) return;
            for (uint32_t k = 1; k < ks; k++)
#pragma unroll
                for (uint32_t n = 0; n < MT; n++) acc[n] += red[((wave + k) * MT + n) * 64 + lane];
        }
        const uint32_t tile = tile_of(i);
        if (tile >= last) return;
        const uint64_t r = (uint64_t)tile * 16 + 4 * g;
#pragma unroll
        for (uint32_t n = 0; n < MT; n++) {
            const uint32_t t = 16 * n + m;
            if (t >= f.rows || f.x_row(t, a.xrows) < 0) continue;
            const uint64_t at = f.row(t) * a.ldy + r;
            if (r + 4 <= a.w_rows)
                store4(a.y, a.y_type, at, acc[n]);
            else
                for (uint32_t k = 0; k < 4; k++)
                    if (r + k < a.w_rows) store_from_f32(a.y, a.y_type, at + k, acc[n][k]);
        }
    };
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t n = 0; n < MT; n++) acc[n] = (v4f){0.f, 0.f, 0.f, 0.f};
    };

    // The next batch, of this tile or of the next round's, is on its way while
    // one is multiplied, the first one while the activations are staged.  Every
    // wave goes through every segment of every round, so all meet the barriers.
    Batch now, then;
    uint32_t i = 0, sg = 0, c0 = kw;
    load(now, 0, 0, kw);
    few_stage<NW, FLOATS>(a, f, 0, seg, nb, sld, codes, scales);
    __syncthreads();
    clear();
    for (;;) {
        uint32_t ni = i, nsg = sg, nc = c0 + PF * ks;
        const bool done = nc >= chunks(sg);
        if (done) {
            nc = kw;
            if (++nsg == nseg) nsg = 0, ni++;
        }
        const bool more = ni < rounds;
        if (more) load(then, ni, nsg, nc);
        multiply(now, sg, c0);
        if (ni != i) {
            finish(i);
            clear();
        }
        if (!more) break;
        if (done && nseg > 1) {
            __syncthreads();
            few_stage<NW, FLOATS>(a, f, nsg * seg, seg, nb, sld, codes, scales);
            __syncthreads();
        }
        now = then, i = ni, sg = nsg, c0 = nc;
    }
}

// Sets of up to 16 * MT rows, by how many groups are there.
template <bool FULL, uint32_t PF, uint32_t MT, uint32_t NW>
__device__ inline void few_groups(const MulArgs &a, const uint8_t *w, const uint8_t *ws,
                                  const FewRange &f, uint32_t first, uint32_t last,
                                  uint32_t block, uint32_t blocks, uint8_t *lds) {
    static_assert(MT <= 2, "one or two groups");
    if (MT == 1 || f.rows <= 16)
        few_rows<FULL, PF, 1, NW, MT == 1>(a, w, ws, f, first, last, block, blocks, lds);
    else
        few_rows<FULL, PF, MT, NW, false>(a, w, ws, f, first, last, block, blocks, lds);
}

__device__ inline uint32_t row_tiles(const MulArgs &a) { return (uint32_t)((a.w_rows + 15) / 16); }

// Dense: grid (blocks, sets of 16 * MT activation rows).
template <bool FULL, uint32_t MT, uint32_t NW>
__global__ __launch_bounds__(64 * NW, MT > 1 ? 4 : 1) void mx4_few_k(MulArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    const uint64_t p0 = (uint64_t)blockIdx.y * 16 * MT;
    const FewRange f = {p0, (uint32_t)min((uint64_t)16 * MT, a.n - p0), 1, nullptr,
                        nullptr};
    few_groups<FULL, 1, MT, NW>(a, a.w, a.ws, f, 0, row_tiles(a), blockIdx.x, a.blocks, lds);
}

// Rows through the experts that the list names; grid (blocks, rows).  GROUP:
// rows of one expert among 256 go together, sixteen at a time, so that its
// weights are read once: the first of them does the work, the others'
// workgroups end.
constexpr size_t kSelList = 4 * 8 + kFewRows * 4;
template <bool FULL, bool GROUP>
__global__ __launch_bounds__(256) void mx4_sel_k(MulArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    uint64_t *same = (uint64_t *)lds;           // which of the 256 rows are of this expert
    uint32_t *list = (uint32_t *)(same + 4);
    const uint32_t p = blockIdx.y, p0 = p & ~255u, q = p0 + threadIdx.x;
    const int32_t e = a.eid[p];
    if (e < 0 || (uint32_t)e >= a.n_expert) return;
    const uint8_t *w = a.w + e * a.w_stride, *ws = a.ws + e * a.ws_stride;
    if constexpr (!GROUP) {
        const FewRange f = {p, 1, a.x_div, nullptr, nullptr};
        few_groups<FULL, 1, 1, 4>(a, w, ws, f, 0, row_tiles(a), blockIdx.x, a.blocks, lds);
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
    FewRange f = {p, rows, a.x_div, nullptr, nullptr};
    if (rows > 1) {
        const uint32_t mine = before(threadIdx.x) - rank;
        if ((same[threadIdx.x >> 6] >> (threadIdx.x & 63u) & 1u) && mine < rows)
            list[mine] = threadIdx.x;
        __syncthreads();
        f.p0 = p0, f.list = list;
    }
    few_groups<FULL, 1, 1, 4>(a, w, ws, f, 0, row_tiles(a), blockIdx.x, a.blocks, lds + kSelList);
}

// ------------------------------------------------------------ rows in tiles
//
// BM activation rows x BN weight rows a workgroup of WM x WN waves, on
// v_mfma_scale_f32_32x32x64_f8f6f4.  K goes in stages of 8 blocks (256
// values): 128 bytes of codes a row, a whole cache line, come by global -> LDS
// copies into one of two buffers while the matrix units work on the other.
// Scales come for four stages at once (32 bytes a row, a quarter of the copies
// a stage): with 8 bytes a row and stage they asked the L2 for as many lines
// as the codes.  Lane (row, half h) of a fragment takes blocks 4h + s of the
// stage (s = 0..3), so one dword holds its scales and step s picks a byte of
// it in the instruction.
//
// LDS places: chunk c (16 bytes) of codes row r at c ^ ((r >> 1) & 7), dword d
// of scales row r at d ^ ((r >> 3) & 7), so that a fragment's reads spread over
// all 64 banks; the copies fill LDS in lane order, so the lanes permute their
// source addresses instead.

typedef float v16f __attribute__((ext_vector_type(16)));

__device__ inline uint32_t tile_swz(uint32_t row) { return (row >> 1) & 7u; }

// Lane i's 16 (4) bytes land at LDS address lds + 16 i (4 i); from a pointer,
// or from a uniform base and a 32-bit offset.  Inline asm, so that the
// compiler adds no wait before the next LDS read.  Nor does it see that a base
// is read: one that a vector instruction wrote (a spilled one read back) needs
// five wait states, which the move and the s_nop 3 are.
__device__ inline void copy16(const void *g, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g),
                 "s"(lds)
                 : "memory", "m0");
}
__device__ inline void copy16(const void *base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off),
                 "s"(base), "s"(lds)
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
// This wave's copies have landed and its LDS reads are done; then the
// workgroup meets.
__device__ inline void stage_barrier() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// LDS: two stages of codes, two windows (four stages) of scales.
template <uint32_t BM, uint32_t BN>
constexpr uint32_t tile_lds() { return (BM + BN) * 2 * (128 + 32); }

// Weight rows [r0, r0 + BN) of w against activation rows [p0, p0 + BM), of
// which those below phi exist; the row read for p is act[p] with GATHER, else
// p.  Rows past either end are read as the last one and not stored.
template <uint32_t BM, uint32_t BN, uint32_t WM, uint32_t WN, bool GATHER>
__device__ inline void tile(const MulArgs &a, const uint8_t *w, const uint8_t *ws, uint64_t r0,
                            int64_t p0, int64_t phi, uint8_t *lds) {
    constexpr uint32_t NW = WM * WN;
    constexpr uint32_t FM = BM / (32 * WM), FN = BN / (32 * WN);
    constexpr uint32_t RA = BM / 8 / NW, RB = BN / 8 / NW;   // 8-row copies of each side a wave
    static_assert(FM && FN && RA && RB, "tile and waves");
    constexpr uint32_t kStage = (BM + BN) * 128, kWindow = (BM + BN) * 32, kScales = 2 * kStage;
    const uint32_t lane = threadIdx.x & 63u, l8 = lane >> 3;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t nb = mx4_blocks(a.cols), sld = mx4_scale_row(nb), nk = (nb + 7) / 8;
    const uint32_t row_bytes = 16u * nb;
    const uint32_t base = (uint32_t)(uintptr_t)lds;     // LDS offset: low half of the address

    // sources of this lane's part of every copy, without the place in K: row
    // pointers with GATHER, else offsets from the tile's first row
    const uint8_t *xc = (const uint8_t *)a.x, *xs = a.xs;
    const uint8_t *xp[GATHER ? RA : 1], *xsp[GATHER ? RA : 1];
    uint32_t xo[RA], wo[RB];
    if (!GATHER) xc += (uint64_t)p0 * row_bytes, xs += (uint64_t)p0 * sld;
    w += r0 * row_bytes, ws += r0 * sld;
    const uint32_t xlast = (uint32_t)min((int64_t)BM, phi - p0) - 1;
    const uint32_t wlast = (uint32_t)min((uint64_t)BN, a.w_rows - r0) - 1;
    auto gathered = [&](uint32_t m) -> uint64_t {
        const int64_t r = a.act ? (int64_t)a.act[p0 + m] : p0 + m;
        return r < 0 || r >= (int64_t)a.xrows ? 0 : (uint64_t)r;
    };
#pragma unroll
    for (uint32_t j = 0; j < RA; j++) {
        const uint32_t m = min((wave * RA + j) * 8 + l8, xlast);
        if constexpr (GATHER) {
            xp[j] = xc + gathered(m) * row_bytes;
            xsp[j] = xs + gathered(min((wave + NW * j) * 8 + l8, xlast)) * sld;
        } else {
            xo[j] = m * row_bytes;
        }
    }
#pragma unroll
    for (uint32_t j = 0; j < RB; j++) wo[j] = min((wave * RB + j) * 8 + l8, wlast) * row_bytes;
    // Part i of FM of stage k's codes; blocks past the last are read as the last.
    const uint32_t c0 = (lane & 7u) ^ (l8 >> 1);        // chunk of an even copy; c0 ^ 4 of an odd
    auto fetch = [&](uint32_t k, uint32_t i) __attribute__((always_inline)) {
        const uint32_t to = base + (k & 1u) * kStage;
        const uint32_t at[2] = {16u * min(8 * k + c0, nb - 1),
                                16u * min(8 * k + (c0 ^ 4u), nb - 1)};
#pragma unroll
        for (uint32_t j = 0; j < RA; j++) {
            if (j % FM != i) continue;
            const uint32_t c = wave * RA + j, d = to + c * 1024;
            if constexpr (GATHER)
                copy16(xp[j] + at[c & 1u], d);
            else
                copy16(xc, xo[j] + at[c & 1u], d);
        }
#pragma unroll
        for (uint32_t j = 0; j < RB; j++) {
            if (j % FM != i) continue;
            const uint32_t c = wave * RB + j;
            copy16(w, wo[j] + at[c & 1u], to + BM * 128 + c * 1024);
        }
    };
    // Quarter q of window v's scales (a side with fewer than four copies a wave
    // makes some of them twice); dwords past the last are read as the last.
    auto fetch_scales = [&](uint32_t v, uint32_t q) __attribute__((always_inline)) {
        const uint32_t to = base + kScales + (v & 1u) * kWindow;
        constexpr uint32_t QA = (RA + 3) / 4, QB = (RB + 3) / 4;
#pragma unroll
        for (uint32_t u = 0; u < QA; u++) {
            const uint32_t i = (q * QA + u) % RA, c = wave + NW * i;
            const uint32_t at = 4u * min(8 * v + ((lane & 7u) ^ (c & 7u)), sld / 4 - 1);
            if constexpr (GATHER) {
                const uint8_t *g = xsp[0];
#pragma unroll
                for (uint32_t j = 1; j < RA; j++) {
                    const uint64_t d = (uint64_t)xsp[j] - (uint64_t)xsp[j - 1];
                    g += i >= j ? d : 0;     // sums, not a choice of places: those would be memory
                }
                copy4(g + at, to + c * 256);
            } else {
                copy4(xs, min(c * 8 + l8, xlast) * sld + at, to + c * 256);
            }
        }
#pragma unroll
        for (uint32_t u = 0; u < QB; u++) {
            const uint32_t c = wave + NW * ((q * QB + u) % RB);
            const uint32_t at = 4u * min(8 * v + ((lane & 7u) ^ (c & 7u)), sld / 4 - 1);
            copy4(ws, min(c * 8 + l8, wlast) * sld + at, to + BM * 32 + c * 256);
        }
    };
    // The last stage, landed: zeros for the activations' blocks past the end.
    auto clear_tail = [&]() __attribute__((always_inline)) {
        const uint32_t first = nb & 7u, st = (nk - 1) & 1u;
        for (uint32_t i = threadIdx.x; i < BM * 8; i += 64 * NW)
            if (((i & 7u) ^ tile_swz(i >> 3)) >= first)
                *(u32x4 *)(lds + st * kStage + 16 * i) = (u32x4){0, 0, 0, 0};
        __syncthreads();
    };
    const uint32_t wm = wave / WN, wn = wave % WN, lr = lane & 31u, h = lane >> 5;
    const uint32_t ra = wm * FM * 32 + lr, rb = wn * FN * 32 + lr;
    uint32_t off[4];
#pragma unroll
    for (uint32_t s = 0; s < 4; s++) off[s] = 16u * ((4 * h + s) ^ tile_swz(lr));

    v16f acc[FM][FN];
#pragma unroll
    for (uint32_t i = 0; i < FM; i++)
#pragma unroll
        for (uint32_t j = 0; j < FN; j++)
#pragma unroll
            for (uint32_t q = 0; q < 16; q++) acc[i][j][q] = 0.f;

    // scales of stage k, a dword a fragment; 1 past the row's end, where the
    // bytes may say NaN
    auto read_scales = [&](uint32_t k, uint32_t *sx, uint32_t *sw) __attribute__((always_inline)) {
        const uint8_t *sc = lds + kScales + ((k >> 2) & 1u) * kWindow;
        const uint32_t d = 2 * (k & 3u) + h;
        const int32_t left = (int32_t)(nb - (8 * k + 4 * h));      // blocks of this lane's four
        const uint32_t in = left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1;
        auto one = [&](uint32_t row, uint32_t r) __attribute__((always_inline)) {
            const uint32_t v = *(const uint32_t *)(sc + row * 32 + 4 * (d ^ ((r >> 3) & 7u)));
            return (v & in) | (0x7f7f7f7fu & ~in);
        };
#pragma unroll
        for (uint32_t i = 0; i < FM; i++) sx[i] = one(ra + 32 * i, ra + 32 * i);
#pragma unroll
        for (uint32_t j = 0; j < FN; j++) sw[j] = one(BM + rb + 32 * j, rb + 32 * j);
    };
    auto read_codes = [&](uint32_t k, uint32_t s, u32x4 *xq, u32x4 *wq)
        __attribute__((always_inline)) {
        const uint8_t *st = lds + (k & 1u) * kStage + off[s];
#pragma unroll
        for (uint32_t i = 0; i < FM; i++) xq[i] = *(const u32x4 *)(st + (ra + 32 * i) * 128);
#pragma unroll
        for (uint32_t j = 0; j < FN; j++) wq[j] = *(const u32x4 *)(st + (BM + rb + 32 * j) * 128);
    };
    auto multiply = [&](auto s_, uint32_t i, const u32x4 *xq, const u32x4 *wq, const uint32_t *sx,
                        const uint32_t *sw) __attribute__((always_inline)) {
        constexpr uint32_t s = decltype(s_)::value;
#pragma unroll
        for (uint32_t j = 0; j < FN; j++)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                widen(wq[j]), widen(xq[i]), acc[i][j], 4, 4, s, (int)sw[j], s, (int)sx[i]);
    };

    // Barrier t says that stage t has landed and that stage t - 1 is read.  It
    // stands before the last products of stage t - 1, whose operands are in
    // registers: they cover the first reads of stage t, and stage t + 1's
    // copies have a whole stage of products to land.  The scheduling barriers
    // keep the reads one step ahead of the products, no further.
    u32x4 xa[FM], wa[FN], xb[FM], wb[FN];
    uint32_t sx[FM], sw[FN], nx[FM], nw[FN];
    const std::integral_constant<uint32_t, 0> s0{};
    const std::integral_constant<uint32_t, 1> s1{};
    const std::integral_constant<uint32_t, 2> s2{};
    const std::integral_constant<uint32_t, 3> s3{};
    auto all = [&](auto s_, const u32x4 *xq, const u32x4 *wq) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t i = 0; i < FM; i++) multiply(s_, i, xq, wq, sx, sw);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto three = [&](uint32_t k) __attribute__((always_inline)) {
        read_codes(k, 1, xb, wb);
        all(s0, xa, wa);
        read_codes(k, 2, xa, wa);
        all(s1, xb, wb);
        read_codes(k, 3, xb, wb);
        all(s2, xa, wa);
    };
    auto next = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t i = 0; i < FM; i++) sx[i] = nx[i];
#pragma unroll
        for (uint32_t j = 0; j < FN; j++) sw[j] = nw[j];
    };

#pragma unroll
    for (uint32_t q = 0; q < 4; q++) fetch_scales(0, q);
#pragma unroll
    for (uint32_t i = 0; i < FM; i++) fetch(0, i);
    stage_barrier();
    if (1 < nk) {
#pragma unroll
        for (uint32_t i = 0; i < FM; i++) fetch(1, i);
        fetch_scales(1, 0);
    } else if (nb & 7u) {
        clear_tail();
    }
    read_scales(0, sx, sw);
    read_codes(0, 0, xa, wa);
    uint32_t k = 0;
    for (; k + 2 < nk; k++) {
        three(k);
        stage_barrier();
        read_scales(k + 1, nx, nw);
        read_codes(k + 1, 0, xa, wa);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (uint32_t i = 0; i < FM; i++) {
            multiply(s3, i, xb, wb, sx, sw);
            fetch(k + 2, i);
            __builtin_amdgcn_sched_barrier(0);
        }
        fetch_scales(((k + 1) >> 2) + 1, (k + 1) & 3u);
        next();
    }
    if (k + 1 < nk) {
        three(k);
        stage_barrier();
        if (nb & 7u) clear_tail();
        read_scales(k + 1, nx, nw);
        read_codes(k + 1, 0, xa, wa);
        all(s3, xb, wb);
        next();
        k++;
    }
    three(k);
    all(s3, xb, wb);

    // Sums of 32 activation rows at a time through LDS (the stages are read),
    // so that a wave stores whole stretches of an output row: lane (row lr, h)
    // holds weight rows 8q + 4h + 0..3 of its fragments.
    constexpr uint32_t kRow = FN * 32 + 4, kLanes = FN * 8;   // floats a row, lanes that store one
    // The largest tile stores past the caches, whatever its output's size.  That
    // pays for outputs that the caches cannot hold and costs below (us through
    // them / past them, bf16 out, alone and with a quantiser that reads it:
    // 16384 rows x 16384 x 1024, 512 MiB, 259 / 222 and 397 / 383; 8192 x 16384
    // x 2048, 256 MiB, 169 / 171 and 253 / 234; 8192 x 8192 x 2048, 128 MiB,
    // 85 / 93 and 113 / 126; 4096 x 8192 x 4096, 64 MiB, 76 / 79 and 91 / 97;
    // 2048 x 8192 x 8192, 32 MiB, 80 / 80 and 83 / 83).
    constexpr bool kStream = BM * BN >= 65536;
    static_assert(NW * 32 * kRow * 4 <= tile_lds<BM, BN>(), "sums fit the stages");
    float *sums = (float *)lds + wave * 32 * kRow;
    const uint64_t rw = r0 + wn * FN * 32 + lane % kLanes * 4;   // weight row of this lane's stores
    const bool whole = r0 + (wn + 1) * FN * 32 <= a.w_rows;
    auto listed = [&](int64_t p) {      // whether row p has an activation row
        return !GATHER || !a.act || (a.act[p] >= 0 && (int64_t)a.act[p] < (int64_t)a.xrows);
    };
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < FM; i++) {
#pragma unroll
        for (uint32_t j = 0; j < FN; j++)
#pragma unroll
            for (uint32_t q = 0; q < 4; q++)
                *(v4f *)(sums + lr * kRow + 32 * j + 8 * q + 4 * h) =
                    (v4f){acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2],
                          acc[i][j][4 * q + 3]};
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const int64_t p1 = p0 + (wm * FM + i) * 32;
        if (whole && p1 + 32 <= phi) {
            constexpr uint32_t kStep = 64 / kLanes;
#pragma unroll
            for (uint32_t u = 0; u < 32 / kStep; u++) {
                const uint32_t m = u * kStep + lane / kLanes;
                const v4f v = *(const v4f *)(sums + m * kRow + lane % kLanes * 4);
                if (listed(p1 + m)) store4<kStream>(a.y, a.y_type, (p1 + m) * a.ldy + rw, v);
            }
        } else {
#pragma unroll 1
            for (uint32_t m = lane / kLanes; m < 32 && p1 + m < phi; m += 64 / kLanes) {
                const int64_t p = p1 + m;
                if (!listed(p)) continue;
                const v4f v = *(const v4f *)(sums + m * kRow + lane % kLanes * 4);
                const uint64_t at = p * a.ldy + rw;
                if (rw + 4 <= a.w_rows)
                    store4(a.y, a.y_type, at, v);
                else
                    for (uint32_t n = 0; n < 4; n++)
                        if (rw + n < a.w_rows) store_from_f32(a.y, a.y_type, at + n, v[n]);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// Tiles of a dense product, `a.blocks` of them, a.m_tiles along the
// activations.  Workgroups go to the eight dies in turn, each with an L2 of
// its own: a die takes a contiguous run of tiles, in groups of kGroup
// activation tiles, so that its L2 holds what its tiles share.
constexpr uint32_t kGroup = 8;
template <uint32_t BM, uint32_t BN, uint32_t WM, uint32_t WN, uint32_t WAVES>
__global__ __launch_bounds__(64 * WM * WN, WAVES) void mx4_dense_k(MulArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    const uint32_t die = blockIdx.x & 7u, i = blockIdx.x >> 3;
    const uint32_t q = a.blocks >> 3, rem = a.blocks & 7u;
    const uint32_t t = die * q + min(die, rem) + i;
    const uint32_t n_tiles = a.blocks / a.m_tiles;
    const uint32_t group = t / (kGroup * n_tiles), in = t - group * kGroup * n_tiles;
    const uint32_t gm = min(kGroup, a.m_tiles - group * kGroup);
    const uint32_t mt = group * kGroup + in % gm, nt = in / gm;
    tile<BM, BN, WM, WN, false>(a, a.w, a.ws, (uint64_t)nt * BN, (int64_t)mt * BM, (int64_t)a.n,
                                lds);
}

// ------------------------------------------------------------- packed rows
//
// Experts differ: of a prompt's, a few take most of the rows and many take a
// handful.  One persistent workgroup a CU goes over two lists: tiles of kIdM
// rows x kIdN weight rows of the experts with more than kIdFew rows (bound by
// the matrix units), and the other experts' 16-row weight tiles, each streamed
// once past all of its expert's rows (bound by memory).  Of the second list a
// workgroup takes one stretch, so that it stages few experts' rows, shorter by
// kIdCost tiles for each large tile that it has (18 of them take as long as
// one; 512 experts' 1024 x 2048 over 4096 tokens, 256 experts' 1280 x 2560 over
// 333: 234 and 122 us at 14, 226 and 118 at 18, 226 and 121 at 22, 230 and 120
// at 26).
// Every second workgroup begins with the streamed tiles, so that memory and
// matrix units work at the same time (188 us all alike, 175 so).
//
// Every workgroup makes the lists by itself, as prefix sums over the experts'
// stretches in LDS (under 5 us with nothing to do): no scratch in memory, no
// launch before, and no workgroups that find nothing to do, of which a grid
// over experts, slices and tiles has tens of thousands (347 us, then 191).
constexpr uint32_t kIdM = 128, kIdN = 256, kIdWM = 2, kIdWN = 4, kIdWaves = kIdWM * kIdWN;
constexpr uint32_t kIdFew = 32, kIdExperts = 1024, kIdCost = 18;
constexpr size_t kIdLists = 2 * (kIdExperts + 1) * 4;

// Sums over a workgroup's threads, before this one and over all.
struct IdCounts {
    uint32_t tiles, few, sets;      // large tiles; streamed sets of kIdFew rows beside them, or alone
    __device__ void add(const IdCounts &o) { tiles += o.tiles, few += o.few, sets += o.sets; }
};
__device__ inline IdCounts block_sums(IdCounts v, IdCounts *tmp, IdCounts *all) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const IdCounts own = v;
#pragma unroll
    for (uint32_t d = 1; d < 64; d *= 2) {
        const IdCounts o = {__shfl_up(v.tiles, d, 64), __shfl_up(v.few, d, 64),
                            __shfl_up(v.sets, d, 64)};
        if (lane >= d) v.add(o);
    }
    if (lane == 63) tmp[wave] = v;
    __syncthreads();
    *all = {0, 0, 0};
    for (uint32_t w = 0; w < kIdWaves; w++) {
        if (w < wave) v.add(tmp[w]);
        all->add(tmp[w]);
    }
    __syncthreads();
    return {v.tiles - own.tiles, v.few - own.few, v.sets - own.sets};
}

// The last e with list[e] <= i, of n + 1 ascending sums.
__device__ inline uint32_t owner(const uint32_t *list, uint32_t n, uint32_t i) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (list[mid] <= i)
            lo = mid;
        else
            hi = mid;
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

template <bool FULL>
__global__ __launch_bounds__(64 * kIdWaves, 2) void mx4_id_k(MulArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    uint32_t *tiles = (uint32_t *)lds, *shares = tiles + kIdExperts + 1;
    uint8_t *work = lds + (kIdLists + 15) / 16 * 16;
    // without a row list, packed row p is activation row p: those past xrows do not exist
    const int64_t end = (int64_t)(a.act ? a.n : min(a.n, a.xrows));
    const uint32_t n = a.n_expert;
    auto stretch = [&](uint32_t e, int64_t *lo) __attribute__((always_inline)) -> int64_t {
        *lo = max(a.bounds[e], 0);
        return min((int64_t)a.bounds[e + 1], end) - *lo;
    };
    constexpr uint32_t kEach = kIdExperts / (64 * kIdWaves);
    IdCounts mine[kEach], sum = {0, 0, 0}, total;
#pragma unroll
    for (uint32_t i = 0; i < kEach; i++) {
        const uint32_t e = threadIdx.x * kEach + i;
        int64_t lo, rows = e < n ? stretch(e, &lo) : 0;
        const uint32_t some = (uint32_t)max(rows, (int64_t)0);
        mine[i] = {some > kIdFew ? (some + kIdM - 1) / kIdM : 0u,
                   some > 0 && some <= kIdFew ? 1u : 0u, (some + kIdFew - 1) / kIdFew};
        sum.add(mine[i]);
    }
    IdCounts at = block_sums(sum, (IdCounts *)work, &total);
    const uint32_t slices = (uint32_t)((a.w_rows + kIdN - 1) / kIdN), per = row_tiles(a);
    // Large tiles, unless streaming every expert in sets of kIdFew rows takes less
    // of the longest workgroup's time, as where there are few of either.
    const uint64_t items = (uint64_t)total.tiles * slices;
    const uint64_t longest = max((items + a.blocks - 1) / a.blocks * kIdCost,
                                 ((uint64_t)total.few * per + items * kIdCost) / a.blocks);
    const bool large = longest <= ((uint64_t)total.sets * per + a.blocks - 1) / a.blocks;
#pragma unroll
    for (uint32_t i = 0; i < kEach; i++) {
        const uint32_t e = threadIdx.x * kEach + i;
        if (e <= n) tiles[e] = at.tiles, shares[e] = large ? at.few : at.sets;
        at.add(mine[i]);
    }
    if (threadIdx.x == 0)
        tiles[n] = total.tiles, shares[n] = large ? total.few : total.sets;
    __syncthreads();
    const uint32_t heavy = large ? total.tiles * slices : 0u;
    // this workgroup's stretch of the others' tiles
    const uint64_t few = (uint64_t)shares[n] * per, all = few + (uint64_t)heavy * kIdCost;
    const uint64_t fair = (all + a.blocks - 1) / a.blocks;
    const uint32_t q = heavy / a.blocks, more = heavy - q * a.blocks;   // large tiles of each
    const uint64_t less = (uint64_t)q * kIdCost;
    const uint64_t s0 = fair > less ? fair - less : 0;                  // with q of them
    const uint64_t s1 = fair > less + kIdCost ? fair - less - kIdCost : 0;
    auto start = [&](uint32_t b) -> uint64_t {
        return min(few, b < more ? b * s1 : more * s1 + (b - more) * s0);
    };
    // every second workgroup of a die takes the streamed tiles first
    for (uint32_t phase = 0; phase < 2; phase++) {
        if (phase == ((blockIdx.x >> 3) & 1u)) {
            for (uint32_t i = blockIdx.x; i < heavy; i += a.blocks) {
                const uint32_t unit = i / slices, part = i - unit * slices;
                const uint32_t e = owner(tiles, n, unit);
                int64_t lo;
                const int64_t rows = stretch(e, &lo), skip = (int64_t)(unit - tiles[e]) * kIdM;
                if (skip < rows)    // always, with bounds that ascend
                    tile<kIdM, kIdN, kIdWM, kIdWN, true>(
                        a, a.w + e * a.w_stride, a.ws + e * a.ws_stride, (uint64_t)part * kIdN,
                        lo + skip, lo + rows, work);
                __syncthreads();    // the next item overwrites what slower waves may still read
            }
            continue;
        }
        const uint64_t end_t = start(blockIdx.x + 1);
        for (uint64_t t = start(blockIdx.x); t < end_t;) {
            const uint32_t unit = (uint32_t)(t / per), first = (uint32_t)(t - (uint64_t)unit * per);
            const uint32_t last = (uint32_t)min((uint64_t)per, first + (end_t - t));
            const uint32_t e = owner(shares, n, unit);
            int64_t lo;
            const int64_t rows = stretch(e, &lo), skip = (int64_t)(unit - shares[e]) * kIdFew;
            const FewRange f = {(uint64_t)(lo + skip),
                                (uint32_t)min((int64_t)kIdFew, rows - skip), 1, a.act, nullptr};
            if (skip >= rows) break;    // never, with bounds that ascend
            few_groups<FULL, 2, kIdFew / 16, kIdWaves>(a, a.w + e * a.w_stride,
                                                       a.ws + e * a.ws_stride, f, first, last, 0,
                                                       1, work);
            t += last - first;
            __syncthreads();    // as above
        }
    }
}

// rows: whether the call has any; without, their pointers may be NULL.
bool mul_ok(const char *who, const MulArgs &a, bool rows) {
    if (!a.w || !a.ws || (rows && (!a.x || !a.y)) || !a.w_rows || !a.cols) {
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
    if (a.x_type == kTypeMx4 ? (rows && !a.xs) || ((uintptr_t)a.x & 15) || ((uintptr_t)a.xs & 3)
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

template <uint32_t BM, uint32_t BN, uint32_t WM, uint32_t WN, uint32_t WAVES>
bool dense_launch(MulArgs &a) {
    static DynLds st;
    constexpr size_t lds = tile_lds<BM, BN>();
    auto k = mx4_dense_k<BM, BN, WM, WN, WAVES>;
    if (!dyn_lds_ok((const void *)k, lds, lds, st, "mx4_dense_k")) return false;
    const uint64_t m = (a.n + BM - 1) / BM, n = (a.w_rows + BN - 1) / BN;
    if (m * n > 0x7fffffffu) {
        set_error("q4mi_mx4_mul: too many tiles");
        return false;
    }
    a.m_tiles = (uint32_t)m, a.blocks = (uint32_t)(m * n);
    k<<<dim3(a.blocks), dim3(64 * WM * WN), lds, stream()>>>(a);
    return launch_ok("mx4_dense_k");
}

// K segment of the few-rows kernels for `rows` activation rows a workgroup of
// `waves`: whole rows where they fit in `room` bytes, else equal parts of whole
// chunks; returns the LDS bytes.
size_t few_fit(MulArgs &a, uint32_t rows, uint32_t groups, uint32_t waves, size_t room) {
    const uint32_t nb = mx4_blocks(a.cols);
    uint32_t parts = 1;
    size_t need;
    do {
        a.seg = ((nb + parts - 1) / parts + 15) / 16 * 16;
        need = (size_t)rows * (few_code_ld(a.seg) + few_scale_ld(a.seg));
        parts++;
    } while (need > room && a.seg > 16);
    return need + (a.ks > 1 ? (size_t)waves * groups * 64 * sizeof(v4f) : 0);
}

// Waves a weight tile: as many as there are chunks, while the whole launch has
// fewer than 8 waves a CU.
uint32_t few_split(const MulArgs &a, uint32_t waves, uint64_t tiles) {
    const uint32_t chunks = (mx4_blocks(a.cols) + 15) / 16;
    uint32_t ks = 1;
    while (ks < waves && ks * 2 <= chunks && tiles * ks < 8ull * cu_count()) ks *= 2;
    return ks;
}

// One group: `rows` (<= 16) activation rows a workgroup, `lists` of them, of
// which about `busy` have work.  One
// chunk a wave is multiplied while one is in flight: two of each are slower
// (three waves a SIMD instead of four: ten experts' 1280 x 2560 8.7 us against
// 7.6, LM head 151936 x 2048 with eight float rows 40.2 against 35.7).  As
// many workgroups as are resident at once, each with the same number of rounds.
template <class F>
bool few_launch(MulArgs &a, uint32_t rows, uint32_t lists, uint32_t busy, size_t extra, F pick,
                const char *name) {
    constexpr uint32_t NW = 4;
    const uint64_t tiles = (a.w_rows + 15) / 16;
    a.ks = few_split(a, NW, tiles * busy);
    const size_t lds = extra + few_fit(a, rows, 1, NW, 40 * 1024);
    const uint64_t sets = (tiles * a.ks + NW - 1) / NW;
    const uint64_t resident = std::max(1u, 4u * cu_count() / busy);
    const uint64_t rounds = (sets + resident - 1) / resident;
    a.blocks = (uint32_t)((sets + rounds - 1) / rounds);
    auto k = pick(mx4_blocks(a.cols) % 16 == 0);
    k<<<dim3(a.blocks, lists), dim3(64 * NW), lds, stream()>>>(a);
    return launch_ok(name);
}
typedef void (*MulKernel)(MulArgs);
MulKernel few_kernel(bool full) { return full ? mx4_few_k<true, 1, 4> : mx4_few_k<false, 1, 4>; }
MulKernel sel_kernel(bool full) {
    return full ? mx4_sel_k<true, false> : mx4_sel_k<false, false>;
}
MulKernel sel_group_kernel(bool full) {
    return full ? mx4_sel_k<true, true> : mx4_sel_k<false, true>;
}

// Two groups: 17 to 32 activation rows, eight waves.
bool few2_launch(MulArgs &a) {
    constexpr uint32_t NW = 8, MT = 2;
    const uint64_t tiles = (a.w_rows + 15) / 16;
    a.ks = few_split(a, NW, tiles);
    // whole rows up to 5632 columns; longer ones a segment at a time, each tile anew
    constexpr size_t kRoom = 100 * 1024, kMost = kRoom + NW * MT * 64 * sizeof(v4f);
    const size_t lds = few_fit(a, (uint32_t)a.n, MT, NW, kRoom);
    const uint32_t per = NW / a.ks;
    a.blocks = (uint32_t)std::min<uint64_t>((tiles + per - 1) / per, 2 * cu_count());
    const bool full = mx4_blocks(a.cols) % 16 == 0;
    auto k = full ? mx4_few_k<true, MT, NW> : mx4_few_k<false, MT, NW>;
    static DynLds st[2];
    if (!dyn_lds_ok((const void *)k, lds, kMost, st[full], "mx4_few_k")) return false;
    k<<<dim3(a.blocks), dim3(64 * NW), lds, stream()>>>(a);
    return launch_ok("mx4_few_k");
}

// Which kernel a dense product takes.  A workgroup's time hardly depends on
// its tile while the chip has room for all of them, so the smallest tile wins
// that still gives at most two workgroups a CU (64 x 64: two and a half);
// measured in us, bf16 out (rows x cols, activation rows):
//   few rows    against 64 x 64:   1024 x 2048, 64: 4.7 / 5.6; 128: 5.5 / 5.7; 192: 6.3 / 5.8;
//                                  4096 x 4096, 32: 7.4 / 8.9; 64: 9.5 / 8.9
//   two groups  against 64 x 64:   8192 x 8192, 17: 13.4 / 20.9; 32: 17.3 / 19.1
//   64 x 64     against 64 x 128:  4096 x 4096, 512: 12.0 / 11.8; 1024: 20.0 / 16.9
//   64 x 128    against 128 x 128: 8192 x 8192, 512: 29.2 / 29.8; 1024: 59.6 / 43.5
//   128 x 128   against 256 x 256: 8192 x 8192, 1024: 43.5 / 54.0; 2048: 86.7 / 71.2
// Past that the two largest are compared by their full rounds: 43 us for two
// 128 x 128 a CU, 71 us for one 256 x 256 (8192 columns).
bool mul_pick(MulArgs &a) {
    const uint64_t cus = cu_count();
    auto tiles = [&](uint64_t bm, uint64_t bn) {
        return ((a.n + bm - 1) / bm) * ((a.w_rows + bn - 1) / bn);
    };
    if (a.n <= kFewRows || tiles(16, 16) <= 2 * cus) {
        const uint32_t sets = (uint32_t)((a.n + kFewRows - 1) / kFewRows);
        return few_launch(a, (uint32_t)std::min<uint64_t>(a.n, kFewRows), sets, sets, 0, few_kernel,
                          "mx4_few_k");
    }
    if (a.n <= 32) return few2_launch(a);
    if (2 * tiles(64, 64) <= 5 * cus) return dense_launch<64, 64, 2, 2, 2>(a);
    if (tiles(64, 128) <= 2 * cus) return dense_launch<64, 128, 1, 4, 2>(a);
    const uint64_t rounds128 = (tiles(128, 128) + 2 * cus - 1) / (2 * cus);
    const uint64_t rounds256 = (tiles(256, 256) + cus - 1) / cus;
    if (3 * rounds128 <= 5 * rounds256) return dense_launch<128, 128, 2, 2, 2>(a);
    return dense_launch<256, 256, 2, 4, 2>(a);
}

bool id_launch(MulArgs &a) {
    // waves a tile while the experts that can have rows do not fill the chip
    const uint32_t tiles = (uint32_t)((a.w_rows + 15) / 16);
    const uint64_t units = std::min<uint64_t>(a.n, a.n_expert) * tiles;
    a.ks = few_split(a, kIdWaves, units);
    const size_t few = few_fit(a, kIdFew, kIdFew / 16, kIdWaves, 112 * 1024);
    const uint64_t slices = (a.w_rows + kIdN - 1) / kIdN;
    if ((a.n / kIdM + a.n_expert) * slices > 0x7fffffffu) {
        set_error("q4mi_mx4_mul_id: too many tiles");
        return false;
    }
    a.blocks = (uint32_t)cu_count();
    constexpr size_t kMost = 160 * 1024;
    const size_t lds = (kIdLists + 15) / 16 * 16 + std::max(few, (size_t)tile_lds<kIdM, kIdN>());
    static DynLds st[2];
    const bool full = mx4_blocks(a.cols) % 16 == 0;
    auto k = full ? mx4_id_k<true> : mx4_id_k<false>;
    if (!dyn_lds_ok((const void *)k, lds, kMost, st[full], "mx4_id_k")) return false;
    k<<<dim3(a.blocks), dim3(64 * kIdWaves), lds, stream()>>>(a);
    return launch_ok("mx4_id_k");
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
    if (!mul_ok("q4mi_mx4_mul", a, n > 0)) return false;
    if (x_type != kTypeMx4 && n > kFloatRows) {
        set_error("q4mi_mx4_mul: %llu float rows not covered (<= %llu; quantise them first)",
                  (unsigned long long)n, (unsigned long long)kFloatRows);
        return false;
    }
    if (!n) return true;
    return mul_pick(a);
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
    if (!mul_ok("q4mi_mx4_mul_sel", a, n > 0)) return false;
    if ((n && !d_eid) || !n_expert || !x_div || n > 65535) {
        set_error("q4mi_mx4_mul_sel: needs a list, experts, x_div >= 1 and at most 65535 rows");
        return false;
    }
    if (!n) return true;
    // Looking for rows of the same expert costs 0.6 us (ten rows of 1024 x 2048:
    // 5.9 against 6.5) and pays where some are likely (105 rows of 2345 x 2144
    // over 3 experts: 53 against 34).
    const uint32_t lists = (uint32_t)n;
    if (4 * n < n_expert) return few_launch(a, 1, lists, lists, 0, sel_kernel, "mx4_sel_k");
    return few_launch(a, std::min(lists, kFewRows), lists,
                      std::min(lists, n_expert + lists / kFewRows), kSelList, sel_group_kernel,
                      "mx4_sel_k");
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
    if (!mul_ok("q4mi_mx4_mul_id", a, total_rows && xrows)) return false;
    if (!d_bounds || !n_expert || n_expert > kIdExperts) {
        set_error("q4mi_mx4_mul_id: needs bounds of 1 to %u experts", kIdExperts);
        return false;
    }
    if (!total_rows || !xrows) return true;
    return id_launch(a);
}

}  // extern "C"

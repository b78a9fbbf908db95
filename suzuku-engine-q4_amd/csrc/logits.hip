// What a decode step does to its logits before it picks tokens: penalties for
// repeated tokens, biases, grammar masks.  For row b and token v, with n_all
// and n_gen the occurrences of v in the row's history and in the part of it
// that the model wrote:
//   z = logits[b][v]
//   z = z > 0 ? z / rep : z * rep            where n_all > 0
//   z = z - freq * n_gen - pres               where n_gen > 0
//   z = z + sum of the row's biases of v, in list order
//   z = -inf                                  where the mask's bit v is 0
//
// A workgroup owns a slice of one row's vocabulary and counts the history's
// tokens of that slice in LDS (integer atomics, so their order does not
// matter): no counters in memory, nothing kept between calls, one launch.
// Every slice reads its row's whole history, sixteen tokens a thread at a time,
// while the slice's own logits and mask are on their way to registers.  Without
// lists the logits' own bytes bound it; with long histories half of the time is
// their counting (64 x 151936, fp32: 13 us without, 27 with up to 32768 tokens a
// row, for which every die's L2 fetches the lists anew: 74 MB read, 39 of them
// logits and masks); one row is a chain of latencies (offsets, history, biases).
#include "mx4.h"
#include "q4mi_internal.h"

using namespace q4mi;

namespace {

struct LogitsArgs {
    const void *x;
    void *out;
    const int32_t *hist, *gen, *bias_ids, *mask_row;
    const int64_t *hist_off, *bias_off;
    const float *pen, *bias;
    const uint32_t *mask;
    uint64_t ld, ldo, mask_ld;
    uint32_t type, vocab, n_mask, slices;
};

constexpr uint32_t kThreads = 512;
constexpr uint32_t kPrompt = 0x80000000u;   // counter bit: the token is in the row's prompt

// Four logits from element i of a row, `left` of them in the slice.
__device__ inline float4 load_four(const LogitsArgs &a, uint64_t i, uint32_t left) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (left >= 4) {
        if (a.type == kTypeF32) {
            const u32x4 q = *(const u32x4_a4 *)((const float *)a.x + i);
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = bits_f32(q[k]);
        } else {
            const u32x2 q = *(const u32x2_a2 *)((const uint16_t *)a.x + i);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint32_t h = k & 1 ? q[k >> 1] >> 16 : q[k >> 1] & 0xffffu;
                v[k] = a.type == kTypeF16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)h)
                                          : bits_f32(h << 16);
            }
        }
    } else {
        for (uint32_t k = 0; k < left; k++) v[k] = load_as_f32(a.x, a.type, i + k);
    }
    return make_float4(v[0], v[1], v[2], v[3]);
}

__device__ inline void store_four(const LogitsArgs &a, uint64_t i, uint32_t left, const float *z) {
    if (left >= 4) {
        if (a.type == kTypeF32) {
            *(u32x4_a4 *)((float *)a.out + i) =
                (u32x4){f32_bits(z[0]), f32_bits(z[1]), f32_bits(z[2]), f32_bits(z[3])};
        } else {
            *(u32x2_a2 *)((uint16_t *)a.out + i) =
                (u32x2){f32_to_16x2(z[0], z[1], a.type), f32_to_16x2(z[2], z[3], a.type)};
        }
    } else {
        for (uint32_t k = 0; k < left; k++) store_from_f32(a.out, a.type, i + k, z[k]);
    }
}

// Occurrences of the slice's tokens in the row's history.
__device__ inline void count_history(const LogitsArgs &a, uint32_t b, uint32_t v0, uint32_t nv,
                                     uint32_t *cnt) {
    const int64_t lo = a.hist_off[b], hi = a.hist_off[b + 1];
    const int64_t wrote = lo + (a.gen ? max(a.gen[b], 0) : 0);
    constexpr uint32_t U = 4;       // loads of four tokens in flight a thread
    for (int64_t i0 = lo + 4 * threadIdx.x; i0 < hi; i0 += 4 * kThreads * U) {
        u32x4 t[U];
#pragma unroll
        for (uint32_t u = 0; u < U; u++) {
            const int64_t i = i0 + 4 * kThreads * u;
            t[u] = (u32x4){~0u, ~0u, ~0u, ~0u};
            if (i + 4 <= hi)
                t[u] = *(const u32x4_a4 *)(a.hist + i);
            else
#pragma unroll
                for (int k = 0; k < 3; k++)
                    if (i + k < hi) t[u][k] = (uint32_t)a.hist[i + k];
        }
#pragma unroll
        for (uint32_t u = 0; u < U; u++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint32_t v = t[u][k] - v0;
                if (v >= nv) continue;      // another slice's, or no token
                if (i0 + 4 * kThreads * u + k >= wrote)
                    atomicAdd(&cnt[v], 1u);
                else
                    atomicOr(&cnt[v], kPrompt);
            }
    }
}

// Sums of the row's biases in list order: every wave goes through the list and
// adds those of the tokens that are its own (v modulo the waves), entries of
// one token among 64 in turn.
__device__ inline void sum_biases(const LogitsArgs &a, int64_t lo, int64_t hi, uint32_t v0,
                                  uint32_t nv, float *add) {
    constexpr uint32_t U = 4, W = kThreads / 64;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    for (int64_t i0 = lo; i0 < hi; i0 += 64 * U) {
        uint32_t t[U];
        float v[U];
#pragma unroll
        for (uint32_t u = 0; u < U; u++) {
            const int64_t i = i0 + 64 * u + lane;
            t[u] = i < hi ? (uint32_t)a.bias_ids[i] : ~0u;
            v[u] = i < hi ? a.bias[i] : 0.f;
        }
#pragma unroll
        for (uint32_t u = 0; u < U; u++) {
            const uint32_t at = t[u] - v0;
            const bool in = at < nv && at % W == wave;  // else another's, or no token
            uint32_t turn = 0;
            for (uint64_t m = __ballot(in); m; m &= m - 1) {
                const uint32_t l = (uint32_t)__builtin_ctzll(m);
                const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)at, (int)l);
                if (in && l < lane && o == at) turn++;
            }
            for (uint32_t k = 0; __ballot(in && turn >= k); k++) {
                if (in && turn == k) add[at] += v[u];
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }
        }
    }
}

}  // namespace

// NG groups of four logits a thread.
template <uint32_t NG>
__global__ __launch_bounds__(kThreads) void logits_k(LogitsArgs a) {
    extern __shared__ __align__(16) uint32_t lds[];
    constexpr uint32_t kSlice = NG * kThreads * 4;
    const uint32_t tid = threadIdx.x;
    const uint32_t b = blockIdx.x / a.slices;
    const uint32_t v0 = (blockIdx.x - b * a.slices) * kSlice;
    const uint32_t nv = min(kSlice, a.vocab - v0);
    float4 x[NG];
    uint32_t bits[NG];
    const uint32_t *mask = nullptr;
    bool none = false;
    if (a.mask) {
        const int32_t r = a.mask_row ? a.mask_row[b] : (int32_t)b;
        none = r >= 0 && (uint32_t)r >= a.n_mask;
        if (r >= 0 && !none) mask = a.mask + (uint64_t)r * a.mask_ld + v0 / 32;
    }
#pragma unroll
    for (uint32_t n = 0; n < NG; n++) {
        const uint32_t i = (n * kThreads + tid) * 4, left = i < nv ? nv - i : 0u;
        x[n] = load_four(a, (uint64_t)b * a.ld + v0 + i, left);
        bits[n] = none ? 0u : mask && left ? mask[i / 32] >> (i & 31u) : 15u;
    }
    const bool counted = a.hist && !(a.pen[3 * b] == 1.f && a.pen[3 * b + 1] == 0.f &&
                                     a.pen[3 * b + 2] == 0.f);
    const int64_t blo = a.bias ? a.bias_off[b] : 0, bhi = a.bias ? a.bias_off[b + 1] : 0;
    const bool biased = bhi > blo;
    // The counters' LDS holds the biases afterwards: half the LDS, and twice the
    // workgroups a CU to hide what each waits for.
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t n = 0; n < NG; n++)
            *(u32x4 *)(lds + (n * kThreads + tid) * 4) = (u32x4){0, 0, 0, 0};
        __syncthreads();
    };
    float z[NG][4];
#pragma unroll
    for (uint32_t n = 0; n < NG; n++)
        z[n][0] = x[n].x, z[n][1] = x[n].y, z[n][2] = x[n].z, z[n][3] = x[n].w;
    if (counted) {
        clear();
        count_history(a, b, v0, nv, lds);
        __syncthreads();
        const float rep = a.pen[3 * b], freq = a.pen[3 * b + 1], pres = a.pen[3 * b + 2];
#pragma unroll
        for (uint32_t n = 0; n < NG; n++) {
            const u32x4 c = *(const u32x4 *)(lds + (n * kThreads + tid) * 4);
            if (!(c[0] | c[1] | c[2] | c[3])) continue;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (!c[k]) continue;
                const float m = (float)(c[k] & ~kPrompt);
                z[n][k] = z[n][k] > 0.f ? z[n][k] / rep : z[n][k] * rep;
                if (m > 0.f) z[n][k] = z[n][k] - freq * m - pres;   // both may be infinite
            }
        }
    }
    if (biased) {
        clear();    // each thread clears what it alone has read
        sum_biases(a, blo, bhi, v0, nv, (float *)lds);
        __syncthreads();
#pragma unroll
        for (uint32_t n = 0; n < NG; n++) {
            const float4 d = *(const float4 *)(lds + (n * kThreads + tid) * 4);
            z[n][0] += d.x, z[n][1] += d.y, z[n][2] += d.z, z[n][3] += d.w;
        }
    }
#pragma unroll
    for (uint32_t n = 0; n < NG; n++) {
        const uint32_t i = (n * kThreads + tid) * 4;
        if (i >= nv) break;
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (!((bits[n] >> k) & 1u)) z[n][k] = -__builtin_inff();
        store_four(a, (uint64_t)b * a.ldo + v0 + i, nv - i, z[n]);
    }
}

extern "C" {

/* Penalties, biases and masks on a batch's logits (see include/q4mi.h). */
bool q4mi_logits_process(const void *d_logits, uint32_t type, uint64_t ld, uint32_t n_rows,
                         uint32_t n_vocab, const int32_t *d_hist, const int64_t *d_hist_off,
                         const int32_t *d_gen, const float *d_pen, const int32_t *d_bias_ids,
                         const float *d_bias, const int64_t *d_bias_off, const uint32_t *d_mask,
                         uint64_t mask_ld, uint32_t n_mask, const int32_t *d_mask_row,
                         void *d_out, uint64_t ld_out) {
    const char *who = "q4mi_logits_process";
    if ((n_rows && (!d_logits || !d_out)) || !n_vocab || n_vocab > (1u << 30)) {
        set_error("%s: bad arguments", who);
        return false;
    }
    if (!is_float_type(type)) {
        set_error("%s: type %u not covered (F32, F16, BF16)", who, type);
        return false;
    }
    if (ld < n_vocab || ld_out < n_vocab || (n_rows && d_out == d_logits && ld != ld_out)) {
        set_error("%s: row strides must cover the vocabulary, and agree in place", who);
        return false;
    }
    if (((uintptr_t)d_logits | (uintptr_t)d_out) & (type_bytes(type) - 1)) {
        set_error("%s: logits must be aligned to their type", who);
        return false;
    }
    if (!n_rows) return true;
    if (!d_pen != !d_hist_off || ((d_hist || d_gen) && !d_pen)) {
        set_error("%s: penalties need their values and the history's offsets", who);
        return false;
    }
    if (!d_bias != !d_bias_ids || (d_bias && !d_bias_off)) {
        set_error("%s: biases need their ids, values and offsets", who);
        return false;
    }
    if (d_mask ? !n_mask || mask_ld < (n_vocab + 31ull) / 32 || (!d_mask_row && n_mask < n_rows)
               : d_mask_row != nullptr) {
        set_error("%s: masks need a row for every state, (n_vocab + 31) / 32 words each", who);
        return false;
    }
    LogitsArgs a = {};
    a.x = d_logits, a.out = d_out, a.hist = d_hist, a.gen = d_gen, a.bias_ids = d_bias_ids;
    a.mask_row = d_mask_row, a.hist_off = d_hist_off, a.bias_off = d_bias_off, a.pen = d_pen;
    a.bias = d_bias, a.mask = d_mask, a.ld = ld, a.ldo = ld_out, a.mask_ld = mask_ld;
    a.type = type, a.vocab = n_vocab, a.n_mask = n_mask;
    // Slices of 2048 tokens until they give every CU four workgroups: then
    // larger ones, which read the history less often.
    const uint64_t least = (n_vocab + 2047ull) / 2048 * n_rows, fill = 4ull * cu_count();
    const uint32_t ng = least <= fill ? 1 : least <= 2 * fill ? 2 : 4;
    const uint32_t slice = ng * kThreads * 4;
    a.slices = (n_vocab + slice - 1) / slice;
    if ((uint64_t)a.slices * n_rows > UINT32_MAX / kThreads) {     // threads of a launch
        set_error("%s: %u rows of %u logits too large", who, n_rows, n_vocab);
        return false;
    }
    const size_t lds = d_hist || d_bias ? (size_t)slice * 4 : 0;
    auto k = ng == 1 ? logits_k<1> : ng == 2 ? logits_k<2> : logits_k<4>;
    k<<<dim3(a.slices * n_rows), dim3(kThreads), lds, stream()>>>(a);
    return launch_ok("logits_k");
}

}  // extern "C"

// What a decode step does to its logits before it picks tokens: penalties for
// repeated tokens, biases, grammar masks.  For row b and token v, with n_all
// and n_gen the occurrences of v in the row's history and in the part of it
// that the model wrote:
//   z = logits[b][v]
//   z = z > 0 ? z / rep : z * rep            where n_all > 0
//   z = z - freq * n_gen - pres * (n_gen > 0)
//   z = z + sum of the row's biases of v, in list order
//   z = -inf                                  where the mask's bit v is 0
//
// A workgroup owns a slice of one row's vocabulary and counts the history's
// tokens of that slice in LDS (integer atomics, so their order does not
// matter): no counters in memory, nothing kept between calls, one launch.
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
    uint32_t type, vocab, n_mask, slices, slice;
};

constexpr uint32_t kPrompt = 0x80000000u;   // counter bit: the token is in the row's prompt

}  // namespace

__global__ __launch_bounds__(256) void logits_k(LogitsArgs a) {
    extern __shared__ uint32_t lds[];
    const uint32_t tid = threadIdx.x;
    const uint32_t b = blockIdx.x / a.slices;
    const uint32_t v0 = (blockIdx.x % a.slices) * a.slice;
    const uint32_t nv = min(a.slice, a.vocab - v0);
    uint32_t *cnt = lds;
    float *add = (float *)(lds + (a.hist ? a.slice : 0u));
    float rep = 1.f, freq = 0.f, pres = 0.f;
    if (a.hist) {
        rep = a.pen[3 * b], freq = a.pen[3 * b + 1], pres = a.pen[3 * b + 2];
    }
    const bool pen = a.hist && !(rep == 1.f && freq == 0.f && pres == 0.f);
    if (pen)
        for (uint32_t i = tid; i < nv; i += 256) cnt[i] = 0;
    if (a.bias)
        for (uint32_t i = tid; i < nv; i += 256) add[i] = 0.f;
    __syncthreads();
    if (pen) {
        const int64_t lo = a.hist_off[b], hi = a.hist_off[b + 1];
        const int64_t wrote = lo + (a.gen ? max(a.gen[b], 0) : 0);
        for (int64_t i = lo + tid; i < hi; i += 256) {
            const uint32_t t = (uint32_t)a.hist[i] - v0;
            if (t < nv) {
                if (i >= wrote)
                    atomicAdd(&cnt[t], 1u);
                else
                    atomicOr(&cnt[t], kPrompt);
            }
        }
    }
    if (a.bias && tid < 64) {
        // one wave, in list order: entries of one token among a wave's 64 are
        // taken in turn
        const int64_t lo = a.bias_off[b], hi = a.bias_off[b + 1];
        for (int64_t i0 = lo; i0 < hi; i0 += 64) {
            const int64_t i = i0 + tid;
            const uint32_t t = i < hi ? (uint32_t)a.bias_ids[i] - v0 : nv;
            const bool in = t < nv;
            const float v = in ? a.bias[i] : 0.f;
            uint32_t turn = 0;
            const uint64_t all = __ballot(in);
            for (uint64_t m = all; m; m &= m - 1) {
                const uint32_t l = (uint32_t)__builtin_ctzll(m);
                const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)t, (int)l);
                if (in && l < tid && o == t) turn++;
            }
            for (uint32_t k = 0; __ballot(in && turn >= k); k++) {
                if (in && turn == k) add[t] += v;
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }
        }
    }
    __syncthreads();
    const uint32_t *mask = nullptr;
    bool none = false;
    if (a.mask) {
        const int32_t r = a.mask_row ? a.mask_row[b] : (int32_t)b;
        none = r >= 0 && (uint32_t)r >= a.n_mask;
        if (r >= 0 && !none) mask = a.mask + (uint64_t)r * a.mask_ld;
    }
    for (uint32_t i = tid; i < nv; i += 256) {
        const uint32_t v = v0 + i;
        float z = load_as_f32(a.x, a.type, (uint64_t)b * a.ld + v);
        if (pen && cnt[i]) {
            const float n = (float)(cnt[i] & ~kPrompt);
            z = z > 0.f ? z / rep : z * rep;
            z = z - freq * n;
            if (n > 0.f) z = z - pres;
        }
        if (a.bias) z += add[i];
        if (none || (mask && !((mask[v >> 5] >> (v & 31u)) & 1u))) z = -__builtin_inff();
        store_from_f32(a.out, a.type, (uint64_t)b * a.ldo + v, z);
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
    if (!d_logits || !d_out || !n_vocab || n_vocab > (1u << 30)) {
        set_error("%s: bad arguments", who);
        return false;
    }
    if (!is_float_type(type)) {
        set_error("%s: type %u not covered (F32, F16, BF16)", who, type);
        return false;
    }
    if (ld < n_vocab || ld_out < n_vocab || (d_out == d_logits && ld != ld_out)) {
        set_error("%s: row strides must cover the vocabulary, and agree in place", who);
        return false;
    }
    if (((uintptr_t)d_logits | (uintptr_t)d_out) & (type_bytes(type) - 1)) {
        set_error("%s: logits must be aligned to their type", who);
        return false;
    }
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
    a.slice = 4096;
    a.slices = (n_vocab + a.slice - 1) / a.slice;
    if ((uint64_t)a.slices * n_rows > 0x7fffffffu) {
        set_error("%s: %u rows of %u logits too large", who, n_rows, n_vocab);
        return false;
    }
    if (!n_rows) return true;
    const size_t bytes = (size_t)a.slice * 4 * ((d_hist ? 1 : 0) + (d_bias ? 1 : 0));
    logits_k<<<dim3(a.slices * n_rows), dim3(256), bytes, stream()>>>(a);
    return launch_ok("logits_k");
}

}  // extern "C"

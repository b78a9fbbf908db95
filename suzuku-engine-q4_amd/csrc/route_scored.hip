// Routing by scores: softmax or sigmoid of the router's logits, a bias for the
// choice, experts in groups of which some stay, top-k, renormalised and scaled
// weights.
//
// Scores, keys and sums are 64-bit: two experts whose keys differ in the last
// bits of an fp32 (with hundreds of experts a few tokens of a thousand have such
// a pair among their picks) come in their true order whatever exp() and the order
// of the sums, so that ids are the same as any other 64-bit computation's.
#include <math.h>

#include "mx4.h"
#include "q4mi_common.h"
#include "q4mi_internal.h"

using namespace q4mi;

namespace {

struct ScoreArgs {
    const void *logits;
    const float *bias, *sg;
    int32_t *ids, *nh;
    float *wts;
    uint64_t ld;
    uint32_t type, n_tok, n_exp, sigmoid, n_group, topk_group, group_top, topk, renorm, ostride;
    int32_t shared;
    float scale;
};

constexpr uint32_t kScoreExperts = 1024, kScoreWaves = 4;

// Wave maximum of a double, on every lane.
template <int CTRL, int ROWS>
__device__ inline double max_dpp(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)b, hi = (uint32_t)(b >> 32);
    const uint32_t l2 = (uint32_t)__builtin_amdgcn_update_dpp((int)lo, (int)lo, CTRL, ROWS, 0xF, false);
    const uint32_t h2 = (uint32_t)__builtin_amdgcn_update_dpp((int)hi, (int)hi, CTRL, ROWS, 0xF, false);
    return fmax(v, __builtin_bit_cast(double, (uint64_t)h2 << 32 | l2));
}
__device__ inline double lane_value(double v, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double,
                              (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), lane) << 32 |
                                  (uint32_t)__builtin_amdgcn_readlane((int)b, lane));
}
__device__ inline double wave_max(double v) {
    v = max_dpp<0x111, 0xF>(v);
    v = max_dpp<0x112, 0xF>(v);
    v = max_dpp<0x114, 0xF>(v);
    v = max_dpp<0x118, 0xF>(v);
    v = max_dpp<0x142, 0xA>(v);
    v = max_dpp<0x143, 0xC>(v);
    return lane_value(v, 63);
}
__device__ inline uint32_t wave_min(uint32_t v) {
#pragma unroll
    for (int d = 32; d; d /= 2) v = min(v, (uint32_t)__shfl_xor((int)v, d, 64));
    return v;
}

}  // namespace

// One wave a token; lane l has experts l, l + 64, ..
template <uint32_t NJ>
__global__ __launch_bounds__(64 * kScoreWaves) void route_scored_k(ScoreArgs a) {
    __shared__ double keys[kScoreWaves][64 * NJ];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63u;
    const uint32_t t = blockIdx.x * kScoreWaves + wave;
    if (t >= a.n_tok) return;
    const uint64_t row = (uint64_t)t * a.ld;
    const double none = -(double)INFINITY;
    // Of the logits +inf counts as the largest finite one, NaN as -inf.
    auto logit = [&](uint32_t e) {
        const float z = load_as_f32(a.logits, a.type, row + e);
        return z != z ? -INFINITY : fminf(z, 3.402823466e38f);
    };
    float z[NJ], top = -INFINITY;
#pragma unroll
    for (uint32_t j = 0; j < NJ; j++) {
        const uint32_t e = lane + 64 * j;
        z[j] = e < a.n_exp ? logit(e) : -INFINITY;
        top = fmaxf(top, z[j]);
    }
    const double zmax = wave_max((double)top);
    double denom = 1.;
    auto score = [&](float x) -> double {
        if (x == -INFINITY) return 0.;
        return a.sigmoid ? 1. / (1. + exp(-(double)x)) : exp((double)x - zmax) / denom;
    };
    if (!a.sigmoid) {
        double sum = 0.;
#pragma unroll
        for (uint32_t j = 0; j < NJ; j++)
            if (z[j] != -INFINITY) sum += exp((double)z[j] - zmax);
        denom = lane_value(q4mi_rsum<64>(sum), 63);
    }
    double key[NJ];
#pragma unroll
    for (uint32_t j = 0; j < NJ; j++) {
        const uint32_t e = lane + 64 * j;
        key[j] = none;
        if (z[j] == -INFINITY) continue;
        double k = a.bias || a.n_group > 1 ? score(z[j]) : 0.;
        if (a.bias) k += (double)a.bias[e];
        if (k == k) key[j] = k;
    }
    if (a.n_group > 1) {
        // lane g ranks group g; a group's keys come through LDS
        const uint32_t size = a.n_exp / a.n_group;
#pragma unroll
        for (uint32_t j = 0; j < NJ; j++) keys[wave][lane + 64 * j] = key[j];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        double best = none;
        if (lane < a.n_group) {
            double b0 = none, b1 = none;
            for (uint32_t i = 0; i < size; i++) {
                const double k = keys[wave][lane * size + i];
                b1 = fmax(b1, fmin(b0, k));
                b0 = fmax(b0, k);
            }
            best = a.group_top > 1 && b1 != none ? b0 + b1 : b0;
        }
        uint64_t stay = 0;
        for (uint32_t i = 0; i < a.topk_group; i++) {
            const double m = wave_max(best);
            if (m == none) break;
            const uint32_t g = wave_min(best == m ? lane : 64u);
            stay |= 1ull << g;
            if (lane == g) best = none;
        }
#pragma unroll
        for (uint32_t j = 0; j < NJ; j++)
            if (!(stay >> (lane + 64 * j) / size & 1)) key[j] = none;
    }
    // Without a bias picks go by the logit: the same order, also of scores that
    // round alike.
    if (!a.bias) {
#pragma unroll
        for (uint32_t j = 0; j < NJ; j++) key[j] = key[j] == none ? none : (double)z[j];
    }
    // the best key, on a tie of the lowest expert, topk times
    int32_t mine = -1;
    for (uint32_t k = 0; k < a.topk; k++) {
        double best = none;
        uint32_t at = 0;
#pragma unroll
        for (uint32_t j = 0; j < NJ; j++)
            if (key[j] > best) best = key[j], at = lane + 64 * j;
        const double m = wave_max(best);
        if (m == none) break;
        const uint32_t e = wave_min(best == m ? at : ~0u);
#pragma unroll
        for (uint32_t j = 0; j < NJ; j++)
            if (e == lane + 64 * j) key[j] = none;
        if (lane == k) mine = (int32_t)e;
    }
    // lane k: weight of pick k
    double w = mine >= 0 ? score(logit((uint32_t)mine)) : 0.;
    if (a.renorm) {
        const double total = lane_value(q4mi_rsum<64>(w), 63);
        w = total > 0. ? w / total : 0.;
    }
    // the shared expert follows the picks that were found
    const uint32_t found = (uint32_t)__popcll(__ballot(mine >= 0));
    const uint64_t out = (uint64_t)t * a.ostride;
    auto put = [&](uint32_t k, int32_t id, float v) { a.ids[out + k] = id, a.wts[out + k] = v; };
    if (lane < a.topk && (a.shared < 0 || lane != found))
        put(lane, mine, (float)(w * (double)a.scale));
    if (lane == 0) {
        if (a.shared >= 0) {
            put(found, a.shared, a.sg ? a.sg[t] : 1.f);
            if (found < a.topk) put(a.topk, -1, 0.f);
        }
        if (a.nh) a.nh[t] = (int32_t)(found + (a.shared >= 0 ? 1u : 0u));
    }
}

namespace {

bool score_ok(const char *who, const ScoreArgs &a) {
    if ((a.n_tok && (!a.logits || !a.ids || !a.wts)) || !a.n_exp || !a.topk) {
        set_error("%s: bad arguments", who);
        return false;
    }
    if (!is_float_type(a.type) || ((uintptr_t)a.logits & (type_bytes(a.type) - 1))) {
        set_error("%s: logits of type %u not covered (F32, F16, BF16, aligned to their type)", who,
                  a.type);
        return false;
    }
    if (((uintptr_t)a.bias | (uintptr_t)a.sg | (uintptr_t)a.ids | (uintptr_t)a.wts |
         (uintptr_t)a.nh) & 3u) {
        set_error("%s: bias, gates and lists must be aligned to 4 bytes", who);
        return false;
    }
    if (a.n_exp > kScoreExperts || a.topk > 64u || a.n_tok > (1u << 24)) {
        set_error("%s: sizes not covered (%u experts, %u picks, 2^24 tokens)", who, kScoreExperts,
                  64u);
        return false;
    }
    if (a.ld < a.n_exp) {
        set_error("%s: row stride below its experts", who);
        return false;
    }
    if (a.sigmoid > 1u) {
        set_error("%s: score %u not covered (0 softmax, 1 sigmoid)", who, a.sigmoid);
        return false;
    }
    if (!a.n_group || a.n_group > 64u || a.n_exp % a.n_group || !a.topk_group ||
        a.topk_group > a.n_group || a.group_top < 1u || a.group_top > 2u) {
        set_error("%s: groups not covered (1 to 64 equal ones, 1 to all of them kept, scored by "
                  "their 1 or 2 best)", who);
        return false;
    }
    if (!isfinite(a.scale)) {
        set_error("%s: scale must be finite", who);
        return false;
    }
    const uint32_t need = a.topk + (a.shared >= 0 ? 1u : 0u);
    if (a.ostride < need) {
        set_error("%s: ostride %u < %u entries per token", who, a.ostride, need);
        return false;
    }
    return true;
}

bool score_launch(const ScoreArgs &a) {
    if (!a.n_tok) return true;
    const dim3 grid((a.n_tok + kScoreWaves - 1) / kScoreWaves), block(64 * kScoreWaves);
    auto k = a.n_exp <= 256 ? route_scored_k<4> : route_scored_k<16>;
    k<<<grid, block, 0, stream()>>>(a);
    return launch_ok("route_scored_k");
}

}  // namespace

extern "C" {

/* Logits to experts and weights (see include/q4mi.h). */
bool q4mi_route_scored(const void *d_logits, uint32_t type, uint64_t ld, uint32_t n_tok,
                       uint32_t n_exp, const float *d_bias, uint32_t sigmoid, uint32_t n_group,
                       uint32_t topk_group, uint32_t group_top, uint32_t topk, bool renorm,
                       float scale, int32_t *d_ids, float *d_wts, int32_t *d_nh, uint32_t ostride,
                       int32_t shared_slot, const float *d_sg) {
    const ScoreArgs a = {d_logits, d_bias, d_sg, d_ids, d_nh, d_wts, ld, type, n_tok, n_exp,
                         sigmoid, n_group, topk_group, group_top, topk, renorm, ostride,
                         shared_slot, scale};
    return score_ok("q4mi_route_scored", a) && score_launch(a);
}

/* The router GEMV ahead of it (see include/q4mi.h). */
bool q4mi_moe_route_scored(const void *d_wr, uint32_t wr_type, const float *d_sgw,
                           const float *d_x, uint32_t n_tok, uint32_t n_embd, uint32_t n_exp,
                           const float *d_bias, uint32_t sigmoid, uint32_t n_group,
                           uint32_t topk_group, uint32_t group_top, uint32_t topk, bool renorm,
                           float scale, float *d_logits, int32_t *d_ids, float *d_wts,
                           int32_t *d_nh, uint32_t ostride, int32_t shared_slot, float *d_sg) {
    const ScoreArgs a = {d_logits, d_bias, d_sgw ? d_sg : nullptr, d_ids, d_nh, d_wts, n_exp,
                         kTypeF32, n_tok, n_exp, sigmoid, n_group, topk_group, group_top, topk,
                         renorm, ostride, shared_slot, scale};
    if (!score_ok("q4mi_moe_route_scored", a)) return false;
    // checked whole before its launch: n_exp as the router takes it, every pointer
    return router_front(d_wr, wr_type, d_sgw, d_x, n_tok, n_embd, n_exp, topk, d_logits, ostride,
                        shared_slot, d_sg, false) &&
           router_front(d_wr, wr_type, d_sgw, d_x, n_tok, n_embd, n_exp, topk, d_logits, ostride,
                        shared_slot, d_sg, true) &&
           score_launch(a);
}

}  // extern "C"

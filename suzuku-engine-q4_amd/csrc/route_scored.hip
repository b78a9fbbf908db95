// Routing by scores: softmax or sigmoid of the router's logits, a bias for the
// choice, experts in groups of which some stay, top-k, renormalised and scaled
// weights.
//
// The picks and weights are those of scores, keys and sums in 64 bits: two experts
// whose keys differ in the last bits of an fp32 (with hundreds of experts a few
// tokens of a thousand have such a pair among their picks) come in their true order
// whatever exp() and the order of the sums.  fp32 keys are used where they are
// further apart than their errors.
#include <math.h>

#include <type_traits>

#include "mx4.h"
#include "q4mi_common.h"
#include "q4mi_internal.h"
#include "route_wave.h"

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

__device__ inline double lane_value(double v, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double,
                              (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), lane) << 32 |
                                  (uint32_t)__builtin_amdgcn_readlane((int)b, lane));
}
// A lane's value moved by DPP; lanes without a source keep their own.
template <int CTRL, int ROWS>
__device__ inline double dpp(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const int lo = (int)(uint32_t)b, hi = (int)(uint32_t)(b >> 32);
    const uint32_t l = (uint32_t)__builtin_amdgcn_update_dpp(lo, lo, CTRL, ROWS, 0xF, false);
    const uint32_t h = (uint32_t)__builtin_amdgcn_update_dpp(hi, hi, CTRL, ROWS, 0xF, false);
    return __builtin_bit_cast(double, (uint64_t)h << 32 | l);
}
// Wave maximum of a double, on every lane.
__device__ inline double wave_max(double v) {
    v = fmax(v, dpp<0x111, 0xF>(v));
    v = fmax(v, dpp<0x112, 0xF>(v));
    v = fmax(v, dpp<0x114, 0xF>(v));
    v = fmax(v, dpp<0x118, 0xF>(v));
    v = fmax(v, dpp<0x142, 0xA>(v));
    v = fmax(v, dpp<0x143, 0xC>(v));
    return lane_value(v, 63);
}
__device__ inline uint32_t wave_min(uint32_t v) { return ~wave_max_u32(~v); }

// exp(x) to about 2^-52: x = n ln 2 + r, |r| <= ln 2 / 2, the Taylor series of
// exp(r) to r^13 (the next term is below 2^-57).  x below -800 gives 0; above 700
// is not asked.
__device__ inline double exp_series(double x) {
    x = fmax(x, -800.);
    const double n = rint(x * 0x1.71547652b82fep+0);        // 1 / ln 2
    double r = fma(n, -0x1.62e42fefa39efp-1, x);            // ln 2 and what it lacks
    r = fma(n, -0x1.abc9e3b39803fp-56, r);
    double s = 1. / 6227020800.;
    s = fma(s, r, 1. / 479001600.);
    s = fma(s, r, 1. / 39916800.);
    s = fma(s, r, 1. / 3628800.);
    s = fma(s, r, 1. / 362880.);
    s = fma(s, r, 1. / 40320.);
    s = fma(s, r, 1. / 5040.);
    s = fma(s, r, 1. / 720.);
    s = fma(s, r, 1. / 120.);
    s = fma(s, r, 1. / 24.);
    s = fma(s, r, 1. / 6.);
    s = fma(s, r, 0.5);
    s = fma(s, r, 1.);
    s = fma(s, r, 1.);
    return __builtin_amdgcn_ldexp(s, (int)n);
}
// 1 / d for 1 <= d < 2^1021: the hardware's estimate and two Newton steps.
__device__ inline double reciprocal(double d) {
    double r = __builtin_amdgcn_rcp(d);
    r = fma(fma(-d, r, 1.), r, r);
    return fma(fma(-d, r, 1.), r, r);
}

}  // namespace

// A group's two best keys, from two parts of it.
__device__ inline void merge2(double &b0, double &b1, double c0, double c1) {
    b1 = fmax(fmin(b0, c0), fmax(b1, c1));
    b0 = fmax(b0, c0);
}
// The same over a group's 2^shift lanes, on each of them: swaps in quads, mirrors
// of halves and rows, then rows.
__device__ inline void merge2_lanes(double &b0, double &b1, uint32_t shift) {
    if (shift > 0) merge2(b0, b1, dpp<0xB1, 0xF>(b0), dpp<0xB1, 0xF>(b1));
    if (shift > 1) merge2(b0, b1, dpp<0x4E, 0xF>(b0), dpp<0x4E, 0xF>(b1));
    if (shift > 2) merge2(b0, b1, dpp<0x141, 0xF>(b0), dpp<0x141, 0xF>(b1));
    if (shift > 3) merge2(b0, b1, dpp<0x140, 0xF>(b0), dpp<0x140, 0xF>(b1));
    if (shift > 4) merge2(b0, b1, __shfl_xor(b0, 16, 64), __shfl_xor(b1, 16, 64));
}

// Where a lane's experts are: with 2^n groups a group is 64 / 2^n lanes' experts,
// else lane l has experts l, l + 64, ..
struct ScorePlaces {
    bool in_lanes;
    uint32_t shift, size, lane;     // 2^shift lanes have `size` adjacent experts
    __device__ ScorePlaces(const ScoreArgs &a, uint32_t l) : lane(l) {
        in_lanes = (a.n_group & (a.n_group - 1)) == 0;
        shift = in_lanes ? 6 - __builtin_ctz(a.n_group) : 6;
        size = in_lanes ? a.n_exp / a.n_group : a.n_exp;
    }
    __device__ uint32_t of(uint32_t l, uint32_t j) const {
        return (l >> shift) * size + (l & ((1u << shift) - 1)) + (j << shift);
    }
    __device__ uint32_t mine(uint32_t j) const { return of(lane, j); }
    __device__ uint32_t last() const { return (lane >> shift) * size + size - 1; }
    __device__ bool is(uint32_t j) const {
        return (lane & ((1u << shift) - 1)) + (j << shift) < size;
    }
};

// Scores of logits in 64 bits: softmax (over a token's, whose largest and sum of
// exponentials are known) or sigmoid.
struct Scores {
    bool softmax;
    double zmax, inv;       // 1 / that sum
    // z above -690 for a sigmoid
    __device__ double near(float z) const {
        return softmax ? exp_series((double)z - zmax) * inv
                       : reciprocal(1. + exp_series(fmin(-(double)z, 700.)));
    }
    // the library's functions, for any logit
    __device__ double any(float z) const {
        if (z == -INFINITY) return 0.;
        return softmax ? exp((double)z - zmax) * inv : 1. / (1. + exp(-(double)z));
    }
};

// Keys in 64 bits, and the groups: of those that do not stay the keys are -inf, of
// those that do the bias's sums or, without a bias, the logits.
template <uint32_t NJ>
__device__ inline void keys_exact(const ScoreArgs &a, const ScorePlaces &at, const float *z,
                                  const float *bias, Scores &score, bool far, float *out) {
    const double none = -(double)INFINITY;
    const uint32_t lane = at.lane, each = a.n_exp / a.n_group;
    double key[NJ];
#pragma unroll
    for (uint32_t j = 0; j < NJ; j++) key[j] = 0.;
#pragma unroll 1
    for (uint32_t j = 0; j < NJ; j++) {
        float x = 0.f;
#pragma unroll
        for (uint32_t u = 0; u < NJ; u++) x = u == j ? z[u] : x;
        const double v = far ? score.any(x) : score.near(x);
#pragma unroll
        for (uint32_t u = 0; u < NJ; u++) key[u] = u == j ? v : key[u];
    }
#pragma unroll
    for (uint32_t j = 0; j < NJ; j++) {
        const double k = key[j] + (a.bias ? (double)bias[j] : 0.);
        key[j] = z[j] != -INFINITY && k == k ? k : none;
    }
    double b0 = none, b1 = none;
    uint32_t own = lane >> at.shift, step = 1u << at.shift;     // this lane's group; lanes each
    if (at.in_lanes) {
#pragma unroll
        for (uint32_t j = 0; j < NJ; j++) merge2(b0, b1, key[j], none);
        merge2_lanes(b0, b1, at.shift);
    } else {
        // lane g ranks group g, whose keys come through LDS
        __shared__ double keys[kScoreWaves][64 * NJ];
        double *mine = keys[threadIdx.x >> 6];
#pragma unroll
        for (uint32_t j = 0; j < NJ; j++) mine[lane + 64 * j] = key[j];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (lane < a.n_group)
            for (uint32_t i = 0; i < each; i++) merge2(b0, b1, mine[lane * each + i], none);
        own = lane, step = 1;
    }
    const double best = a.group_top > 1 && b1 != none ? b0 + b1 : b0;
    uint32_t before = 0;        // groups ahead of this lane's
    for (uint32_t g = 0; g < a.n_group; g++) {
        const double o = lane_value(best, (int)(g * step));
        before += o > best || (o == best && g < own) ? 1u : 0u;
    }
    const uint64_t stay = __ballot(before < a.topk_group && best != none);
#pragma unroll
    for (uint32_t j = 0; j < NJ; j++) {
        const uint32_t g = at.in_lanes ? lane : at.mine(j) / each;
        out[j] = key[j] == none || !(stay >> (g & 63u) & 1) ? -INFINITY
                 : a.bias                                  ? (float)key[j]
                                                           : z[j];
    }
}

// The same in 32 bits; false if two groups are nearer than their errors.  `room`
// covers those of two scores.
template <uint32_t NJ>
__device__ inline bool keys_fast(const ScoreArgs &a, const ScorePlaces &at, const float *z,
                                 const float *bias, float zmax, float room, float *key) {
    const float none = -INFINITY;
    constexpr float kLog2e = 1.44269504f;
    if (a.sigmoid) {
#pragma unroll
        for (uint32_t j = 0; j < NJ; j++)
            key[j] = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-z[j] * kLog2e));
    } else {
        float sum = 0.f;
#pragma unroll
        for (uint32_t j = 0; j < NJ; j++) {
            key[j] = __builtin_amdgcn_exp2f((z[j] - zmax) * kLog2e);
            sum += key[j];
        }
        sum = q4mi_rsum<64>(sum);
        const float inv = __builtin_amdgcn_rcpf(
            bits_f32((uint32_t)__builtin_amdgcn_readlane((int)f32_bits(sum), 63)));
#pragma unroll
        for (uint32_t j = 0; j < NJ; j++) key[j] *= inv;
    }
    if (a.bias) {
#pragma unroll
        for (uint32_t j = 0; j < NJ; j++) key[j] += bias[j];
    }
#pragma unroll
    for (uint32_t j = 0; j < NJ; j++) key[j] = z[j] == none ? none : fmaxf(key[j], none);  // NaN
    if (a.n_group == 1) return true;
    float b0 = none, b1 = none;
    auto merge = [](float &x0, float &x1, float y0, float y1) {
        x1 = fmaxf(fminf(x0, y0), fmaxf(x1, y1));
        x0 = fmaxf(x0, y0);
    };
    auto moved = [](auto ctrl, float v) {
        return bits_f32((uint32_t)__builtin_amdgcn_update_dpp((int)f32_bits(v), (int)f32_bits(v),
                                                              decltype(ctrl)::value, 0xF, 0xF, false));
    };
#pragma unroll
    for (uint32_t j = 0; j < NJ; j++) merge(b0, b1, key[j], none);
    const std::integral_constant<int, 0xB1> swap1{};       // as merge2_lanes
    const std::integral_constant<int, 0x4E> swap2{};
    const std::integral_constant<int, 0x141> half{};
    const std::integral_constant<int, 0x140> whole{};
    if (at.shift > 0) merge(b0, b1, moved(swap1, b0), moved(swap1, b1));
    if (at.shift > 1) merge(b0, b1, moved(swap2, b0), moved(swap2, b1));
    if (at.shift > 2) merge(b0, b1, moved(half, b0), moved(half, b1));
    if (at.shift > 3) merge(b0, b1, moved(whole, b0), moved(whole, b1));
    if (at.shift > 4) merge(b0, b1, __shfl_xor(b0, 16, 64), __shfl_xor(b1, 16, 64));
    const float best = a.group_top > 1 && b1 != none ? b0 + b1 : b0;
    // what it is at least and at most (of two keys that cancel the errors stay)
    const float off = room + (fabsf(b0) + (b1 != none ? fabsf(b1) : 0.f)) * 0x1p-22f;
    const float low = best == none ? none : best - off, high = best == none ? none : best + off;
    uint32_t ahead = 0, near = 0;   // groups ahead of this lane's for certain, and perhaps
    for (uint32_t g = 0; g < a.n_group; g++) {
        const int from = (int)(g << at.shift);
        const float olow = bits_f32((uint32_t)__builtin_amdgcn_readlane((int)f32_bits(low), from));
        const float ohigh =
            bits_f32((uint32_t)__builtin_amdgcn_readlane((int)f32_bits(high), from));
        ahead += olow > high ? 1u : 0u;
        near += g != at.lane >> at.shift && !(ohigh < low) ? 1u : 0u;
    }
    const bool stays = ahead < a.topk_group && best != none;
    const bool sure = best == none || ahead >= a.topk_group || near < a.topk_group;
    if (!a.bias) {
#pragma unroll
        for (uint32_t j = 0; j < NJ; j++) key[j] = z[j];
    }
#pragma unroll
    for (uint32_t j = 0; j < NJ; j++) key[j] = stays ? key[j] : none;
    return __all(sure);
}

// Lane k: the token's pick k, ties to the lowest expert, or -1, by keys in fp32
// (-inf: none) that are off by at most half of gap + 2^-22 of their size, or not at
// all (gap 0: equal ones may differ in 64 bits).  exact(e): expert e's key there.
//
// A key is an unsigned number of the same order (-inf: below kFinite) whose lowest
// bits give way to the lane's slot.  Finds go on until one is behind the last pick for certain; if
// some of them are not apart, their 64-bit keys, after ready(), give their order.
template <uint32_t NJ, class Ready, class Exact>
__device__ inline int32_t pick_experts(const ScoreArgs &a, const ScorePlaces &at, const float *key,
                                       float gap, Ready ready,
                                       Exact exact) {
    const double none = -(double)INFINITY;
    const uint32_t lane = at.lane;
    constexpr uint32_t kSlot = NJ - 1, kFinite = 0x00800000;
    const float part = gap > 0.f ? 0x1p-22f : 0.f;
    // the highest and lowest that a key stands for
    auto above = [](uint32_t m) { return key2f(m | kSlot); };
    auto below = [](uint32_t m) { return key2f(m & ~kSlot); };
    uint32_t high[NJ];
#pragma unroll
    for (uint32_t j = 0; j < NJ; j++) high[j] = (f2key(key[j]) & ~kSlot) | (kSlot - j);
    // a lane's in descending order (odd-even merge sort): its best is the first
#pragma unroll
    for (uint32_t p = 1; p < NJ; p *= 2)
#pragma unroll
        for (uint32_t q = p; q >= 1; q /= 2)
#pragma unroll
            for (uint32_t j = q % p; j + q < NJ; j += 2 * q)
#pragma unroll
                for (uint32_t i = 0; i < q; i++)
                    if (i + j + q < NJ && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
                        const uint32_t x = high[i + j], y = high[i + j + q];
                        high[i + j] = max(x, y), high[i + j + q] = min(x, y);
                    }
    // lane k of these: find k's key (0: none) and the lane that had it
    uint32_t key_of = 0, lane_of = 0, k = 0;
    float end = 0.f;        // finds below this are behind the last pick
    bool done = false;
    for (; k < 64; k++) {
        const uint32_t m = wave_max_u32(high[0]);
        if (m < kFinite || (k >= a.topk && above(m) < end)) {
            done = true;
            break;
        }
        if (k + 1 == a.topk) end = below(m) - (gap + fabsf(below(m)) * part);
        const uint32_t who = (uint32_t)__builtin_ctzll(__ballot(high[0] == m));
        key_of = lane == k ? m : key_of;
        lane_of = lane == k ? who : lane_of;
        const uint32_t won = lane == who ? ~0u : 0u;        // the winner's list moves up
#pragma unroll
        for (uint32_t j = 0; j < NJ; j++)
            high[j] = (j + 1 < NJ ? high[j + 1] & won : 0u) | (high[j] & ~won);
    }
    int32_t pick = key_of ? (int32_t)at.of(lane_of, kSlot - (key_of & kSlot)) : -1;
    if (done) {
        const uint32_t next = (uint32_t)__shfl_down((int)key_of, 1, 64);
        const float own = below(key_of);
        const bool apart = lane + 1 >= k || above(next) < own - (gap + fabsf(own) * part);
        if (__all(apart)) return pick;
        ready();
        // the finds hold the picks: lane i takes the one that i others are ahead of
        const double mine = pick < 0 ? none : exact((uint32_t)pick);
        uint32_t before = 0;
        for (uint32_t i = 0; i < k; i++) {
            const double o = lane_value(mine, (int)i);
            const int32_t e = __builtin_amdgcn_readlane(pick, (int)i);
            before += o > mine || (o == mine && e < pick) ? 1u : 0u;
        }
        int32_t sorted = -1;
        for (uint32_t i = 0; i < k; i++) {
            const uint32_t to = (uint32_t)__builtin_amdgcn_readlane((int)before, (int)i);
            sorted = lane == to ? __builtin_amdgcn_readlane(pick, (int)i) : sorted;
        }
        return sorted;
    }
    // More near ones than lanes, and always with 64 picks, where no find is left to be
    // behind them: the best key, on a tie of the lowest expert, topk times (8192 x 512,
    // us: 62 picks 40 with a bias; 63, some of whose tokens come here, 257; 64 711, 299
    // without a bias).
    ready();
    uint32_t alive = 0;
#pragma unroll
    for (uint32_t j = 0; j < NJ; j++) alive |= key[j] == -INFINITY ? 0u : 1u << j;
    pick = -1;
    for (k = 0; k < a.topk; k++) {
        double best = none;
        uint32_t e = 0;
#pragma unroll 1
        for (uint32_t j = 0; j < NJ; j++) {
            const double v = alive >> j & 1 ? exact(at.mine(j)) : none;
            if (v > best || (v == best && v != none && at.mine(j) < e)) best = v, e = at.mine(j);
        }
        const double m = wave_max(best);
        if (m == none) break;
        const uint32_t first = wave_min(best == m ? e : ~0u);
#pragma unroll 1
        for (uint32_t j = 0; j < NJ; j++)
            if (first == at.mine(j)) alive &= ~(1u << j);
        if (lane == k) pick = (int32_t)first;
    }
    return pick;
}

// One wave a token, NJ experts a lane.
//
// 8192 tokens x 512 experts occupy the chip once, and what bounds that is the
// number of instructions a wave, and then the last token's chain of them.  So
// scores are computed only where they decide (with a bias or groups), in fp32 with
// the hardware's exponential where that settles the groups, and 64-bit ones of the
// picks alone where those are near each other.
//
// Measured at 8192 tokens, fp32 logits: 512 experts, 10 picks with bias and 4 of 8
// groups 17 us (55 us with 64-bit scores of every expert; 14.6 us where no keys are
// near), without either 11.3 us (1.5 TB/s), 128 experts 7 us; one token 3.6 to 5 us; 480
// experts in 8 groups 16.3, in 12 (no lanes' own, so 64-bit scores of every expert) 36.  8 waves a SIMD, at the
// price of spills in the 64-bit path, against 5 without: 11.8 against 12.4 us
// without bias and groups, 8.7 against 9.7 us for 256 experts with a bias.
template <uint32_t NJ>
__global__ __launch_bounds__(64 * kScoreWaves, NJ <= 8 ? 8 : 4) void route_scored_k(ScoreArgs a) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t t = blockIdx.x * kScoreWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (t >= a.n_tok) return;
    const uint64_t row = (uint64_t)t * a.ld;
    const ScorePlaces at(a, lane);
    // Of the logits +inf counts as the largest finite one, NaN as -inf.
    auto counted = [](float z) { return z != z ? -INFINITY : fminf(z, 3.402823466e38f); };
    // All loads go out before the first is used, with one choice of the type for
    // them, at 32-bit offsets from the row; a lane without a jth expert reads the last
    // one's place of its group.
    float z[NJ], bias[NJ];
    uint32_t off[NJ];
#pragma unroll
    for (uint32_t j = 0; j < NJ; j++) off[j] = at.is(j) ? at.mine(j) : at.last();
    if (a.type == kTypeF32) {
        const char *base = (const char *)a.logits + row * 4;
#pragma unroll
        for (uint32_t j = 0; j < NJ; j++) z[j] = *(const float *)(base + off[j] * 4u);
    } else {
        const char *base = (const char *)a.logits + row * 2;
        uint16_t q[NJ];
#pragma unroll
        for (uint32_t j = 0; j < NJ; j++) q[j] = *(const uint16_t *)(base + off[j] * 2u);
#pragma unroll
        for (uint32_t j = 0; j < NJ; j++)
            z[j] = a.type == kTypeF16 ? (float)__builtin_bit_cast(_Float16, q[j])
                                      : bits_f32((uint32_t)q[j] << 16);
    }
    if (a.bias) {
#pragma unroll
        for (uint32_t j = 0; j < NJ; j++)
            bias[j] = *(const float *)((const char *)a.bias + off[j] * 4u);
    }
#pragma unroll
    for (uint32_t j = 0; j < NJ; j++) z[j] = at.is(j) ? counted(z[j]) : -INFINITY;
    const bool softmax = !a.sigmoid;
    float zmax = 0.f;
    if (softmax) {
        float top = z[0];
#pragma unroll
        for (uint32_t j = 1; j < NJ; j++) top = fmaxf(top, z[j]);
        zmax = key2f(wave_max_u32(f2key(top)));
    }
    Scores score = {softmax, (double)zmax, 1.};
    bool far = false;       // a sigmoid below 2^-1000
    bool settled = false;
    auto settle = [&]() {   // what 64-bit scores need besides
        if (settled) return;
        settled = true;
        if (softmax) {
            double sum = 0.;
#pragma unroll
            for (uint32_t j = 0; j < NJ; j++) sum += exp_series((double)z[j] - score.zmax);
            score.inv = 1. / lane_value(q4mi_rsum<64>(sum), 63);
        } else {
#pragma unroll
            for (uint32_t j = 0; j < NJ; j++) far |= z[j] < -690.f && z[j] != -INFINITY;
            far = __any(far);
        }
    };
    float key[NJ], gap = 0.f;
#pragma unroll
    for (uint32_t j = 0; j < NJ; j++) key[j] = z[j];
    if (a.bias || a.n_group > 1) {
        // errors of a sigmoid (four roundings, the hardware's exponential and
        // reciprocal within an ulp: under 2^-22), and of a softmax score, whose
        // sum has up to 22 roundings in a row: under 2^-18.8
        const float room = softmax ? 0x1p-17f : 0x1p-20f;
        if (a.bias) gap = room;
        if (!at.in_lanes || !keys_fast<NJ>(a, at, z, bias, zmax, room, key)) {
            settle();
            keys_exact<NJ>(a, at, z, bias, score, far, key);
            gap = 0.f;
        }
    }
    auto logit = [&](uint32_t e) { return counted(load_as_f32(a.logits, a.type, row + e)); };
    auto ready = [&]() {
        if (a.bias) settle();
    };
    int32_t mine = pick_experts<NJ>(a, at, key, gap, ready, [&](uint32_t e) -> double {
        const float x = logit(e);
        if (!a.bias) return (double)x;
        return score.any(x) + (double)a.bias[e];
    });
    if (lane >= a.topk) mine = -1;
    if (softmax && !a.renorm) settle();     // of renormalised weights it cancels out
    // lane k: weight of pick k
    double w = mine >= 0 ? score.any(logit((uint32_t)mine)) : 0.;
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
    const uint32_t a_lane = (a.n_exp + 63) / 64;    // with equal groups no lane has more
    auto k = a_lane <= 1   ? route_scored_k<1>
             : a_lane <= 2 ? route_scored_k<2>
             : a_lane <= 4 ? route_scored_k<4>
             : a_lane <= 8 ? route_scored_k<8>
                           : route_scored_k<16>;
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

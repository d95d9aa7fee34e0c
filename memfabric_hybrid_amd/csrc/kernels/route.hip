/*
 * Routing by groups of experts, and its gradient.
 *
 * s = sigmoid(l) or softmax(l); c = s + bias decides, s weighs. A token's experts are the K largest c of its best groups, ties to the lower
 * index; its weights are their s, over their sum if asked for, times a factor.
 *
 * The picks turn on the difference of two c, however small, so they are those of 64 bits. But 32 bits tell almost everything apart: a wave takes the
 * groups, and in them a few candidates more than there are picks, by choices of 32 bits (without a bias by the logits, whose order is that of the
 * scores), and ranks the candidates, one to a lane, by their choices in 64 bits, of whose scores the weights are made. A row whose groups are
 * closer than the rounding of 32 bits (one in some thousands) is worked out in 64 bits from the start. What bounds it is the number of
 * instructions: 8192 tokens, 256 experts in eight groups, 13.4 us; all rows in 64 bits 19.6; picks by rounds of arg-max in 32 bits 21.8.
 */
#include "zbal_device.h"
#include "zbal_hip_kernels.h"

namespace {

constexpr int kMaxExperts = 1024, kMaxGroups = 64, kMaxTopk = 32;
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));

enum { SCORE_SIGMOID = 0, SCORE_SOFTMAX = 1, GROUP_BY_TOP2 = 0, GROUP_BY_MAX = 1 };

__device__ __forceinline__ float logit_at(const void *p, int dtype, int64_t i)
{
    if (dtype == ZDT_FP32) return static_cast<const float *>(p)[i];
    const uint16_t h = static_cast<const uint16_t *>(p)[i];
    return dtype == ZDT_BF16 ? zb_bf16_to_f32(h) : zb_fp16_to_f32(h);
}

template <int CTRL> __device__ __forceinline__ int swapped(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true); }
template <int CTRL> __device__ __forceinline__ float swapped(float v) { return __int_as_float(swapped<CTRL>(__float_as_int(v))); }
template <int CTRL> __device__ __forceinline__ double swapped(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)swapped<CTRL>((int)(uint32_t)u), hi = (uint32_t)swapped<CTRL>((int)(uint32_t)(u >> 32));
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
/* over each run of LANES lanes, to all of them: neighbours, pairs, the halves of eight and of sixteen mirrored, then the rest */
template <int LANES, typename V, typename F> __device__ __forceinline__ V over_lanes(V v, F join)
{
    v = join(v, swapped<0xB1>(v));
    v = join(v, swapped<0x4E>(v));
    v = join(v, swapped<0x141>(v));
    v = join(v, swapped<0x140>(v));
    if constexpr (LANES >= 32) v = join(v, __shfl_xor(v, 16, 64));
    if constexpr (LANES >= 64) v = join(v, __shfl_xor(v, 32, 64));
    return v;
}

__device__ __forceinline__ double lane_f64(double v, int lane)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint64_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
    return __builtin_bit_cast(double, hi << 32 | lo);
}
struct RouteParams {
    const void *logits;
    int dtype, tokens, experts, topk, groups, kept, score, by_max, renormalize;
    double scale;
    const float *bias;
    void *idx;
    int idx_i64;
    float *w;
    int log2_lanes;              /* of a group's lanes: 64 over the groups, rounded down to a power of two */
};

/* sum of lanes 0 .. n - 1 in their order */
__device__ __forceinline__ double first_lanes_sum_f64(double v, int n)
{
    double sum = 0.0;
    for (int k = 0; k < n; ++k) sum += lane_f64(v, k);
    return sum;
}

struct Candidate {
    float logit, bias;
    int expert, pad;
};

/* slot `slot` of a token's picks */
__device__ __forceinline__ void put_pick(const RouteParams &p, int t, int slot, int pick, double weight, double sum)
{
    if (p.renormalize) weight = sum > 0.0 ? weight / sum : 0.0;
    if (slot < p.topk) {
        const int64_t at = (int64_t)t * p.topk + slot;
        if (p.idx_i64) static_cast<int64_t *>(p.idx)[at] = pick;
        else static_cast<int32_t *>(p.idx)[at] = pick;
        p.w[at] = (float)(weight * p.scale);
    }
}

/*
 * A token's row has a wave. A group has `lanes` consecutive lanes, and a lane SLOTS of its experts, `lanes` apart: what a group needs is a reduction
 * inside it, and the lowest index of equal experts is in the lowest lane's group, there in the lowest slot, there in the lowest lane.
 */
template <int SLOTS> struct RouteRow {
    const RouteParams &p;
    const int t, lane, per, group, sub;
    float l[SLOTS], mx;

    __device__ __forceinline__ RouteRow(const RouteParams &p_, int t_, int lane_)
        : p(p_), t(t_), lane(lane_), per(p_.experts / p_.groups), group(lane_ >> p_.log2_lanes), sub(lane_ & ((1 << p_.log2_lanes) - 1))
    {
        mx = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) {
            l[i] = mine(i) ? logit_at(p.logits, p.dtype, (int64_t)t * p.experts + expert_of(i)) : -__builtin_inff();
            mx = fmaxf(mx, l[i]);
        }
    }
    __device__ __forceinline__ int expert_of(int i) const { return group * per + (i << p.log2_lanes) + sub; }
    __device__ __forceinline__ bool mine(int i) const { return group < p.groups && (i << p.log2_lanes) + sub < per; }
    /* number of groups with a larger score, or an equal one and a lower index */
    template <typename V> __device__ __forceinline__ int rank_of_group(V score) const
    {
        int rank = 0;
        for (int g = 0; g < p.groups; ++g) {
            V o;
            if constexpr (sizeof(V) == 8) o = lane_f64(score, g << p.log2_lanes);
            else o = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(score), g << p.log2_lanes));
            rank += o > score || (o == score && g < group) ? 1 : 0;
        }
        return rank;
    }

    /* everything in 64 bits */
    __device__ void exact()
    {
        const double none = -__builtin_inf();
        double s[SLOTS], c[SLOTS];
        if (p.score == SCORE_SOFTMAX) {
            const float top = zb_wave_reduce_dpp<true>(mx);
            double part = 0.0;
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) {
                s[i] = mine(i) ? exp((double)l[i] - (double)top) : 0.0;
                part += s[i];
            }
            const double sum = over_lanes<64>(part, [](double a, double b) { return a + b; });
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) s[i] /= sum;
        } else {
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) s[i] = 1.0 / (1.0 + exp(-(double)l[i]));
        }
        /* what may be picked: an expert whose logit is not minus infinity and whose choice is neither that nor no number */
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) {
            c[i] = s[i];
            if (p.bias && mine(i)) c[i] += (double)p.bias[expert_of(i)];
            if (!(mine(i) && l[i] > -__builtin_inff() && c[i] > none)) c[i] = none;
        }
        if (p.groups > 1) {
            double b1 = c[0], b2 = none;
#pragma unroll
            for (int i = 1; i < SLOTS; ++i) {
                b2 = fmax(b2, fmin(b1, c[i]));
                b1 = fmax(b1, c[i]);
            }
            for (int off = 1; off < 1 << p.log2_lanes; off <<= 1) {
                const double o1 = __shfl_xor(b1, off, 64), o2 = __shfl_xor(b2, off, 64);
                b2 = fmax(fmin(b1, o1), fmax(b2, o2));
                b1 = fmax(b1, o1);
            }
            if (rank_of_group(p.by_max || b2 == none ? b1 : b1 + b2) >= p.kept)
#pragma unroll
                for (int i = 0; i < SLOTS; ++i) c[i] = none;
        }
        /* K rounds of arg-max; lane k keeps the k-th pick */
        int pick = -1;
        double weight = 0.0;
        for (int k = 0; k < p.topk; ++k) {
            double best = c[0];
#pragma unroll
            for (int i = 1; i < SLOTS; ++i) best = fmax(best, c[i]);
            best = over_lanes<64>(best, [](double a, double b) { return fmax(a, b); });
            if (best == none) break;
            int e = 0x7fffffff;
            double es = 0.0;
#pragma unroll
            for (int i = SLOTS - 1; i >= 0; --i)
                if (c[i] == best) { e = expert_of(i); es = s[i]; }
            const int lowest = over_lanes<64>(e, [](int a, int b) { return a < b ? a : b; });
            const int owner = __ffsll((long long)__ballot(e == lowest)) - 1;
            es = lane_f64(es, owner);
#pragma unroll
            for (int i = 0; i < SLOTS; ++i)
                if (expert_of(i) == lowest && mine(i)) c[i] = none;
            if (lane == k) { pick = lowest; weight = es; }
        }
        put_pick(p, t, lane, pick, weight, p.renormalize ? first_lanes_sum_f64(weight, p.topk) : 0.0);
    }

    /*
     * By 32 bits as far as they decide; false, with nothing written, where they do not.
     *
     * How far choices of 32 bits may be off, in steps of 2^-24. A sigmoid: 2 |l| of its exponential for the rounding of the argument, which its slope makes 0.45, the
     * exponential's own 2 a quarter of that, sum and quotient 3: under 4. A softmax: 3 |l - max| of the score, which is at most exp(l - max), so 1.1; its
     * exponential, quotient and product 6: under 7.1, with the sum in 64 bits (without a bias the sum's error is a common factor of all choices, and changes no order).
     * The choice's own rounding: 1 of its size. So 8.1 of the larger of one and the choice. Two choices in question are 16.2 apart at most, and 1 for what
     * the limit itself is rounded by: kStep is 64. A group's sum is off by what its two choices are, whose sizes a bias may make far larger than the sum, and
     * the rounding of the sum and of its bounds, 2 of the two sizes: 10.1 of each size, where kOff is 16.
     */
    __device__ bool quick(Candidate *candidates)
    {
        constexpr float kStep = 0x1p-18f, kOff = 0x1p-20f;
        const float none = -__builtin_inff();
        const bool by_logit = p.bias == nullptr;       /* the order of the logits is that of the scores */
        float key[SLOTS], c[SLOTS], b[SLOTS], top = 0.0f;
        double sum = 1.0;
        if (p.score == SCORE_SOFTMAX) {
            top = zb_wave_reduce_dpp<true>(mx);
            float part = 0.0f;
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) {
                c[i] = mine(i) ? __builtin_amdgcn_exp2f((l[i] - top) * 1.44269504f) : 0.0f;
                part += c[i];
            }
            /* over the sum of the picks' scores, the sum of all cancels */
            if (!by_logit || !p.renormalize) {
                double d = 0.0;
#pragma unroll
                for (int i = 0; i < SLOTS; ++i) d += mine(i) ? exp((double)l[i] - (double)top) : 0.0;
                sum = over_lanes<64>(d, [](double a, double b) { return a + b; });
                part = (float)sum;
            } else {
                part = zb_wave_reduce_dpp<false>(part);
            }
            const float over = __builtin_amdgcn_rcpf(part);
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) c[i] *= over;
        } else {
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) c[i] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(l[i] * -1.44269504f));
        }
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) {
            b[i] = !by_logit && mine(i) ? p.bias[expert_of(i)] : 0.0f;
            c[i] += b[i];
            const bool ok = mine(i) && l[i] > none && c[i] > none;
            key[i] = ok ? (by_logit ? l[i] : c[i]) : none;
            if (!ok) c[i] = none;
        }
        if (p.groups > 1) {
            float b1 = p.by_max ? key[0] : c[0], b2 = none;
#pragma unroll
            for (int i = 1; i < SLOTS; ++i) {
                const float v = p.by_max ? key[i] : c[i];
                b2 = fmaxf(b2, fminf(b1, v));
                b1 = fmaxf(b1, v);
            }
            auto join = [&](float o1, float o2) __attribute__((always_inline)) {
                b2 = fmaxf(fminf(b1, o1), fmaxf(b2, o2));
                b1 = fmaxf(b1, o1);
            };
            if (p.log2_lanes > 0) join(swapped<0xB1>(b1), swapped<0xB1>(b2));        /* quads: neighbours, then pairs */
            if (p.log2_lanes > 1) join(swapped<0x4E>(b1), swapped<0x4E>(b2));
            if (p.log2_lanes > 2) join(swapped<0x141>(b1), swapped<0x141>(b2));      /* the halves of eight and of sixteen lanes, mirrored */
            if (p.log2_lanes > 3) join(swapped<0x140>(b1), swapped<0x140>(b2));
            if (p.log2_lanes > 4) join(__shfl_xor(b1, 16, 64), __shfl_xor(b2, 16, 64));
            const bool two = !p.by_max && b2 > none, exact_keys = p.by_max && by_logit;
            /* a sum past the lowest number is still more than a group that has no experts */
            const float score = two ? fmaxf(b1 + b2, -3.402823466e38f) : b1;
            const bool keep = rank_of_group(score) < p.kept && group < p.groups;
            /* the least that a group kept can be against the most that one of the others can be; logits are what they are */
            float off = b1 > none && !exact_keys ? kOff * fmaxf(1.0f, fabsf(b1)) : 0.0f;
            if (two) off += kOff * fmaxf(1.0f, fabsf(b2));
            const float least = -zb_wave_reduce_dpp<true>(keep ? off - score : none), most = zb_wave_reduce_dpp<true>(keep || group >= p.groups ? none : score + off);
            const float gap = least - most, apart = exact_keys ? kStep * fmaxf(1.0f, fmaxf(fabsf(least), fabsf(most))) : 0.0f;
            /* equal logits are a tie, for the lower index, if the next ones above have scores of 64 bits above theirs */
            const bool tie = exact_keys && gap == 0.0f && fabsf(least) > 0x1p-10f && least < 20.0f && least - top > -600.0f;
            if (most > none && !(gap > apart) && !tie) return false;
            if (!keep)
#pragma unroll
                for (int i = 0; i < SLOTS; ++i) key[i] = none;
        }
        /* a value that the topk largest reach and not many more: halving the interval from the least to the largest */
        float high = key[0], low = key[0] > none ? key[0] : __builtin_inff();
#pragma unroll
        for (int i = 1; i < SLOTS; ++i) {
            high = fmaxf(high, key[i]);
            low = fminf(low, key[i] > none ? key[i] : __builtin_inff());
        }
        high = zb_wave_reduce_dpp<true>(high);
        low = -zb_wave_reduce_dpp<true>(-low);
        if (high == __builtin_inff()) return false;    /* nothing to halve */
        uint64_t has[SLOTS];
        auto reach = [&](float v) __attribute__((always_inline)) {       /* v is finite, or no number */
            int n = 0;
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) {
                has[i] = __ballot(key[i] >= v);
                n += __popcll(has[i]);
            }
            return n;
        };
        if (high == none) low = 0.0f;                  /* nothing to pick */
        int count = reach(low);
        const int enough = p.topk + 4;
        for (int i = 0; i < 40 && count > enough; ++i) {
            /* the first step leaves out what is far below, as a masked value is */
            const float mid = fmaxf(0.5f * (low + high), i == 0 ? high - 32.0f : low);
            if (!(mid > low && mid < high)) break;
            const int n = reach(mid);
            if (n >= p.topk) { low = mid; count = n; }
            else high = mid;
        }
        /* and what rounding may have left below it */
        count = reach(fmaxf(low - kStep * fmaxf(1.0f, fabsf(low)), -3.402823466e38f));
        if (count > 64) return false;
        int before = 0;
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) {
            const int at = before + __builtin_amdgcn_mbcnt_hi((uint32_t)(has[i] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)has[i], 0));
            if (has[i] >> lane & 1) candidates[at] = {l[i], b[i], expert_of(i), 0};
            before += __popcll(has[i]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        /* lane k has candidate k: its score and choice in 64 bits, and its rank among them */
        const bool there = lane < count;
        const Candidate mine_k = candidates[there ? lane : 0];
        double score = 0.0, choice = -__builtin_inf();
        if (there) {
            score = p.score == SCORE_SIGMOID ? 1.0 / (1.0 + exp(-(double)mine_k.logit)) : exp((double)mine_k.logit - (double)top) / sum;
            choice = by_logit ? score : score + (double)mine_k.bias;
        }
        /* logits so far out that scores of 64 bits are equal where they are not: others may belong here by their index */
        const bool far = p.score == SCORE_SIGMOID ? !(mine_k.logit < 20.0f && mine_k.logit > -600.0f) : !(mine_k.logit - top > -600.0f);
        if (__ballot(there && far) != 0) return false;
        int rank = 0;
        for (int k = 0; k < count; ++k) {
            const double o = lane_f64(choice, k);
            const int e = __builtin_amdgcn_readlane(mine_k.expert, k);
            rank += o > choice || (o == choice && e < mine_k.expert) ? 1 : 0;
        }
        const bool picked = there && rank < p.topk;
        double total = 0.0;
        if (p.renormalize)
            for (uint64_t left = __ballot(picked); left != 0; left &= left - 1) total += lane_f64(score, __ffsll((long long)left) - 1);
        /* the picks' slots, then those that are left over */
        if (picked || (lane >= count && lane < p.topk)) put_pick(p, t, picked ? rank : lane, picked ? mine_k.expert : -1, picked ? score : 0.0, total);
        return true;
    }
};

template <int SLOTS>
__global__ void __launch_bounds__(256)
group_route_kernel(RouteParams p)
{
    const int t = blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6);
    if (t >= p.tokens) return;                   /* whole waves leave together */
    __shared__ Candidate candidates[4][64];
    RouteRow<SLOTS> row(p, t, threadIdx.x & 63);
    if (!row.quick(candidates[threadIdx.x >> 6])) row.exact();
}

struct RouteBackParams {
    const float *grad;
    const void *logits;
    int dtype, tokens, experts, topk, score, renormalize;
    double scale;
    ExpertIds idx;
    void *out;
};

__device__ __forceinline__ void put_logit(void *p, int dtype, int64_t i, float v)
{
    if (dtype == ZDT_FP32) static_cast<float *>(p)[i] = v;
    else static_cast<uint16_t *>(p)[i] = (uint16_t)(dtype == ZDT_BF16 ? zb_f32_to_bf16(v) : zb_f32_to_fp16(v));
}

/* 2^y, y <= 0, to 2^-32: the whole part is the exponent, the rest, up to a half, goes through the polynomial that meets 2^f in the eight Chebyshev nodes. No number: 0 */
__device__ __forceinline__ double exp2_of(double y)
{
    y = fmax(y, -1400.0);
    const double n = __builtin_rint(y), f = y - n;
    double v = 1.5303699001378845e-05;
    v = __builtin_fma(v, f, 0.00015469729140704658);
    v = __builtin_fma(v, f, 0.0013333478480888061);
    v = __builtin_fma(v, f, 0.009618025613598036);
    v = __builtin_fma(v, f, 0.055504109063177154);
    v = __builtin_fma(v, f, 0.24022651213495422);
    v = __builtin_fma(v, f, 0.6931471805568341);
    v = __builtin_fma(v, f, 0.9999999999595622);
    return __builtin_amdgcn_ldexp(v, (int)n);
}

/*
 * Lane k of a token's LANES has its k-th pick: d_k = dL/ds_k is scale g_k, or, where the weights are over their sum S, scale / S (g_k -
 * sum_j g_j s_j / S). An expert's D is the sum over its picks (the first of them adds up in order, should an expert be there twice).
 * sigmoid: dl = D s (1 - s), nothing where there is no pick. softmax: dl = s (D - sum D s): with weights over their sum, sum D s is zero and
 * nothing but the picks has a gradient either; else every logit has one. A row that has no pick has a gradient of zeros whatever its logits, and so has
 * one whose logits are all minus infinity, where a softmax is no number.
 *
 * All of it is in 64 bits, rounded once (exponentials, their sum and the last product in 32: 0.2 us less where a row has 128 experts, 1.6 of 10.1 for 4096 tokens of
 * 1024, and twice the error). The picks' part is the same number of instructions for one token as for four, so a wave has as many tokens as
 * their picks and a sixteenth of their logits leave room for; the logits are read once, four at a time, and stay in registers. 16384 tokens, 128 experts,
 * softmax over all: 6.9 us, one token to a wave 16.7; 8192 tokens, 256 experts, sigmoid: 4.2 and 7.9.
 */
constexpr int kBackLogits = 16;                  /* of a lane */
constexpr double kLog2e = 1.4426950408889634;
constexpr int kUnpicked = 0x7fc05eed;            /* a place of the row that no pick has written: a NaN that arithmetic does not make */

template <int LANES, bool VEC>
__global__ void __launch_bounds__(256)
group_route_backward_kernel(RouteBackParams p)
{
    constexpr int V = VEC ? 4 : 1;
    extern __shared__ float rows[];              /* [256 / LANES][experts] */
    const int sub = threadIdx.x & (LANES - 1), r = threadIdx.x / LANES, own = blockIdx.x * (256 / LANES) + r;
    const bool live = own < p.tokens;            /* the others repeat the last token, and store nothing */
    const int t = live ? own : p.tokens - 1;
    float *row = rows + r * p.experts;
    const int64_t base = (int64_t)t * p.experts;
    const bool dense = p.score == SCORE_SOFTMAX && !p.renormalize;
    const float none = -__builtin_inff();
    auto plus = [](auto a, auto b) __attribute__((always_inline)) { return a + b; };
    auto larger = [](float a, float b) __attribute__((always_inline)) { return fmaxf(a, b); };

    const float unpicked = dense ? __int_as_float(kUnpicked) : 0.0f;
    float x[kBackLogits], mx = none;
#pragma unroll
    for (int c = 0; c < kBackLogits / V; ++c) {
        const int at = (c * LANES + sub) * V;
        if (at >= p.experts) continue;
        if constexpr (VEC) *reinterpret_cast<f32x4 *>(row + at) = f32x4{unpicked, unpicked, unpicked, unpicked};
        else row[at] = unpicked;
    }
    int e = -1;
    double g = 0.0, s = 0.0;
    float l = none;
    if (sub < p.topk) {
        e = p.idx[(int64_t)t * p.topk + sub];
        if (e < 0 || e >= p.experts) e = -1;
    }
    if (e >= 0) {
        g = (double)p.grad[(int64_t)t * p.topk + sub] * p.scale;
        l = logit_at(p.logits, p.dtype, base + e);
    }
    double sum = 1.0, ex[kBackLogits];
    if (dense) {
#pragma unroll
        for (int c = 0; c < kBackLogits / V; ++c) {
            const int at = (c * LANES + sub) * V;
#pragma unroll
            for (int j = 0; j < V; ++j) x[c * V + j] = none;
            if (at >= p.experts) continue;
            if constexpr (!VEC) x[c] = logit_at(p.logits, p.dtype, base + at);
            else if (p.dtype == ZDT_FP32) {
                const f32x4 v = *reinterpret_cast<const f32x4 *>(static_cast<const float *>(p.logits) + base + at);
#pragma unroll
                for (int j = 0; j < V; ++j) x[c * V + j] = v[j];
            } else {
                const u16x4 v = *reinterpret_cast<const u16x4 *>(static_cast<const uint16_t *>(p.logits) + base + at);
#pragma unroll
                for (int j = 0; j < V; ++j) x[c * V + j] = p.dtype == ZDT_BF16 ? zb_bf16_to_f32(v[j]) : zb_fp16_to_f32(v[j]);
            }
        }
#pragma unroll
        for (int i = 0; i < kBackLogits; ++i) mx = fmaxf(mx, x[i]);
        mx = over_lanes<LANES>(mx, larger);
        const bool none_picked = over_lanes<LANES>(e, [](int a, int b) __attribute__((always_inline)) { return a > b ? a : b; }) < 0;
        double part = 0.0;
        if (none_picked || mx == none) {
#pragma unroll
            for (int i = 0; i < kBackLogits; ++i) ex[i] = 0.0;
            part = 1.0 / LANES;
        } else {
#pragma unroll
            for (int c = 0; c < kBackLogits / V; ++c) {
                if (c * LANES * V >= p.experts) continue;            /* nobody's */
#pragma unroll
                for (int i = c * V; i < c * V + V; ++i) {
                    ex[i] = exp2_of(__builtin_fma((double)x[i], kLog2e, (double)mx * -kLog2e));
                    part += ex[i];
                }
            }
            bool nan = false;
#pragma unroll
            for (int i = 0; i < kBackLogits; i += 2) nan = nan || __builtin_isunordered(x[i], x[i + 1]);
            if (nan) part = __builtin_nan("");
        }
        sum = over_lanes<LANES>(part, plus);
    } else if (p.score == SCORE_SOFTMAX) {
        mx = over_lanes<LANES>(l, larger);                   /* the other logits cancel */
    }
    if (e >= 0) s = p.score == SCORE_SIGMOID ? 1.0 / (1.0 + exp(-(double)l)) : (l == none ? 0.0 : exp((double)l - (double)mx) / sum);
    double d = g;
    if (p.renormalize) {
        const double total = over_lanes<LANES>(s, plus), gs = over_lanes<LANES>(g * s, plus);
        d = e >= 0 && total > 0.0 ? (g - gs / total) / total : 0.0;
    }
    const double c = dense ? over_lanes<LANES>(d * s, plus) : 0.0, rest = -c / sum;

    /* an expert that is there twice: its place in the row holds one lane's number only */
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (e >= 0) row[e] = __int_as_float(sub);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    bool first = e >= 0;
    double all = d;
    if (__ballot(e >= 0 && __float_as_int(row[e >= 0 ? e : 0]) != sub) != 0) {
        for (int k = 0; k < p.topk; ++k) {
            const int ek = __shfl(e, k, LANES);
            const double dk = __shfl(d, k, LANES);
            if (ek == e && k != sub) {
                if (k < sub) first = false;
                else all += dk;
            }
        }
    }
    if (p.score == SCORE_SIGMOID) all *= s * (1.0 - s);
    else all = dense ? s * (all - c) : all * s;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (first) row[e] = (float)all;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int k = 0; k < kBackLogits / V; ++k) {
        const int at = (k * LANES + sub) * V;
        if (at >= p.experts || !live) continue;
        f32x4 v;
        if constexpr (VEC) v = *reinterpret_cast<const f32x4 *>(row + at);
        else v[0] = row[at];
        if (dense)
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = __float_as_int(v[j]) == kUnpicked ? (float)(ex[k * V + j] * rest) : v[j];
        if constexpr (!VEC) put_logit(p.out, p.dtype, base + at, v[0]);
        else if (p.dtype == ZDT_FP32) *reinterpret_cast<f32x4 *>(static_cast<float *>(p.out) + base + at) = v;
        else {
            u16x4 h;
#pragma unroll
            for (int j = 0; j < V; ++j) h[j] = (uint16_t)(p.dtype == ZDT_BF16 ? zb_f32_to_bf16(v[j]) : zb_f32_to_fp16(v[j]));
            *reinterpret_cast<u16x4 *>(static_cast<uint16_t *>(p.out) + base + at) = h;
        }
    }
}

template <int LANES> void launch_backward(const RouteBackParams &p, bool vec, hipStream_t stream)
{
    const dim3 grid((unsigned)((p.tokens + 256 / LANES - 1) / (256 / LANES))), block(256);
    const size_t lds = (size_t)p.experts * (256 / LANES) * sizeof(float);
    if (vec) zb_launch(group_route_backward_kernel<LANES, true>, grid, block, lds, stream, p);
    else zb_launch(group_route_backward_kernel<LANES, false>, grid, block, lds, stream, p);
}

} // namespace

extern "C" int32_t zbalhip_group_route(const zbalhip_group_route_t *d, void *topk_idx, int32_t idx_is_i64, float *topk_w, void *stream)
{
    if (!d || d->tokens < 0 || d->tokens > ZBALHIP_ROUTE_MAX_TOKENS || d->experts <= 0 || d->experts > kMaxExperts || d->topk <= 0 || d->topk > kMaxTopk ||
        d->topk > d->experts || d->groups <= 0 || d->groups > kMaxGroups || d->experts % d->groups != 0 || d->kept_groups <= 0 ||
        d->kept_groups > d->groups || d->topk > d->kept_groups * (d->experts / d->groups) || (d->score & ~1) || (d->group_score & ~1))
        return ZBALHIP_INVALID;
    if (d->dtype != ZDT_FP32 && d->dtype != ZDT_BF16 && d->dtype != ZDT_FP16) return ZBALHIP_INVALID;
    if (d->tokens == 0) return ZBALHIP_OK;
    if (!d->logits || !topk_idx || !topk_w) return ZBALHIP_INVALID;
    RouteParams p = {d->logits, d->dtype, (int)d->tokens, (int)d->experts, (int)d->topk, (int)d->groups, (int)d->kept_groups, d->score,
                     d->group_score, d->renormalize, d->scale, d->bias, topk_idx, idx_is_i64, topk_w, 6};
    while ((p.groups << p.log2_lanes) > 64) --p.log2_lanes;
    const int lanes = 1 << p.log2_lanes, slots = (p.experts / p.groups + lanes - 1) / lanes;
    const dim3 grid((unsigned)((d->tokens + 3) / 4)), block(256);
    hipStream_t st = (hipStream_t)stream;
    if (slots <= 1) zb_launch(group_route_kernel<1>, grid, block, 0, st, p);
    else if (slots <= 2) zb_launch(group_route_kernel<2>, grid, block, 0, st, p);
    else if (slots <= 4) zb_launch(group_route_kernel<4>, grid, block, 0, st, p);
    else if (slots <= 8) zb_launch(group_route_kernel<8>, grid, block, 0, st, p);
    else if (slots <= 16) zb_launch(group_route_kernel<16>, grid, block, 0, st, p);
    else zb_launch(group_route_kernel<32>, grid, block, 0, st, p);
    return zbalhip_check_launch();
}

extern "C" int32_t zbalhip_group_route_backward(const zbalhip_group_route_t *d, const float *grad_w, const void *topk_idx,
                                                int32_t idx_is_i64, void *grad_logits, void *stream)
{
    if (!d || d->tokens < 0 || d->tokens > ZBALHIP_ROUTE_MAX_TOKENS || d->experts <= 0 || d->experts > kMaxExperts || d->topk <= 0 || d->topk > kMaxTopk ||
        (d->score & ~1))
        return ZBALHIP_INVALID;
    if (d->dtype != ZDT_FP32 && d->dtype != ZDT_BF16 && d->dtype != ZDT_FP16) return ZBALHIP_INVALID;
    if (d->tokens == 0) return ZBALHIP_OK;
    if (!d->logits || !topk_idx || !grad_w || !grad_logits) return ZBALHIP_INVALID;
    const RouteBackParams p = {grad_w, d->logits, d->dtype, (int)d->tokens, (int)d->experts, (int)d->topk, d->score, d->renormalize,
                               d->scale, expert_ids(topk_idx, idx_is_i64 != 0, true), grad_logits};
    const uintptr_t both = (uintptr_t)p.logits | (uintptr_t)p.out;
    const bool vec = p.experts % 4 == 0 && both % (p.dtype == ZDT_FP32 ? 16 : 8) == 0;
    if (p.topk <= 16 && p.experts <= 16 * kBackLogits) launch_backward<16>(p, vec, (hipStream_t)stream);
    else if (p.experts <= 32 * kBackLogits) launch_backward<32>(p, vec, (hipStream_t)stream);
    else launch_backward<64>(p, vec, (hipStream_t)stream);
    return zbalhip_check_launch();
}

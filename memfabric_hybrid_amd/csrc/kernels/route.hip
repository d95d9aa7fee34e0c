/*
 * Routing by groups of experts, and its gradient.
 *
 * s = sigmoid(l) or softmax(l); c = s + bias decides, s weighs. A token's experts are the K largest c of its best groups, ties to the lower
 * index; its weights are their s, over their sum if asked for, times a factor. The picks turn on the difference of two c, however
 * small, so scores, choices and their sums are held in 64 bits, where the vector units are as fast as in 32.
 */
#include "zbal_device.h"
#include "zbal_hip_kernels.h"

namespace {

constexpr int kMaxExperts = 1024, kMaxGroups = 64, kMaxTopk = 32;
enum { SCORE_SIGMOID = 0, SCORE_SOFTMAX = 1, GROUP_BY_TOP2 = 0, GROUP_BY_MAX = 1 };

__device__ __forceinline__ float logit_at(const void *p, int dtype, int64_t i)
{
    if (dtype == ZDT_FP32) return static_cast<const float *>(p)[i];
    const uint16_t h = static_cast<const uint16_t *>(p)[i];
    return dtype == ZDT_BF16 ? zb_bf16_to_f32(h) : zb_fp16_to_f32(h);
}

__device__ __forceinline__ double shfl_xor_f64(double v, int mask) { return __shfl_xor(v, mask, 64); }
__device__ __forceinline__ double lane_f64(double v, int lane)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint64_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
    return __builtin_bit_cast(double, hi << 32 | lo);
}
__device__ __forceinline__ double wave_max_f64(double v)
{
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = fmax(v, shfl_xor_f64(v, off));
    return v;
}
__device__ __forceinline__ double wave_sum_f64(double v)
{
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += shfl_xor_f64(v, off);
    return v;
}

struct RouteParams {
    const void *logits;
    int dtype, tokens, experts, topk, groups, kept, score, by_max, renormalize;
    double scale;
    const float *bias;
    void *idx;
    int idx_i64;
    float *w;
    int lanes;                   /* of a group: 64 over the groups, rounded down to a power of two */
};

/*
 * One wave per token. A group has `lanes` consecutive lanes, and a lane SLOTS of its experts, `lanes` apart: what a group needs is a
 * reduction inside it.
 */
template <int SLOTS>
__global__ void __launch_bounds__(256)
group_route_kernel(RouteParams p)
{
    const int lane = threadIdx.x & 63;
    const int t = blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6);
    if (t >= p.tokens) return;                   /* whole waves leave together */
    const double none = -__builtin_inf();
    const int per = p.experts / p.groups, group = lane / p.lanes, sub = lane % p.lanes;
    double s[SLOTS], c[SLOTS];
    float l[SLOTS];
    auto expert_of = [&](int i) __attribute__((always_inline)) { return group * per + i * p.lanes + sub; };
    auto mine = [&](int i) __attribute__((always_inline)) { return group < p.groups && i * p.lanes + sub < per; };
    float mx = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
        l[i] = mine(i) ? logit_at(p.logits, p.dtype, (int64_t)t * p.experts + expert_of(i)) : -__builtin_inff();
        mx = fmaxf(mx, l[i]);
    }
    if (p.score == SCORE_SOFTMAX) {
        mx = zb_wave_reduce_dpp<true>(mx);
        double part = 0.0;
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) {
            s[i] = mine(i) ? exp((double)l[i] - (double)mx) : 0.0;
            part += s[i];
        }
        const double sum = wave_sum_f64(part);
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
        for (int off = 1; off < p.lanes; off <<= 1) {
            const double o1 = shfl_xor_f64(b1, off), o2 = shfl_xor_f64(b2, off);
            b2 = fmax(fmin(b1, o1), fmax(b2, o2));
            b1 = fmax(b1, o1);
        }
        const double score = p.by_max || b2 == none ? b1 : b1 + b2;
        int rank = 0;
        for (int g = 0; g < p.groups; ++g) {
            const double o = lane_f64(score, g * p.lanes);
            rank += o > score || (o == score && g < group) ? 1 : 0;
        }
        if (rank >= p.kept)
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
        best = wave_max_f64(best);
        if (best == none) break;
        int e = 0x7fffffff;
        double es = 0.0;
#pragma unroll
        for (int i = SLOTS - 1; i >= 0; --i)
            if (c[i] == best) { e = expert_of(i); es = s[i]; }
        int lowest = e;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            const int o = __shfl_xor(lowest, off, 64);
            lowest = o < lowest ? o : lowest;
        }
        const int owner = __ffsll((long long)__ballot(e == lowest)) - 1;
        es = lane_f64(es, owner);
#pragma unroll
        for (int i = 0; i < SLOTS; ++i)
            if (expert_of(i) == lowest && mine(i)) c[i] = none;
        if (lane == k) { pick = lowest; weight = es; }
    }
    if (p.renormalize) {
        const double sum = wave_sum_f64(weight);
        weight = sum > 0.0 ? weight / sum : 0.0;
    }
    if (lane < p.topk) {
        const int64_t at = (int64_t)t * p.topk + lane;
        if (p.idx_i64) static_cast<int64_t *>(p.idx)[at] = pick;
        else static_cast<int32_t *>(p.idx)[at] = pick;
        p.w[at] = (float)(weight * p.scale);
    }
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

/*
 * One wave per token, lane k its k-th pick: d_k = dL/ds_k is scale g_k, or, where the weights are over their sum S, scale / S (g_k -
 * sum_j g_j s_j / S). An expert's D is the sum over its picks (the first of them adds up in order, should an expert be there twice).
 * sigmoid: dl = D s (1 - s), nothing where there is no pick. softmax: dl = s (D - sum D s): with weights over their sum, sum D s is zero and
 * nothing but the picks has a gradient either; else every logit has one.
 */
__global__ void __launch_bounds__(256)
group_route_backward_kernel(RouteBackParams p)
{
    extern __shared__ float rows[];              /* [4][experts] */
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t = blockIdx.x * (blockDim.x >> 6) + wave;
    if (t >= p.tokens) return;
    float *row = rows + wave * p.experts;
    const int64_t base = (int64_t)t * p.experts;
    const bool dense = p.score == SCORE_SOFTMAX && !p.renormalize;
    for (int e = lane; e < p.experts; e += 64) row[e] = 0.0f;
    int e = -1;
    double g = 0.0, s = 0.0;
    float l = 0.0f;
    if (lane < p.topk) {
        e = p.idx[(int64_t)t * p.topk + lane];
        if (e < 0 || e >= p.experts) e = -1;
    }
    if (e >= 0) {
        g = (double)p.grad[(int64_t)t * p.topk + lane] * p.scale;
        l = logit_at(p.logits, p.dtype, base + e);
    }
    float mx = 0.0f;
    double sum = 1.0;
    if (p.score == SCORE_SOFTMAX) {
        mx = -__builtin_inff();
        if (p.renormalize) mx = e >= 0 ? l : mx;         /* the other logits cancel */
        else for (int i = lane; i < p.experts; i += 64) mx = fmaxf(mx, logit_at(p.logits, p.dtype, base + i));
        mx = zb_wave_reduce_dpp<true>(mx);
        if (e >= 0) s = exp((double)l - (double)mx);
        if (!p.renormalize) {
            float part = 0.0f;
            for (int i = lane; i < p.experts; i += 64) part += expf(logit_at(p.logits, p.dtype, base + i) - mx);
            sum = wave_sum_f64((double)part);
            s /= sum;
        }
    } else if (e >= 0) {
        s = 1.0 / (1.0 + exp(-(double)l));
    }
    double d = g;
    if (p.renormalize) {
        const double total = wave_sum_f64(s), gs = wave_sum_f64(g * s);
        d = e >= 0 && total > 0.0 ? (g - gs / total) / total : 0.0;
    }
    double all = d;
    bool first = e >= 0;
    for (int k = 0; k < p.topk; ++k) {
        const int ek = __builtin_amdgcn_readlane(e, k);
        const double dk = lane_f64(d, k);
        if (ek == e && k != lane) {
            if (k < lane) first = false;
            else all += dk;
        }
    }
    double c = 0.0;
    if (p.score == SCORE_SIGMOID) all *= s * (1.0 - s);
    else if (dense) c = wave_sum_f64(first ? all * s : 0.0);
    else all *= s;
    if (first) row[e] = (float)all;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int i = lane; i < p.experts; i += 64) {
        float v = row[i];
        if (dense) v = expf(logit_at(p.logits, p.dtype, base + i) - mx) * (float)(((double)v - c) / sum);
        put_logit(p.out, p.dtype, base + i, v);
    }
}

} // namespace

extern "C" int32_t zbalhip_group_route(const zbalhip_group_route_t *d, void *topk_idx, int32_t idx_is_i64, float *topk_w, void *stream)
{
    if (!d || d->tokens < 0 || d->tokens > 0x7fffffff || d->experts <= 0 || d->experts > kMaxExperts || d->topk <= 0 || d->topk > kMaxTopk ||
        d->topk > d->experts || d->groups <= 0 || d->groups > kMaxGroups || d->experts % d->groups != 0 || d->kept_groups <= 0 ||
        d->kept_groups > d->groups || d->topk > d->kept_groups * (d->experts / d->groups) || (d->score & ~1) || (d->group_score & ~1))
        return ZBALHIP_INVALID;
    if (d->dtype != ZDT_FP32 && d->dtype != ZDT_BF16 && d->dtype != ZDT_FP16) return ZBALHIP_INVALID;
    if (d->tokens == 0) return ZBALHIP_OK;
    if (!d->logits || !topk_idx || !topk_w) return ZBALHIP_INVALID;
    RouteParams p = {d->logits, d->dtype, (int)d->tokens, (int)d->experts, (int)d->topk, (int)d->groups, (int)d->kept_groups, d->score,
                     d->group_score, d->renormalize, d->scale, d->bias, topk_idx, idx_is_i64, topk_w, 64};
    while (p.lanes * p.groups > 64) p.lanes >>= 1;
    const int slots = (p.experts / p.groups + p.lanes - 1) / p.lanes;
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
    if (!d || d->tokens < 0 || d->tokens > 0x7fffffff || d->experts <= 0 || d->experts > kMaxExperts || d->topk <= 0 || d->topk > kMaxTopk ||
        (d->score & ~1))
        return ZBALHIP_INVALID;
    if (d->dtype != ZDT_FP32 && d->dtype != ZDT_BF16 && d->dtype != ZDT_FP16) return ZBALHIP_INVALID;
    if (d->tokens == 0) return ZBALHIP_OK;
    if (!d->logits || !topk_idx || !grad_w || !grad_logits) return ZBALHIP_INVALID;
    const RouteBackParams p = {grad_w, d->logits, d->dtype, (int)d->tokens, (int)d->experts, (int)d->topk, d->score, d->renormalize,
                               d->scale, expert_ids(topk_idx, idx_is_i64 != 0, true), grad_logits};
    zb_launch(group_route_backward_kernel, dim3((unsigned)((d->tokens + 3) / 4)), dim3(256), (size_t)p.experts * 16, (hipStream_t)stream, p);
    return zbalhip_check_launch();
}

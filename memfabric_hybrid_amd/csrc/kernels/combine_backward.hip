/*
 * The combine's gradient. out[t] = sum_k w[t, k] y[row(t, k)], so the row of a pick gets w[t, k] g[t], and its weight <g[t], y[row(t, k)]>.
 *
 * A stream of three tensors of rows: bound by the memory's bandwidth. One workgroup per token; a lane keeps sixteen bytes of the
 * token's gradient and asks for those of up to eight picks' rows at once, writes their gradients, and adds up the products in 32
 * bits; the workgroup's sums meet at the end of a row, always in the same order.
 */
#include "zbal_device.h"
#include "zbal_hip_kernels.h"

namespace {

constexpr int kMaxTopk = 32, kGroup = 8, kMaxWaves = 16;

template <int DT>
__global__ void __launch_bounds__(1024)
combine_backward_kernel(const uint16_t *__restrict__ grad, const uint16_t *__restrict__ y, int64_t y_rows, const int32_t *__restrict__ base,
                        const float *__restrict__ w, ExpertIds topk_idx, const int32_t *__restrict__ rank_in_expert, int hidden, int topk,
                        int experts, uint16_t *__restrict__ grad_y, float *__restrict__ grad_w)
{
    __shared__ float sums[kMaxWaves][kGroup];
    const int t = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    /* lane k resolves pick k; a pick that went nowhere, or whose row the tensors do not hold, has no gradient */
    int64_t row = -1;
    float wk = 0.0f;
    if (lane < topk) {
        const int e = topk_idx[(int64_t)t * topk + lane];
        const int32_t rk = rank_in_expert[(int64_t)t * topk + lane];
        wk = w[(int64_t)t * topk + lane];
        if (e >= 0 && e < experts && rk >= 0) {
            row = (int64_t)base[e] + rk;
            if (row < 0 || row >= y_rows) row = -1;
        }
    }
    const uint32_t row_lo = (uint32_t)row, row_hi = (uint32_t)((uint64_t)row >> 32);
    const u32x4 *g_row = reinterpret_cast<const u32x4 *>(grad + (int64_t)t * hidden);
    for (int first = 0; first < topk; first += kGroup) {
        int64_t at[kGroup];
        float wu[kGroup], dot[kGroup];
#pragma unroll
        for (int u = 0; u < kGroup; ++u) {
            const int k = first + u;
            at[u] = -1;
            dot[u] = 0.0f;
            if (k < topk) {
                at[u] = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)row_hi, k) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)row_lo, k));
                wu[u] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(wk), k));
            }
        }
        for (int c = threadIdx.x; c < hidden / 8; c += blockDim.x) {
            const u32x4 g = g_row[c];
            u32x4 v[kGroup];
#pragma unroll
            for (int u = 0; u < kGroup; ++u)
                if (at[u] >= 0) v[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(y + at[u] * hidden) + c);
            float gf[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                gf[2 * i] = zb_half_to_f32<DT>(g[i] & 0xffffu);
                gf[2 * i + 1] = zb_half_to_f32<DT>(g[i] >> 16);
            }
#pragma unroll
            for (int u = 0; u < kGroup; ++u) {
                if (at[u] < 0) continue;
                u32x4 o;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    dot[u] = __builtin_fmaf(zb_half_to_f32<DT>(v[u][i] & 0xffffu), gf[2 * i], dot[u]);
                    dot[u] = __builtin_fmaf(zb_half_to_f32<DT>(v[u][i] >> 16), gf[2 * i + 1], dot[u]);
                    o[i] = zb_pack2_half<DT>(wu[u] * gf[2 * i], wu[u] * gf[2 * i + 1]);
                }
                __builtin_nontemporal_store(o, reinterpret_cast<u32x4 *>(grad_y + at[u] * hidden) + c);
            }
        }
#pragma unroll
        for (int u = 0; u < kGroup; ++u) dot[u] = zb_wave_reduce_dpp<false>(dot[u]);
        __syncthreads();                         /* the group before has been added up */
        if (lane == 0)
#pragma unroll
            for (int u = 0; u < kGroup; ++u) sums[wave][u] = dot[u];
        __syncthreads();
        if (threadIdx.x < kGroup && first + (int)threadIdx.x < topk) {
            float s = 0.0f;
            for (int i = 0; i < waves; ++i) s += sums[i][threadIdx.x];
            grad_w[(int64_t)t * topk + first + threadIdx.x] = s;
        }
    }
}

} // namespace

extern "C" int32_t zbalhip_combine_backward(const void *grad, const void *y, int64_t y_rows, int32_t dtype, const int32_t *base,
                                            const float *w, const void *topk_idx, int32_t idx_is_i64, const int32_t *send_token_idx,
                                            int64_t tokens, int64_t hidden, int64_t topk, int64_t experts, void *grad_y, float *grad_w,
                                            void *stream)
{
    if (dtype != ZDT_BF16 && dtype != ZDT_FP16) return ZBALHIP_INVALID;
    if (tokens < 0 || tokens > ZBALHIP_ROUTE_MAX_TOKENS || hidden <= 0 || hidden % 8 != 0 || hidden > 0x7fffffff || topk <= 0 || topk > kMaxTopk ||
        experts <= 0 || experts > 0x7fffffff || y_rows < 0)
        return ZBALHIP_INVALID;
    if (tokens == 0) return ZBALHIP_OK;
    if (!grad || !y || !base || !w || !topk_idx || !send_token_idx || !grad_y || !grad_w) return ZBALHIP_INVALID;
    int64_t threads = (hidden / 8 + 63) / 64 * 64;
    const int64_t most = tokens < 1024 ? 1024 : 256;
    if (threads > most) threads = most;
    const ExpertIds ids = expert_ids(topk_idx, idx_is_i64 != 0);
    const dim3 grid((unsigned)tokens), block((unsigned)threads);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == ZDT_BF16)
        zb_launch(combine_backward_kernel<ZDT_BF16>, grid, block, 0, st, (const uint16_t *)grad, (const uint16_t *)y, y_rows, base, w, ids, send_token_idx,
                  (int)hidden, (int)topk, (int)experts, (uint16_t *)grad_y, grad_w);
    else
        zb_launch(combine_backward_kernel<ZDT_FP16>, grid, block, 0, st, (const uint16_t *)grad, (const uint16_t *)y, y_rows, base, w, ids, send_token_idx,
                  (int)hidden, (int)topk, (int)experts, (uint16_t *)grad_y, grad_w);
    return zbalhip_check_launch();
}

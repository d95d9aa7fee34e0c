/*
 * The products of the experts for few rows, weights with consecutive k.
 *
 * A token's products read every weight once, and nothing else takes time: 2048 x 7168, one row, are 29 MB, 4.7 us at what a large read reaches. Weights that
 * only one wave needs gain nothing from the LDS: a lane loads the eight k of its column straight into the fragment that the matrix
 * instruction takes. What counts is bytes under way: a workgroup has sixteen columns only, its four waves take every fourth 64 k (a line of each
 * of the sixteen rows of W), 32 loads of a lane at a time, and add up their sums through the LDS, in order. One row of 2048 x 7168: 8.0 us,
 * over weights that change from call to call; timed side by side, 9.5 against 11.3 of 16 x 64 tiles through the LDS. More rows, or experts, are enough workgroups for
 * wider tiles, which read their rows fewer times.
 */
#ifndef ZBAL_EXPERT_ROWS_H_
#define ZBAL_EXPERT_ROWS_H_

#include "zbal_expert_tile.h"

namespace {

/* NT sub-tiles of sixteen columns: one, or the gate's and the up columns; BATCH: k in steps of 64 that a wave asks for at a time */
template <int DT, int NT, int WAVES, int BATCH = 8 / NT>
__global__ void __launch_bounds__(WAVES * 64)
expert_gemm_rows_kernel(XgemmParams p)
{
    constexpr int LD = NT * 16 + 1;
    __shared__ x_sum_t<DT> sums[WAVES][16][LD];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quad = lane >> 4;
    const int cols = p.n_half ? p.n_half : p.N, n_tiles = (cols + 15) / 16;
    const XTile t = x_locate<16>(p, n_tiles, blockIdx.x, XSLOTS);
    if (t.expert < 0) return;
    const int n0 = t.n_tile * 16;

    /* rows and columns past the end repeat the last one; their sums go nowhere */
    const int row = t.row_begin + (lane & 15), col = n0 + (lane & 15);
    const uint16_t *a = p.a + (int64_t)(row < t.row_end ? row : t.row_end - 1) * p.lda;
    const uint16_t *b = p.b + t.expert * p.b_stride + (int64_t)(col < cols ? col : cols - 1) * p.ldb;
    const int64_t up = (int64_t)p.n_half * p.ldb;

    /* what int8's epilogue reads, for the element that the lane will finish, asked for in front of the operands */
    const int r_out = tid >> 4, c_out = n0 + (tid & 15);
    const int64_t at = t.row_begin + r_out, first = (int64_t)t.expert * p.N;
    const bool mine = tid < 256 && at < t.row_end && c_out < cols;
    float row_scale = 0.0f, col_scale[2] = {0.0f, 0.0f}, bias[2] = {0.0f, 0.0f}, residual = 0.0f;
    if (x_is_i8<DT> && mine) {
        row_scale = p.a_scale[at];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            col_scale[i] = x_load<ZDT_BF16>(p.b_scale, p.b_scale_f32, first + i * p.n_half + c_out);
            if (p.bias) bias[i] = x_load<DT>(p.bias, p.bias_f32, first + i * p.n_half + c_out);
        }
        if (p.residual) residual = x_load<DT>(p.residual, p.out_f32, at * p.ldo + c_out);
    }
    x_sums_t<DT> acc[NT];
    for (auto &v : acc) v = x_sums_t<DT>{0, 0, 0, 0};
    for (int k0 = wave * 64; k0 < p.K; k0 += WAVES * 64 * BATCH) {
        u32x4 fa[BATCH][2], fb[NT][BATCH][2];
#pragma unroll
        for (int c = 0; c < BATCH; ++c)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int k = k0 + c * WAVES * 64 + s * 32 + quad * 8, at = k < p.K ? k : 0;
#pragma unroll
                for (int i = 0; i < NT; ++i) fb[i][c][s] = *reinterpret_cast<const u32x4 *>(b + i * up + at);
                fa[c][s] = *reinterpret_cast<const u32x4 *>(a + at);
            }
#pragma unroll
        for (int c = 0; c < BATCH; ++c)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const bool in = k0 + c * WAVES * 64 + s * 32 + quad * 8 < p.K;
                const u32x4 none = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < NT; ++i) acc[i] = x_mfma<DT>(in ? fb[i][c][s] : none, in ? fa[c][s] : none, acc[i]);
            }
    }
    /* a lane has columns 4 (l / 16) .. + 3 of row l % 16 */
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sums[wave][lane & 15][i * 16 + quad * 4 + j] = acc[i][j];
    __syncthreads();
    const int r = tid >> 4, c = tid & 15;
    if (!mine) return;
    x_sum_t<DT> z[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int w = 0; w < WAVES; ++w) z[i] += sums[w][r][i * 16 + c];
    if constexpr (x_is_i8<DT>) {
        float v[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) v[i] = (float)z[i] * col_scale[i] * row_scale + bias[i];
        x_store<DT>(p.out, p.out_f32, at * p.ldo + c_out, (NT > 1 ? x_silu(v[0]) * v[1] : x_activate(p.act, v[0])) + residual);
    } else {
        x_finish<DT>(p, t.expert, at, c_out, z[0], z[1]);
    }
}

} // namespace

#endif /* ZBAL_EXPERT_ROWS_H_ */

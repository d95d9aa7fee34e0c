/*
 * The experts' products in half precision: rows sorted by expert times the experts' weights, with bias, activation and residual
 * in the epilogue, and the gradients of the rows, the weights, the bias and the pre-activation.
 */
#include <cmath>

#include "zbal_expert_rows.h"
#include "zbal_expert_wide.h"

namespace {

/*
 * Any sizes: operands pass through registers, sixteen bytes at a time from wherever they start (two bytes' alignment), the last
 * elements of a row or column one by one.
 */
template <int DT, bool REDUCE, bool B_TR, int TM, int TN, int WM, int WN, bool SHORT>
__global__ void __launch_bounds__(WM * WN * 64)
expert_gemm_any_kernel(XgemmParams p)
{
    constexpr int THREADS = WM * WN * 64, MT = TM / WM / 16, NT = TN / WN / 16;
    constexpr int A_CHUNKS = TM * 8 / THREADS, B_CHUNKS = TN * 8 / THREADS;
    static_assert(A_CHUNKS * THREADS == TM * 8 || TM * 8 < THREADS, "every thread moves as many chunks");
    constexpr int AC = A_CHUNKS > 0 ? A_CHUNKS : 1;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[(TM + TN) * 128];
    uint8_t *lds_a = lds, *lds_b = lds + TM * 128;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;
    typedef u32x4 __attribute__((aligned(2))) loose_t;

    const int cols = p.n_half ? p.n_half : p.N, tile_cols = p.n_half ? TN / 2 : TN, n_tiles = (cols + tile_cols - 1) / tile_cols;
    int expert, m0, m_end, n0, k_begin, k_end;
    const int split = p.splits > 1 ? blockIdx.y : 0;
    if constexpr (REDUCE) {
        const int m_tiles = (p.M + TM - 1) / TM, per = m_tiles * n_tiles;
        expert = blockIdx.x / per;
        const int in = blockIdx.x - expert * per;
        m0 = in % m_tiles * TM;
        m_end = p.M;
        n0 = in / m_tiles * tile_cols;
        const XSpan s = x_rows_of(p, expert);
        k_begin = s.begin;
        k_end = s.end;
    } else {
        const XTile t = x_locate<TM>(p, n_tiles, blockIdx.x, XSLOTS);
        if (t.expert < 0) return;
        expert = t.expert;
        m0 = t.row_begin;
        m_end = t.row_end;
        n0 = t.n_tile * tile_cols;
        k_begin = 0;
        k_end = p.K;
    }
    if (p.splits > 1) {          /* whole steps for everyone, in order */
        const int steps = (k_end - k_begin + XBK - 1) / XBK, each = (steps + p.splits - 1) / p.splits;
        const int from = k_begin + split * each * XBK;
        k_end = k_end - from > each * XBK ? from + each * XBK : k_end;
        k_begin = from < k_end ? from : k_end;
    }
    const uint16_t *b = p.b + (REDUCE ? 0 : expert * p.b_stride);

    /* tile column -> column of B; columns past the end of their half are none */
    auto b_col = [&](int c, int *end) __attribute__((always_inline)) {
        if (!p.n_half) { *end = p.N; return n0 + c; }
        *end = c < TN / 2 ? p.n_half : p.N;
        return c < TN / 2 ? n0 + c : p.n_half + n0 + c - TN / 2;
    };
    /*
     * Eight elements from column `col` of a row: a piece that ends past `end` is taken from its last eight and shifted, so that all loads are alike
     * and under way together (one by one, the last columns' tiles took twice as long as the others: 1021 x 1001 x 1531 in 64 x 64, with gelu, bias and residual, 27 us, 41).
     */
    struct Piece { u32x4 v; int away; };         /* elements to shift out; eight: nothing is left */
    auto eight = [&](const uint16_t *row, int col, int end, bool there) __attribute__((always_inline)) -> Piece {
        if constexpr (SHORT) {
            u32x4 v = {0, 0, 0, 0};
            for (int i = 0; there && i < 8 && col + i < end; ++i) v[i >> 1] |= (uint32_t)row[col + i] << ((i & 1) * 16);
            return {v, 0};
        } else {
            const int from = col < end - 8 ? col : end - 8, away = col - from;
            return {*reinterpret_cast<const loose_t *>(row + from), !there || away > 8 ? 8 : away};
        }
    };
    auto shifted = [&](const Piece &c) __attribute__((always_inline)) -> u32x4 {
        if (c.away == 0) return c.v;
        const int bits = (c.away & 3) * 16;
        uint64_t lo = (uint64_t)c.v[1] << 32 | c.v[0], hi = (uint64_t)c.v[3] << 32 | c.v[2];
        if (c.away >= 4) { lo = hi; hi = 0; }
        if (c.away >= 8) lo = 0;
        if (bits) { lo = lo >> bits | hi << (64 - bits); hi >>= bits; }
        return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
    };
    auto load_a = [&](int c, int k0) __attribute__((always_inline)) -> Piece {
        if constexpr (REDUCE) {
            const int k = k0 + c / (TM / 8), m = m0 + c % (TM / 8) * 8;
            return eight(p.a + (int64_t)(k < k_end ? k : k_end - 1) * p.lda, m, m_end, k < k_end);
        } else {
            const int row = m0 + (c >> 3), k = k0 + (c & 7) * 8;
            return eight(p.a + (int64_t)(row < m_end ? row : m_end - 1) * p.lda, k, k_end, row < m_end);
        }
    };
    auto load_b = [&](int c, int k0) __attribute__((always_inline)) -> Piece {
        int end;
        if constexpr (REDUCE || B_TR) {
            const int k = k0 + c / (TN / 8), n = b_col(c % (TN / 8) * 8, &end);
            return eight(b + (int64_t)(k < k_end ? k : k_end - 1) * p.ldb, n, end, k < k_end);
        } else {
            const int n = b_col(c >> 3, &end), k = k0 + (c & 7) * 8;
            return eight(b + (int64_t)(n < end ? n : end - 1) * p.ldb, k, k_end, n < end);
        }
    };

    f32x4 acc[MT][NT], bias_acc[REDUCE ? (MT > NT ? MT : NT) : 1];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (auto &v : bias_acc) v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    /* the tiles of the other operand's first columns sum this one's, as a product with ones */
    const bool bias_b = REDUCE && p.bias_side == 1 && m0 == 0 && wm == 0, bias_a = REDUCE && p.bias_side == 2 && n0 == 0 && wn == 0;
    const uint32_t one2 = DT == ZDT_BF16 ? 0x3f803f80u : 0x3c003c00u;
    const u32x4 ones = {one2, one2, one2, one2};

    /* two steps' pieces are under way while a third is multiplied, where registers leave room for it and for a second workgroup */
    constexpr int AHEAD = TM * TN > 64 * 128 ? 1 : 2;
    Piece ra[AHEAD][AC], rb[AHEAD][B_CHUNKS];
    const bool a_mine = A_CHUNKS > 0 || tid < TM * 8;
    auto fetch = [&](Piece(&pa)[AC], Piece(&pb)[B_CHUNKS], int k0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < AC; ++i)
            if (a_mine) pa[i] = load_a(tid + i * THREADS, k0);
#pragma unroll
        for (int i = 0; i < B_CHUNKS; ++i) pb[i] = load_b(tid + i * THREADS, k0);
    };
    auto step = [&](Piece(&pa)[AC], Piece(&pb)[B_CHUNKS], int k0) __attribute__((always_inline)) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < AC; ++i)
            if (a_mine) {
                const int c = tid + i * THREADS;
                *reinterpret_cast<u32x4 *>(lds_a + (REDUCE ? tr_at<TM>(c / (TM / 8), c % (TM / 8)) : kc_at(c >> 3, c & 7))) = shifted(pa[i]);
            }
#pragma unroll
        for (int i = 0; i < B_CHUNKS; ++i) {
            const int c = tid + i * THREADS;
            *reinterpret_cast<u32x4 *>(lds_b + (REDUCE || B_TR ? tr_at<TN>(c / (TN / 8), c % (TN / 8)) : kc_at(c >> 3, c & 7))) = shifted(pb[i]);
        }
        __syncthreads();
        fetch(pa, pb, k0 + AHEAD * XBK);          /* past the end: the last pieces again, and none of them used */
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            u32x4 fa[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const int r = wm * (MT * 16) + mt * 16;
                fa[mt] = REDUCE ? tr_fragment<TM>(lds_a, r, s, lane) : kc_fragment(lds_a, r, s, lane);
                if (bias_a) bias_acc[mt] = x_mfma<DT>(ones, fa[mt], bias_acc[mt]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int c = !p.n_half ? wn * (NT * 16) + nt * 16
                                        : (nt < NT / 2 ? wn * (NT * 8) + nt * 16 : TN / 2 + wn * (NT * 8) + (nt - NT / 2) * 16);
                const u32x4 fb = REDUCE || B_TR ? tr_fragment<TN>(lds_b, c, s, lane) : kc_fragment(lds_b, c, s, lane);
                if (bias_b) bias_acc[nt] = x_mfma<DT>(fb, ones, bias_acc[nt]);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) acc[mt][nt] = x_mfma<DT>(fb, fa[mt], acc[mt][nt]);
            }
        }
    };
    if (k_begin < k_end) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) fetch(ra[i], rb[i], k_begin + i * XBK);
        for (int k0 = k_begin; k0 < k_end; k0 += AHEAD * XBK)
#pragma unroll
            for (int i = 0; i < AHEAD; ++i)
                if (k0 + i * XBK < k_end) step(ra[i], rb[i], k0 + i * XBK);
    }

    /* a lane has columns 4 (l / 16) .. + 3 of row l % 16 of every sub-tile */
    const int q4 = (lane >> 4) * 4;
    if constexpr (REDUCE) {
        auto put = [&](int j, int end, float v) __attribute__((always_inline)) {
            if (j >= end) return;
            if (p.splits > 1) p.bias_partial[split * p.bias_ldp + j] = v;
            else x_store<DT>(p.bias_grad, p.out_f32, (int64_t)expert * end + j, v);
        };
        if (bias_b && (lane & 15) == 0)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                for (int i = 0; i < 4; ++i) put(n0 + wn * (NT * 16) + nt * 16 + q4 + i, p.N, bias_acc[nt][i]);
        if (bias_a && lane < 16)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) put(m0 + wm * (MT * 16) + mt * 16 + lane, p.M, bias_acc[mt][0]);
    }
    /*
     * Through the LDS, a row sub-tile of every wave at a time: neighbouring lanes then have neighbouring columns, whose loads and stores are one
     * access each, and several of them under way (1021 x 1001 x 1531, gelu, bias and residual, from the sums' own lanes, one after the other: 33 us more).
     */
    constexpr int LD = TN + 1, ROWS = WM * 16;
    static_assert(ROWS * LD * 4 <= (TM + TN) * 128, "sums fit the operands' place");
    float *sums = reinterpret_cast<float *>(lds);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int c = !p.n_half ? wn * (NT * 16) + nt * 16 : (nt < NT / 2 ? wn * (NT * 8) + nt * 16 : TN / 2 + wn * (NT * 8) + (nt - NT / 2) * 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[(wm * 16 + (lane & 15)) * LD + c + q4 + i] = acc[mt][nt][i];
        }
        __syncthreads();
#pragma unroll 4
        for (int i = tid; i < ROWS * TN; i += THREADS) {
            const int r = i / TN, c = i % TN, row = m0 + r / 16 * (MT * 16) + mt * 16 + r % 16;
            const bool up = p.n_half && c >= TN / 2;
            const int j = n0 + (up ? c - TN / 2 : c);
            if (row >= m_end || j >= cols) continue;
            const float z = sums[r * LD + c];
            if (p.splits > 1) p.partial[((int64_t)split * (REDUCE ? p.M : p.rows) + row) * p.ldp + j + (up ? p.n_half : 0)] = z;
            else if constexpr (REDUCE) x_store<DT>(p.out, p.out_f32, expert * p.out_stride + row * p.ldo + j, z);
            else if (!up) x_finish<DT>(p, expert, row, j, z, p.n_half ? sums[r * LD + TN / 2 + c] : 0.0f);
        }
    }
}

/* the sums of a product split along k, in order, and what the epilogue does with them; one expert. Four columns a lane */
template <int DT, bool REDUCE>
__global__ void __launch_bounds__(256)
expert_join_kernel(XgemmParams p)
{
    const int cols = p.n_half ? p.n_half : p.N, quads = (cols + 3) / 4;
    const int rows = REDUCE ? p.M : x_rows_of(p, 0).end;
    const int64_t plane = (int64_t)(REDUCE ? p.M : p.rows) * p.ldp, total = (int64_t)rows * quads;
    const bool whole = p.ldo % 4 == 0 && p.N % 4 == 0 && p.n_half % 4 == 0;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int row = (int)(i / quads), j = (int)(i - (int64_t)row * quads) * 4;
        const float *from = p.partial + (int64_t)row * p.ldp + j;
        f32x4 z = {0.0f, 0.0f, 0.0f, 0.0f}, up = z;
        if (whole) {
            for (int s = 0; s < p.splits; ++s) {
                z += *reinterpret_cast<const f32x4 *>(from + s * plane);
                if (p.n_half) up += *reinterpret_cast<const f32x4 *>(from + s * plane + p.n_half);
            }
            if constexpr (REDUCE) x_store4<DT>(p.out, p.out_f32, row * p.ldo + j, z);
            else x_finish4<DT>(p, 0, row, j, z, up);
        } else {
            for (int c = 0; c < 4 && j + c < cols; ++c) {
                float zc = 0.0f, uc = 0.0f;
                for (int s = 0; s < p.splits; ++s) {
                    zc += from[s * plane + c];
                    if (p.n_half) uc += from[s * plane + p.n_half + c];
                }
                if constexpr (REDUCE) x_store<DT>(p.out, p.out_f32, row * p.ldo + j + c, zc);
                else x_finish<DT>(p, 0, row, j + c, zc, uc);
            }
        }
    }
    if constexpr (REDUCE) {
        const int n = p.bias_side == 1 ? p.N : (p.bias_side == 2 ? p.M : 0);
        for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x) {
            float z = 0.0f;
            for (int s = 0; s < p.splits; ++s) z += p.bias_partial[s * p.bias_ldp + i];
            x_store<DT>(p.bias_grad, p.out_f32, i, z);
        }
    }
}

/*
 * The pre-activation's gradient: dz = dy act'(z), for swiglu of both halves; with no activation the rounding of a gradient in 32 bits.
 * A stream of the three tensors, V elements to a lane: 16384 x 7168 out of 32 bits 137 us at eight (5.1 TB/s), 174 one by one; gelu, which reads z besides, 196
 * (one by one 225, where eight took 192).
 */
template <int DT, int V>
__global__ void __launch_bounds__(256)
expert_slope_kernel(XgemmParams p, const void *__restrict__ dy, int dy_f32, const uint16_t *__restrict__ z, uint16_t *__restrict__ dz)
{
    typedef uint16_t halves __attribute__((ext_vector_type(V)));
    typedef float floats __attribute__((ext_vector_type(V), aligned(V * 4 < 16 ? 4 : 16)));
    const int cols = (p.n_half ? p.n_half : p.N) / V, rows = p.counts ? x_rows_of(p, p.experts - 1).end : p.rows;
    const int64_t n = (int64_t)rows * cols, first = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int step = gridDim.x * blockDim.x, step_rows = step / cols, step_cols = step - step_rows * cols;
    int64_t row = first / cols;
    int col = (int)(first - row * cols);
    for (int64_t i = first; i < n; i += step) {
        float d[V];
        if (dy_f32) {
            const floats v = reinterpret_cast<const floats *>(dy)[i];
#pragma unroll
            for (int k = 0; k < V; ++k) d[k] = v[k];
        } else {
            const halves v = reinterpret_cast<const halves *>(dy)[i];
#pragma unroll
            for (int k = 0; k < V; ++k) d[k] = zb_half_to_f32<DT>(v[k]);
        }
        if (p.act == ACT_SWIGLU) {
            const int64_t at = row * 2 * cols + col;
            const halves gs = reinterpret_cast<const halves *>(z)[at], us = reinterpret_cast<const halves *>(z)[at + cols];
            halves dg, du;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float g = zb_half_to_f32<DT>(gs[k]), u = zb_half_to_f32<DT>(us[k]);
                dg[k] = (uint16_t)zb_f32_to_half<DT>(d[k] * u * x_slope(ACT_SILU, g));
                du[k] = (uint16_t)zb_f32_to_half<DT>(d[k] * x_silu(g));
            }
            reinterpret_cast<halves *>(dz)[at] = dg;
            reinterpret_cast<halves *>(dz)[at + cols] = du;
        } else {
            halves v;
            if (p.act == ACT_NONE) {
#pragma unroll
                for (int k = 0; k < V; ++k) v[k] = (uint16_t)zb_f32_to_half<DT>(d[k]);
            } else {
                const halves zs = reinterpret_cast<const halves *>(z)[i];
#pragma unroll
                for (int k = 0; k < V; ++k) v[k] = (uint16_t)zb_f32_to_half<DT>(d[k] * x_slope(p.act, zb_half_to_f32<DT>(zs[k])));
            }
            reinterpret_cast<halves *>(dz)[i] = v;
        }
        row += step_rows;
        col += step_cols;
        if (col >= cols) { col -= cols; ++row; }
    }
}

template <int DT> void launch_slope(const XgemmParams &p, const void *dy, int dy_f32, const uint16_t *z, uint16_t *dz, hipStream_t st)
{
    const int cols = p.n_half ? p.n_half : p.N;
    const bool wide = cols % 8 == 0;             /* the tensors themselves are aligned */
    const int64_t groups = ((int64_t)p.rows * cols / (wide ? 8 : 1) + 255) / 256;
    const dim3 grid((unsigned)(groups < 4096 ? groups : 4096));
    if (wide) zb_launch(expert_slope_kernel<DT, 8>, grid, dim3(256), 0, st, p, dy, dy_f32, z, dz);
    else zb_launch(expert_slope_kernel<DT, 1>, grid, dim3(256), 0, st, p, dy, dy_f32, z, dz);
}

template <int DT, bool REDUCE, bool B_TR, int TM, int TN, int WM, int WN, bool SHORT = false>
void launch_any(const XgemmParams &p, hipStream_t st)
{
    const int cols = p.n_half ? p.n_half : p.N, tile_cols = p.n_half ? TN / 2 : TN;
    const int64_t n_tiles = (cols + tile_cols - 1) / tile_cols;
    int64_t blocks;
    if (REDUCE) {
        blocks = (int64_t)p.experts * ((p.M + TM - 1) / TM) * n_tiles;
    } else {
        /* every expert may end with a tile that is not full */
        const int64_t most = p.rows / TM + p.experts;
        blocks = (most < p.rows ? most : p.rows) * n_tiles;
        blocks = (blocks + 7) / 8 * 8;
    }
    zb_launch(expert_gemm_any_kernel<DT, REDUCE, B_TR, TM, TN, WM, WN, SHORT>, dim3((unsigned)blocks, (unsigned)p.splits), dim3(WM * WN * 64), 0, st, p);
}

/* workgroups of a product of rows sorted by expert: as many as there can be tiles */
template <int TM> unsigned tiles_of_cols(const XgemmParams &p, int tile_cols)
{
    const int cols = p.n_half ? p.n_half : p.N;
    const int64_t n_tiles = (cols + tile_cols - 1) / tile_cols, most = p.rows / TM + p.experts;    /* every expert may end with a tile that is not full */
    return (unsigned)(((most < p.rows ? most : p.rows) * n_tiles + 7) / 8 * 8);
}

template <bool REDUCE, int TM, int TN> unsigned tiles_of(const XgemmParams &p)
{
    if (REDUCE) return (unsigned)(((int64_t)p.experts * ((p.M + TM - 1) / TM) * ((p.N + TN - 1) / TN) + 7) / 8 * 8);
    return tiles_of_cols<TM>(p, p.n_half ? TN / 2 : TN);
}

template <int DT, bool REDUCE, bool B_TR, int TM, int TN, int WM, int WN, int STAGES>
void launch_direct(const XgemmParams &p, hipStream_t st)
{
    zb_launch(expert_gemm_kernel<DT, REDUCE, B_TR, TM, TN, WM, WN, STAGES>, dim3(tiles_of<REDUCE, TM, TN>(p), (unsigned)p.splits), dim3(WM * WN * 64), 0, st, p);
}

template <int DT> void launch_rows(const XgemmParams &p, hipStream_t st)
{
    /* eight waves where four have more than one batch of loads */
    const dim3 grid(tiles_of_cols<16>(p, 16)), four(256), eight(512);
    if (p.n_half) {
        if (p.K > 1024) zb_launch(expert_gemm_rows_kernel<DT, 2, 8>, grid, eight, 0, st, p);
        else zb_launch(expert_gemm_rows_kernel<DT, 2, 4>, grid, four, 0, st, p);
    } else {
        if (p.K > 2048) zb_launch(expert_gemm_rows_kernel<DT, 1, 8>, grid, eight, 0, st, p);
        else zb_launch(expert_gemm_rows_kernel<DT, 1, 4>, grid, four, 0, st, p);
    }
}

template <int DT, bool REDUCE, bool B_TR> void launch_wide(XgemmParams p, hipStream_t st)
{
    p.through_lds = !REDUCE && (p.bias || p.residual || p.preact || (p.act != ACT_NONE && p.act != ACT_SWIGLU));
    unsigned blocks = tiles_of<REDUCE, 256, 256>(p);
    if (!p.through_lds && blocks > XW_CUS) blocks = XW_CUS;
    const dim3 grid(blocks), block(512);
    if constexpr (REDUCE) {
        if (p.bias_side == 1) zb_launch(expert_gemm_wide_kernel<DT, REDUCE, B_TR, 1>, grid, block, 0, st, p);
        else if (p.bias_side == 2) zb_launch(expert_gemm_wide_kernel<DT, REDUCE, B_TR, 2>, grid, block, 0, st, p);
        else zb_launch(expert_gemm_wide_kernel<DT, REDUCE, B_TR, 0>, grid, block, 0, st, p);
    } else {
        zb_launch(expert_gemm_wide_kernel<DT, REDUCE, B_TR>, grid, block, 0, st, p);
    }
}

/* every row of the operands and outputs starts at a multiple of eight elements */
inline bool rows_are_aligned(const XgemmParams &p) { return p.lda % 8 == 0 && p.ldb % 8 == 0 && p.ldo % 8 == 0 && p.N % 8 == 0 && p.n_half % 8 == 0; }

/* how a product is cut: the tiles, and the parts along k whose sums a second launch adds up */
enum Cut { CUT_WIDE, CUT_128, CUT_64_128, CUT_64, CUT_32, CUT_16, CUT_ANY, CUT_ANY_64, CUT_ANY_16, CUT_SHORT, CUT_ROWS };
struct Plan {
    Cut cut;
    int splits;
    int64_t bytes;               /* of workspace */
};

/*
 * The cut that takes least time by what a step of 64 k takes on a CU, `alone` with one tile there and `full` with as many as run side by side
 * (us). Measured, best by this rule / the next: 32 experts of 7168 x 4096: 128 rows each wide 375 / 128 480, 32 rows 64 x 128 318 / 32 x 128 359;
 * one matrix: 4096 x 7168 x 256 128 in four parts 31 / 64 x 128 in four 33 / 64 x 64 whole 40; 2048 x 4096 x 2048 128 43 / 64 x 128 52; 1024 x 2048 x
 * 2048 64 x 64 17.7 / 128 20.2; 64 x 2048 x 7168 16 x 64 11.5 / 64 x 64 13.1. Weights' gradients end in large stores, which only the wide tiles overlap with
 * products: 32 experts of 7168 x 4096, 128 rows each, wide 432 / 128 1009. Parts along k, for one expert, cost their sums twice through the memory, and a launch.
 * Where the weights' stream is what takes the time, wide tiles read longer pieces of rows whose columns are consecutive (16 rows over 32 experts of 7168 x
 * 4096: wide 139, 32 x 128 148, 16 x 64 162; k consecutive 145, 136, 137).
 */
Plan plan_product(const XgemmParams &p, bool reduce, bool b_cols)
{
    struct Kind { Cut cut; int tm, tn, at_once; double alone, full; };
    static const Kind kinds[] = {{CUT_WIDE, 256, 256, 1, 1.5, 1.5}, {CUT_128, 128, 128, 1, 0.57, 0.57}, {CUT_64_128, 64, 128, 2, 0.55, 0.75},
                                 {CUT_64, 64, 64, 2, 0.4, 0.45}, {CUT_32, 32, 128, 2, 0.35, 0.5}, {CUT_16, 16, 64, 2, 0.2, 0.27},
                                 {CUT_ROWS, 16, 16, 4, 0.1, 0.15}};
    static const Kind any[] = {{CUT_ANY, 128, 128, 2, 1.8, 2.2}, {CUT_ANY_64, 64, 64, 4, 0.75, 1.6}, {CUT_ANY_16, 16, 128, 4, 0.8, 1.8}};
    if ((reduce ? p.M : p.K) < 8 || (p.n_half ? p.n_half : p.N) < 8) return {CUT_SHORT, 1, 0};
    const bool aligned = rows_are_aligned(p);
    const Kind *list = aligned ? kinds : any;
    const int count = !aligned ? 3 : (b_cols ? 6 : 7);
    const double steps = ((reduce ? (double)p.rows / p.experts : p.K) + XBK - 1) / XBK, per_expert = (double)p.rows / p.experts;
    const double reached = p.rows < p.experts ? p.rows : p.experts;
    const int cols = p.n_half ? p.n_half : p.N, rows = reduce ? p.M : p.rows;
    Plan plan = {list[0].cut, 1, 0};
    double best = 0.0;
    for (int i = 0; i < count; ++i) {
        const Kind &k = list[i];
        if (reduce && k.tm < 64) continue;
        const int tile_cols = p.n_half && k.cut != CUT_ROWS ? k.tn / 2 : k.tn;
        const double n_tiles = (cols + tile_cols - 1) / tile_cols;
        double m_tiles = reduce ? (double)p.experts * ((p.M + k.tm - 1) / k.tm) : (p.rows + k.tm - 1) / k.tm;
        if (!reduce && p.experts > 1) {      /* every expert ends with half a tile, on average */
            m_tiles = p.experts * (per_expert / k.tm + 0.5);
            if (m_tiles < reached) m_tiles = reached;
        }
        const double tiles = m_tiles * n_tiles;
        for (int splits = 1; splits <= 8; splits *= 2) {
            if (splits > 1 && (p.experts > 1 || k.cut == CUT_WIDE || k.cut == CUT_ROWS || steps / splits < 4 || tiles * splits > 512)) break;
            const double each = tiles * splits, per_round = 256.0 * k.at_once;
            const double beside = each < per_round ? ceil(each / 256.0) - 1.0 : k.at_once - 1.0;       /* that share a CU with one */
            double us = (k.at_once == 1 ? k.full : k.alone + (k.full - k.alone) * fmax(beside, 0.0) / (k.at_once - 1)) * ceil(each / per_round) * ceil(steps / splits);
            if (k.cut == CUT_WIDE && !reduce && per_expert <= 128) us *= 0.6;      /* tiles without a second half */
            /* an epilogue of stores in every round, which takes no time beside the next tile's steps in the wide kernel */
            if (reduce) us += ceil(each / per_round) * (k.cut == CUT_WIDE ? 1.0 : 8.0);
            if (splits > 1) us += 4.0 + (double)splits * rows * p.N * 8 / 5e6;
            const double stream = !b_cols ? 5.3e6 : (k.tn == 256 ? 5.3e6 : (k.tn == 128 ? 5.0e6 : 4.5e6));       /* bytes a us */
            const double memory = reached * p.b_stride * 2 / stream;
            if (us < memory) us = memory;
            if (best == 0.0 || us < best * 0.97) {
                best = us;
                plan.cut = k.cut;
                plan.splits = splits;
            }
        }
    }
    if (plan.splits > 1) {
        const int64_t ldp = (p.N + 3) / 4 * 4, bias_ldp = ((p.M > p.N ? p.M : p.N) + 3) / 4 * 4;
        plan.bytes = plan.splits * (rows * ldp + (reduce ? bias_ldp : 0)) * 4;
    }
    return plan;
}

template <int DT, bool REDUCE, bool B_TR> void launch_product(XgemmParams p, void *workspace, int64_t workspace_bytes, hipStream_t st)
{
    Plan plan = plan_product(p, REDUCE, REDUCE || B_TR);
    if (plan.bytes > workspace_bytes || !workspace) plan.splits = 1;
    if (plan.splits > 1) {
        p.splits = plan.splits;
        p.ldp = (p.N + 3) / 4 * 4;
        p.partial = (float *)workspace;
        p.bias_partial = p.partial + (int64_t)p.splits * (REDUCE ? p.M : p.rows) * p.ldp;
        p.bias_ldp = ((p.M > p.N ? p.M : p.N) + 3) / 4 * 4;
    }
    switch (plan.cut) {
        case CUT_WIDE: launch_wide<DT, REDUCE, B_TR>(p, st); break;
        case CUT_128: launch_direct<DT, REDUCE, B_TR, 128, 128, 2, 4, 4>(p, st); break;
        case CUT_64_128: launch_direct<DT, REDUCE, B_TR, 64, 128, 2, 2, 3>(p, st); break;
        case CUT_64: launch_direct<DT, REDUCE, B_TR, 64, 64, 2, 2, 4>(p, st); break;
        case CUT_ANY: launch_any<DT, REDUCE, B_TR, 128, 128, 2, 2>(p, st); break;
        case CUT_SHORT: launch_any<DT, REDUCE, B_TR, 64, 64, 2, 2, true>(p, st); break;
        case CUT_ANY_64: launch_any<DT, REDUCE, B_TR, 64, 64, 2, 2>(p, st); break;
        case CUT_ROWS:
            if constexpr (!REDUCE && !B_TR) launch_rows<DT>(p, st);
            break;
        default:
            if constexpr (!REDUCE) {
                if (plan.cut == CUT_32) launch_direct<DT, REDUCE, B_TR, 32, 128, 2, 2, 4>(p, st);
                else if (plan.cut == CUT_16) launch_direct<DT, REDUCE, B_TR, 16, 64, 1, 2, 8>(p, st);
                else launch_any<DT, REDUCE, B_TR, 16, 128, 1, 4>(p, st);
            }
    }
    if (p.splits > 1) {
        const int cols = p.n_half ? p.n_half : p.N, rows = REDUCE ? p.M : p.rows;
        const int64_t quads = (int64_t)rows * ((cols + 3) / 4);
        const unsigned blocks = (unsigned)((quads + 255) / 256 < 4096 ? (quads + 255) / 256 : 4096);
        zb_launch(expert_join_kernel<DT, REDUCE>, dim3(blocks), dim3(256), 0, st, p);
    }
}

template <bool REDUCE> void launch_types(const XgemmParams &p, int dtype, bool b_tr, void *ws, int64_t ws_bytes, hipStream_t st)
{
    if (dtype == ZDT_BF16) {
        if (b_tr) launch_product<ZDT_BF16, REDUCE, true>(p, ws, ws_bytes, st);
        else if constexpr (!REDUCE) launch_product<ZDT_BF16, REDUCE, false>(p, ws, ws_bytes, st);
    } else {
        if (b_tr) launch_product<ZDT_FP16, REDUCE, true>(p, ws, ws_bytes, st);
        else if constexpr (!REDUCE) launch_product<ZDT_FP16, REDUCE, false>(p, ws, ws_bytes, st);
    }
}

bool linear_sizes_ok(const zbalhip_expert_linear_t *d)
{
    if (!d || d->rows < 0 || d->k <= 0 || d->n <= 0 || d->experts <= 0 || d->experts > 1024) return false;
    if (d->dtype != ZDT_BF16 && d->dtype != ZDT_FP16) return false;
    if (d->activation < ACT_NONE || d->activation > ACT_SWIGLU || (d->activation == ACT_SWIGLU && d->n % 2 != 0)) return false;
    /* the numbers of tiles stay in 32 bits */
    return d->rows <= ZBALHIP_EXPERT_MAX_ROWS && d->k <= ZBALHIP_EXPERT_MAX_WIDTH && d->n <= ZBALHIP_EXPERT_MAX_WIDTH;
}

XgemmParams common_params(const zbalhip_expert_linear_t *d)
{
    XgemmParams p = {};
    p.counts = d->counts;
    p.counts_i64 = d->counts_are_i64;
    p.experts = (int)d->experts;
    p.rows = (int)d->rows;
    p.splits = 1;
    return p;
}

/* the three products as tiles know them; tensors that the plan does not turn on are set where they are launched */
XgemmParams forward_params(const zbalhip_expert_linear_t *d)
{
    XgemmParams p = common_params(d);
    p.lda = d->k;
    p.b = (const uint16_t *)d->weight;
    p.ldb = d->weight_is_nk ? d->k : d->n;
    p.b_stride = d->k * d->n;
    p.K = (int)d->k;
    p.N = (int)d->n;
    p.act = d->activation;
    p.n_half = d->activation == ACT_SWIGLU ? p.N / 2 : 0;
    p.ldo = p.n_half ? p.n_half : p.N;
    return p;
}

XgemmParams rows_gradient_params(const zbalhip_expert_linear_t *d)
{
    XgemmParams p = common_params(d);
    p.lda = d->n;
    p.b = (const uint16_t *)d->weight;
    p.ldb = d->weight_is_nk ? d->k : d->n;
    p.b_stride = d->k * d->n;
    p.K = (int)d->n;
    p.N = (int)d->k;
    p.ldo = d->k;
    return p;
}

XgemmParams weights_gradient_params(const zbalhip_expert_linear_t *d)
{
    XgemmParams p = common_params(d);
    p.lda = d->weight_is_nk ? d->n : d->k;
    p.ldb = d->weight_is_nk ? d->k : d->n;
    p.M = (int)p.lda;
    p.N = (int)p.ldb;
    p.ldo = p.N;
    p.out_stride = d->k * d->n;
    return p;
}

} // namespace

extern "C" int64_t zbalhip_expert_linear_workspace(const zbalhip_expert_linear_t *d, int32_t backward)
{
    if (!linear_sizes_ok(d)) return -1;
    if (d->rows == 0) return 0;
    if (!backward) return plan_product(forward_params(d), false, !d->weight_is_nk).bytes;
    /* one after the other in the same memory */
    const int64_t a = plan_product(rows_gradient_params(d), false, d->weight_is_nk != 0).bytes, b = plan_product(weights_gradient_params(d), true, true).bytes;
    return a > b ? a : b;
}

extern "C" int32_t zbalhip_expert_linear(const zbalhip_expert_linear_t *d, const void *x, const void *bias, int32_t bias_is_f32,
                                         const void *residual, void *y, int32_t y_is_f32, void *preact, void *workspace,
                                         int64_t workspace_bytes, void *stream)
{
    if (!linear_sizes_ok(d) || !d->weight || (d->experts > 1 && !d->counts)) return ZBALHIP_INVALID;
    if (d->rows == 0) return ZBALHIP_OK;
    if (!x || !y) return ZBALHIP_INVALID;
    XgemmParams p = forward_params(d);
    p.a = (const uint16_t *)x;
    p.out = y;
    p.out_f32 = y_is_f32;
    p.bias = bias;
    p.bias_f32 = bias_is_f32;
    p.residual = residual;
    p.preact = (uint16_t *)preact;
    launch_types<false>(p, d->dtype, !d->weight_is_nk, workspace, workspace_bytes, (hipStream_t)stream);
    return zbalhip_check_launch();
}

extern "C" int32_t zbalhip_expert_linear_backward(const zbalhip_expert_linear_t *d, const void *grad, int32_t grad_is_f32, const void *x,
                                                  const void *preact, void *grad_x, void *grad_weight, void *grad_bias,
                                                  int32_t weight_grad_is_f32, void *grad_preact, void *workspace,
                                                  int64_t workspace_bytes, void *stream)
{
    if (!linear_sizes_ok(d) || !d->weight || (d->experts > 1 && !d->counts)) return ZBALHIP_INVALID;
    const bool rounds = d->activation != ACT_NONE || grad_is_f32;
    if (d->rows > 0 && (!grad || (grad_weight && !x) || (d->activation != ACT_NONE && !preact) || (rounds && !grad_preact))) return ZBALHIP_INVALID;
    if (grad_bias && !grad_weight) return ZBALHIP_INVALID;
    if (!grad_x && !grad_weight && !(rounds && d->rows > 0)) return ZBALHIP_OK;
    hipStream_t st = (hipStream_t)stream;
    const uint16_t *dz = (const uint16_t *)grad;
    if (rounds && d->rows > 0) {
        XgemmParams p = common_params(d);
        p.N = (int)d->n;
        p.act = d->activation;
        p.n_half = d->activation == ACT_SWIGLU ? p.N / 2 : 0;
        if (d->dtype == ZDT_BF16) launch_slope<ZDT_BF16>(p, grad, grad_is_f32, (const uint16_t *)preact, (uint16_t *)grad_preact, st);
        else launch_slope<ZDT_FP16>(p, grad, grad_is_f32, (const uint16_t *)preact, (uint16_t *)grad_preact, st);
        dz = (const uint16_t *)grad_preact;
    }
    if (grad_x && d->rows > 0) {
        XgemmParams p = rows_gradient_params(d);
        p.a = dz;
        p.out = grad_x;
        launch_types<false>(p, d->dtype, d->weight_is_nk != 0, workspace, workspace_bytes, st);
    }
    if (grad_weight) {           /* also of experts without rows: zeros */
        XgemmParams p = weights_gradient_params(d);
        p.a = d->weight_is_nk ? dz : (const uint16_t *)x;
        p.b = d->weight_is_nk ? (const uint16_t *)x : dz;
        p.out = grad_weight;
        p.out_f32 = weight_grad_is_f32;
        p.bias_grad = grad_bias;
        p.bias_side = grad_bias ? (d->weight_is_nk ? 2 : 1) : 0;
        launch_types<true>(p, d->dtype, true, workspace, workspace_bytes, st);
    }
    return zbalhip_check_launch();
}

/*
 * The experts' products for many rows: 256 x 256 tiles, 64 k per step, eight waves, one persistent workgroup per CU.
 *
 * The waves are two row groups x four column ranges of 64; a row group has every other sixteen rows, so that a tile that is not
 * full leaves both the same work. A wave keeps a step's eight column fragments in registers and streams its row fragments past them. A stage
 * of the LDS is handed back in two parts, the columns and the first 128 rows by the middle of a step, the other rows by its end, and each
 * part is refilled for the step after next as soon as the barrier there has been passed: every transfer has a step and a half to arrive, in
 * two stages. Either barrier stands in front of a sub-tile whose operands are in registers already. The steps of one tile follow those of the one before
 * without a gap; what a tile stores is on its way while the next one is multiplied.
 */
#ifndef ZBAL_EXPERT_WIDE_H_
#define ZBAL_EXPERT_WIDE_H_

#include "zbal_expert_direct.h"

namespace {

constexpr int XW_CUS = 256;

/* BIAS (REDUCE): the operand whose columns are summed for the bias's gradient besides, 1 = b, 2 = a, 0 = none */
template <int DT, bool REDUCE, bool B_TR, int BIAS = 0>
__global__ void __launch_bounds__(512, 2)
expert_gemm_wide_kernel(XgemmParams p)
{
    constexpr int TM = 256, TN = 256, MT = 8, NT = 4, WAVES = 8, STAGE = (TM + TN) * 128;
    constexpr bool A_COLS = REDUCE, B_COLS = REDUCE || B_TR;
    __shared__ __attribute__((aligned(131072))) uint8_t smem[2 * STAGE];
    __shared__ __attribute__((aligned(16))) uint8_t lds_out[WAVES * 2048];
    __shared__ int lds_rows[1025], lds_tiles[1025];              /* rows, and row tiles, before expert e */
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 2, wn = wave & 3;
    const int E = p.experts;

    if (wave == 0) {
        uint32_t run = 0, tiles = 0;
        for (int base = 0; base < E; base += 64) {
            const int e = base + lane;
            const uint32_t c = e < E ? x_count(p, e) : 0, incl = __builtin_elementwise_add_sat(run, x_scan(c));
            const XSpan s = x_span(p, incl - c, incl);
            const uint32_t mt = (uint32_t)(s.end - s.begin + TM - 1) / TM, mt_incl = tiles + (uint32_t)zb_wave_scan_dpp((int)mt);
            if (e < E) {
                lds_rows[e] = s.begin;
                lds_tiles[e] = (int)(mt_incl - mt);
                if (e == E - 1) { lds_rows[E] = s.end; lds_tiles[E] = (int)mt_incl; }
            }
            run = (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
            tiles = (uint32_t)__builtin_amdgcn_readlane((int)mt_incl, 63);
        }
    }
    __syncthreads();

    /*
     * XCD x (workgroups x, x + 8, ...) has a contiguous run of tiles, its workgroups take consecutive ones of it: expert by expert, in
     * blocks of four row tiles by eight column tiles, so that what runs at the same time shares operands in the L2, and no line of
     * them with more than seven others (4096 x 7168 x 4096, columns consecutive: sixteen by two 431000 cycles, four by eight 363000).
     */
    const int cols = p.n_half ? p.n_half : p.N, tile_cols = p.n_half ? TN / 2 : TN, n_tiles = (cols + tile_cols - 1) / tile_cols;
    const int m_tiles = (p.M + TM - 1) / TM;
    const int total = REDUCE ? E * m_tiles * n_tiles : __builtin_amdgcn_readfirstlane(lds_tiles[E]) * n_tiles;
    const int chunk = (total + 7) / 8, slots = (int)gridDim.x >> 3, xcd = blockIdx.x & 7;
    const int id0 = xcd * chunk + (int)(blockIdx.x >> 3), id_end = (xcd + 1) * chunk < total ? (xcd + 1) * chunk : total;
    if (id0 >= id_end) return;
    struct Tile { int expert, m0, m_end, n0, k_begin, k_end; };
    /* bands of up to four row tiles, as even as they go; in each, groups of eight column tiles, row tile fastest */
    auto in_bands = [&](int in, int mt, int *m, int *n) __attribute__((always_inline)) {
        const int bands = (mt + 3) / 4, high = (mt + bands - 1) / bands, band = in / (high * n_tiles), rest = in - band * high * n_tiles;
        const int rows = mt - band * high < high ? mt - band * high : high, g = rest / (rows * 8), in_g = rest - g * rows * 8;
        *m = band * high + in_g % rows;
        *n = g * 8 + in_g / rows;
    };
    /*
     * The K loop takes all registers. What only the change of a tile needs is worked out there anew, from the lane's number and from the launch's
     * arguments in memory, neither of which the compiler can then keep through the loop.
     */
    auto fresh_lane = [&]() __attribute__((always_inline)) { int l = lane; asm volatile("" : "+v"(l)); return l; };
    typedef const XgemmParams __attribute__((address_space(4))) *args_t;
    auto fresh_args = []() __attribute__((always_inline)) { auto *a = __builtin_amdgcn_kernarg_segment_ptr(); asm volatile("" : "+s"(a)); return (args_t)a; };
    auto uni = [](int v) __attribute__((always_inline)) { return __builtin_amdgcn_readfirstlane(v); };
    auto tile_at = [&](int id) __attribute__((always_inline)) -> Tile {
        Tile t;
        const args_t p = fresh_args();
        if constexpr (REDUCE) {
            const int per = m_tiles * n_tiles;
            t.expert = id / per;
            int m, n;
            in_bands(id - t.expert * per, m_tiles, &m, &n);
            t.m0 = m * TM;
            t.m_end = p->M - t.m0 > TM ? t.m0 + TM : p->M;
            t.n0 = n * tile_cols;
            t.k_begin = uni(lds_rows[t.expert]);
            t.k_end = uni(lds_rows[t.expert + 1]);
        } else {
            const int q = id / n_tiles;
            int lo = 0, hi = E;                                 /* lds_tiles[lo] <= q < lds_tiles[hi] */
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (uni(lds_tiles[mid]) <= q) lo = mid;
                else hi = mid;
            }
            const int first = uni(lds_tiles[lo]), mt_e = uni(lds_tiles[lo + 1]) - first, in = id - first * n_tiles;
            const int begin = uni(lds_rows[lo]), end = uni(lds_rows[lo + 1]);
            int m, n;
            in_bands(in, mt_e, &m, &n);
            t.expert = lo;
            t.m0 = begin + m * TM;
            t.m_end = end - t.m0 > TM ? t.m0 + TM : end;
            t.n0 = n * tile_cols;
            t.k_begin = 0;
            t.k_end = p->K;
        }
        return t;
    };

    /*
     * ---- transfers: where the stream of steps that are brought stands ----
     * KiB wave + 8 j of an operand's 32; A's first 128 rows (columns) are its first half. Consecutive columns lie as two blocks of 128 (A), or
     * as one of 256 (B), by rows of k.
     */
    uint32_t a_off[4], b_off[4];
    uint64_t a_base = 0, b_base = 0, b_base2 = 0;
    int a_bytes = 0, b_bytes = 0;                               /* k consecutive: from the base to the last row's end; else what the first column of a tile takes off */
    int bring_id = id0, bring_left = 0;                         /* k left of its tile, this step's among them */
    const int lda2 = (int)p.lda * 2, ldb2 = (int)p.ldb * 2;
    const int kc_r = wave * 8 + (lane >> 3), kc_c = (lane & 7) ^ kc_key(kc_r);
    const int64_t a_step = A_COLS ? (int64_t)XBK * p.lda * 2 : XBK * 2, b_step = B_COLS ? (int64_t)XBK * p.ldb * 2 : XBK * 2;
    auto aim = [&]() __attribute__((always_inline)) {
        const Tile t = tile_at(bring_id);
        const args_t p = fresh_args();
        const int lane = fresh_lane();
        const int kc_r = wave * 8 + (lane >> 3), kc_c = (lane & 7) ^ kc_key(kc_r);
        bring_left = t.k_end - t.k_begin;
        if constexpr (A_COLS) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = (wave + 8 * (j & 1)) * 4 + (lane >> 4), slot = lane & 15;
                const int c = (j >> 1) * 128 + ((((slot >> 1) ^ tr_key<128>(k)) << 1) + (slot & 1)) * 8;
                a_off[j] = t.m0 + c < t.m_end ? (uint32_t)(k * (int)p->lda + c) * 2 : XNOWHERE;
            }
            a_base = (uint64_t)(uintptr_t)(p->a + (int64_t)t.k_begin * p->lda + t.m0);
            a_bytes = t.m0 * 2;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) a_off[j] = (uint32_t)((kc_r + 64 * j) * (int)p->lda) * 2 + kc_c * 16;
            a_base = (uint64_t)(uintptr_t)(p->a + (int64_t)t.m0 * p->lda);
            a_bytes = (t.m_end - t.m0) * lda2;
        }
        const uint16_t *b = p->b + (REDUCE ? 0 : t.expert * p->b_stride);
        if constexpr (B_COLS) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = (wave + 8 * j) * 2 + (lane >> 5), slot = lane & 31;
                const int c = ((((slot >> 1) ^ tr_key<256>(k)) << 1) + (slot & 1)) * 8;
                const bool up = p->n_half && c >= TN / 2;
                const int from = up ? p->n_half + c - TN / 2 : c, end = up || !p->n_half ? p->N : p->n_half;
                b_off[j] = t.n0 + from < end ? (uint32_t)(k * (int)p->ldb + from) * 2 : XNOWHERE;
            }
            b_base = (uint64_t)(uintptr_t)(b + (int64_t)t.k_begin * p->ldb + t.n0);
            b_bytes = t.n0 * 2;
        } else {
            /* gate rows in the first half of the parts, up rows in the second, from a descriptor of their own */
#pragma unroll
            for (int j = 0; j < 4; ++j) b_off[j] = (uint32_t)((kc_r + 64 * (p->n_half ? j & 1 : j)) * (int)p->ldb) * 2 + kc_c * 16;
            const int rows = cols - t.n0 < TN ? cols - t.n0 : TN;
            b_base = (uint64_t)(uintptr_t)(b + (int64_t)t.n0 * p->ldb);
            b_base2 = b_base + (uint64_t)p->n_half * p->ldb * 2;     /* without halves the same */
            b_bytes = rows * ldb2;
        }
    };
    auto words = [&](uint64_t base, bool by_k, int bytes, int ld2) __attribute__((always_inline)) -> u32x4 {
        if (by_k) {                                             /* rows of k: as many as are left */
            const int rows = bring_left < XBK ? bring_left : XBK;
            bytes = rows > 0 ? rows * ld2 - bytes : 0;
        }
        return u32x4{(uint32_t)uni((int)(uint32_t)base), (uint32_t)uni((int)(uint32_t)(base >> 32)), (uint32_t)uni(bytes), 0x00020000u};
    };
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(x_lds(smem) + wave * 1024);
    auto in_step = [&](bool by_k, uint32_t off) __attribute__((always_inline)) -> uint32_t { return by_k || kc_c * 8 < bring_left ? off : XNOWHERE; };
    auto bring_a = [&](int stage, int j) __attribute__((always_inline)) {
        x_dma16(words(a_base, A_COLS, a_bytes, lda2), in_step(A_COLS, a_off[j]), lds0 + stage * STAGE + j * 8192);
    };
    auto bring_b = [&](int stage, int j) __attribute__((always_inline)) {
        x_dma16(words(!B_COLS && j >= 2 ? b_base2 : b_base, B_COLS, b_bytes, ldb2), in_step(B_COLS, b_off[j]), lds0 + stage * STAGE + TM * 128 + j * 8192);
    };
    auto bring_first = [&](int stage) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) bring_b(stage, j);
        bring_a(stage, 0);
        bring_a(stage, 1);
    };
    /* the last transfer of a step; then on to the next step, or to the first of the next tile, or to nothing at all */
    auto bring_last = [&](int stage) __attribute__((always_inline)) {
        bring_a(stage, 3);
        a_base += a_step;
        b_base += b_step;
        b_base2 += b_step;
        if (!A_COLS) a_bytes -= XBK * 2;
        if (!B_COLS) b_bytes -= XBK * 2;
        bring_left -= XBK;
        if (bring_left <= 0) {
            bring_id += slots;
            if (bring_id < id_end) aim();
            else bring_left = a_bytes = b_bytes = 0;
        }
    };
    /* one part has landed for everybody and nobody reads the one before it any more: the two parts since, eight transfers, may be on their way */
    auto landed = [&]() __attribute__((always_inline)) { asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

    auto col_of = [&](int nt) __attribute__((always_inline)) {
        return !p.n_half ? wn * 64 + nt * 16 : (nt < NT / 2 ? wn * 32 + nt * 16 : TN / 2 + wn * 32 + (nt - NT / 2) * 16);
    };
    /*
     * Where a lane's fragments begin, in the stage in use: what differs between sub-tiles and halves of a step is a constant, where the
     * places of consecutive k or columns are exchanged within a row an exclusive or. Columns: sub-tiles 0 and 1, then 2 and 3 (up).
     */
    const int j16 = lane & 15, g16 = lane >> 4;
    uint32_t at_a[2], at_b[4];
    {
        const uint32_t base = x_lds(smem);
        if constexpr (A_COLS) {
            const int k = g16 * 8 + (j16 >> 2);
            at_a[0] = base + k * 256 + ((wm ^ tr_key<128>(k)) << 5) + (j16 & 3) * 8;
            at_a[1] = 0;
        } else {
            at_a[0] = base + kc_at(wm * 16 + j16, g16);
            at_a[1] = at_a[0] ^ 64;
        }
        const uint32_t first = base + TM * 128;
        if constexpr (B_COLS) {
            const int k = g16 * 8 + (j16 >> 2), key = tr_key<256>(k);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) at_b[nt] = first + k * 512 + (((col_of(nt) >> 4) ^ key) << 5) + (j16 & 3) * 8;
        } else {
            at_b[0] = first + kc_at(col_of(0) + j16, g16);
            at_b[1] = at_b[0] ^ 64;
            at_b[2] = first + kc_at(col_of(2) + j16, g16);
            at_b[3] = at_b[2] ^ 64;
        }
    }
    auto other_stage = [&]() __attribute__((always_inline)) {
        at_a[0] ^= STAGE;
        if (!A_COLS) at_a[1] ^= STAGE;
#pragma unroll
        for (int i = 0; i < 4; ++i) at_b[i] ^= STAGE;
    };
    static_assert(STAGE == 65536, "stages a power of two apart");
    typedef const u32x4 __attribute__((address_space(3))) *lds128_t;
    typedef s16x4_t __attribute__((address_space(3))) *lds64_t;
    auto transposed = [&](uint32_t at, int row) __attribute__((always_inline)) -> u32x4 {
        const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds64_t)(uintptr_t)at));
        const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds64_t)(uintptr_t)(at + 4 * row)));
        return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
    auto load_b = [&](int s, int nt) __attribute__((always_inline)) -> u32x4 {
        if constexpr (B_COLS) return transposed(at_b[nt] + s * 16384, 512);
        else return *(lds128_t)(uintptr_t)(at_b[(nt >> 1) * 2 + s] + (nt & 1) * 2048);
    };
    auto load_a = [&](int s, int mt) __attribute__((always_inline)) -> u32x4 {
        if constexpr (A_COLS) return transposed((at_a[0] ^ ((mt & 3) << 6)) + (mt >> 2) * 16384 + s * 8192, 256);
        else return *(lds128_t)(uintptr_t)(at_a[s] + mt * 4096);
    };

    aim();
    bring_first(0);
    bring_a(0, 2);
    bring_last(0);
    bring_first(1);
    bring_a(1, 2);
    landed();
    int stage = 0;
    u32x4 fb[2][NT], fa[2][2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) fb[s][nt] = load_b(s, nt);
        fa[0][s] = load_a(s, 0);
    }
    const uint32_t one2 = DT == ZDT_BF16 ? 0x3f803f80u : 0x3c003c00u;
    const u32x4 ones = {one2, one2, one2, one2};

    for (int id = id0; id < id_end; id += slots) {
        const Tile t = tile_at(id);
        f32x4 acc[MT][NT], bias_acc[BIAS == 1 ? NT : (BIAS == 2 ? MT : 1)];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (auto &v : bias_acc) v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        /* the tiles of the other operand's first columns do it, as a product with ones */
        const bool bias_b = BIAS == 1 && t.m0 == 0 && wm == 0, bias_a = BIAS == 2 && t.n0 == 0 && wn == 0;

        auto sums_of_columns = [&]() __attribute__((always_inline)) {
            if constexpr (BIAS == 1)
                if (bias_b)
#pragma unroll
                    for (int s = 0; s < 2; ++s)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) bias_acc[nt] = x_mfma<DT>(fb[s][nt], ones, bias_acc[nt]);
        };
        /*
         * A row sub-tile's products, and between them up to two transfers: asked for all at once they fill the queue to the caches, and a wave that
         * waits at its end multiplies nothing. RENEW: each column fragment is replaced by the next step's behind its last use.
         */
        auto multiply = [&](int mt, auto renew, auto transfer1, auto transfer2) __attribute__((always_inline)) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                if constexpr (BIAS == 2)
                    if (bias_a) bias_acc[mt] = x_mfma<DT>(ones, fa[mt & 1][s], bias_acc[mt]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    acc[mt][nt] = x_mfma<DT>(fb[s][nt], fa[mt & 1][s], acc[mt][nt]);
                    if (decltype(renew)::value) fb[s][nt] = load_b(s, nt);
                    if (s == 0 && nt == 1) { __builtin_amdgcn_sched_barrier(0); transfer1(); __builtin_amdgcn_sched_barrier(0); }
                    if (s == 1 && nt == 1) { __builtin_amdgcn_sched_barrier(0); transfer2(); __builtin_amdgcn_sched_barrier(0); }
                }
            }
        };
        auto ask = [&](int mt) __attribute__((always_inline)) {
#pragma unroll
            for (int s = 0; s < 2; ++s) fa[mt & 1][s] = load_a(s, mt);
        };
        /* what is asked for stays in front of the products that it arrives behind */
        auto keep = []() __attribute__((always_inline)) { __builtin_amdgcn_sched_barrier(0); };
        auto none = []() {};
        const std::false_type same = {};
        const std::true_type renew = {};
        int left = t.k_end - t.k_begin;
        if (t.m_end - t.m0 > TM / 2) {
            do {
                sums_of_columns();
                ask(1);
                keep();
                multiply(0, same, [&]() __attribute__((always_inline)) { bring_last(stage ^ 1); }, none);
                keep();
#pragma unroll
                for (int mt = 1; mt < 3; ++mt) {
                    ask(mt + 1);
                    keep();
                    multiply(mt, same, none, none);
                    keep();
                }
                landed();
                ask(4);
                keep();
                multiply(3, same, [&]() __attribute__((always_inline)) { bring_b(stage, 0); }, [&]() __attribute__((always_inline)) { bring_b(stage, 1); });
                keep();
                ask(5);
                keep();
                multiply(4, same, [&]() __attribute__((always_inline)) { bring_b(stage, 2); }, [&]() __attribute__((always_inline)) { bring_b(stage, 3); });
                keep();
                ask(6);
                keep();
                multiply(5, same, [&]() __attribute__((always_inline)) { bring_a(stage, 0); }, none);
                keep();
                ask(7);
                keep();
                multiply(6, same, [&]() __attribute__((always_inline)) { bring_a(stage, 1); }, none);
                keep();
                landed();
                other_stage();
                ask(0);
                keep();
                multiply(7, renew, [&]() __attribute__((always_inline)) { bring_a(stage, 2); }, none);
                keep();
                stage ^= 1;
                left -= XBK;
            } while (left > 0);
        } else {                                                /* the other rows are none */
            do {
                sums_of_columns();
                ask(1);
                keep();
                multiply(0, same, [&]() __attribute__((always_inline)) { bring_last(stage ^ 1); }, none);
                keep();
                ask(2);
                keep();
                multiply(1, same, none, none);
                keep();
                ask(3);
                keep();
                multiply(2, same, none, none);
                keep();
                landed();
                bring_first(stage);
                keep();
                multiply(3, same, none, none);
                keep();
                landed();
                other_stage();
                bring_a(stage, 2);
                ask(0);
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) fb[s][nt] = load_b(s, nt);
                stage ^= 1;
                left -= XBK;
            } while (left > 0);
        }

        /* ---- epilogue: a lane has columns 4 (l / 16) .. + 3 of row l % 16 of every sub-tile ---- */
        const int q4 = (lane >> 4) * 4;
        if constexpr (BIAS == 1) {
            if (bias_b && (lane & 15) == 0)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int j = t.n0 + wn * 64 + nt * 16 + q4 + i;
                        if (j < p.N) x_store<DT>(p.bias_grad, p.out_f32, (int64_t)t.expert * p.N + j, bias_acc[nt][i]);
                    }
        }
        if constexpr (BIAS == 2) {
            if (bias_a && lane < 16)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const int j = t.m0 + mt * 32 + wm * 16 + lane;
                    if (j < p.M) x_store<DT>(p.bias_grad, p.out_f32, (int64_t)t.expert * p.M + j, bias_acc[mt][0]);
                }
        }
        if (REDUCE || !p.through_lds) {
            /* the weights' gradient is not read again soon */
            const args_t p = fresh_args();
            const int lane = fresh_lane(), first_col = t.n0 + (p->n_half ? wn * 32 : wn * 64), row0 = t.m0 + wm * 16;
            const uint32_t own = uni((int)(x_lds(lds_out) + wave * 2048));
            auto *to = static_cast<uint8_t *>(p->out) + ((REDUCE ? t.expert * p->out_stride : 0) + (int64_t)row0 * p->ldo + first_col) * (p->out_f32 ? 4 : 2);
            if (!REDUCE && p->n_half)
                x_lines_out<DT, MT, NT / 2, 32, 0>(own, to, p->out_f32, (int)p->ldo, t.m_end - row0, cols - first_col, lane, [&](int mt, int i) __attribute__((always_inline)) {
                    f32x4 y;
#pragma unroll
                    for (int c = 0; c < 4; ++c) y[c] = x_silu(acc[mt][i][c]) * acc[mt][i + NT / 2][c];
                    return y;
                });
            else
                x_lines_out<DT, MT, NT, 32, REDUCE ? 2 : 0>(own, to, p->out_f32, (int)p->ldo, t.m_end - row0, cols - first_col, lane,
                                                            [&](int mt, int i) __attribute__((always_inline)) { return acc[mt][i]; });
        } else if constexpr (!REDUCE) {
            /* the launch has a workgroup per tile, and what was brought behind its last step is nothing: the stages are free */
            constexpr int PASS = 2, ROWS = PASS * 32, LD = TN + 4;
            static_assert(ROWS * LD * 4 <= 2 * STAGE, "sums fit the stages");
            float *sums = reinterpret_cast<float *>(smem);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
            for (int pass = 0; pass < MT / PASS; ++pass) {
                __syncthreads();
#pragma unroll
                for (int h = 0; h < PASS; ++h)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        *reinterpret_cast<f32x4 *>(sums + (h * 32 + wm * 16 + (lane & 15)) * LD + col_of(nt) + q4) = acc[pass * PASS + h][nt];
                __syncthreads();
                const int quads = tile_cols / 4;
#pragma unroll 1
                for (int i = tid; i < ROWS * quads; i += WAVES * 64) {
                    const int r = i / quads, c = (i - r * quads) * 4, j = t.n0 + c, row = t.m0 + pass * ROWS + r;
                    if (row >= t.m_end || j >= cols) continue;
                    const f32x4 z = *reinterpret_cast<const f32x4 *>(sums + r * LD + c);
                    f32x4 up = {0.0f, 0.0f, 0.0f, 0.0f};
                    if (p.n_half) up = *reinterpret_cast<const f32x4 *>(sums + r * LD + TN / 2 + c);
                    x_finish4<DT>(p, t.expert, row, j, z, up);
                }
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");             /* nothing lands in the LDS of whoever comes next */
}

} // namespace

#endif /* ZBAL_EXPERT_WIDE_H_ */

/*
 * The experts' products where every row of the operands starts at a 16-byte boundary, in half precision every row of outputs and every half of swiglu's columns, too (int8's
 * outputs, scales, bias and residual may have any width): operands go from memory to the LDS without passing
 * through registers (buffer loads with the LDS as their target), in a ring of stages, all but one of which are on their way while one is
 * multiplied. For tiles so small, or so few, that the time of a step is that of a transfer.
 *
 * What the buffer descriptor does besides: rows past the tile's end, and k past the last, lie behind its end and arrive as zeros, so that neither
 * another expert's rows nor what lies behind a tensor is ever multiplied. Columns past the end, and the chunks of a last step that is not full,
 * ask for an offset that no descriptor has.
 */
#ifndef ZBAL_EXPERT_DIRECT_H_
#define ZBAL_EXPERT_DIRECT_H_

#include "zbal_expert_tile.h"

namespace {

constexpr uint32_t XNOWHERE = 0x80000000u;

__device__ __forceinline__ uint32_t x_lds(const void *p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p; }

/*
 * 16 bytes for every lane, lane l's to lds_wave_addr + 16 l. A scalar register written by a vector instruction wants five wait states
 * before a vector-memory instruction reads it, which the compiler does not see to inside the text: the move to M0 is one, `s_nop 3` are four.
 */
__device__ __forceinline__ void x_dma16(const u32x4 &buffer, uint32_t lane_off, uint32_t lds_wave_addr)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(lds_wave_addr), "v"(lane_off), "s"(buffer)
                 : "memory", "m0");
}

__device__ __forceinline__ void *x_uniform_address(const void *v)
{
    const uint64_t u = (uint64_t)(uintptr_t)v;
    return (void *)(uintptr_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(u >> 32)) << 32 |
                               (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)u));
}

/*
 * A wave's sums to memory: MT row sub-tiles, ROW_STEP rows from one to the next, of OS column sub-tiles side by side, which `value`(mt, i) gives
 * (columns 4 (l / 16) .. + 3 of row l % 16). `out` is where the wave's first row and column go, `rows` and `cols` how many there are from there
 * on (none or fewer, too).
 * By way of two KiB of LDS that are the wave's own, sixteen rows of up to 128 bytes, 16-byte chunk c of row r in slot c ^ (r & 7): a store then
 * writes whole lines, or the longest pieces that there are, instead of 32 or 64 bytes of sixteen rows. Rows past the last lie behind the buffer's
 * end, columns past the last go nowhere. CACHE 2: the streaming hint.
 */
template <int DT, int MT, int OS, int ROW_STEP, int CACHE, typename V>
__device__ __forceinline__ void x_lines_out(uint32_t own, void *out, int f32, int ldo, int rows, int cols, int lane, V value)
{
    typedef const u32x4 __attribute__((address_space(3))) *lds128_t;
    typedef f32x4 __attribute__((address_space(3))) *lds_f_t;
    typedef u32x2 __attribute__((address_space(3))) *lds_h_t;
    const int width = f32 ? 4 : 2, ldo_b = ldo * width, j16 = lane & 15, g16 = lane >> 4;
    const int bytes = rows > 0 && cols > 0 ? (rows - 1) * ldo_b + cols * width : 0;
    const __amdgpu_buffer_rsrc_t to = __builtin_amdgcn_make_buffer_rsrc(x_uniform_address(out), 0, __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
    auto group = [&](auto g_tag, auto f32_tag) __attribute__((always_inline)) {
        constexpr int G = decltype(g_tag)::value;                     /* sub-tiles to a line */
        constexpr bool F32 = decltype(f32_tag)::value;
        constexpr int ROW = G * (F32 ? 64 : 32), LANES = ROW / 16, AT_ONCE = 64 / LANES;      /* bytes and lanes of a row, rows of a store */
        const int r_out = lane / LANES, c_out = lane % LANES;
        const uint32_t from = own + r_out * 128 + ((c_out ^ (r_out & 7)) << 4), put = own + j16 * 128, key = j16 & 7;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            if (mt * ROW_STEP >= rows) continue;
#pragma unroll
            for (int i0 = 0; i0 < OS; i0 += G) {
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    const f32x4 v = value(mt, i0 + i);
                    if constexpr (F32) *(lds_f_t)(uintptr_t)(put + (((i * 4 + g16) ^ key) << 4)) = v;
                    else *(lds_h_t)(uintptr_t)(put + (((i * 2 + (g16 >> 1)) ^ key) << 4) + (g16 & 1) * 8) =
                        u32x2{zb_pack2_half<x_half<DT>>(v[0], v[1]), zb_pack2_half<x_half<DT>>(v[2], v[3])};
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                const int at = i0 * (F32 ? 64 : 32) + c_out * 16;
                const bool some = at < cols * width && r_out < 16, in = some && (!x_is_i8<DT> || at + 16 <= cols * width);
                const uint32_t off = in ? (uint32_t)((mt * ROW_STEP + r_out) * ldo_b + at) : XNOWHERE;
                __builtin_amdgcn_raw_buffer_store_b128(*(lds128_t)(uintptr_t)from, to, (int)off, 0, CACHE);
                if constexpr (AT_ONCE < 16)
                    __builtin_amdgcn_raw_buffer_store_b128(*(lds128_t)(uintptr_t)(from + 1024), to, (int)(in ? off + 8 * ldo_b : XNOWHERE), 0, CACHE);
                if (x_is_i8<DT> && some && !in)              /* a row's last sixteen bytes, not all of which are its own */
#pragma unroll
                    for (int half = 0; half < (AT_ONCE < 16 ? 2 : 1); ++half)
#pragma unroll
                        for (int e = 0; e < 16 / (F32 ? 4 : 2) - 1; ++e) {
                            const uint32_t src = from + half * 1024 + e * (F32 ? 4 : 2), at_e = (uint32_t)((mt * ROW_STEP + r_out + half * 8) * ldo_b + at + e * width);
                            if (at + e * width >= cols * width) continue;
                            if constexpr (F32) __builtin_amdgcn_raw_buffer_store_b32(*(const uint32_t __attribute__((address_space(3))) *)(uintptr_t)src, to, (int)at_e, 0, CACHE);
                            else __builtin_amdgcn_raw_buffer_store_b16(*(const uint16_t __attribute__((address_space(3))) *)(uintptr_t)src, to, (int)at_e, 0, CACHE);
                        }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }
        }
    };
    if (f32) group(std::integral_constant<int, OS < 2 ? OS : 2>{}, std::true_type{});
    else group(std::integral_constant<int, OS < 4 ? OS : 4>{}, std::false_type{});
}

/* all but this wave's last N transfers have landed, and nobody reads the stage before any more */
template <int N> __device__ __forceinline__ void x_turn() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory"); }

template <int DT, bool REDUCE, bool B_TR, int TM, int TN, int WM, int WN, int STAGES>
__global__ void __launch_bounds__(WM * WN * 64)
expert_gemm_kernel(XgemmParams p)
{
    constexpr int WAVES = WM * WN, MT = TM / WM / 16, NT = TN / WN / 16;
    constexpr int A_PARTS = TM / 8 / WAVES, B_PARTS = TN / 8 / WAVES;         /* KiB per wave and step */
    static_assert(A_PARTS >= 1 && B_PARTS >= 1 && A_PARTS * WAVES * 8 == TM && B_PARTS * WAVES * 8 == TN, "every wave moves as much");
    constexpr bool A_COLS = REDUCE, B_COLS = REDUCE || B_TR;                  /* the operand's columns are consecutive */
    static_assert((!A_COLS || TM >= 64) && (!B_COLS || TN >= 64), "the key of consecutive columns wants four units at least");
    static_assert(WAVES % 2 == 0, "a wave's rows of every part have the same key");
    constexpr int STAGE = (TM + TN) * 128;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[STAGES * STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;

    const int cols = p.n_half ? p.n_half : p.N, tile_cols = p.n_half ? TN / 2 : TN, n_tiles = (cols + tile_cols - 1) / tile_cols;
    int expert, m0, m_end, n0, k_begin, k_end;
    const int split = p.splits > 1 ? blockIdx.y : 0;
    if constexpr (REDUCE) {
        const int m_tiles = (p.M + TM - 1) / TM, per = m_tiles * n_tiles;
        /* XCD x has a contiguous run of tiles (experts one after the other), so that what it works on shares columns in its L2 */
        const int total = p.experts * per, chunk = (total + 7) / 8, logical = (int)(blockIdx.x & 7) * chunk + (int)(blockIdx.x >> 3);
        if ((int)(blockIdx.x >> 3) >= chunk || logical >= total) return;
        expert = logical / per;
        const int in = logical - expert * per, group = 8 * m_tiles, g = in / group, rest = in - g * group;
        m0 = rest % m_tiles * TM;
        m_end = p.M;
        n0 = (g * 8 + rest / m_tiles) * tile_cols;
        const XSpan s = x_rows_of(p, expert);
        k_begin = s.begin;
        k_end = s.end;
    } else {
        const XTile t = x_locate<TM>(p, n_tiles, blockIdx.x, 32);
        if (t.expert < 0) return;
        expert = t.expert;
        m0 = t.row_begin;
        m_end = t.row_end;
        n0 = t.n_tile * tile_cols;
        k_begin = 0;
        k_end = p.K;
    }
    if (p.splits > 1) {
        const int steps = (k_end - k_begin + XBK - 1) / XBK, each = (steps + p.splits - 1) / p.splits;
        const int from = k_begin + split * each * XBK;
        k_end = k_end - from > each * XBK ? from + each * XBK : k_end;
        k_begin = from < k_end ? from : k_end;
    }

    /* ---- transfers: part j of a stage is KiB wave + WAVES j of it ---- */
    uint32_t a_off[A_PARTS], b_off[B_PARTS];
    int a_chunk = 0, b_chunk = 0;          /* the lane's first k within a step, for the last one */
    uint64_t a_base, b_base;
    int a_bytes, b_bytes;                  /* k consecutive: from the base to the last row's end; else what the first column takes off a row */
    int left = k_end - k_begin;            /* k from the step that is brought next on */
    const int lda2 = (int)p.lda * 2, ldb2 = (int)p.ldb * 2;
    const int64_t a_step = A_COLS ? (int64_t)XBK * p.lda * 2 : XBK * 2, b_step = B_COLS ? (int64_t)XBK * p.ldb * 2 : XBK * 2;
    /* columns consecutive: KiB i holds rows of k, PER_KB of them */
    auto cols_off = [&](auto w_tag, int i, int *k) __attribute__((always_inline)) -> int {
        constexpr int W = decltype(w_tag)::value, PER_KB = 512 / W, LANES = 64 / PER_KB;
        *k = i * PER_KB + lane / LANES;
        const int slot = lane % LANES;
        return ((((slot >> 1) ^ tr_key<W>(*k)) << 1) + (slot & 1)) * 8;       /* column of the tile */
    };
    if constexpr (A_COLS) {
#pragma unroll
        for (int j = 0; j < A_PARTS; ++j) {
            int k;
            const int c = cols_off(std::integral_constant<int, TM>{}, wave + WAVES * j, &k);
            a_off[j] = m0 + c < m_end ? (uint32_t)(k * p.lda + c) * 2 : XNOWHERE;
        }
        a_base = (uint64_t)(uintptr_t)(p.a + (int64_t)k_begin * p.lda + m0);
        a_bytes = m0 * 2;
    } else {
#pragma unroll
        for (int j = 0; j < A_PARTS; ++j) {
            const int r = (wave + WAVES * j) * 8 + (lane >> 3), c = (lane & 7) ^ kc_key(r);
            a_off[j] = (uint32_t)(r * p.lda) * 2 + c * 16;
            a_chunk = c * 8;               /* WAVES is even, so the same for every j */
        }
        a_base = (uint64_t)(uintptr_t)(p.a + (int64_t)m0 * p.lda + k_begin);
        a_bytes = (m_end - m0 < TM ? m_end - m0 : TM) * lda2 - k_begin * 2;
    }
    const uint16_t *b = p.b + (REDUCE ? 0 : expert * p.b_stride);
    if constexpr (B_COLS) {
#pragma unroll
        for (int j = 0; j < B_PARTS; ++j) {
            int k;
            const int c = cols_off(std::integral_constant<int, TN>{}, wave + WAVES * j, &k);
            const bool up = p.n_half && c >= TN / 2;
            const int from = up ? p.n_half + c - TN / 2 : c, end = up || !p.n_half ? p.N : p.n_half;
            b_off[j] = n0 + from < end ? (uint32_t)(k * p.ldb + from) * 2 : XNOWHERE;
        }
        b_base = (uint64_t)(uintptr_t)(b + (int64_t)k_begin * p.ldb + n0);
        b_bytes = n0 * 2;
    } else {
        /* gate rows in the first half of the parts, up rows in the second, from a descriptor of their own */
#pragma unroll
        for (int j = 0; j < B_PARTS; ++j) {
            const int r = (wave + WAVES * j) * 8 + (lane >> 3), c = (lane & 7) ^ kc_key(r);
            b_off[j] = (uint32_t)((p.n_half && j >= B_PARTS / 2 ? r - TN / 2 : r) * p.ldb) * 2 + c * 16;
            b_chunk = c * 8;
        }
        b_base = (uint64_t)(uintptr_t)(b + (int64_t)n0 * p.ldb + k_begin);
        b_bytes = (cols - n0 < TN ? cols - n0 : TN) * ldb2 - k_begin * 2;
    }
    const uint64_t up = !B_COLS && p.n_half ? (uint64_t)p.n_half * p.ldb * 2 : 0;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(x_lds(smem) + wave * 1024);
    auto words = [&](uint64_t base, bool by_k, int bytes, int ld2) __attribute__((always_inline)) -> u32x4 {
        if (by_k) bytes = (left < XBK ? left : XBK) * ld2 - bytes;            /* rows of k: as many as are left */
        if (left <= 0) bytes = 0;                                              /* behind the last step nothing is brought, by transfers of the same number */
        return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)base), (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(base >> 32)),
                     (uint32_t)__builtin_amdgcn_readfirstlane(bytes), 0x00020000u};
    };
    auto bring_next = [&](int stage) __attribute__((always_inline)) {
        const u32x4 aw = words(a_base, A_COLS, a_bytes, lda2), bw = words(b_base, B_COLS, b_bytes, ldb2);
        const u32x4 bw2 = B_COLS ? bw : words(b_base + up, false, b_bytes, ldb2);
        const uint32_t to = lds0 + stage * STAGE;
        const bool a_in = A_COLS || a_chunk < left, b_in = B_COLS || b_chunk < left;
#pragma unroll
        for (int j = 0; j < A_PARTS; ++j) x_dma16(aw, a_in ? a_off[j] : XNOWHERE, to + j * (WAVES * 1024));
#pragma unroll
        for (int j = 0; j < B_PARTS; ++j) x_dma16(!B_COLS && j >= B_PARTS / 2 ? bw2 : bw, b_in ? b_off[j] : XNOWHERE, to + TM * 128 + j * (WAVES * 1024));
        a_base += a_step;
        b_base += b_step;
        if (!A_COLS) a_bytes -= XBK * 2;
        if (!B_COLS) b_bytes -= XBK * 2;
        left -= XBK;
    };

    x_sums_t<DT> acc[MT][NT], bias_acc[REDUCE ? (MT > NT ? MT : NT) : 1];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = x_sums_t<DT>{0, 0, 0, 0};
    for (auto &v : bias_acc) v = x_sums_t<DT>{0, 0, 0, 0};
    const bool bias_b = REDUCE && p.bias_side == 1 && m0 == 0 && wm == 0, bias_a = REDUCE && p.bias_side == 2 && n0 == 0 && wn == 0;
    const uint32_t one2 = DT == ZDT_BF16 ? 0x3f803f80u : 0x3c003c00u;
    const u32x4 ones = {one2, one2, one2, one2};
    /* where a wave's column sub-tiles lie: with swiglu, the second half of them are the up columns of the first */
    auto col_of = [&](int nt) __attribute__((always_inline)) {
        return !p.n_half ? wn * (NT * 16) + nt * 16 : (nt < NT / 2 ? wn * (NT * 8) + nt * 16 : TN / 2 + wn * (NT * 8) + (nt - NT / 2) * 16);
    };

    constexpr int PASS = MT % 2 == 0 && WM * 32 * (TN + 4) * 4 <= STAGES * STAGE ? 2 : 1, ROWS = WM * PASS * 16, LD = TN + 4, QUADS = TN / 4;
    /*
     * What int8's epilogue reads, asked for in front of the first transfers: behind the last products it would be waited for, twice (1021 x 1001 x 1531 with gelu, bias and
     * residual, its copies included, 24.6 us behind them, 17.6 in front; 15.8 with what the epilogue below gained since).
     */
    constexpr int TURNS = ROWS * QUADS / (WAVES * 64), ROW_STEP = WAVES * 64 / QUADS;
    static_assert(!x_is_i8<DT> || (TURNS % 2 == 0 && TURNS * WAVES * 64 == ROWS * QUADS && ROW_STEP * QUADS == WAVES * 64), "a lane has the same columns in every turn");
    const int q_col = tid % QUADS * 4, q_row = tid / QUADS, q_j = n0 + q_col;      /* its first of four columns of the tile, not of the up ones, and its first row of a pass */
    const int q_there = p.splits == 1 && q_col < (p.n_half ? TN / 2 : TN) ? cols - q_j : 0;                    /* columns of it */
    auto row_of = [&](int pass, int r) __attribute__((always_inline)) { return m0 + r / (PASS * 16) * (MT * 16) + pass * (PASS * 16) + r % (PASS * 16); };
    XScales<MT, NT> scales;
    u32x4 bias4 = {0, 0, 0, 0}, bias_up4 = bias4, residual4[x_is_i8<DT> ? MT / PASS * TURNS : 1];
    if constexpr (x_is_i8<DT>) {
        if (p.splits == 1)
            x_load_scales(scales, p.a_scale, p.b_scale, p.b_scale_f32, (int64_t)expert * p.N, m_end, [&](int mt) { return m0 + wm * (MT * 16) + mt * 16 + (lane & 15); }, [&](int nt) {
                const bool up = p.n_half && nt >= NT / 2;
                const int j = n0 + wn * (p.n_half ? NT * 8 : NT * 16) + (up ? nt - NT / 2 : nt) * 16 + (lane >> 4) * 4;
                return XCols{j + (up ? p.n_half : 0), cols - j};
            });
        if (p.bias) {
            bias4 = x_raw4<DT>(p.bias, p.bias_f32, (int64_t)expert * p.N + q_j, q_there);
            if (p.n_half) bias_up4 = x_raw4<DT>(p.bias, p.bias_f32, (int64_t)expert * p.N + p.n_half + q_j, q_there);
        }
        /* one branch for all of them, so that nothing comes between the loads */
        auto bring_residual = [&](int f32, int n) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < MT / PASS * TURNS; ++i) {
                const int row = row_of(i / TURNS, q_row + i % TURNS * ROW_STEP);
                residual4[i] = x_raw4<DT>(p.residual, f32, (row < m_end ? row : m_end - 1) * p.ldo + q_j, n);
            }
        };
        if (p.residual) {
            if (q_there < 4) {
                if (q_there > 0) bring_residual(p.out_f32, q_there);
            } else if (p.out_f32) {
                bring_residual(1, 4);
            } else {
                bring_residual(0, 4);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) bring_next(i);
    int stage = 0;
    for (int steps = (left + (STAGES - 1) * XBK + XBK - 1) / XBK; steps > 0; --steps) {
        x_turn<(STAGES - 2) * (A_PARTS + B_PARTS)>();
        const uint8_t *la = smem + stage * STAGE, *lb = la + TM * 128;
        u32x4 fa[2][MT], fb[2][NT];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) fb[s][nt] = B_COLS ? tr_fragment<TN>(lb, col_of(nt), s, lane) : kc_fragment(lb, col_of(nt), s, lane);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const int r = wm * (MT * 16) + mt * 16;
                fa[s][mt] = A_COLS ? tr_fragment<TM>(la, r, s, lane) : kc_fragment(la, r, s, lane);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        bring_next(stage == 0 ? STAGES - 1 : stage - 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            if (bias_b)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) bias_acc[REDUCE ? nt : 0] = x_mfma<DT>(fb[s][nt], ones, bias_acc[REDUCE ? nt : 0]);
            if (bias_a)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) bias_acc[REDUCE ? mt : 0] = x_mfma<DT>(ones, fa[s][mt], bias_acc[REDUCE ? mt : 0]);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = x_mfma<DT>(fb[s][nt], fa[s][mt], acc[mt][nt]);
        }
        stage = stage + 1 == STAGES ? 0 : stage + 1;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

    /* ---- epilogue: a lane has columns 4 (l / 16) .. + 3 of row l % 16 of every sub-tile; in half precision cols is a multiple of 8 ---- */
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
#pragma unroll
                for (int i = 0; i < 4; ++i) put(n0 + wn * (NT * 16) + nt * 16 + q4 + i, p.N, bias_acc[nt][i]);
        if (bias_a && lane < 16)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) put(m0 + wm * (MT * 16) + mt * 16 + lane, p.M, bias_acc[mt][0]);
    }
    const int cols_left = cols - n0 - wn * (p.n_half ? NT * 8 : NT * 16), row0 = m0 + wm * (MT * 16), rows_left = m_end - row0;
    const uint32_t own = __builtin_amdgcn_readfirstlane(x_lds(smem) + wave * 2048);
    static_assert(WAVES * 2048 <= STAGES * STAGE, "every wave has its own");
    /* parts' sums stay integers until they are joined */
    if constexpr (x_is_i8<DT>)
        if (p.splits == 1) x_scale_tile(acc, scales);
    const bool plain = REDUCE || p.splits > 1 || (!p.bias && !p.residual && !p.preact && (p.act == ACT_NONE || p.act == ACT_SWIGLU));
    if (plain) {
        __syncthreads();
        if (p.splits > 1) {
            const int parts_left = x_is_i8<DT> ? (cols_left + 3) & ~3 : cols_left;       /* rows of sums are padded to four */
            float *to = p.partial + ((int64_t)split * (REDUCE ? p.M : p.rows) + row0) * p.ldp + (cols - cols_left);
            if (NT > 1 && p.n_half) {
                x_lines_out<DT, MT, (NT > 1 ? NT / 2 : 1), 16, 0>(own, to, 1, (int)p.ldp, rows_left, parts_left, lane, [&](int mt, int i) { return x_value(acc[mt][i]); });
                x_lines_out<DT, MT, (NT > 1 ? NT / 2 : 1), 16, 0>(own, to + (x_is_i8<DT> ? p.up_at : p.n_half), 1, (int)p.ldp, rows_left, parts_left, lane, [&](int mt, int i) { return x_value(acc[mt][i + NT / 2]); });
            } else {
                x_lines_out<DT, MT, NT, 16, 0>(own, to, 1, (int)p.ldp, rows_left, parts_left, lane, [&](int mt, int i) { return x_value(acc[mt][i]); });
            }
            return;
        }
        auto *to = static_cast<uint8_t *>(p.out) + ((REDUCE ? expert * p.out_stride : 0) + (int64_t)row0 * p.ldo + (cols - cols_left)) * (p.out_f32 ? 4 : 2);
        if (NT > 1 && p.n_half)
            x_lines_out<DT, MT, (NT > 1 ? NT / 2 : 1), 16, 0>(own, to, p.out_f32, (int)p.ldo, rows_left, cols_left, lane, [&](int mt, int i) {
                f32x4 y;
#pragma unroll
                for (int c = 0; c < 4; ++c) y[c] = x_silu(x_value(acc[mt][i])[c]) * x_value(acc[mt][i + NT / 2])[c];
                return y;
            });
        else
            x_lines_out<DT, MT, NT, 16, 0>(own, to, p.out_f32, (int)p.ldo, rows_left, cols_left, lane, [&](int mt, int i) { return x_value(acc[mt][i]); });
        return;
    }
    if constexpr (REDUCE) return;
    /*
     * Everything else through the LDS, up to two row sub-tiles of every wave at a time, so that the activations' code is there once: rows of TN
     * sums, and four more for the banks.
     */
    static_assert(ROWS * LD * 4 <= STAGES * STAGE, "sums fit the stages");
    float *sums = reinterpret_cast<float *>(smem);
#pragma unroll
    for (int pass = 0; pass < MT / PASS; ++pass) {
        __syncthreads();
#pragma unroll
        for (int h = 0; h < PASS; ++h)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                *reinterpret_cast<f32x4 *>(sums + (wm * (PASS * 16) + h * 16 + (lane & 15)) * LD + col_of(nt) + q4) = x_value(acc[pass * PASS + h][nt]);
        __syncthreads();
        if constexpr (x_is_i8<DT>) {
            /* two rows at a time, the types chosen outside the loop (1021 x 1008 x 1536 with residual 10.1 -> 9.7 us, with gelu, bias and residual 11.3 -> 10.8) */
            auto rows_out = [&](auto in_32_bits, auto with_residual) __attribute__((always_inline)) {
                constexpr bool F32 = decltype(in_32_bits)::value, RESIDUAL = decltype(with_residual)::value;
                u32x4 waiting[RESIDUAL ? TURNS : 1];
                if constexpr (RESIDUAL)
#pragma unroll
                    for (int i = 0; i < TURNS; ++i) waiting[i] = residual4[pass * TURNS + i];
                const f32x4 b = x_of_raw4<DT>(bias4, p.bias_f32), bu = x_of_raw4<DT>(bias_up4, p.bias_f32);
#pragma unroll 1
                for (int i = 0; i < TURNS; i += 2) {
                    if (q_there <= 0) continue;
                    f32x4 z[2], up[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float *from = sums + (q_row + (i + h) * ROW_STEP) * LD + q_col;
                        z[h] = *reinterpret_cast<const f32x4 *>(from) + b;
                        if (p.n_half) up[h] = *reinterpret_cast<const f32x4 *>(from + TN / 2) + bu;
                    }
                    x_activate_all<2>(p, z, up);
                    if constexpr (RESIDUAL) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) z[h] += x_of_raw4<DT>(waiting[h], F32);
#pragma unroll
                        for (int k = 2; k < TURNS; ++k) waiting[k - 2] = waiting[k];
                    }
                    auto out = [&](int n) __attribute__((always_inline)) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int row = row_of(pass, q_row + (i + h) * ROW_STEP);
                            if (row < m_end) x_put4<DT>(p.out, F32, row * p.ldo + q_j, n, z[h]);
                        }
                    };
                    if (q_there >= 4) out(4);
                    else out(q_there);
                }
            };
            const std::true_type yes = {};
            const std::false_type no = {};
            if (p.out_f32) p.residual ? rows_out(yes, yes) : rows_out(yes, no);
            else p.residual ? rows_out(no, yes) : rows_out(no, no);
            continue;
        }
#pragma unroll 1
        for (int i = tid; i < ROWS * QUADS; i += WAVES * 64) {
            const int r = i / QUADS, c = i % QUADS * 4;
            const int row = row_of(pass, r);
            if (row >= m_end) continue;
            const f32x4 z = *reinterpret_cast<const f32x4 *>(sums + r * LD + c);
            const bool up = p.n_half && c >= TN / 2;
            const int j = n0 + (up ? c - TN / 2 : c);
            if (j >= cols) continue;
            if (!up) {
                f32x4 other = {0.0f, 0.0f, 0.0f, 0.0f};
                if (p.n_half) other = *reinterpret_cast<const f32x4 *>(sums + r * LD + TN / 2 + c);
                x_finish4<DT>(p, expert, row, j, z, other);
            }
        }
    }
}

} // namespace

#endif /* ZBAL_EXPERT_DIRECT_H_ */

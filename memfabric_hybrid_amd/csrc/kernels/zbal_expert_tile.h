/*
 * What the half-precision and int8 products of the experts share: the parameter block, where a workgroup's tile lies, how operands lie in
 * the LDS and come out of it as matrix-instruction fragments, and the epilogues.
 *
 * Three products are tiles of the same kind, C[m, n] = sum over k of A[m, k] B[k, n]:
 *   forward          Y = X W        A rows are tokens (k consecutive), B = W, k or n consecutive
 *   rows' gradient   dX = dZ W^T    the same with W's other order
 *   weights'         dW_e = X_e^T dZ_e, k runs over the expert's rows, m and n are consecutive in memory ("REDUCE")
 *
 * An operand whose k is consecutive lies in the LDS as rows of 64 k (128 bytes), one whose m or n is consecutive as rows of the
 * tile's width, 64 of them; the latter is read with ds_read_b64_tr_b16, which hands every lane four k of its column.
 *
 * In int8 both operands have consecutive k, and two of them are one element of 16 bits to all that moves them: the matrix instruction takes the same
 * sixteen bytes of a lane, in the same places, for twice as many k, and adds up 32-bit integers, which no order of the sums can change.
 */
#ifndef ZBAL_EXPERT_TILE_H_
#define ZBAL_EXPERT_TILE_H_

#include "zbal_device.h"
#include "zbal_hip_kernels.h"

namespace {

constexpr int XBK = 64;          /* k per step */
constexpr int XSLOTS = 64;       /* workgroups an XCD runs at a time (32 CUs), for the tile order */

enum { ACT_NONE = 0, ACT_RELU, ACT_SILU, ACT_GELU, ACT_GELU_TANH, ACT_SWIGLU };

struct XgemmParams {
    const uint16_t *a, *b;
    int64_t lda, ldb, b_stride;  /* elements from row to row, and from expert to expert of b */
    const void *counts;          /* [experts] rows of each expert, int32 or int64; null: one expert has all rows */
    int counts_i64, experts;
    int rows;                    /* of the token-side tensors */
    int M, N, K;                 /* M: REDUCE only; K: not REDUCE */
    int n_half;                  /* swiglu: N / 2, where the up columns start; else 0 */
    void *out;
    int64_t ldo, out_stride;
    int out_f32, act;
    const void *bias;            /* [experts, N] */
    int bias_f32;
    const void *residual;        /* of out's type and shape */
    uint16_t *preact;            /* [rows, N] */
    const float *a_scale;        /* int8: [rows] */
    const void *b_scale;         /* int8: [experts, N], fp32 or bf16 */
    int b_scale_f32;
    void *bias_grad;             /* REDUCE: [experts, bias_n], of out's type */
    int bias_side;               /* REDUCE: the operand whose columns it sums: 1 = b, 2 = a */
    float *partial;              /* split along k: [splits][rows of C][ldp] sums instead of out, and [splits][bias_ldp] of the bias's */
    float *bias_partial;
    int64_t ldp, bias_ldp;
    int up_at;                   /* where the up columns start in a row of parts' sums */
    int splits;
    int through_lds;             /* the wide kernel's epilogue: more than a swiglu, with a workgroup per tile */
};

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));

/* the operands' type in DT: bf16, fp16, or int8 with the 16-bit type of the outputs */
constexpr int XI8 = 0x100;
template <int DT> constexpr bool x_is_i8 = (DT & XI8) != 0;
template <int DT> constexpr int x_half = DT & ~XI8;
template <int DT> using x_sum_t = std::conditional_t<x_is_i8<DT>, int32_t, float>;
template <int DT> using x_sums_t = std::conditional_t<x_is_i8<DT>, i32x4, f32x4>;

template <int DT> __device__ __forceinline__ x_sums_t<DT> x_mfma(const u32x4 &rows, const u32x4 &cols, const x_sums_t<DT> &c)
{
    if constexpr (x_is_i8<DT>)
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, rows), __builtin_bit_cast(i32x4, cols), c, 0, 0, 0);
    else if constexpr (DT == ZDT_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, rows), __builtin_bit_cast(bf16x8_t, cols), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, rows), __builtin_bit_cast(f16x8_t, cols), c, 0, 0, 0);
}

/* ---- operands in the LDS ------------------------------------------------------------------------------------------- */

/*
 * k consecutive: row r at +128 r, its 16-byte chunk c in slot c ^ key(r). Sixteen lanes that read one chunk of sixteen rows touch
 * every 16 bytes of the 64 banks once: rows are half of the banks' width, so the key leaves the lowest bit of r to the address.
 */
__device__ __forceinline__ constexpr int kc_key(int r) { return (r >> 1) & 7; }
__device__ __forceinline__ constexpr int kc_at(int r, int c) { return r * 128 + ((c ^ kc_key(r)) << 4); }

/*
 * m or n consecutive, W of them in a row of k: 32-byte units (sixteen columns), unit u of row k in place u ^ key. Half a wave reads a
 * unit of eight rows, k = 0-3 and 8-11 of a group of sixteen; the key spreads them over the banks (256 bytes: eight units, or four of either
 * row parity where W is 64).
 */
template <int W> __device__ __forceinline__ constexpr int tr_key(int k)
{
    return W >= 128 ? ((k & 3) | ((k >> 3) & 1) << 2) : (((k >> 1) & 1) | ((k >> 3) & 1) << 1);
}
template <int W> __device__ __forceinline__ constexpr int tr_at(int k, int c) { return k * (W * 2) + (((c >> 1) ^ tr_key<W>(k)) << 5) + ((c & 1) << 4); }

/* fragment of rows r0 .. r0 + 15, k = 32 s ..: lane l has row l % 16 and the eight k from 8 (l / 16) */
__device__ __forceinline__ u32x4 kc_fragment(const uint8_t *tile, int r0, int s, int lane)
{
    return *reinterpret_cast<const u32x4 *>(tile + kc_at(r0 + (lane & 15), s * 4 + (lane >> 4)));
}

/* the same of columns c0 .. c0 + 15 (c0 a multiple of 16): two transposing reads of four k each */
template <int W> __device__ __forceinline__ u32x4 tr_fragment(const uint8_t *tile, int c0, int s, int lane)
{
    const int j = lane & 15, k = s * 32 + (lane >> 4) * 8 + (j >> 2);
    const uint8_t *at = tile + k * (W * 2) + (((c0 >> 4) ^ tr_key<W>(k)) << 5) + (j & 3) * 8;     /* k + 4 has the same key */
    typedef s16x4_t __attribute__((address_space(3))) *lds_t;
    const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(uintptr_t)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)at);
    const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(uintptr_t)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)(at + 4 * (W * 2)));
    const u32x2 l2 = __builtin_bit_cast(u32x2, lo), h2 = __builtin_bit_cast(u32x2, hi);
    return u32x4{l2[0], l2[1], h2[0], h2[1]};
}

/* ---- whose rows ---------------------------------------------------------------------------------------------------- */

__device__ __forceinline__ uint32_t x_count(const XgemmParams &p, int e)
{
    if (!p.counts) return (uint32_t)p.rows;
    const int64_t c = p.counts_i64 ? static_cast<const int64_t *>(p.counts)[e] : (int64_t)static_cast<const int32_t *>(p.counts)[e];
    return c < 0 ? 0u : (c > p.rows ? (uint32_t)p.rows : (uint32_t)c);
}

/* inclusive sum over the lanes, stopping at the largest number instead of wrapping round */
__device__ __forceinline__ uint32_t x_scan(uint32_t v)
{
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t o = __shfl_up(v, off, 64);
        if ((int)(threadIdx.x & 63) >= off) v = __builtin_elementwise_add_sat(v, o);
    }
    return v;
}

/* counts are taken as they come: none is less than nothing, and no expert's rows end behind the tensors' last */
struct XSpan { int begin, end; };
__device__ __forceinline__ XSpan x_span(const XgemmParams &p, uint32_t before, uint32_t incl)
{
    const uint32_t r = (uint32_t)p.rows;
    return {(int)(before < r ? before : r), (int)(incl < r ? incl : r)};
}

/* rows of expert e, for a whole wave */
__device__ __forceinline__ XSpan x_rows_of(const XgemmParams &p, int e)
{
    if (p.experts == 1) return x_span(p, 0, x_count(p, 0));
    const int lane = threadIdx.x & 63;
    uint32_t run = 0;
    for (int base = 0;; base += 64) {
        const uint32_t c = base + lane < p.experts ? x_count(p, base + lane) : 0;
        const uint32_t incl = x_scan(c);
        if (e < base + 64) {
            const uint32_t end = __builtin_elementwise_add_sat(run, (uint32_t)__builtin_amdgcn_readlane((int)incl, e - base));
            const uint32_t own = (uint32_t)__builtin_amdgcn_readlane((int)c, e - base);
            /* a sum that stopped at the largest number is past the last row either way */
            return x_span(p, end - own, end);
        }
        run = __builtin_elementwise_add_sat(run, (uint32_t)__builtin_amdgcn_readlane((int)incl, 63));
    }
}

/* where the last expert's rows end, for a whole wave: all counts are loaded at once. A lane's sum that stops at the last row leaves the result what it is */
__device__ __forceinline__ int x_rows_in_all(const XgemmParams &p)
{
    uint32_t sum = 0;
    for (int e = threadIdx.x & 63; e < p.experts; e += 64) sum += x_count(p, e);
    const uint32_t r = (uint32_t)p.rows, all = (uint32_t)zb_wave_sum_dpp((int)(sum < r ? sum : r));
    return (int)(all < r ? all : r);
}

struct XTile { int expert, row_begin, row_end, n_tile; };

/*
 * Tile `id` of the order in which XCD x (workgroups x, x + 8, ...) has a contiguous run of tiles: expert by expert, in groups of all
 * the expert's row tiles by up to eight column tiles, row tile fastest, so that what runs at the same time on an XCD shares operands in
 * its L2. expert -1: there is no such tile. Every wave works it out for itself from the counts.
 */
template <int TM> __device__ __forceinline__ XTile x_locate(const XgemmParams &p, int n_tiles, int id, int slots)
{
    const int lane = threadIdx.x & 63;
    auto tiles_of = [&](uint32_t before, uint32_t incl) { const XSpan s = x_span(p, before, incl); return (uint32_t)(s.end - s.begin + TM - 1) / TM; };
    /* tile r of an expert's */
    auto place = [&](int expert, int begin, int end, int mt, int r) __attribute__((always_inline)) -> XTile {
        int group = slots / mt;
        group = group < 1 ? 1 : (group > 8 ? 8 : group);
        const int per = mt * group, g = r / per, in = r - g * per, from = begin + in % mt * TM;
        return {expert, from, end - from > TM ? from + TM : end, g * group + in / mt};
    };
    if (p.experts == 1) {
        const XSpan s = x_rows_of(p, 0);
        const int mt = (s.end - s.begin + TM - 1) / TM, total = mt * n_tiles, chunk = (total + 7) / 8, logical = (id & 7) * chunk + (id >> 3);
        if ((id >> 3) >= chunk || logical >= total) return {-1, 0, 0, 0};
        return place(0, s.begin, s.end, mt, logical);
    }
    uint32_t run = 0, tiles = 0;
    for (int base = 0; base < p.experts; base += 64) {
        const uint32_t c = base + lane < p.experts ? x_count(p, base + lane) : 0;
        const uint32_t incl = __builtin_elementwise_add_sat(run, x_scan(c));
        tiles += (uint32_t)zb_wave_sum_dpp((int)tiles_of(incl - c, incl));
        run = (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
    }
    const int total = (int)tiles * n_tiles, chunk = (total + 7) / 8, logical = (id & 7) * chunk + (id >> 3);
    if ((id >> 3) >= chunk || logical >= total) return {-1, 0, 0, 0};
    const int q = logical / n_tiles;                         /* a row tile of the expert wanted */
    run = 0;
    uint32_t first = 0;
    for (int base = 0; base < p.experts; base += 64) {
        const uint32_t c = base + lane < p.experts ? x_count(p, base + lane) : 0;
        const uint32_t incl = __builtin_elementwise_add_sat(run, x_scan(c));
        const uint32_t mt = tiles_of(incl - c, incl), mt_incl = first + (uint32_t)zb_wave_scan_dpp((int)mt);
        const uint64_t owner = __ballot(mt_incl > (uint32_t)q);
        if (owner != 0) {
            const int l = __ffsll((long long)owner) - 1;
            const int mt_e = __builtin_amdgcn_readlane((int)mt, l);
            const int first_e = __builtin_amdgcn_readlane((int)mt_incl, l) - mt_e;
            const XSpan s = x_span(p, incl - c, incl);
            const int begin = __builtin_amdgcn_readlane(s.begin, l), end = __builtin_amdgcn_readlane(s.end, l);
            return place(base + l, begin, end, mt_e, logical - first_e * n_tiles);
        }
        first = (uint32_t)__builtin_amdgcn_readlane((int)mt_incl, 63);
        run = (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
    }
    return {-1, 0, 0, 0};
}

/* ---- activations --------------------------------------------------------------------------------------------------- */

__device__ __forceinline__ float x_sigmoid(float z) { return 1.0f / (1.0f + __expf(-z)); }
__device__ __forceinline__ float x_silu(float z) { return z / (1.0f + __expf(-z)); }

/*
 * The normal distribution's integral up to z and exp(-z^2 / 2), which gelu and its slope are made of. With x = |z| the tail is R(x) exp(-x^2 / 2), and
 * R(x) (1 + 0.31 x) hardly changes: a polynomial of the ninth degree in w = 0.31 x / (1 + 0.31 x) that meets it in the ten Chebyshev nodes of x = 0 .. 16 is good to
 * 2^-26. The square's rounding and its product's with log2 e go back into the exponential, so that the tail, and gelu far below zero, keep their relative precision:
 * within 7 steps of 2^-24 from -12 to 12, where 1 + erf is off by a step of one (1.6e3 steps of gelu(-3.5)). gelu's rms error for normally distributed z is 0.37
 * steps. The library's erfc and exp are as good, and cost 4096 x 2048 x 4096 with gelu 94 us instead of 81, the gradient's stream of 16384 x 7168 217 instead of 196.
 */
struct XNormal { float integral, bell; };
__device__ __forceinline__ XNormal x_normal(float z)
{
    const float x = fminf(fabsf(z), 16.0f), d = __builtin_fmaf(x, 0.31f, 1.0f);
    float r = __builtin_amdgcn_rcpf(d);
    r = __builtin_fmaf(r, __builtin_fmaf(-d, r, 1.0f), r);
    const float w = x * 0.31f * r;
    float v = 0x1.432956p-6f;
    v = __builtin_fmaf(v, w, -0x1.471c64p-4f);
    v = __builtin_fmaf(v, w, 0x1.97a3d4p-4f);
    v = __builtin_fmaf(v, w, -0x1.f1cbecp-7f);
    v = __builtin_fmaf(v, w, 0x1.2af4c6p-7f);
    v = __builtin_fmaf(v, w, -0x1.0bbb48p-3f);
    v = __builtin_fmaf(v, w, -0x1.41443cp-6f);
    v = __builtin_fmaf(v, w, 0x1.0e21a6p-1f);
    v = __builtin_fmaf(v, w, -0x1.92e5d4p-1f);
    v = __builtin_fmaf(v, w, 0x1.0p-1f);
    v *= r;
    const float h = x * x, low = __builtin_fmaf(x, x, -h), a = h * -0.721347511f;
    const float rest = __builtin_fmaf(low, -0.721347511f, __builtin_fmaf(h, -9.62981517e-09f, __builtin_fmaf(h, -0.721347511f, -a)));
    const float e = __builtin_amdgcn_exp2f(a), bell = __builtin_fmaf(e, rest * 0.693147181f, e);
    return {z < 0.0f ? v * bell : __builtin_fmaf(-v, bell, 1.0f), bell};
}
/* 0.5 (1 + tanh u) is the sigmoid of 2 u */
__device__ __forceinline__ float x_gelu_gate(float z) { return x_sigmoid(1.5957691216057308f * (z + 0.044715f * z * z * z)); }

__device__ __forceinline__ float x_activate(int act, float z)
{
    switch (act) {
        case ACT_RELU: return z > 0.0f ? z : (z == z ? 0.0f : z);
        case ACT_SILU: return x_silu(z);
        case ACT_GELU: return z * x_normal(z).integral;
        case ACT_GELU_TANH: return z * x_gelu_gate(z);
        default: return z;
    }
}

/* its derivative */
__device__ __forceinline__ float x_slope(int act, float z)
{
    switch (act) {
        case ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
        case ACT_SILU: {
            const float s = x_sigmoid(z);
            return s * (1.0f + z * (1.0f - s));
        }
        case ACT_GELU: {
            const XNormal n = x_normal(z);
            return __builtin_fmaf(z * 0.39894228040143268f, n.bell, n.integral);
        }
        case ACT_GELU_TANH: {
            const float s = x_gelu_gate(z), w = s * (1.0f - s);
            return w == 0.0f ? s : s + z * w * 1.5957691216057308f * (1.0f + 0.134145f * z * z);        /* far out z^2 is infinite */
        }
        default: return 1.0f;
    }
}

template <int DT> __device__ __forceinline__ float x_load(const void *p, int f32, int64_t i)
{
    return f32 ? static_cast<const float *>(p)[i] : zb_half_to_f32<x_half<DT>>(static_cast<const uint16_t *>(p)[i]);
}
template <int DT> __device__ __forceinline__ void x_store(void *p, int f32, int64_t i, float v)
{
    if (f32) static_cast<float *>(p)[i] = v;
    else static_cast<uint16_t *>(p)[i] = (uint16_t)zb_f32_to_half<x_half<DT>>(v);
}

/* one value of the output from its sums: bias, activation, residual, one rounding. `j`: output column */
template <int DT> __device__ __forceinline__ void x_finish(const XgemmParams &p, int expert, int64_t row, int j, float z, float up)
{
    if (p.bias) {
        z += x_load<DT>(p.bias, p.bias_f32, (int64_t)expert * p.N + j);
        if (p.n_half) up += x_load<DT>(p.bias, p.bias_f32, (int64_t)expert * p.N + p.n_half + j);
    }
    if (p.preact) {
        p.preact[row * p.N + j] = (uint16_t)zb_f32_to_half<x_half<DT>>(z);
        if (p.n_half) p.preact[row * p.N + p.n_half + j] = (uint16_t)zb_f32_to_half<x_half<DT>>(up);
    }
    float y = p.n_half ? x_silu(z) * up : x_activate(p.act, z);
    if (p.residual) y += x_load<DT>(p.residual, p.out_f32, row * p.ldo + j);
    x_store<DT>(p.out, p.out_f32, row * p.ldo + j, y);
}

/*
 * Four values, where every row of outputs, bias and residual starts at a multiple of four and is one of four long. In int8 rows start, and end, anywhere, which
 * loads and stores of several elements allow; what is less than four is not loaded or stored here.
 */
typedef f32x4 __attribute__((aligned(4))) x_floats_t;
typedef u32x2 __attribute__((aligned(2))) x_halves_t;
template <int DT> __device__ __forceinline__ f32x4 x_load4(const void *p, int f32, int64_t i)
{
    if (f32) {
        if constexpr (x_is_i8<DT>) return *reinterpret_cast<const x_floats_t *>(static_cast<const float *>(p) + i);
        else return *reinterpret_cast<const f32x4 *>(static_cast<const float *>(p) + i);
    }
    u32x2 h;
    if constexpr (x_is_i8<DT>) h = *reinterpret_cast<const x_halves_t *>(static_cast<const uint16_t *>(p) + i);
    else h = *reinterpret_cast<const u32x2 *>(static_cast<const uint16_t *>(p) + i);
    constexpr int H = x_half<DT>;
    return f32x4{zb_half_to_f32<H>(h[0] & 0xffffu), zb_half_to_f32<H>(h[0] >> 16), zb_half_to_f32<H>(h[1] & 0xffffu), zb_half_to_f32<H>(h[1] >> 16)};
}
template <int DT> __device__ __forceinline__ void x_store4(void *p, int f32, int64_t i, const f32x4 &v)
{
    if constexpr (x_is_i8<DT>) {
        if (f32) *reinterpret_cast<x_floats_t *>(static_cast<float *>(p) + i) = v;
        else *reinterpret_cast<x_halves_t *>(static_cast<uint16_t *>(p) + i) = u32x2{zb_pack2_half<x_half<DT>>(v[0], v[1]), zb_pack2_half<x_half<DT>>(v[2], v[3])};
    } else if (f32) *reinterpret_cast<f32x4 *>(static_cast<float *>(p) + i) = v;
    else *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(p) + i) = u32x2{zb_pack2_half<x_half<DT>>(v[0], v[1]), zb_pack2_half<x_half<DT>>(v[2], v[3])};
}
template <int DT> __device__ __forceinline__ void x_finish4(const XgemmParams &p, int expert, int64_t row, int j, f32x4 z, f32x4 up)
{
    if (p.bias) {
        z += x_load4<DT>(p.bias, p.bias_f32, (int64_t)expert * p.N + j);
        if (p.n_half) up += x_load4<DT>(p.bias, p.bias_f32, (int64_t)expert * p.N + p.n_half + j);
    }
    if (p.preact) {
        x_store4<DT>(p.preact, 0, row * p.N + j, z);
        if (p.n_half) x_store4<DT>(p.preact, 0, row * p.N + p.n_half + j, up);
    }
    f32x4 y;
    for (int i = 0; i < 4; ++i) y[i] = p.n_half ? x_silu(z[i]) * up[i] : x_activate(p.act, z[i]);
    if (p.residual) y += x_load4<DT>(p.residual, p.out_f32, row * p.ldo + j);
    x_store4<DT>(p.out, p.out_f32, row * p.ldo + j, y);
}

/* ---- int8: sums of integers and their scales ----------------------------------------------------------------------- */

/* a sum as the value that it stands for (half precision: it is that). `j`: column of W */
template <int DT> __device__ __forceinline__ float x_scaled(const XgemmParams &p, int expert, int64_t row, int j, x_sum_t<DT> sum)
{
    if constexpr (x_is_i8<DT>) return (float)sum * x_load<ZDT_BF16>(p.b_scale, p.b_scale_f32, (int64_t)expert * p.N + j) * p.a_scale[row];
    else return sum;
}
template <int DT> __device__ __forceinline__ f32x4 x_scaled4(const XgemmParams &p, int expert, int64_t row, int j, const x_sums_t<DT> &sum)
{
    if constexpr (x_is_i8<DT>) return __builtin_convertvector(sum, f32x4) * x_load4<XI8 | ZDT_BF16>(p.b_scale, p.b_scale_f32, (int64_t)expert * p.N + j) * p.a_scale[row];
    else return sum;
}

/*
 * The scales of a lane's sub-tiles. row(mt): the row that it has there, nobody's from row_end on; col(nt): the first of its four columns and how many of them there
 * are.
 */
struct XCols { int first, there; };
template <int MT, int NT> struct XScales { float rows[MT]; f32x4 cols[NT]; };
template <int MT, int NT, typename Row, typename Col>
__device__ __forceinline__ void x_load_scales(XScales<MT, NT> &s, const float *a_scale, const void *b_scale, int b_scale_f32, int64_t first_scale, int row_end, Row row, Col col)
{
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) s.rows[mt] = a_scale[row(mt) < row_end ? row(mt) : row_end - 1];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const XCols c = col(nt);
        s.cols[nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (c.there >= 4) {
            s.cols[nt] = x_load4<XI8 | ZDT_BF16>(b_scale, b_scale_f32, first_scale + c.first);
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (i < c.there) s.cols[nt][i] = x_load<ZDT_BF16>(b_scale, b_scale_f32, first_scale + c.first + i);
        }
    }
}
/* integers become the bits of the values that they stand for, where they are */
template <int MT, int NT> __device__ __forceinline__ void x_scale_tile(i32x4 (&acc)[MT][NT], const XScales<MT, NT> &s)
{
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) acc[mt][nt] = __builtin_bit_cast(i32x4, __builtin_convertvector(acc[mt][nt], f32x4) * s.cols[nt] * s.rows[mt]);
}
/* four values as they lie in memory, so that what is asked for early is waited for late; at the end of a row `there` of them */
template <int DT> __device__ __forceinline__ u32x4 x_raw4(const void *p, int f32, int64_t i, int there)
{
    u32x4 r = {0, 0, 0, 0};
    if (there >= 4) {
        if (f32) return __builtin_bit_cast(u32x4, (f32x4)*reinterpret_cast<const x_floats_t *>(static_cast<const float *>(p) + i));
        const u32x2 h = *reinterpret_cast<const x_halves_t *>(static_cast<const uint16_t *>(p) + i);
        r[0] = h[0];
        r[1] = h[1];
        return r;
    }
    if (there <= 0) return r;
    /* all three loads are made, of the first element where there is no other, and are under way together */
    uint32_t v[3];
    if (f32) {
#pragma unroll
        for (int k = 0; k < 3; ++k) v[k] = static_cast<const uint32_t *>(p)[k < there ? i + k : i];
        return u32x4{v[0], there > 1 ? v[1] : 0, there > 2 ? v[2] : 0, 0};
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) v[k] = static_cast<const uint16_t *>(p)[k < there ? i + k : i];
    r[0] = there > 1 ? v[1] << 16 | v[0] : v[0];
    r[1] = there > 2 ? v[2] : 0;
    return r;
}
template <int DT> __device__ __forceinline__ f32x4 x_of_raw4(const u32x4 &r, int f32)
{
    constexpr int H = x_half<DT>;
    if (f32) return __builtin_bit_cast(f32x4, r);
    return f32x4{zb_half_to_f32<H>(r[0] & 0xffffu), zb_half_to_f32<H>(r[0] >> 16), zb_half_to_f32<H>(r[1] & 0xffffu), zb_half_to_f32<H>(r[1] >> 16)};
}

/* the bias of a lane's columns, as it lies in memory, and its addition to the bits of the values that integers have become */
template <int DT, int NT, typename Col>
__device__ __forceinline__ void x_load_bias(u32x4 (&b)[NT], const void *bias, int bias_f32, int64_t first, Col col)
{
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) b[nt] = x_raw4<DT>(bias, bias_f32, first + col(nt).first, col(nt).there);
}
template <int DT, int MT, int NT> __device__ __forceinline__ void x_add_bias(i32x4 (&acc)[MT][NT], const u32x4 (&b)[NT], int bias_f32)
{
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) acc[mt][nt] = __builtin_bit_cast(i32x4, __builtin_bit_cast(f32x4, acc[mt][nt]) + x_of_raw4<DT>(b[nt], bias_f32));
}

/* T times four values behind the activation, which is chosen once for all of them, so that their chains of operations run side by side; z and up have their biases */
template <int T> __device__ __forceinline__ void x_activate_all(const XgemmParams &p, f32x4 (&z)[T], const f32x4 (&up)[T])
{
    auto all = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int k = 0; k < 4; ++k) z[t][k] = f(z[t][k], up[t][k]);
    };
    if (p.n_half) return all([](float v, float u) __attribute__((always_inline)) { return x_silu(v) * u; });
    switch (p.act) {
        case ACT_RELU: return all([](float v, float) __attribute__((always_inline)) { return x_activate(ACT_RELU, v); });
        case ACT_SILU: return all([](float v, float) __attribute__((always_inline)) { return x_activate(ACT_SILU, v); });
        case ACT_GELU: return all([](float v, float) __attribute__((always_inline)) { return x_activate(ACT_GELU, v); });
        case ACT_GELU_TANH: return all([](float v, float) __attribute__((always_inline)) { return x_activate(ACT_GELU_TANH, v); });
        default: return;
    }
}
/* four values of the output, `there` of them */
template <int DT> __device__ __forceinline__ void x_put4(void *p, int f32, int64_t i, int there, const f32x4 &y)
{
    if (there >= 4) {
        x_store4<DT>(p, f32, i, y);
    } else {
#pragma unroll
        for (int k = 0; k < 3; ++k)
            if (k < there) x_store<DT>(p, f32, i + k, y[k]);
    }
}
__device__ __forceinline__ f32x4 x_value(const f32x4 &v) { return v; }
__device__ __forceinline__ f32x4 x_value(const i32x4 &v) { return __builtin_bit_cast(f32x4, v); }

} // namespace

#endif /* ZBAL_EXPERT_TILE_H_ */

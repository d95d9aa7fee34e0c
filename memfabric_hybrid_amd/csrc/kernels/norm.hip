/*
 * Rows of tokens between the products: the root-mean-square norm with the residual's addition and its gradient, and activations,
 * with an output in int8 and a scale for each row.
 *
 * A row is read once: its elements stay in registers (eight to a piece, up to eight pieces to a lane) from the loads over the row's
 * sum of squares and its largest element to the stores. Pieces start wherever their row starts; the last one of a row whose length is not a
 * multiple of eight goes element by element.
 */
#include "zbal_expert_tile.h"

namespace {

constexpr int N_LANES = 512, N_MOST_LANES = 1024, N_PIECES = 8;      /* lanes of a row, those of one that 512 cannot hold (32768 elements), and pieces of a lane */

/* ---- eight elements ------------------------------------------------------------------------------------------------ */

template <int DT> __device__ __forceinline__ float n_load1(const void *p, int64_t i)
{
    if constexpr (DT == ZDT_FP32) return static_cast<const float *>(p)[i];
    else return zb_half_to_f32<DT>(static_cast<const uint16_t *>(p)[i]);
}
template <int DT> __device__ __forceinline__ void n_store1(void *p, int64_t i, float v)
{
    if constexpr (DT == ZDT_FP32) static_cast<float *>(p)[i] = v;
    else static_cast<uint16_t *>(p)[i] = (uint16_t)zb_f32_to_half<DT>(v);
}

typedef u32x4 __attribute__((aligned(2))) n_halves_t;
typedef f32x4 __attribute__((aligned(4))) n_floats_t;
typedef u32x2 __attribute__((aligned(1))) n_bytes_t;

/* as they lie in memory, so that a piece that waits takes no more registers than it must */
template <int DT> struct Piece {
    u32x4 w[DT == ZDT_FP32 ? 2 : 1];
    __device__ __forceinline__ float operator[](int i) const
    {
        if constexpr (DT == ZDT_FP32) return __uint_as_float(w[i >> 2][i & 3]);
        else return zb_half_to_f32<DT>(i & 1 ? w[0][i >> 1] >> 16 : w[0][i >> 1] & 0xffffu);
    }
};

/* elements at .. at + 7 of which `n` are there; zeros for the others */
template <int DT> __device__ __forceinline__ Piece<DT> n_load(const void *p, int64_t at, int n)
{
    Piece<DT> r = {};
    if (n >= 8) {
        if constexpr (DT == ZDT_FP32) {
            r.w[0] = __builtin_bit_cast(u32x4, (f32x4)*reinterpret_cast<const n_floats_t *>(static_cast<const float *>(p) + at));
            r.w[1] = __builtin_bit_cast(u32x4, (f32x4)*reinterpret_cast<const n_floats_t *>(static_cast<const float *>(p) + at + 4));
        } else {
            r.w[0] = *reinterpret_cast<const n_halves_t *>(static_cast<const uint16_t *>(p) + at);
        }
        return r;
    }
#pragma unroll
    for (int i = 0; i < 7; ++i)
        if (i < n) {
            if constexpr (DT == ZDT_FP32) r.w[i >> 2][i & 3] = static_cast<const uint32_t *>(p)[at + i];
            else r.w[0][i >> 1] |= (uint32_t)static_cast<const uint16_t *>(p)[at + i] << ((i & 1) * 16);
        }
    return r;
}

template <int DT> __device__ __forceinline__ void n_store(void *p, int64_t at, int n, const float (&v)[8])
{
    if (n >= 8) {
        if constexpr (DT == ZDT_FP32) {
            *reinterpret_cast<n_floats_t *>(static_cast<float *>(p) + at) = f32x4{v[0], v[1], v[2], v[3]};
            *reinterpret_cast<n_floats_t *>(static_cast<float *>(p) + at + 4) = f32x4{v[4], v[5], v[6], v[7]};
        } else {
            *reinterpret_cast<n_halves_t *>(static_cast<uint16_t *>(p) + at) =
                u32x4{zb_pack2_half<DT>(v[0], v[1]), zb_pack2_half<DT>(v[2], v[3]), zb_pack2_half<DT>(v[4], v[5]), zb_pack2_half<DT>(v[6], v[7])};
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 7; ++i)
        if (i < n) n_store1<DT>(p, at + i, v[i]);
}

/* four numbers of at most 127 (and a rounding), to the nearest integers: the addition of 1.5 * 2^23 leaves them in the low bits */
__device__ __forceinline__ uint32_t n_pack4(float a, float b, float c, float d)
{
    constexpr float MAGIC = 12582912.0f;
    const uint32_t ab = __builtin_amdgcn_perm(__float_as_uint(b + MAGIC), __float_as_uint(a + MAGIC), 0x0c0c0400);
    const uint32_t cd = __builtin_amdgcn_perm(__float_as_uint(d + MAGIC), __float_as_uint(c + MAGIC), 0x04000c0c);
    return ab | cd;
}
__device__ __forceinline__ void n_store_int8(uint8_t *p, int64_t at, int n, const float (&v)[8])
{
    const u32x2 q = {n_pack4(v[0], v[1], v[2], v[3]), n_pack4(v[4], v[5], v[6], v[7])};
    if (n >= 8) {
        *reinterpret_cast<n_bytes_t *>(p + at) = q;
        return;
    }
#pragma unroll
    for (int i = 0; i < 7; ++i)
        if (i < n) p[at + i] = (uint8_t)(q[i >> 2] >> ((i & 3) * 8));
}

/* ---- rows ---------------------------------------------------------------------------------------------------------- */

/*
 * The lanes of a row: `waves` whole waves, and as many rows side by side in a workgroup as there are groups of them. What a round of rows leaves
 * in the LDS lies in one of two places in turn: who is a barrier ahead writes the other one.
 */
struct Lanes {
    int lane, of_row, group, waves, rows;     /* of_row: this lane's place among its row's */
    __device__ __forceinline__ Lanes() : lane(threadIdx.x & 63), of_row(threadIdx.x), group(threadIdx.y), waves(blockDim.x >> 6), rows(blockDim.y) {}
    __device__ __forceinline__ int slot() const { return __builtin_amdgcn_readfirstlane(group * waves + (of_row >> 6)); }
};

template <int N> struct RowSums { float v[N]; };

/* sums over a row's lanes, in all of them; always in the same order */
template <int N> __device__ __forceinline__ RowSums<N> row_sum(RowSums<N> s, const Lanes &l, float (*red)[N])
{
#pragma unroll
    for (int i = 0; i < N; ++i) s.v[i] = zb_wave_reduce_dpp<false>(s.v[i]);
    if (l.waves == 1) return s;
    if (l.lane == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) red[l.slot()][i] = s.v[i];
    __syncthreads();
    RowSums<N> r = {};
    for (int w = 0; w < l.waves; ++w)
#pragma unroll
        for (int i = 0; i < N; ++i) r.v[i] += red[l.group * l.waves + w][i];
    return r;
}

/*
 * The largest magnitude of a row, as its bits: ordered like the numbers, infinity above them and every NaN above that, so that neither is lost.
 */
__device__ __forceinline__ uint32_t n_magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t n_max(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t row_max(uint32_t m, const Lanes &l, uint32_t *red)
{
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) m = n_max(m, (uint32_t)__shfl_xor((int)m, off, 64));
    if (l.waves == 1) return m;
    if (l.lane == 0) red[l.slot()] = m;
    __syncthreads();
    m = 0;
    for (int w = 0; w < l.waves; ++w) m = n_max(m, red[l.group * l.waves + w]);
    return m;
}

/*
 * scale = max / 127, and what the row is multiplied by: 127 / max. The scale is a normal number (2^-126 at least, so that the factor is finite),
 * 0 for a row of zeros, and NaN where the row holds an infinity or a NaN: then nothing that is computed from it looks sound.
 */
struct RowScale { float scale, by; };
__device__ __forceinline__ RowScale row_scale(uint32_t max_bits)
{
    const float max = __uint_as_float(max_bits);
    if (max_bits >= 0x7f800000u) return {__uint_as_float(0x7fc00000u), 0.0f};
    if (max_bits == 0) return {0.0f, 0.0f};
    if (max < 127.0f * 0x1p-126f) return {0x1p-126f, 0x1p126f};
    return {max / 127.0f, 127.0f / max};
}

/* ---- the norm ------------------------------------------------------------------------------------------------------ */

struct NormParams {
    const void *x, *residual, *weight;
    void *y, *total;
    uint8_t *q;
    float *scales;
    const void *grad, *grad_total;    /* the gradient's */
    void *grad_x;
    float *partial;                   /* [row groups of the launch][ldp]: the sums of their rows for the weight's gradient */
    void *grad_weight;                /* of a workgroup alone */
    int weight_grad_f32;
    int64_t rows;
    int width, ldp, weight_f32;
    float eps, per_width;             /* 1 / width */
};

__device__ __forceinline__ float n_rsqrt(float mean_square, float eps) { return 1.0f / __builtin_sqrtf(mean_square + eps); }

/*
 * Eight elements of the weight, ones without one: of the rows' type (W is DT) or of 32 bits. A lane has the same columns of every row, so they are asked for in front of the
 * first row, and are there when its sum is: what the norm gains by that, whose workgroups have one round of rows up to 2^20 of them. The gradient's have many and load them once.
 */
template <int W> __device__ __forceinline__ Piece<W> n_weight(const NormParams &p, int at)
{
    if (p.weight) return n_load<W>(p.weight, at, p.width - at);
    Piece<W> ones;
    constexpr uint32_t one = W == ZDT_FP32 ? 0x3f800000u : (W == ZDT_BF16 ? 0x3f803f80u : 0x3c003c00u);
    for (auto &v : ones.w) v = u32x4{one, one, one, one};
    return ones;
}

template <int DT, int W, int C, int L>
__global__ void __launch_bounds__(L)
rms_norm_kernel(NormParams p)
{
    __shared__ float sums[2][16][1];
    __shared__ uint32_t maxima[2][16];
    const Lanes l;
    Piece<W> w[C];
#pragma unroll
    for (int c = 0; c < C; ++c) w[c] = n_weight<W>(p, (l.of_row + c * (int)blockDim.x) * 8);
    int turn = 0;
    for (int64_t base = (int64_t)blockIdx.x * l.rows; base < p.rows; base += (int64_t)gridDim.x * l.rows, turn ^= 1) {
        const int64_t row = base + l.group, at = row * p.width;
        const bool live = row < p.rows;
        int there[C];
        float h[C][8];
        {
            Piece<DT> x[C], r[C];
#pragma unroll
            for (int c = 0; c < C; ++c) {
                there[c] = live ? p.width - (l.of_row + c * (int)blockDim.x) * 8 : 0;
                x[c] = n_load<DT>(p.x, at + (l.of_row + c * (int)blockDim.x) * 8, there[c]);
                if (p.residual) r[c] = n_load<DT>(p.residual, at + (l.of_row + c * (int)blockDim.x) * 8, there[c]);
            }
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) h[c][i] = p.residual ? x[c][i] + r[c][i] : x[c][i];
        }
        RowSums<1> s = {};
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) s.v[0] = __builtin_fmaf(h[c][i], h[c][i], s.v[0]);
        if (p.total)
#pragma unroll
            for (int c = 0; c < C; ++c) n_store<DT>(p.total, at + (l.of_row + c * (int)blockDim.x) * 8, there[c], h[c]);
        s = row_sum<1>(s, l, sums[turn]);
        const float r = n_rsqrt(s.v[0] * p.per_width, p.eps);
        uint32_t most = 0;
#pragma unroll
        for (int c = 0; c < C; ++c) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                h[c][i] = h[c][i] * r * w[c][i];              /* zeros where the row has ended, or NaN where it has one */
                most = n_max(most, n_magnitude(h[c][i]));
            }
            if (p.y) n_store<DT>(p.y, at + (l.of_row + c * (int)blockDim.x) * 8, there[c], h[c]);
        }
        if (p.q) {
            const RowScale to = row_scale(row_max(most, l, maxima[turn]));
            if (live && l.of_row == 0) p.scales[row] = to.scale;
#pragma unroll
            for (int c = 0; c < C; ++c) {
#pragma unroll
                for (int i = 0; i < 8; ++i) h[c][i] *= to.by;
                n_store_int8(p.q, at + (l.of_row + c * (int)blockDim.x) * 8, there[c], h[c]);
            }
        }
    }
}

/*
 * With n = h r and d = g w: dh = r (d - n mean(d n)) + the sum's own gradient, and the weight's gradient is the sum over rows of g n. Both means of a row
 * come from one reduction, of h^2 and of d h. A lane has the same columns of every row that its workgroup takes, so the
 * weight's sums stay in registers until the last of them; a second launch adds up the workgroups', in order. ALONE: one workgroup has all rows, side by side
 * in its lanes, and adds up their sums itself.
 */
template <int DT, int W, int C, int L, bool ALONE>
__global__ void __launch_bounds__(L)
rms_norm_backward_kernel(NormParams p)
{
    static_assert(!ALONE || C == 1, "a row is a piece to a lane");
    __shared__ float columns[ALONE ? L * 8 : 1];
    __shared__ float sums[2][16][2];
    const Lanes l;
    Piece<W> w[C];
#pragma unroll
    for (int c = 0; c < C; ++c) w[c] = n_weight<W>(p, (l.of_row + c * (int)blockDim.x) * 8);
    float dw[C][8];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[c][i] = 0.0f;
    /* where registers allow, the next row's pieces are on their way while this one's are summed up, and its gradient stored (16384 x 2048 58 -> 53 us, in half the workgroups) */
    constexpr bool AHEAD = C <= 2;
    struct Row { Piece<DT> h[C], g[C], t[C]; };
    auto load = [&](Row &r, int64_t row) __attribute__((always_inline)) {
        const int64_t at = row * p.width;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int col = (l.of_row + c * (int)blockDim.x) * 8, there = row < p.rows ? p.width - col : 0;
            r.h[c] = n_load<DT>(p.x, at + col, there);
            r.g[c] = n_load<DT>(p.grad, at + col, there);
            if (p.grad_total) r.t[c] = n_load<DT>(p.grad_total, at + col, there);
        }
    };
    const int64_t first = (int64_t)blockIdx.x * l.rows, step = (int64_t)gridDim.x * l.rows;
    int turn = 0;
    Row now, next;
    if (AHEAD) load(now, first + l.group);
    for (int64_t base = first; base < p.rows; base += step, turn ^= 1) {
        const int64_t row = base + l.group, at = row * p.width;
        if (!AHEAD) load(now, row);
        else if (base + step < p.rows) load(next, row + step);
        RowSums<2> s = {};
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                s.v[0] = __builtin_fmaf(now.h[c][i], now.h[c][i], s.v[0]);
                s.v[1] = __builtin_fmaf(now.g[c][i] * w[c][i], now.h[c][i], s.v[1]);
            }
        s = row_sum<2>(s, l, sums[turn]);
        const float r = n_rsqrt(s.v[0] * p.per_width, p.eps), mean = s.v[1] * p.per_width * r;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int col = (l.of_row + c * (int)blockDim.x) * 8;
            float d[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float n = now.h[c][i] * r;
                d[i] = r * __builtin_fmaf(-n, mean, now.g[c][i] * w[c][i]);
                if (p.grad_total) d[i] += now.t[c][i];
                dw[c][i] = __builtin_fmaf(now.g[c][i], n, dw[c][i]);
            }
            n_store<DT>(p.grad_x, at + col, row < p.rows ? p.width - col : 0, d);
        }
        if (AHEAD) now = next;
    }
    if constexpr (ALONE) {
        const int per_row = blockDim.x * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) columns[l.group * per_row + l.of_row * 8 + i] = dw[0][i];
        __syncthreads();
        for (int col = l.group * (int)blockDim.x + l.of_row; col < p.width; col += blockDim.x * blockDim.y) {
            float sum = 0.0f;
            for (int g = 0; g < l.rows; ++g) sum += columns[g * per_row + col];
            if (p.weight_grad_f32) static_cast<float *>(p.grad_weight)[col] = sum;
            else n_store1<DT>(p.grad_weight, col, sum);
        }
        return;
    }
    if (!p.partial) return;
    float *to = p.partial + ((int64_t)blockIdx.x * l.rows + l.group) * p.ldp;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int at = (l.of_row + c * (int)blockDim.x) * 8;
        n_store<ZDT_FP32>(to, at, p.width - at, dw[c]);
    }
}

/*
 * Sums of `count` rows of ldp floats, 32 columns (a line) to a workgroup and every 128th row to a lane, then in two steps through the LDS: few columns are few
 * workgroups, so that each has to have many rows under way. out f32, or of type DT.
 */
template <int DT>
__global__ void __launch_bounds__(1024)
rms_norm_join_kernel(const float *__restrict__ partial, int count, int ldp, int width, int out_f32, void *__restrict__ out)
{
    __shared__ f32x4 sums[128][8], some[8][8];
    const int quad = threadIdx.x & 7, first = threadIdx.x >> 3, col = (blockIdx.x * 8 + quad) * 4;
    f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
    if (col < ldp)
#pragma unroll 8
        for (int i = first; i < count; i += 128) s += *reinterpret_cast<const f32x4 *>(partial + (int64_t)i * ldp + col);
    sums[first][quad] = s;
    __syncthreads();
    if (first < 8) {
        s = sums[first][quad];
#pragma unroll
        for (int i = 1; i < 16; ++i) s += sums[first + i * 8][quad];
        some[first][quad] = s;
    }
    __syncthreads();
    if (first != 0) return;
#pragma unroll
    for (int i = 1; i < 8; ++i) s += some[i][quad];
    for (int i = 0; i < 4 && col + i < width; ++i) {
        if (out_f32) static_cast<float *>(out)[col + i] = s[i];
        else n_store1<DT>(out, col + i, s[i]);
    }
}

/* ---- activations in int8 ------------------------------------------------------------------------------------------- */

/*
 * silu in a dozen cycles: an exponential of two and a reciprocal, each a step off (2^-23), and the exponential's argument rounded: about |z| 2^-24 besides, as in the products'
 * epilogue. Zero from about -88 down, where the exponential ends (silu(-88) is -5.3e-37). For swiglu, whose kernel is a stream: with the division of the products' epilogue the vector
 * units took longer than the memory (32768 x 4096: 78 us, now 57). silu alone has that division, chosen element by element (97 us, 65 of bytes).
 */
__device__ __forceinline__ float n_silu(float z) { return z * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f)); }

/* ACT: ACT_NONE, ACT_SWIGLU, or ACT_SILU for whichever of the others the parameters name */
template <int DT, int ACT, int C, int L>
__global__ void __launch_bounds__(L)
quantize_rows_kernel(XgemmParams p, const void *__restrict__ x, uint8_t *__restrict__ q, float *__restrict__ scales)
{
    __shared__ uint32_t maxima[2][16];
    const Lanes l;
    const int cols = p.n_half ? p.n_half : p.N, rows = p.counts ? x_rows_of(p, p.experts - 1).end : p.rows;
    int turn = 0;
    for (int64_t base = (int64_t)blockIdx.x * l.rows; base < rows; base += (int64_t)gridDim.x * l.rows, turn ^= 1) {
        const int64_t row = base + l.group, at = row * p.N;
        const bool live = row < rows;
        int there[C];
        Piece<DT> z[C], up[ACT == ACT_SWIGLU ? C : 1];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int col = (l.of_row + c * (int)blockDim.x) * 8;
            there[c] = live ? cols - col : 0;
            z[c] = n_load<DT>(x, at + col, there[c]);
            if constexpr (ACT == ACT_SWIGLU) up[c] = n_load<DT>(x, at + cols + col, there[c]);
        }
        float y[C][8];
        uint32_t most = 0;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if constexpr (ACT == ACT_NONE) y[c][i] = z[c][i];
                else if constexpr (ACT == ACT_SWIGLU) y[c][i] = n_silu(z[c][i]) * up[c][i];
                else y[c][i] = x_activate(p.act, z[c][i]);
                most = n_max(most, n_magnitude(y[c][i]));    /* where the row has ended there are zeros, and all activations of zero are that */
            }
        const RowScale to = row_scale(row_max(most, l, maxima[turn]));
        if (live && l.of_row == 0) scales[row] = to.scale;
#pragma unroll
        for (int c = 0; c < C; ++c) {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[c][i] *= to.by;
            n_store_int8(q, row * cols + (l.of_row + c * (int)blockDim.x) * 8, there[c], y[c]);
        }
    }
}

/* ---- launches ------------------------------------------------------------------------------------------------------ */

/*
 * Lanes and pieces of a row of `width` elements: one piece to a lane up to `most` lanes, then more; rows side by side in 256 lanes. A gradient of more than 16384
 * elements, and a norm of more than 32768, has more in hand than its registers hold, and is slower for it.
 */
struct Shape {
    int pieces, groups;
    unsigned lanes;
    dim3 block() const { return dim3(lanes, groups); }
    unsigned blocks(int64_t rows, int64_t most) const
    {
        const int64_t n = (rows + groups - 1) / groups;
        return (unsigned)(n < most ? n : most);
    }
};
inline Shape shape_of(int64_t width, int most)
{
    const int64_t pieces = (width + 7) / 8;
    Shape s = {1, 1, 0};
    while (s.pieces < N_PIECES && (pieces + s.pieces - 1) / s.pieces > most) s.pieces *= 2;
    s.lanes = (unsigned)(((pieces + s.pieces - 1) / s.pieces + 63) / 64 * 64);
    s.groups = s.lanes >= 256 ? 1 : 256 / (int)s.lanes;
    return s;
}

/*
 * Few rows have a lane to a piece as far as that goes; many of them more rows side by side on a CU. us with 512 / 256 lanes, bf16, over inputs that change, norm alone and int8 rows
 * without an activation: 4096 columns, 512 rows 4.1 / 4.0 and 3.8 / 3.8, 1024 5.5 / 5.0 and 4.7 / 4.6, 2048 8.0 / 7.3 and 7.2 / 6.2, 2560 9.3 / 8.4 and 8.5 / 7.7, 8192 29.6 / 22.9 and
 * 22.5 / 18.2; 7168, 256 rows 3.6 / 4.0 and 3.9 / 3.8, 2560 16.0 / 15.3 and 12.1 / 11.8, 8192 43.0 / 38.6 and 29.8 / 29.1; 8192, 2560 16.2 / 16.3 and 12.8 / 12.5, 8192 44.2 / 42.2 and
 * 31.8 / 31.8. With residual and int8 besides (4096 x 7168 42.4 / 43.1) and from 14336 columns on (8192 rows 84.9 / 94.2 and 62.1 / 64.4) half the lanes are a few percent slower.
 */
inline Shape forward_shape(int64_t width, int64_t rows) { return shape_of(width, rows > 2048 ? 256 : N_LANES); }

/* f(pieces, most lanes) as integral constants */
template <typename F> void with_shape(const Shape &s, F f)
{
    const std::integral_constant<int, N_LANES> lanes = {};
    switch (s.pieces) {
        case 1: f(std::integral_constant<int, 1>{}, lanes); break;
        case 2: f(std::integral_constant<int, 2>{}, lanes); break;
        case 4: f(std::integral_constant<int, 4>{}, lanes); break;
        default:
            if (s.lanes <= N_LANES) f(std::integral_constant<int, 8>{}, lanes);
            else f(std::integral_constant<int, 8>{}, std::integral_constant<int, N_MOST_LANES>{});
    }
}
template <typename F> void with_type(int dtype, F f)
{
    switch (dtype) {
        case ZDT_BF16: f(std::integral_constant<int, ZDT_BF16>{}); break;
        case ZDT_FP16: f(std::integral_constant<int, ZDT_FP16>{}); break;
        default: f(std::integral_constant<int, ZDT_FP32>{});
    }
}

constexpr int64_t N_MOST_BLOCKS = 1 << 20;           /* of 1024 lanes: a launch is less than 2^32 lanes */

bool norm_ok(const zbalhip_rms_norm_t *d)
{
    if (!d || d->tokens < 0 || d->tokens > ZBALHIP_EXPERT_MAX_ROWS || d->hidden <= 0 || d->hidden > ZBALHIP_EXPERT_MAX_WIDTH) return false;
    if (d->dtype != ZDT_BF16 && d->dtype != ZDT_FP16 && d->dtype != ZDT_FP32) return false;
    return d->eps > 0.0f && d->eps < __builtin_inff();
}

NormParams norm_params(const zbalhip_rms_norm_t *d)
{
    NormParams p = {};
    p.x = d->x;
    p.residual = d->residual;
    p.weight = d->weight;
    p.weight_f32 = d->weight_is_f32;
    p.rows = d->tokens;
    p.width = (int)d->hidden;
    p.ldp = (p.width + 3) / 4 * 4;
    p.eps = d->eps;
    p.per_width = 1.0f / (float)d->hidden;
    return p;
}

/*
 * Workgroups of the gradient's launch, each with sums of its own: 512 lanes a CU (twice that where a row is not asked for ahead of its time), the same number on every CU, are
 * enough for the memory, and sums of two rows at least cost less than their rows once every CU has one. us at 256 / 512 / 1024 workgroups: 16384 x 2048 67 / 52 / 56;
 * 4096 x 7168 (of 448 lanes) 48 / 52 / 58, 292 of them 63; 1000 x 1024 8.6 / 11.0 / 11.0.
 */
Shape backward_shape(const zbalhip_rms_norm_t *d)
{
    return shape_of(d->hidden, N_LANES);
}
unsigned backward_blocks(const zbalhip_rms_norm_t *d)
{
    const Shape s = backward_shape(d);
    const int64_t rounds = (d->tokens + s.groups - 1) / s.groups, each = (s.pieces <= 2 ? 512 : 1024) / (int64_t)(s.lanes * s.groups);
    const int64_t full = each > 1 ? each * 256 : 256, most = full < (rounds + 1) / 2 ? full : (rounds + 1) / 2;
    return s.blocks(d->tokens, most > 256 ? most : 256);
}
/* rows that one workgroup is through with before a second launch would have begun: a round takes 0.6 to 2 us, a launch 2.3 (32 x 512 6.2 -> 4.5 us) */
int backward_alone(const zbalhip_rms_norm_t *d)
{
    const Shape s = backward_shape(d);
    const int groups = N_MOST_LANES / (int)s.lanes;
    return s.pieces == 1 && d->tokens > 0 && d->tokens <= (int64_t)groups * 2 ? groups : 0;
}

} // namespace

extern "C" int32_t zbalhip_rms_norm(const zbalhip_rms_norm_t *d, void *y, void *total, int8_t *q, float *scales, void *stream)
{
    if (!norm_ok(d) || (q && !scales)) return ZBALHIP_INVALID;
    if (d->tokens == 0) return ZBALHIP_OK;
    if (!d->x || (!y && !total && !q)) return ZBALHIP_INVALID;
    NormParams p = norm_params(d);
    p.y = y;
    p.total = total;
    p.q = (uint8_t *)q;
    p.scales = scales;
    const Shape s = forward_shape(d->hidden, d->tokens);
    with_type(d->dtype, [&](auto dt) {
        with_shape(s, [&](auto c, auto l) {
            constexpr int DT = decltype(dt)::value, C = decltype(c)::value, L = decltype(l)::value;
            const dim3 grid(s.blocks(p.rows, N_MOST_BLOCKS));
            if (p.weight && p.weight_f32) zb_launch(rms_norm_kernel<DT, ZDT_FP32, C, L>, grid, s.block(), 0, (hipStream_t)stream, p);
            else zb_launch(rms_norm_kernel<DT, DT, C, L>, grid, s.block(), 0, (hipStream_t)stream, p);
        });
    });
    return zbalhip_check_launch();
}

extern "C" int64_t zbalhip_rms_norm_backward_workspace(const zbalhip_rms_norm_t *d)
{
    if (!norm_ok(d)) return -1;
    return backward_alone(d) ? 0 : (int64_t)backward_blocks(d) * backward_shape(d).groups * ((d->hidden + 3) / 4 * 4) * 4;
}

extern "C" int32_t zbalhip_rms_norm_backward(const zbalhip_rms_norm_t *d, const void *grad, const void *grad_total, void *grad_x, void *grad_weight,
                                             int32_t weight_grad_is_f32, void *workspace, int64_t workspace_bytes, void *stream)
{
    if (!norm_ok(d)) return ZBALHIP_INVALID;
    if (d->tokens > 0 && (!d->x || !grad || !grad_x)) return ZBALHIP_INVALID;
    if (d->tokens == 0 && !grad_weight) return ZBALHIP_OK;
    const int64_t need = grad_weight && d->tokens > 0 ? zbalhip_rms_norm_backward_workspace(d) : 0;
    if (need > 0 && (!workspace || workspace_bytes < need)) return ZBALHIP_INVALID;
    NormParams p = norm_params(d);
    p.grad = grad;
    p.grad_total = grad_total;
    p.grad_x = grad_x;
    p.partial = grad_weight ? (float *)workspace : nullptr;
    hipStream_t st = (hipStream_t)stream;
    const int groups = grad_weight ? backward_alone(d) : 0;
    if (groups) {
        p.grad_weight = grad_weight;
        p.weight_grad_f32 = weight_grad_is_f32;
        const dim3 block(backward_shape(d).lanes, groups);
        with_type(d->dtype, [&](auto dt) {
            constexpr int DT = decltype(dt)::value;
            if (p.weight && p.weight_f32) zb_launch(rms_norm_backward_kernel<DT, ZDT_FP32, 1, N_MOST_LANES, true>, dim3(1), block, 0, st, p);
            else zb_launch(rms_norm_backward_kernel<DT, DT, 1, N_MOST_LANES, true>, dim3(1), block, 0, st, p);
        });
        return zbalhip_check_launch();
    }
    const Shape s = backward_shape(d);
    const unsigned blocks = backward_blocks(d);
    if (d->tokens > 0)
        with_type(d->dtype, [&](auto dt) {
            with_shape(s, [&](auto c, auto l) {
                constexpr int DT = decltype(dt)::value, C = decltype(c)::value, L = decltype(l)::value;
                if (p.weight && p.weight_f32) zb_launch(rms_norm_backward_kernel<DT, ZDT_FP32, C, L, false>, dim3(blocks), s.block(), 0, st, p);
                else zb_launch(rms_norm_backward_kernel<DT, DT, C, L, false>, dim3(blocks), s.block(), 0, st, p);
            });
        });
    if (grad_weight)
        with_type(d->dtype, [&](auto dt) {
            zb_launch(rms_norm_join_kernel<decltype(dt)::value>, dim3((unsigned)(p.ldp + 31) / 32), dim3(1024), 0, st, p.partial, (int)(blocks * s.groups), p.ldp,
                      p.width, weight_grad_is_f32, grad_weight);
        });
    return zbalhip_check_launch();
}

extern "C" int32_t zbalhip_quantize_rows(const zbalhip_quantize_rows_t *d, const void *x, int8_t *q, float *scales, void *stream)
{
    if (!d || d->rows < 0 || d->rows > ZBALHIP_EXPERT_MAX_ROWS || d->width <= 0 || d->width > ZBALHIP_EXPERT_MAX_WIDTH) return ZBALHIP_INVALID;
    if (d->dtype != ZDT_BF16 && d->dtype != ZDT_FP16 && d->dtype != ZDT_FP32) return ZBALHIP_INVALID;
    if (d->activation < ACT_NONE || d->activation > ACT_SWIGLU || (d->activation == ACT_SWIGLU && d->width % 2 != 0)) return ZBALHIP_INVALID;
    if (d->counts && (d->experts <= 0 || d->experts > 1024)) return ZBALHIP_INVALID;
    if (d->rows == 0) return ZBALHIP_OK;
    if (!x || !q || !scales) return ZBALHIP_INVALID;
    XgemmParams p = {};
    p.counts = d->counts;
    p.counts_i64 = d->counts_are_i64;
    p.experts = d->counts ? (int)d->experts : 1;
    p.rows = (int)d->rows;
    p.N = (int)d->width;
    p.act = d->activation;
    p.n_half = d->activation == ACT_SWIGLU ? p.N / 2 : 0;
    const Shape s = forward_shape(p.n_half ? p.n_half : p.N, d->rows);
    const dim3 grid(s.blocks(d->rows, N_MOST_BLOCKS));
    with_type(d->dtype, [&](auto dt) {
        with_shape(s, [&](auto c, auto l) {
            constexpr int DT = decltype(dt)::value, C = decltype(c)::value, L = decltype(l)::value;
            if (p.act == ACT_NONE) zb_launch(quantize_rows_kernel<DT, ACT_NONE, C, L>, grid, s.block(), 0, (hipStream_t)stream, p, x, (uint8_t *)q, scales);
            else if (p.act == ACT_SWIGLU) zb_launch(quantize_rows_kernel<DT, ACT_SWIGLU, C, L>, grid, s.block(), 0, (hipStream_t)stream, p, x, (uint8_t *)q, scales);
            else zb_launch(quantize_rows_kernel<DT, ACT_SILU, C, L>, grid, s.block(), 0, (hipStream_t)stream, p, x, (uint8_t *)q, scales);
        });
    });
    return zbalhip_check_launch();
}

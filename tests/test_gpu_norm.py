"""The root-mean-square norm with its int8 output and gradient, and activations in int8, against plain forms in 64 bits: one element to the widest
rows, lengths that no piece divides, every type, weight and output, rows that nothing sound can come of, rows of nobody."""
import ctypes

import pytest
import torch

from memfabric_hybrid_amd import capi
from memfabric_hybrid_amd.buffer import Buffer

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
ACTIVATIONS = ["none", "relu", "silu", "gelu", "gelu_tanh", "swiglu"]
U = 2.0 ** -24
EPS = 1e-6
SIZES = [(1, 1), (1, 8), (3, 7), (6, 64), (2, 100), (5, 511), (9, 512), (3, 513), (70, 1024), (9, 1531), (33, 2048), (5, 4096), (2, 4104), (3, 7168), (2, 8191),
         (3, 16392), (2, 33000), (2, 65536)]


@pytest.fixture(scope="module")
def buf():
    b = Buffer()
    yield b
    torch.cuda.synchronize()
    b.close()


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """half of the smallest step of a type"""
    return 2.0 ** -25 if dtype == torch.float16 else 1e-37


def close(got, want, err, dtype):
    """one rounding to the type of a value that is `err` off"""
    assert got.dtype == dtype
    bad = (got.double() - want).abs() > half_step(dtype) * (want.abs() + err) + err + tiny(dtype)
    assert not bad.any(), (bad.sum().item(), ((got.double() - want).abs() / (want.abs() + err + 1e-300)).max().item())


def make(tokens, hidden, dtype, seed, weight="same"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = torch.exp(torch.randn((tokens, 1), device="cuda", generator=g))
    x = (torch.randn((tokens, hidden), device="cuda", generator=g) * rows).to(dtype)
    w = None if weight is None else torch.randn((hidden,), device="cuda", generator=g).to(dtype if weight == "same" else torch.float32)
    return g, x, w


def norm64(h, w, eps=EPS):
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return y if w is None else y * w.double()


# A row's squares are summed by chains of up to 64 in a lane, 6 steps of a wave and 16 waves, of sums of two roundings: 90 steps, halved by the root; the mean, eps, the
# root, the reciprocal, h, and two products are 8 more.
ERR = 53 * U


def check_int8(q, scales, y, err):
    """y: in 64 bits, `err` (relative) off. Both the largest and the element may be, and the quotient and product are rounded."""
    amax = y.abs().amax(-1)
    want = torch.where(amax > 0, torch.clamp(amax / 127, min=2.0 ** -126), 0.0)
    assert ((scales.double() - want).abs() <= (err + 2 * U) * want).all()
    steps = torch.where(want > 0, 1 / want, 0.0)[:, None] * y
    off = (q.double() - steps).abs()
    assert (off <= 0.5 + 127 * (2 * err + 4 * U)).all(), off.max().item()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,hidden", SIZES)
def test_norm(buf, tokens, hidden, dtype):
    for weight, residual, int8, norm in (("same", True, True, True), ("fp32", False, True, False), (None, True, False, True), ("same", False, False, True)):
        g, x, w = make(tokens, hidden, dtype, tokens + hidden, weight)
        r = torch.randn((tokens, hidden), device="cuda", generator=g).to(dtype) if residual else None
        y, q, scales, total = buf.rms_norm(x, w, r, EPS, int8, norm)
        assert (y is None) == (not norm) and (q is None) == (scales is None) == (not int8) and (total is None) == (not residual)
        h = x.double() + (r.double() if residual else 0)
        if residual:
            close(total, h, U * h.abs(), dtype)
        want = norm64(h, w)
        # where x and the residual cancel, the sum's own rounding is what it is
        if norm:
            close(y, want, ERR * want.abs(), dtype)
        if int8:
            assert q.dtype == torch.int8 and scales.dtype == torch.float32 and scales.shape == (tokens,)
            check_int8(q, scales, want, ERR)


# from 2049 rows on a row has half as many lanes and twice as many pieces
MANY_ROWS = [(2049, 1531), (3000, 2100), (2500, 4104), (4096, 7168), (2048, 7168), (2200, 8200), (2049, 16392), (2100, 33000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,hidden", MANY_ROWS)
def test_norm_of_many_rows(buf, tokens, hidden, dtype):
    for weight, residual, int8, norm in (("same", True, True, True), ("fp32", False, True, False)):
        g, x, w = make(tokens, hidden, dtype, tokens + hidden, weight)
        r = torch.randn((tokens, hidden), device="cuda", generator=g).to(dtype) if residual else None
        y, q, scales, total = buf.rms_norm(x, w, r, EPS, int8, norm)
        h = x.double() + (r.double() if residual else 0)
        if residual:
            close(total, h, U * h.abs(), dtype)
        want = norm64(h, w)
        if norm:
            close(y, want, ERR * want.abs(), dtype)
        check_int8(q, scales, want, ERR)


def test_more_rounds_of_rows_than_one(buf):
    """A launch has 2^20 workgroups at most: rows past them, and those that the same workgroups had before, are what they are in a call of their own. Rows of
    three waves, one to a workgroup, and of one wave, four to a workgroup."""
    for rows, width in (((1 << 20) + 40000, 1032), ((1 << 22) + 90000, 72)):
        more = rows % (1 << 20)
        x = torch.empty((rows, width), device="cuda", dtype=torch.bfloat16).normal_()
        x *= torch.exp2((torch.arange(rows, device="cuda") * 7 % 13 - 6).to(torch.bfloat16))[:, None]      # neighbours of other sizes
        w = torch.randn((width,), device="cuda").to(torch.bfloat16)
        parts = (slice(0, more), slice(rows - 2 * more, rows))
        got = buf.rms_norm(x, w, None, EPS, True, True)
        for part in parts:
            want = buf.rms_norm(x[part].clone(), w, None, EPS, True, True)
            assert all(torch.equal(a[part], b) for a, b in zip(got[:3], want[:3]))
        del got, want
        for act in ("none", "silu"):
            got = buf.quantize_rows(x, activation=act)
            for part in parts:
                assert all(torch.equal(a[part], b) for a, b in zip(got, buf.quantize_rows(x[part].clone(), activation=act)))
            del got
        count = rows - more // 2
        got = buf.quantize_rows(x, torch.tensor([count], device="cuda"))
        part = slice(rows - 2 * more, count)
        assert all(torch.equal(a[part], b) for a, b in zip(got, buf.quantize_rows(x[part].clone())))
        del x, got
    rows = (1 << 20) + 20000
    x = torch.empty((rows, 2064), device="cuda", dtype=torch.bfloat16).normal_()
    got = buf.quantize_rows(x, activation="swiglu")
    for part in (slice(0, 20000), slice(rows - 40000, rows)):
        assert all(torch.equal(a[part], b) for a, b in zip(got, buf.quantize_rows(x[part].clone(), activation="swiglu")))


def test_eps_and_the_norms_own_types(buf):
    for eps in (1e-12, 1e-5, 1.0, 1e6):
        g, x, w = make(5, 640, torch.float32, 3)
        x[1] *= 1e-6
        want = norm64(x.double(), w, float(torch.tensor(eps, dtype=torch.float32)))
        close(buf.rms_norm(x, w, eps=eps)[0], want, ERR * want.abs(), torch.float32)


def test_rows_of_nothing_sound(buf):
    """zeros have the scale 0, infinities and NaN reach their own row's results and no other's, in every output"""
    for dtype in TYPES:
        for hidden in (96, 1531, 7168):
            g, x, w = make(9, hidden, dtype, 5)
            r = torch.randn((9, hidden), device="cuda", generator=g).to(dtype)
            clean = buf.rms_norm(x, w, r, EPS, True, True)
            x2, r2 = x.clone(), r.clone()
            x2[1], r2[1] = 0, 0
            x2[3, hidden - 1] = float("nan")
            r2[5, 0] = float("inf")
            x2[7, 17], r2[7, 17] = float("inf"), float("-inf")
            y, q, scales, total = buf.rms_norm(x2, w, r2, EPS, True, True)
            for row in (0, 2, 4, 6, 8):
                for a, b in zip((y, q, scales, total), clean):
                    assert torch.equal(a[row], b[row])
            assert (y[1] == 0).all() and (q[1] == 0).all() and scales[1] == 0
            assert torch.isnan(scales[[3, 5, 7]]).all() and torch.isnan(y[[3, 7]]).all() and torch.isnan(y[5, 0])
            # a NaN or an infinity that comes from the weight
            w2 = w.clone()
            w2[hidden // 2] = float("nan")
            assert torch.isnan(buf.rms_norm(x, w2, None, EPS, True, False)[2]).all()
            z = x.clone()
            z[4, hidden // 3], z[6, hidden - 1] = float("inf"), float("nan")
            q, scales = buf.quantize_rows(z)
            assert torch.isnan(scales[[4, 6]]).all() and torch.isfinite(scales[[0, 1, 2, 3, 5, 7, 8]]).all()


def test_small_rows_keep_a_normal_scale(buf):
    """magnitudes whose 127th part is no normal number: the scale stays at 2^-126, and the elements within half of it"""
    x = torch.randn((6, 200), device="cuda") * torch.tensor([[2.0 ** -118], [2.0 ** -120], [2.0 ** -126], [2.0 ** -140], [2.0 ** -149], [1.0]], device="cuda")
    q, scales = buf.quantize_rows(x)
    check_int8(q, scales, x.double(), 0.0)
    assert (scales >= 2.0 ** -126).all() and (q[0].abs() > 20).any()
    y, q, scales, _ = buf.rms_norm(x, None, None, 1.0, True, True)
    check_int8(q[:5], scales[:5], x[:5].double(), 1e-6)


# ---- gradients -----------------------------------------------------------------------------------------------------------

def backward_case(buf, tokens, hidden, dtype, weight, total, wgrad, seed=0):
    g, x, w = make(tokens, hidden, dtype, seed + tokens + hidden, weight)
    grad = torch.randn((tokens, hidden), device="cuda", generator=g).to(dtype)
    gt = torch.randn((tokens, hidden), device="cuda", generator=g).to(dtype) if total else None
    gx, gw = buf.rms_norm_backward(grad, x, w, gt, EPS, wgrad)
    h, wd = x.double(), torch.ones((hidden,), device="cuda", dtype=torch.float64) if w is None else w.double()
    r = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
    n, d = h * r, grad.double() * wd
    mean = (d * n).mean(-1, keepdim=True)
    want = r * (d - n * mean)
    # r is 53 steps off (see above); the sum of d h is one chain of 90 steps of its terms' sizes, times r; then half a dozen roundings
    size = r * (d.abs() + n.abs() * (d * n).abs().mean(-1, keepdim=True))
    err = 260 * U * size
    if total:
        want = want + gt.double()
        err = err + U * want.abs()
    close(gx, want, err, dtype)
    terms = grad.double() * n
    # a lane's rows, a thread's partial sums, sixteen threads' and n's own steps
    steps = (tokens / 1024 + 1) + 256 + 16 + 56
    close(gw, terms.sum(0), steps * U * terms.abs().sum(0), wgrad or dtype)
    return gx, gw


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,hidden", SIZES + [(5000, 64), (2100, 1030), (1100, 2048), (0, 72), (96, 512), (97, 512), (77, 64), (41, 1025), (12, 4090), (13, 4090), (18, 2000)])
def test_gradients(buf, tokens, hidden, dtype):
    backward_case(buf, tokens, hidden, dtype, "same", True, None)
    backward_case(buf, tokens, hidden, dtype, "fp32", False, torch.float32)
    backward_case(buf, tokens, hidden, dtype, None, True, torch.float32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,hidden", [(700, 7168), (1100, 4104), (3000, 4104), (600, 8200), (1500, 12000), (600, 16392), (900, 24001), (300, 40000), (600, 33000)])
def test_gradients_of_several_rows_to_a_workgroup_and_pieces_to_a_lane(buf, tokens, hidden, dtype):
    """two, four and eight pieces, the latter in 512 lanes and in 1024, over rows that a workgroup takes one after the other"""
    backward_case(buf, tokens, hidden, dtype, "same", True, None)
    backward_case(buf, tokens, hidden, dtype, "fp32", False, torch.float32)


def test_what_is_not_asked_for(buf):
    g, x, w = make(50, 640, torch.bfloat16, 1)
    grad = torch.randn_like(x)
    gx, gw = buf.rms_norm_backward(grad, x, w)
    only, none = buf.rms_norm_backward(grad, x, w, need_weight=False)
    assert none is None and torch.equal(only, gx)


def test_gradients_against_differences(buf):
    """d/dx, d/dresidual and d/dweight of <a, y> + <b, total> by steps of the forward call in 32 bits"""
    tokens, hidden, step = 3, 24, 2.0 ** -6
    g, x, w = make(tokens, hidden, torch.float32, 2)
    x, r = torch.randn((2, tokens, hidden), device="cuda", generator=g)
    a, b = torch.randn((2, tokens, hidden), device="cuda", generator=g)

    def f(x, r, w):
        y, _, _, total = buf.rms_norm(x, w, r, EPS)
        return ((y.double() * a.double()).sum() + (total.double() * b.double()).sum()).item()

    total = buf.rms_norm(x, w, r, EPS)[3]
    gx, gw = buf.rms_norm_backward(a, total, w, b, EPS)
    scale = (1 / total.double().pow(2).mean(-1).sqrt()).max().item()
    for i, j in ((0, 0), (2, 23), (1, 7), (2, 5)):
        for t, grad in ((x, gx[i, j]), (r, gx[i, j]), (w, gw[j])):
            at = (j,) if t.dim() == 1 else (i, j)
            up, down = t.clone(), t.clone()
            up[at] += step
            down[at] -= step
            diff = (f(*[up if t is v else v for v in (x, r, w)]) - f(*[down if t is v else v for v in (x, r, w)])) / (2 * step)
            # y's third derivative in an element is below 15 scale^3 |w|, over all terms below sqrt(hidden) |a|; 32 bits of y of size 5 over a step
            size = a.norm().item() * w.abs().max().item() * 15 * scale ** 3
            assert abs(diff - grad.item()) <= step ** 2 / 6 * size + 60 * U * 5 * a.abs().sum().item() / step


# ---- activations in int8 -------------------------------------------------------------------------------------------------

def act64(z, name):
    F = torch.nn.functional
    return {"none": lambda: z, "relu": lambda: torch.relu(z), "silu": lambda: F.silu(z), "gelu": lambda: F.gelu(z),
            "gelu_tanh": lambda: F.gelu(z, approximate="tanh"),
            "swiglu": lambda: F.silu(z[:, :z.shape[1] // 2]) * z[:, z.shape[1] // 2:]}[name]()


def quantize_case(buf, rows, width, dtype, act, counts=None, count_dtype=torch.int32):
    g = torch.Generator(device="cuda").manual_seed(rows + width)
    x = (torch.randn((rows, width), device="cuda", generator=g) * torch.exp(torch.randn((rows, 1), device="cuda", generator=g))).to(dtype)
    ct = None if counts is None else torch.tensor(counts, device="cuda", dtype=count_dtype)
    q, scales = buf.quantize_rows(x, ct, act)
    n = rows
    if counts is not None:
        n = 0
        for c in counts:
            n = min(rows, n + max(0, min(int(c), rows)))
    y = act64(x[:n].double(), act)
    amax = y.abs().amax(-1) if n else y.new_zeros((0,))
    # an activation is a dozen operations of 32 bits, and gelu's tail or tanh a step of one, times z: far below zero its relative error is more, but not that of the
    # row's largest. In steps of the scale:
    z = x[:n].double().abs()
    z = z[:, :z.shape[1] // 2] if act == "swiglu" else z
    err = 0 if act == "none" else 16 * U * y.abs() + (8 * U * z if act.startswith("gelu") else 0)
    worst = err.amax(-1) if act != "none" and n else 0 * amax
    want = torch.where(amax > 0, torch.clamp(amax / 127, min=2.0 ** -126), 0.0)
    assert ((scales[:n].double() - want).abs() <= worst / 127 + 2 * U * want).all()
    steps = torch.where(want > 0, 1 / want, 0.0)[:, None]
    assert ((q[:n].double() - y * steps).abs() <= 0.5 + 2 * (worst[:, None] * steps) + 127 * 4 * U).all()
    return x, q, scales, n


@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("rows,width", [(1, 2), (3, 14), (5, 64), (2, 130), (9, 1024), (4, 1030), (300, 2048), (3, 4096), (7, 6130), (2, 65536)])
def test_quantize(buf, rows, width, act):
    for dtype in TYPES:
        quantize_case(buf, rows, width, dtype, act)


@pytest.mark.parametrize("rows,width,act", [(2049, 1030, "none"), (3000, 2100, "silu"), (2100, 6130, "swiglu"), (4096, 4096, "relu"), (2500, 16392, "gelu"), (2048, 16384, "swiglu"),
                                            (2049, 33000, "none"), (2100, 65536, "swiglu"), (2500, 8200, "gelu_tanh")])
def test_quantize_many_rows(buf, rows, width, act):
    for dtype in TYPES:
        quantize_case(buf, rows, width, dtype, act)


@pytest.mark.parametrize("counts", [[0, 0, 0], [5, 0, 30], [40, 20, 0], [-3, 10, 1 << 30], [1], [0] * 1000 + [7] * 24])
def test_quantized_rows_of_nobody_stay(buf, counts):
    for act, width in (("swiglu", 528), ("silu", 130)):
        for dtype in (torch.int32, torch.int64):
            quantize_case(buf, 50, width, torch.bfloat16, act, counts, dtype)
        cols = width // 2 if act == "swiglu" else width
        x = torch.randn((50, width), device="cuda").to(torch.bfloat16)
        n = 0
        for c in counts:
            n = min(50, n + max(0, min(c, 50)))
        x[n:] = float("nan")
        q, scales = torch.full((50, cols), 77, device="cuda", dtype=torch.int8), torch.full((50,), 77.0, device="cuda")
        ct = torch.tensor(counts, device="cuda", dtype=torch.int32)
        d = capi.QuantizeRows(ct.data_ptr(), 0, capi.DT_BF16, capi.ACTIVATIONS[act], 50, width, len(counts))
        assert capi.load().zbalhip_quantize_rows(ctypes.byref(d), x.data_ptr(), q.data_ptr(), scales.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
        assert (q[n:] == 77).all() and (scales[n:] == 77).all() and torch.isfinite(scales[:n]).all()


# ---- calls ---------------------------------------------------------------------------------------------------------------

def test_empty_batches(buf):
    x = torch.empty((0, 64), device="cuda", dtype=torch.bfloat16)
    w = torch.ones((64,), device="cuda", dtype=torch.bfloat16)
    y, q, scales, total = buf.rms_norm(x, w, x, EPS, True)
    assert y.shape == q.shape == total.shape == (0, 64) and scales.shape == (0,)
    gx, gw = buf.rms_norm_backward(x, x, w)
    assert gx.shape == (0, 64) and (gw == 0).all()
    q, scales = buf.quantize_rows(x, activation="swiglu")
    assert q.shape == (0, 32) and scales.shape == (0,)


def test_past_32_bits_of_offset(buf):
    """more than 2^31 elements: the last rows are what they are on their own"""
    tokens, hidden = 33000, 65536
    x = torch.empty((tokens, hidden), device="cuda", dtype=torch.bfloat16).normal_()
    w = torch.randn((hidden,), device="cuda").to(torch.bfloat16)
    y, q, scales, _ = buf.rms_norm(x, w, None, EPS, True, True)
    for rows in (slice(0, 2), slice(tokens - 2, tokens)):
        a = buf.rms_norm(x[rows].clone(), w, None, EPS, True, True)
        assert torch.equal(y[rows], a[0]) and torch.equal(q[rows], a[1]) and torch.equal(scales[rows], a[2])
    del y, q
    gx = buf.rms_norm_backward(x, x, w, need_weight=False)[0]
    assert torch.equal(gx[-2:], buf.rms_norm_backward(x[-2:].clone(), x[-2:].clone(), w, need_weight=False)[0])
    del gx
    q, scales = buf.quantize_rows(x)
    a = buf.quantize_rows(x[-2:].clone())
    assert torch.equal(q[-2:], a[0]) and torch.equal(scales[-2:], a[1])


@pytest.mark.parametrize("tokens,hidden", [(1, 7168), (300, 520), (3000, 1031)])
def test_the_same_every_time_and_captured(buf, tokens, hidden):
    g, x, w = make(tokens, hidden, torch.bfloat16, 7)
    r, x2 = torch.randn_like(x), torch.randn_like(x)
    xin = x.clone()

    def step(x):
        y, q, scales, total = buf.rms_norm(x, w, r, EPS, True)
        return (y, q, scales, total) + tuple(buf.rms_norm_backward(y, total, w, x, EPS, torch.float32)) + tuple(buf.quantize_rows(y, activation="silu"))

    want = step(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(xin)
        aside = step(x)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(aside, want))
    graph, again = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(xin)
    with torch.cuda.graph(again):
        got2 = step(xin)
    for src in (x, x2, x):
        xin.copy_(src)
        graph.replay()
        again.replay()
        want = step(src)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a, b) for a, b in zip(got2, want))


def test_the_sum_in_place(buf):
    """through the C entry: the next residual in the memory of the last one"""
    g, x, w = make(40, 1000, torch.bfloat16, 8)
    r = torch.randn_like(x)
    want = buf.rms_norm(x, w, r, EPS)
    for on in (r.clone(), x.clone()):
        y = torch.empty_like(x)
        xi, ri = (x, on) if not torch.equal(on, x) else (on, r)
        t = capi.tensor_info
        code = capi.load().zbal_moe_rms_norm(t(xi), t(w), t(ri), EPS, t(y), t(on), None, None, buf.runtime.comm, capi.stream_ptr(), 0)
        assert code == 0
        assert torch.equal(y, want[0]) and torch.equal(on, want[3])


@pytest.mark.parametrize("tokens,hidden", [(3, 600), (700, 4104), (2100, 520)])
def test_the_gradient_in_place(buf, tokens, hidden):
    """through the kernel's entry: the rows' gradient in the memory of the one that comes in, or of the sum's"""
    g, x, w = make(tokens, hidden, torch.bfloat16, 9)
    grad, total = torch.randn_like(x), torch.randn_like(x)
    gx, gw = buf.rms_norm_backward(grad, x, w, total, EPS, torch.float32)
    lib, stream = capi.load(), torch.cuda.current_stream().cuda_stream
    d = capi.RmsNorm(x.data_ptr(), None, w.data_ptr(), capi.DT_BF16, 0, tokens, hidden, EPS)
    size = lib.zbalhip_rms_norm_backward_workspace(ctypes.byref(d))
    ws = torch.empty((max(size, 16),), dtype=torch.uint8, device="cuda")
    for on_grad in (True, False):
        a, b, got = grad.clone(), total.clone(), torch.empty_like(gw)
        on = a if on_grad else b
        assert lib.zbalhip_rms_norm_backward(ctypes.byref(d), a.data_ptr(), b.data_ptr(), on.data_ptr(), got.data_ptr(), 1, ws.data_ptr(), size, stream) == 0
        assert torch.equal(on, gx) and torch.equal(got, gw)


def test_refusals(buf):
    bf = lambda *s: torch.ones(s, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    x, w = bf(4, 64), bf(64)
    wide = bf(4, 128)
    for call in (lambda: buf.rms_norm(wide[:, :64], w), lambda: buf.rms_norm(bf(64), w), lambda: buf.rms_norm(x, bf(63)), lambda: buf.rms_norm(x, bf(1, 64)),
                 lambda: buf.rms_norm(x, w, bf(3, 64)), lambda: buf.rms_norm(x, w, x.cpu()), lambda: buf.rms_norm_backward(bf(4, 63), x, w),
                 lambda: buf.rms_norm_backward(x, x, w, bf(4, 65)), lambda: buf.rms_norm_backward(x, x, w, weight_grad_dtype=torch.float16),
                 lambda: buf.quantize_rows(wide[:, :64]), lambda: buf.quantize_rows(bf(64)), lambda: buf.quantize_rows(x, activation="tanh")):
        with pytest.raises(ValueError):
            call()
    for call, text in ((lambda: buf.rms_norm(x, w.half()), "weight"), (lambda: buf.rms_norm(x, w, x.float()), "residual"), (lambda: buf.rms_norm(x, w, eps=0.0), "eps"),
                       (lambda: buf.rms_norm(x, w, eps=float("nan")), "eps"), (lambda: buf.rms_norm(x, w, eps=-1.0), "eps"), (lambda: buf.rms_norm(x, w, eps=1e300), "eps"),
                       (lambda: buf.rms_norm(x, w, need_norm=False), "no output"), (lambda: buf.rms_norm(x.to(torch.int8), None), "type"), (lambda: buf.rms_norm(bf(2, 65537)), "out of range"),
                       (lambda: buf.rms_norm(bf(4, 65)[1:], None), "aligned"), (lambda: buf.rms_norm_backward(x.float(), x, w), "grad"),
                       (lambda: buf.rms_norm_backward(x, x, w, x.half()), "gradTotal"), (lambda: buf.quantize_rows(bf(4, 63), activation="swiglu"), "even"),
                       (lambda: buf.quantize_rows(x, torch.ones((1025,), device="cuda", dtype=torch.int32)), "experts"),
                       (lambda: buf.quantize_rows(x, torch.ones((2,), device="cuda")), "tokensPerExpert"), (lambda: buf.quantize_rows(bf(2, 65538)), "out of range")):
        with pytest.raises(capi.ZbalError, match=text):
            call()
    with pytest.raises(TypeError):
        buf.rms_norm_backward(None, x, w)

"""The experts' products and their gradients against plain forms in 64 bits: one row to many, sizes that no tile, chunk or register divides, both
weight orders, every activation and part of the epilogue, experts without rows, counts that are wrong, rows that are nobody's."""
import ctypes

import pytest
import torch

from memfabric_hybrid_amd import capi
from memfabric_hybrid_amd.buffer import Buffer

pytestmark = pytest.mark.gpu
ACTIVATIONS = ["none", "relu", "silu", "gelu", "gelu_tanh", "swiglu"]
U = 2.0 ** -24


@pytest.fixture(scope="module")
def buf():
    b = Buffer()
    yield b
    torch.cuda.synchronize()
    b.close()


def act64(z, name):
    F = torch.nn.functional
    return {"none": lambda: z, "relu": lambda: torch.relu(z), "silu": lambda: F.silu(z), "gelu": lambda: F.gelu(z),
            "gelu_tanh": lambda: F.gelu(z, approximate="tanh"),
            "swiglu": lambda: F.silu(z[:, :z.shape[1] // 2]) * z[:, z.shape[1] // 2:]}[name]()


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def spans(counts, rows):
    out, at = [], 0
    for c in counts:
        end = min(rows, at + max(0, min(int(c), rows)))
        out.append((at, end))
        at = end
    return out


def make(rows, E, K, N, dtype, seed, transposed=False, counts=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, K), device="cuda", generator=g).to(dtype)
    w = (torch.randn((E, N, K) if transposed else (E, K, N), device="cuda", generator=g) * K ** -0.5).to(dtype)
    if counts is None:
        p = torch.rand((E,), generator=torch.Generator().manual_seed(seed)) + 0.05
        if E > 3:
            p[1] = 0.0
        counts = torch.bincount(torch.multinomial(p, rows, replacement=True, generator=torch.Generator().manual_seed(seed)), minlength=E).tolist() \
            if rows else [0] * E
    return g, x, w, counts


def products(x, w, counts, transposed):
    """(z, the sum of the products' magnitudes) in 64 bits; rows of nobody are left out at the end"""
    zs, mags = [], []
    for e, (a, b) in enumerate(spans(counts, x.shape[0])):
        we = w[e].double().t() if transposed else w[e].double()
        zs.append(x[a:b].double() @ we)
        mags.append(x[a:b].double().abs() @ we.abs())
    return torch.cat(zs), torch.cat(mags)


def forward_case(buf, rows, E, K, N, dtype, act="none", bias=None, residual=False, out_dtype=None, transposed=False, preact=False, counts=None, seed=0,
                 count_dtype=torch.int32):
    g, x, w, counts = make(rows, E, K, N, dtype, seed + rows + K + N, transposed, counts)
    cols = N // 2 if act == "swiglu" else N
    od = out_dtype or dtype
    b = torch.randn((E, N), device="cuda", generator=g).to(bias) if bias is not None else None
    r = torch.randn((rows, cols), device="cuda", generator=g).to(od) if residual else None
    out = torch.full((rows, cols), 77.0, device="cuda", dtype=od)
    ct = None if counts == "all" else torch.tensor(counts, dtype=count_dtype, device="cuda")
    if counts == "all":
        counts = [rows]
    got = buf.expert_linear(x, w, ct, b, act, r, out_dtype, transposed, preact, out)
    got, gotz = got if preact else (got, None)
    assert got.data_ptr() == out.data_ptr()
    z, mag = products(x, w, counts, transposed)
    n = z.shape[0]
    err = (K + 2) * U * mag
    if b is not None:
        be = torch.cat([b[e].double().expand(q - p, N) for e, (p, q) in enumerate(spans(counts, rows))])
        z = z + be
        err = err + U * z.abs()
    y = act64(z, act)
    if act == "swiglu":
        h = N // 2
        ge, ue, gate, up = err[:, :h], err[:, h:], z[:, :h], z[:, h:]
        err_y = 1.1 * ge * (up.abs() + ue) + act64(gate, "silu").abs() * ue
    else:
        err_y = 1.13 * err                       # no slope is steeper
    # an activation is a dozen operations of 32 bits; gelu's 1 + erf or tanh loses a step of one, times z
    err_y = err_y + 16 * U * y.abs() + (8 * U * z.abs()[:, :cols] if act.startswith("gelu") else 0)
    if r is not None:
        y = y + r[:n].double()
        err_y = err_y + U * y.abs()
    tiny = 2.0 ** -25 if od == torch.float16 else 1e-37
    far = (got[:n].double() - y).abs() - (half_step(od) * (y.abs() + err_y) + err_y + tiny)
    assert far.max().item() <= 0 if far.numel() else True, (far.max().item(), (far > 0).sum().item())
    assert (out[n:] == 77.0).all()
    if preact:
        bad = (gotz[:n].double() - z).abs() > half_step(dtype) * (z.abs() + err) + err + tiny
        assert not bad.any()
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("rows,K,N", [(1, 1, 1), (1, 64, 128), (2, 7, 9), (3, 65, 130), (15, 200, 72), (16, 256, 128), (17, 1001, 515), (64, 512, 384),
                                      (127, 96, 1000), (129, 1024, 264), (300, 333, 777), (513, 2048, 520), (1, 7168, 256), (2, 2048, 4096)])
def test_dense(buf, rows, K, N, dtype, transposed):
    forward_case(buf, rows, 1, K, N, dtype, transposed=transposed, counts="all")


@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("rows,K,N", [(1, 320, 256), (5, 104, 40), (33, 130, 66), (200, 512, 512), (700, 264, 1032)])
def test_epilogues(buf, rows, K, N, act):
    forward_case(buf, rows, 1, K, N, torch.bfloat16, act, counts="all", transposed=rows % 2 == 0)
    forward_case(buf, rows, 1, K, N, torch.float16, act, bias=torch.float32, residual=True, preact=True, counts="all")
    forward_case(buf, rows, 1, K, N, torch.bfloat16, act, bias=torch.bfloat16, residual=True, out_dtype=torch.float32, counts="all")


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("rows,E,K,N,act", [(16, 32, 256, 256, "swiglu"), (8, 64, 200, 130, "silu"), (100, 4, 96, 200, "none"), (333, 7, 128, 256, "swiglu"),
                                            (700, 65, 64, 72, "gelu"), (3000, 8, 320, 520, "swiglu"), (2000, 130, 128, 128, "none"), (40, 1024, 64, 64, "relu"),
                                            (9000, 5, 256, 384, "none")])
def test_grouped(buf, rows, E, K, N, act, transposed):
    forward_case(buf, rows, E, K, N, torch.bfloat16, act, transposed=transposed, bias=torch.float32, count_dtype=torch.int64)
    forward_case(buf, rows, E, K, N, torch.float16, act, transposed=transposed, residual=True)


# sizes that are cut into every kind of tiles and parts, for many workgroups a CU; the last rows, columns and k of each are ragged
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("rows,E,K,N", [(8200, 1, 136, 4104), (4033, 64, 200, 4104), (1280, 20, 136, 2056), (1200, 40, 72, 1928), (900, 3, 264, 1160),
                                        (4100, 1, 2056, 264), (70, 1, 2120, 520), (2100, 1, 4097, 250), (1030, 2, 266, 2050), (200, 60, 130, 1026), (5000, 3, 131, 1029),
                                        (1, 1, 4104, 2056), (1, 1, 1104, 4104), (17, 2, 2056, 4104), (5, 3, 1032, 72), (3, 5, 1048, 80)])
def test_every_cut(buf, rows, E, K, N, transposed):
    counts = "all" if E == 1 else None
    forward_case(buf, rows, E, K, N, torch.bfloat16, transposed=transposed, counts=counts, out_dtype=torch.float32)
    forward_case(buf, rows, E, K, N, torch.float16, "silu", bias=torch.float16, residual=True, preact=True, transposed=transposed, counts=counts, seed=1)
    if N % 2 == 0:
        forward_case(buf, rows, E, K, N, torch.bfloat16, "swiglu", transposed=transposed, counts=counts, seed=2)
        forward_case(buf, rows, E, K, N, torch.float16, "swiglu", bias=torch.float32, residual=True, preact=True, transposed=transposed, counts=counts, seed=3)


@pytest.mark.parametrize("counts", [[0, 0, 0, 0], [0, 0, 0, 50], [50, 0, 0, 0], [10, 10, 10, 10], [-5, 20, -(1 << 31), 10], [30, 1 << 30, 7, (1 << 31) - 1],
                                    [1, 47, 1, 1], [20, 20, 20, 20]])
@pytest.mark.parametrize("N", [128, 130])
def test_counts(buf, counts, N):
    """empty experts, rows of nobody, negative counts (none), counts past the last row (cut off there)"""
    forward_case(buf, 50, 4, 128, N, torch.bfloat16, "silu", counts=counts)
    forward_case(buf, 50, 4, 128, N, torch.bfloat16, "none", counts=counts, count_dtype=torch.int64)


def test_counts_past_32_bits(buf):
    forward_case(buf, 300, 3, 64, 64, torch.bfloat16, counts=[100, 1 << 40, 5], count_dtype=torch.int64)
    forward_case(buf, 300, 3, 64, 64, torch.bfloat16, counts=[100, -(1 << 40), 50], count_dtype=torch.int64)


def test_one_row_does_not_see_the_others(buf):
    """infinities and NaN of a row, an expert and rows of nobody stay where they are"""
    for rows, E, K, N in ((48, 3, 128, 128), (600, 3, 136, 264), (600, 3, 133, 261)):
        g, x, w, counts = make(rows, E, K, N, torch.bfloat16, 1, counts=[rows // 3, rows // 3 - 4, rows // 3 - 6])
        ct = torch.tensor(counts, device="cuda")
        clean = buf.expert_linear(x, w, ct)
        n = sum(counts)
        x2, w2 = x.clone(), w.clone()
        x2[3], x2[n:] = float("nan"), float("inf")
        w2[1] = float("nan")
        dirty = buf.expert_linear(x2, w2, ct)
        same = [r for r in range(n) if r != 3 and not counts[0] <= r < counts[0] + counts[1]]
        assert torch.equal(clean[same], dirty[same]) and torch.isnan(dirty[3]).all()
        assert torch.isnan(dirty[counts[0]:counts[0] + counts[1]]).all()
        dw = buf.expert_linear_backward(clean, x2, w, ct, need_x=False)[1]
        dwc = buf.expert_linear_backward(clean, x, w, ct, need_x=False)[1]
        assert torch.equal(dw[1:], dwc[1:]) and torch.isnan(dw[0]).all()


# ---- gradients -----------------------------------------------------------------------------------------------------------

def backward_case(buf, rows, E, K, N, dtype, act="none", bias=True, transposed=False, wgrad=None, grad_dtype=None, counts=None, seed=0):
    g, x, w, counts = make(rows, E, K, N, dtype, seed + rows + K + N, transposed, counts)
    cols = N // 2 if act == "swiglu" else N
    dy = torch.randn((rows, cols), device="cuda", generator=g).to(grad_dtype or dtype)
    z = torch.randn((rows, N), device="cuda", generator=g).to(dtype) if act != "none" else None
    ct = None if counts == "all" else torch.tensor(counts, dtype=torch.int32, device="cuda")
    counts = [rows] if counts == "all" else counts
    gx, gw, gb, gz = buf.expert_linear_backward(dy, x, w, ct, act, z, transposed, bias, wgrad)
    wt = wgrad or dtype
    assert gx.dtype == dtype and gw.dtype == wt and gw.shape == w.shape and (gb is None) == (not bias)
    sp = spans(counts, rows)
    n = sp[-1][1]
    d = dy.double()
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-37
    if act != "none":
        zz = z.double().requires_grad_()
        act64(zz, act).backward(d)
        d = zz.grad
        d2, z2 = dy.double().abs(), z.double()
        # slopes are up to 1.13, made of a dozen terms of 32 bits; gelu's have terms of z
        size = 1.2 * (torch.cat([d2 * z2[:, cols:].abs(), d2 * z2[:, :cols].abs()], 1) if act == "swiglu" else d2 * (1 + z2.abs()))
        assert ((gz[:n].double() - d[:n]).abs() <= half_step(dtype) * d[:n].abs() + 24 * U * (size + d2.repeat(1, N // cols))[:n] + tiny).all()
    elif gz is not None:
        assert torch.equal(gz[:n], dy[:n].to(dtype))
    dz = (gz if gz is not None else dy)[:n].double()         # the tensor that the products take
    for e, (a, b) in enumerate(sp):
        we, xe, de = w[e].double(), x[a:b].double(), dz[a:b]
        wt_e = we if transposed else we.t()
        want, mag = de @ wt_e, de.abs() @ wt_e.abs()
        assert ((gx[a:b].double() - want).abs() <= half_step(dtype) * want.abs() + 1.01 * (N + 2) * U * mag + tiny).all()
        l, r = (de, xe) if transposed else (xe, de)
        want, mag = l.t() @ r, l.abs().t() @ r.abs()
        assert ((gw[e].double() - want).abs() <= half_step(wt) * want.abs() + 1.01 * (b - a + 2) * U * mag + tiny).all(), e
        if bias:
            want, mag = de.sum(0), de.abs().sum(0)
            got = (gb[e] if gb.dim() == 2 else gb).double()
            assert ((got - want).abs() <= half_step(wt) * want.abs() + 1.01 * (b - a + 2) * U * mag + tiny).all()
    return gx, gw, gb, gz


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("rows,E,K,N", [(1, 1, 1, 1), (1, 1, 128, 128), (3, 1, 9, 7), (65, 1, 72, 200), (200, 1, 264, 520), (333, 1, 515, 130), (1000, 1, 1024, 256),
                                        (50, 8, 64, 128), (777, 5, 136, 264), (900, 9, 130, 66), (4000, 4, 320, 512)])
def test_gradients(buf, rows, E, K, N, transposed):
    backward_case(buf, rows, E, K, N, torch.bfloat16, transposed=transposed)
    backward_case(buf, rows, E, K, N, torch.float16, transposed=transposed, wgrad=torch.float32)


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("rows,E,K,N", [(2049, 1, 1544, 1536), (1030, 1, 1216, 3336), (1030, 1, 3336, 1216), (8201, 1, 256, 264), (8200, 1, 250, 129), (3000, 3, 1040, 1288), (2500, 3, 1031, 1290),
                                        (2049, 20, 520, 776), (129, 1, 2056, 4104), (4941, 8, 8, 5640)])
def test_gradients_of_every_cut(buf, rows, E, K, N, transposed):
    counts = "all" if E == 1 else None
    backward_case(buf, rows, E, K, N, torch.bfloat16, transposed=transposed, counts=counts)
    backward_case(buf, rows, E, K, N, torch.float16, "silu", transposed=transposed, counts=counts, wgrad=torch.float32, grad_dtype=torch.float32)
    backward_case(buf, rows, E, K, N, torch.bfloat16, transposed=transposed, counts=counts, bias=False, seed=1)


@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("rows,E,K,N", [(7, 1, 64, 40), (130, 3, 200, 66), (600, 4, 256, 512)])
def test_gradients_of_activations(buf, rows, E, K, N, act):
    backward_case(buf, rows, E, K, N, torch.bfloat16, act)
    backward_case(buf, rows, E, K, N, torch.float16, act, wgrad=torch.float32, transposed=True)
    backward_case(buf, rows, E, K, N, torch.bfloat16, act, grad_dtype=torch.float32, bias=False)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_slopes_far_out(buf, act):
    """nothing becomes infinite or no number where the activation has long been straight"""
    z = torch.tensor([[-3e38, -1e30, -1e20, -300.0, -40.0, -12.0, 0.0, -0.0, 12.0, 40.0, 300.0, 1e20, 1e30, 3e38, 1e-30, -1e-30]], device="cuda").to(torch.bfloat16)
    x, w = torch.zeros((1, 8), device="cuda", dtype=torch.bfloat16), torch.zeros((8, 16), device="cuda", dtype=torch.bfloat16)
    gz = buf.expert_linear_backward(torch.ones_like(z), x, w, activation=act, preact=z)[3]
    want = torch.tensor([[0.0] * 6 + [0.5] * 2 + [1.0] * 6 + [0.5] * 2], device="cuda")
    assert (gz.float() - want).abs().max() < 2.0 ** -9 + 13 * 7e-6        # a rounding; silu's slope at -12 is -11 exp(-12)
    y = buf.expert_linear(x, w, bias=z[0].float(), activation=act)
    exact = act64(z.double(), act)
    assert ((y.double() - exact).abs() <= 2.0 ** -8 * exact.abs() + 8 * U * z.double().abs().clamp(max=12)).all()


def test_gelu_keeps_its_precision(buf):
    """Outputs of 32 bits, in steps of 2^-24 of themselves: the tail's polynomial 0.2 by its fit, 5 by its roundings; reciprocal and product 2; the bell's
    exponential 2, its argument's rest and their sum 2; product, difference and the product with z 3."""
    z = torch.linspace(-12.5, 12.5, 100001, device="cuda").view(1, -1)[:, :65536].contiguous()
    z = torch.cat([z, -z])
    x, w = torch.zeros((1, 8), device="cuda", dtype=torch.float16), torch.zeros((8, 65536), device="cuda", dtype=torch.float16)
    for row in z:
        y = buf.expert_linear(x, w, bias=row, activation="gelu", out_dtype=torch.float32)[0].double()
        r = row.double()
        want = 0.5 * r * torch.special.erfc(r * -(0.5 ** 0.5))
        assert ((y - want).abs() <= 16 * U * want.abs() + 1e-37).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gelus_slope_keeps_its_precision(buf, dtype):
    """every value of the type from 2^-8 to 8, either sign: one rounding, and terms of 32 bits as large as the integral and the bell are there"""
    z = torch.arange(1 << 15, dtype=torch.int32).to(torch.int16).view(dtype)
    z = z[(z >= 2.0 ** -8) & (z <= 8)]
    z = torch.cat([-z, z]).view(1, -1).cuda()
    z = z[:, :z.shape[1] // 8 * 8].contiguous()
    N = z.shape[1]
    x, w = torch.zeros((1, 8), device="cuda", dtype=dtype), torch.zeros((8, N), device="cuda", dtype=dtype)
    gz = buf.expert_linear_backward(torch.ones_like(z), x, w, activation="gelu", preact=z)[3].double()
    r = z.double()
    integral, bell = 0.5 * torch.special.erfc(r * -(0.5 ** 0.5)), r.abs() * torch.exp(-0.5 * r * r) * 0.3989422804014327
    want = integral + torch.sign(r) * bell
    err = U * (14 * integral + 8 * bell + want.abs())
    half = torch.exp2(torch.frexp(want.abs() + err).exponent.double()) * half_step(dtype) / 2             # of a step where the result lies
    assert ((gz - want).abs() <= half + err + (2.0 ** -25 if dtype == torch.float16 else 1e-37)).all()


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("rows,E,K,N", [(9, 2, 64, 128), (1, 1, 7, 5), (70, 1, 2120, 520), (1200, 40, 72, 1928), (4033, 64, 200, 4104), (900, 3, 264, 1160), (1030, 2, 266, 2050), (17, 2, 2056, 4104),
                                        (1, 1, 4104, 2056), (4100, 1, 2056, 264), (8200, 1, 136, 4104)])
def test_every_preactivation_is_written_and_no_other(buf, rows, E, K, N, transposed):
    """through the kernels' own entry, into tensors that hold NaN: the rows of experts become numbers within the sums' rounding, the rows of nobody stay"""
    for act, name in ((2, "silu"), (5, "swiglu")):
        if name == "swiglu" and N % 2:
            continue
        g, x, w, counts = make(rows, E, K, N, torch.float16, 9, transposed)
        if rows > 1:                                             # the last rows are nobody's
            last = max(range(E), key=lambda e: counts[e])
            counts[last] -= 1
        cols = N // 2 if name == "swiglu" else N
        nan = float("nan")
        y, z = torch.full((rows, cols), nan, device="cuda", dtype=torch.float16), torch.full((rows, N), nan, device="cuda", dtype=torch.float16)
        ct = torch.tensor(counts, dtype=torch.int32, device="cuda")
        d = capi.ExpertLinear(w.data_ptr(), int(transposed), capi.DT_FP16, ct.data_ptr(), 0, act, rows, K, N, E)
        lib = capi.load()
        size = lib.zbalhip_expert_linear_workspace(ctypes.byref(d), 0)
        ws = torch.empty((max(size, 16),), dtype=torch.uint8, device="cuda")
        code = lib.zbalhip_expert_linear(ctypes.byref(d), x.data_ptr(), None, 0, None, y.data_ptr(), 0, z.data_ptr(), ws.data_ptr(), size,
                                         torch.cuda.current_stream().cuda_stream)
        assert code == 0
        want, mag = products(x, w, counts, transposed)
        n = want.shape[0]
        err = (K + 2) * U * mag
        assert ((z[:n].double() - want).abs() <= half_step(torch.float16) * (want.abs() + err) + err + 2.0 ** -25).all()
        assert torch.isfinite(y[:n]).all() and torch.isnan(y[n:]).all() and torch.isnan(z[n:]).all()


@pytest.mark.parametrize("counts", [[0, 0, 0], [0, 0, 90], [90, 0, 0], [20, 30, 10], [-4, 70, 1 << 30]])
@pytest.mark.parametrize("K,N", [(128, 128), (66, 130)])
def test_gradient_counts(buf, counts, K, N):
    """experts without rows have gradients of zero; rows of nobody have none and give none"""
    gx, gw, gb, gz = backward_case(buf, 90, 3, K, N, torch.bfloat16, "silu", counts=counts)
    for e, (a, b) in enumerate(spans(counts, 90)):
        if a == b:
            assert (gw[e] == 0).all() and (gb[e] == 0).all()


def test_the_most_experts(buf):
    """tiles of a kind that holds every expert's place"""
    for transposed in (False, True):
        forward_case(buf, 20000, 1024, 264, 256, torch.bfloat16, transposed=transposed)
        backward_case(buf, 20000, 1024, 264, 256, torch.bfloat16, transposed=transposed)
    counts = [0] * 1024
    counts[1023] = 300
    forward_case(buf, 300, 1024, 264, 256, torch.float16, "silu", bias=torch.float32, counts=counts)
    backward_case(buf, 300, 1024, 264, 256, torch.float16, "silu", counts=counts)


def test_no_rows(buf):
    w = torch.randn((2, 64, 128), device="cuda").to(torch.bfloat16)
    x, ct = torch.empty((0, 64), device="cuda", dtype=torch.bfloat16), torch.zeros((2,), dtype=torch.int32, device="cuda")
    assert buf.expert_linear(x, w, ct).shape == (0, 128)
    gx, gw, gb, _ = buf.expert_linear_backward(torch.empty((0, 128), device="cuda", dtype=torch.bfloat16), x, w, ct, bias=True)
    assert gx.shape == (0, 64) and (gw == 0).all() and (gb == 0).all()


def test_gradients_against_differences(buf):
    """d/dw and d/dx of <r, y> by steps of the forward call, its outputs in 32 bits. K is small enough for a step to be far above the sums' rounding"""
    for act in ("silu", "gelu", "swiglu"):
        K, N, rows, h = 8, 16, 4, 2.0 ** -4
        g, x, w, _ = make(rows, 1, K, N, torch.float16, 3, counts=[rows])
        x, w = (x * 8).round() / 8, (w * 16).round() / 16          # so that a step of h is exact
        cols = N // 2 if act == "swiglu" else N
        r = torch.randn((rows, cols), device="cuda", generator=g).half()
        f = lambda x, w: (buf.expert_linear(x, w, None, None, act, out_dtype=torch.float32).double() * r.double()).sum().item()  # noqa: E731
        z = buf.expert_linear(x, w, None, None, act, return_preact=True)[1]
        gx, gw, _, _ = buf.expert_linear_backward(r, x, w, None, act, z, weight_grad_dtype=torch.float32)
        for at in ((0, 0), (3, 7), (2, 5)):
            for t, grad, pos in ((x, gx, at), (w, gw, (0, at[1], 2 * at[0]))):
                up, down = t.clone(), t.clone()
                up[pos] += h
                down[pos] -= h
                diff = (f(up, w) - f(down, w)) / (2 * h) if t is x else (f(x, up) - f(x, down)) / (2 * h)
                # third derivatives of up to 1 (an entry moves z by h times one of the other operand, up to 3) times h^2 / 6, summed over
                # up to N terms of size |r|, and the half-precision roundings of z, dz and the gradient
                assert abs(diff - grad[pos].item()) <= 16 * (h * h * 9 / 6 + 4 * 2.0 ** -11) * r.abs().max().item()


# ---- calls ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,E,K,N", [(4, 1, 2048, 512), (40, 8, 256, 512), (2000, 4, 512, 520), (500, 1, 4096, 128), (8200, 1, 256, 264),
                                        (1000, 1, 1001, 333), (9000, 8, 136, 2048)])
def test_the_same_every_time_and_captured(buf, rows, E, K, N):
    g, x, w, counts = make(rows, E, K, N, torch.bfloat16, 5)
    ct = torch.tensor(counts, dtype=torch.int32, device="cuda")
    x2 = torch.randn_like(x)
    xin = x.clone()
    b = torch.randn((E, N), device="cuda")

    def step(x):
        y, z = buf.expert_linear(x, w, ct, b, "silu", return_preact=True)
        return (y, z) + tuple(buf.expert_linear_backward(y, x, w, ct, "silu", z, bias=True))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(xin)
        aside = step(x)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(aside, step(x)))
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
        assert all(torch.equal(p, q) for p, q in zip(got, want)) and all(torch.equal(p, q) for p, q in zip(got2, want))


def test_two_streams_at_once(buf):
    """calls that run side by side share nothing"""
    g, x, w, _ = make(64, 1, 4096, 512, torch.bfloat16, 6)
    xs = [torch.randn_like(x) for _ in range(4)]
    want = [buf.expert_linear(v, w) for v in xs]
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for v, s in zip(xs, streams):
            with torch.cuda.stream(s):
                got.append(buf.expert_linear(v, w))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want[i % 4]) for i, a in enumerate(got))


def test_residual_in_place(buf):
    for rows, K, N in ((3, 2048, 512), (300, 256, 264)):
        g, x, w, _ = make(rows, 1, K, N, torch.bfloat16, 7)
        r = torch.randn((rows, N), device="cuda").to(torch.bfloat16)
        want = buf.expert_linear(x, w, residual=r)
        assert torch.equal(buf.expert_linear(x, w, residual=r, out=r), want)


def test_refusals(buf):
    g, x, w, _ = make(12, 2, 64, 128, torch.bfloat16, 8)
    ct = torch.tensor([6, 6], dtype=torch.int32, device="cuda")
    bad = [dict(tokens_per_expert=None), dict(tokens_per_expert=ct[:1]), dict(tokens_per_expert=ct.short()), dict(tokens_per_expert=ct.cpu()),
           dict(x=x.float()), dict(x=x.half()), dict(x=x[:, :63].contiguous()), dict(x=x.t()), dict(x=x.cpu()), dict(x=x[0]), dict(x=x.reshape(-1)[1:1 + 11 * 64].view(11, 64)),
           dict(weight=w.half()), dict(weight=w.transpose(1, 2)), dict(weight=w[:, :, 0]), dict(bias=torch.zeros((128,), device="cuda")),
           dict(bias=torch.zeros((2, 128), device="cuda").half()), dict(bias=torch.zeros((2, 127), device="cuda")), dict(activation="tanh"),
           dict(residual=torch.zeros((12, 127), device="cuda").to(x.dtype)), dict(residual=torch.zeros((12, 128), device="cuda")),
           dict(out_dtype=torch.float16), dict(out=torch.zeros((12, 128), device="cuda")), dict(out=torch.zeros((11, 128), device="cuda").to(x.dtype)),
           dict(weight=w[:, :, :127].contiguous(), activation="swiglu"), dict(transposed=True)]
    for kw in bad:
        args = dict(x=x, weight=w, tokens_per_expert=ct)
        args.update(kw)
        with pytest.raises((ValueError, KeyError, RuntimeError)):
            buf.expert_linear(**args)
    sq = torch.randn((12, 64, 64), device="cuda").to(torch.bfloat16)[:2].contiguous()
    with pytest.raises(capi.ZbalError):
        buf.expert_linear(x, sq, ct, out=x)
    y, z = buf.expert_linear(x, w, ct, activation="silu", return_preact=True)
    bad = [dict(preact=None), dict(preact=z[:, :64].contiguous()), dict(preact=z.half()), dict(grad=y[:11]), dict(grad=y.half()), dict(grad=y.cpu()),
           dict(weight_grad_dtype=torch.float16), dict(need_weight=False, bias=True), dict(tokens_per_expert=None)]
    for kw in bad:
        args = dict(grad=y, x=x, weight=w, tokens_per_expert=ct, activation="silu", preact=z)
        args.update(kw)
        with pytest.raises((ValueError, KeyError, RuntimeError)):
            buf.expert_linear_backward(**args)

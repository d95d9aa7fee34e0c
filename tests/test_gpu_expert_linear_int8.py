"""The experts' int8 products against plain forms in 64 bits: one row to many, sizes that no tile or piece divides, every activation and part of the epilogue, experts
without rows, counts that are wrong, rows of nobody; and a layer that is made of the operators around the int8 exchange."""
import pytest
import torch

from int8_cuts import CASES
from memfabric_hybrid_amd import capi
from memfabric_hybrid_amd.buffer import Buffer

pytestmark = pytest.mark.gpu
ACTIVATIONS = ["none", "relu", "silu", "gelu", "gelu_tanh", "swiglu"]
TYPES = [torch.bfloat16, torch.float16, torch.float32]
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


def make(rows, E, K, N, seed, counts=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randint(-128, 128, (rows, K), device="cuda", generator=g, dtype=torch.int8)
    w = torch.randint(-128, 128, (E, N, K), device="cuda", generator=g, dtype=torch.int8)
    xs = (torch.rand((rows,), device="cuda", generator=g) + 0.1) / 64
    ws = (torch.rand((E, N), device="cuda", generator=g) + 0.1) * K ** -0.5 / 64
    if counts is None:
        p = torch.rand((E,), generator=torch.Generator().manual_seed(seed)) + 0.05
        if E > 3:
            p[1] = 0.0
        counts = torch.bincount(torch.multinomial(p, rows, replacement=True, generator=torch.Generator().manual_seed(seed)), minlength=E).tolist()
    return g, x, xs, w, ws, counts


def product64(x, xs, w, ws, counts):
    return torch.cat([(x[a:b].double() @ w[e].double().t()) * ws[e].double() * xs[a:b, None].double() for e, (a, b) in enumerate(spans(counts, x.shape[0]))])


def case(buf, rows, E, K, N, out=torch.bfloat16, act="none", bias=None, residual=False, scale_type=torch.float32, counts=None, count_dtype=torch.int32, seed=0):
    g, x, xs, w, ws, counts = make(rows, E, K, N, seed + rows + K + N, None if counts == "all" else counts)
    ws = ws.to(scale_type)
    cols = N // 2 if act == "swiglu" else N
    b = torch.randn((E, N), device="cuda", generator=g).to(bias) if bias is not None else None
    r = torch.randn((rows, cols), device="cuda", generator=g).to(out) if residual else None
    y = torch.full((rows, cols), 77.0, device="cuda", dtype=out)
    ct = None if E == 1 and sum(counts) == rows else torch.tensor(counts, dtype=count_dtype, device="cuda")
    got = buf.expert_linear_int8(x, xs, w, ws, ct, b, act, r, out, y)
    assert got.data_ptr() == y.data_ptr()
    z = product64(x, xs, w, ws, counts)
    n = z.shape[0]
    err = 3 * U * z.abs()                        # the sum, which is exact, rounded to 32 bits, and two products
    if b is not None:
        z = z + torch.cat([b[e].double().expand(q - p, N) for e, (p, q) in enumerate(spans(counts, rows))])
        err = err + U * z.abs()
    v = act64(z, act)
    if act == "swiglu":
        h = N // 2
        ge, ue, gate, up = err[:, :h], err[:, h:], z[:, :h], z[:, h:]
        err_y = 1.1 * ge * (up.abs() + ue) + act64(gate, "silu").abs() * ue
    else:
        err_y = 1.13 * err                       # no slope is steeper
    # an activation is a dozen operations of 32 bits; gelu's tail or tanh a step of one, times z
    err_y = err_y + 16 * U * v.abs() + (8 * U * z.abs()[:, :cols] if act.startswith("gelu") else 0)
    if r is not None:
        v = v + r[:n].double()
        err_y = err_y + U * v.abs()
    tiny = 2.0 ** -25 if out == torch.float16 else 1e-37
    far = (got[:n].double() - v).abs() - (half_step(out) * (v.abs() + err_y) + err_y + tiny)
    assert far.max().item() <= 0 if far.numel() else True, (far.max().item(), (far > 0).sum().item())
    assert (y[n:] == 77.0).all()
    return got


@pytest.mark.parametrize("rows,K,N", [(1, 1, 1), (1, 15, 9), (1, 16, 128), (2, 17, 9), (3, 65, 130), (5, 31, 64), (15, 400, 72), (16, 512, 128), (17, 2001, 515), (64, 1024, 384),
                                      (127, 192, 1000), (129, 2048, 264), (300, 333, 777), (513, 4096, 520), (1, 7168, 256), (2, 2048, 4096)])
def test_dense(buf, rows, K, N):
    for out in TYPES:
        case(buf, rows, 1, K, N, out)


@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("rows,K,N", [(1, 640, 256), (5, 104, 40), (33, 131, 66), (200, 512, 512), (700, 528, 1032)])
def test_epilogues(buf, rows, K, N, act):
    case(buf, rows, 1, K, N, torch.bfloat16, act)
    case(buf, rows, 1, K, N, torch.float16, act, bias=torch.float32, residual=True)
    case(buf, rows, 1, K, N, torch.float16, act, bias=torch.float16, scale_type=torch.bfloat16)
    case(buf, rows, 1, K, N, torch.float32, act, bias=torch.bfloat16, residual=True)


@pytest.mark.parametrize("rows,E,K,N,act", [(16, 32, 512, 256, "swiglu"), (8, 64, 200, 130, "silu"), (100, 4, 96, 200, "none"), (333, 7, 256, 256, "swiglu"),
                                            (700, 65, 128, 72, "gelu"), (3000, 8, 640, 520, "swiglu"), (2000, 130, 256, 128, "none"), (40, 1024, 64, 64, "relu"),
                                            (9000, 5, 512, 384, "none")])
def test_grouped(buf, rows, E, K, N, act):
    case(buf, rows, E, K, N, torch.bfloat16, act, bias=torch.float32, count_dtype=torch.int64)
    case(buf, rows, E, K, N, torch.float16, act, residual=True, scale_type=torch.bfloat16)
    case(buf, rows, E, K, N, torch.float32, act)


# sizes that are cut into every kind of tiles and parts, for many workgroups a CU; the last rows, columns and k of each are ragged
@pytest.mark.parametrize("rows,E,K,N", [(8200, 1, 272, 4104), (4033, 64, 400, 4104), (1280, 20, 272, 2056), (1200, 40, 144, 1928), (900, 3, 528, 1160), (4100, 1, 4112, 264),
                                        (70, 1, 4240, 520), (2100, 1, 8193, 250), (1030, 2, 530, 2050), (200, 60, 258, 1026), (5000, 3, 261, 1029), (1, 1, 8208, 2056),
                                        (1, 1, 2208, 4104), (17, 2, 4112, 4104), (5, 3, 2064, 72), (3, 5, 2096, 80)])
def test_every_cut(buf, rows, E, K, N):
    case(buf, rows, E, K, N, torch.float32)
    case(buf, rows, E, K, N, torch.float16, "silu", bias=torch.float16, residual=True, seed=1)
    if N % 2 == 0:
        case(buf, rows, E, K, N, torch.bfloat16, "swiglu", seed=2)
        case(buf, rows, E, K, N, torch.float16, "swiglu", bias=torch.float32, residual=True, seed=3)


# what the rule gives each kind of tiles, whole and in parts, aligned rows and rows that are copied, or multiplied as they lie; columns that end anywhere
@pytest.mark.parametrize("rows,E,K,N,act", [
    (1915, 1, 144, 2157, "none"), (1130, 20, 176, 3078, "swiglu"), (2130, 1, 175, 1880, "swiglu"), (2100, 1, 296, 1815, "none"),                      # 128 x 128
    (15, 20, 736, 1983, "none"), (3505, 1, 1616, 114, "swiglu"), (327, 1, 1890, 1280, "swiglu"),                                                     # 16 x 64
    (27, 20, 16, 2865, "none"), (4597, 1, 5168, 80, "none"), (564, 1, 4416, 248, "none"), (1066, 1, 7744, 226, "swiglu"), (337, 1, 6032, 350, "none"),     # 32 x 128
    (10, 20, 224, 2071, "none"), (1429, 1, 6096, 280, "swiglu"), (711, 1, 6100, 271, "none"), (434, 1, 8196, 568, "swiglu"), (2722, 1, 6416, 35, "none"),   # 64 x 64
    (639, 20, 16, 2198, "none"), (4564, 20, 16, 394, "swiglu"), (921, 20, 52, 3888, "none"),                                                         # 64 x 128
    (2222, 8, 16, 1697, "none"), (1917, 20, 16, 1836, "swiglu"), (7187, 1, 20, 772, "swiglu"), (3816, 1, 17, 1485, "none"),                          # 256 x 256
    (1835, 3, 17, 2147, "none"), (5613, 1, 18, 778, "swiglu"), (68, 1, 1727, 2674, "none"), (1, 1, 3644, 2302, "none"), (1, 1, 3537, 2120, "swiglu"),  # as they lie
    (1, 1, 4115, 1105, "none"), (2511, 8, 17, 787, "none"), (8692, 1, 1775, 12, "none"), (5719, 1, 3268, 10, "swiglu"), (1336, 1, 8604, 9, "none"),
    (9, 20, 16, 2855, "none"), (1449, 20, 16, 630, "swiglu"), (2988, 20, 18, 1166, "swiglu"), (492, 20, 16, 3895, "none"), (1273, 20, 21, 2236, "swiglu"),   # rings of two
    (7156, 1, 16, 162, "none"), (2689, 1, 17, 1190, "none"), (5751, 1, 16, 222, "swiglu"), (1023, 1, 19, 3212, "swiglu"),
    (405, 8, 400, 3862, "none"), (2323, 1, 385, 974, "swiglu"), (706, 1, 532, 1700, "swiglu"), (497, 1, 1582, 406, "none"), (1087, 1, 5264, 364, "none"),     # and again of the others
    (2679, 1, 6640, 154, "none"), (373, 1, 2245, 1004, "swiglu"), (23, 20, 752, 2010, "none"), (103, 20, 880, 1734, "swiglu"), (8529, 1, 528, 29, "none"),
    (4160, 8, 16, 1906, "none"), (3910, 20, 16, 2148, "swiglu"), (5363, 8, 17, 1580, "none"), (4598, 20, 17, 2180, "swiglu"), (7939, 3, 272, 457, "none"),
    (1249, 1, 272, 3070, "swiglu"), (2163, 1, 257, 1734, "swiglu"), (123, 1, 5072, 3718, "none"), (18, 1, 7552, 3577, "none"),
    (7, 3, 1040, 77, "none"), (9, 2, 2064, 90, "swiglu"), (5, 4, 528, 131, "none"), (30, 3, 3104, 46, "swiglu")])                                      # 16 columns
def test_every_kind_of_the_rule(buf, rows, E, K, N, act):
    case(buf, rows, E, K, N, torch.float32, act)
    case(buf, rows, E, K, N, torch.float16, "silu" if act == "none" else act, bias=torch.float16, residual=True, seed=1)
    case(buf, rows, E, K, N, torch.bfloat16, act, bias=torch.float32, scale_type=torch.bfloat16, seed=2)


@pytest.mark.parametrize("cut,rows,E,K,N,act", CASES)
def test_every_kind_by_its_name(buf, cut, rows, E, K, N, act):
    import ctypes
    d = capi.ExpertLinearInt8(None, None, 1, 0, None, capi.ACTIVATIONS[act], capi.DT_FP32, rows, K, N, E)
    parts, copied = ctypes.c_int32(), ctypes.c_int32()
    assert (capi.load().zbalhip_expert_linear_int8_plan(ctypes.byref(d), ctypes.byref(parts), ctypes.byref(copied)).decode(), parts.value, copied.value) == cut
    plain = act == "none"
    case(buf, rows, E, K, N, torch.float32, act)
    case(buf, rows, E, K, N, torch.float16, "silu" if plain else act, bias=torch.float16, residual=True, seed=1)
    case(buf, rows, E, K, N, torch.bfloat16, act, bias=torch.float32, scale_type=torch.bfloat16, seed=2)
    case(buf, rows, E, K, N, torch.float32, "gelu" if plain else act, residual=True, count_dtype=torch.int64, seed=3)
    if plain:
        case(buf, rows, E, K, N, torch.bfloat16, "gelu_tanh", seed=4)


@pytest.mark.parametrize("cut,rows,E,K,N,act", CASES)
def test_every_kind_with_rows_of_nobody_and_in_place(buf, cut, rows, E, K, N, act):
    """rows past the last expert's, whose scales and residuals are NaN, stay what they are; the residual's rows are read before they are written"""
    n = rows * 2 // 3
    counts = [n] if E == 1 else [0] + [n // (E - 1)] * (E - 1)
    n = sum(counts)
    g, x, xs, w, ws, _ = make(rows, E, K, N, 7, counts)
    r = torch.randn((rows, N // 2 if act == "swiglu" else N), device="cuda", generator=g)
    xs[n:], r[n:] = float("nan"), float("nan")
    ct, b = torch.tensor(counts, dtype=torch.int32, device="cuda"), torch.randn((E, N), device="cuda", generator=g)
    whole = buf.expert_linear_int8(x[:n].clone(), xs[:n].clone(), w, ws, ct, b, "silu" if act == "none" else act, r[:n].clone(), torch.float32)
    out = torch.full_like(r, 77.0)
    buf.expert_linear_int8(x, xs, w, ws, ct, b, "silu" if act == "none" else act, r, torch.float32, out)
    assert torch.equal(out[:n], whole) and (out[n:] == 77.0).all()
    buf.expert_linear_int8(x, xs, w, ws, ct, b, "silu" if act == "none" else act, r, torch.float32, r)
    assert torch.equal(r[:n], whole) and torch.isnan(r[n:]).all()


@pytest.mark.parametrize("counts", [[0, 0, 0, 0], [0, 0, 0, 50], [50, 0, 0, 0], [10, 10, 10, 10], [-5, 20, -(1 << 31), 10], [30, 1 << 30, 7, (1 << 31) - 1],
                                    [1, 47, 1, 1], [20, 20, 20, 20]])
@pytest.mark.parametrize("K,N", [(128, 128), (130, 131)])
def test_counts(buf, counts, K, N):
    """empty experts, rows of nobody, negative counts (none), counts past the last row (cut off there)"""
    case(buf, 50, 4, K, N, torch.bfloat16, "silu", counts=counts)
    case(buf, 50, 4, K, N, torch.bfloat16, counts=counts, count_dtype=torch.int64)


@pytest.mark.parametrize("rows,K,N,act", [(5, 640, 256, "none"), (40, 133, 66, "silu"), (711, 6100, 271, "none"), (1066, 7744, 226, "swiglu"), (700, 528, 1032, "gelu"),
                                          (1, 3644, 2302, "none"), (4100, 272, 2053, "silu"), (4100, 256, 2056, "none"), (2000, 4099, 1003, "none")])
@pytest.mark.parametrize("share", [0, 0.4, 1, 5])
def test_one_experts_count(buf, rows, K, N, act, share):
    """one expert that has fewer rows than there are, or claims more, in every kind of tile and in parts"""
    case(buf, rows, 1, K, N, torch.bfloat16, act, counts=[int(rows * share)], residual=act != "none", seed=4)


def test_sums_are_exact(buf):
    """all products at their largest: 2^14 each, 2^30 in all, and values that differ in the last bit of a sum of 2^24"""
    for K in (65536, 65535):
        x = torch.full((3, K), -128, device="cuda", dtype=torch.int8)
        x[1] = 127
        w = torch.full((2, 24, K), -128, device="cuda", dtype=torch.int8)
        one, ones = torch.ones((3,), device="cuda"), torch.ones((2, 24), device="cuda")
        y = buf.expert_linear_int8(x, one, w, ones, torch.tensor([1, 2], device="cuda"), out_dtype=torch.float32)
        want = torch.tensor([[16384.0 * K], [-16256.0 * K], [16384.0 * K]], device="cuda", dtype=torch.float64)
        assert torch.equal(y, want.float().expand(3, 24))
    K = 1024                                    # 1040 * 16129 = 2^24 - 3056, far from a multiple of anything
    x = torch.full((1, K + 16), 127, device="cuda", dtype=torch.int8)
    w = torch.full((32, K + 16), 127, device="cuda", dtype=torch.int8)
    w[torch.arange(32), torch.arange(32)] = torch.arange(95, 127, device="cuda", dtype=torch.int8)
    y = buf.expert_linear_int8(x, torch.ones((1,), device="cuda"), w, torch.ones((32,), device="cuda"), out_dtype=torch.float32)
    assert torch.equal(y[0].double(), (K + 16) * 16129.0 - 127.0 * torch.arange(32, 0, -1, device="cuda").double())


def test_one_row_does_not_see_the_others(buf):
    """a NaN or infinity in a row's or a column's scale stays there"""
    for rows, E, K, N in ((48, 3, 256, 128), (600, 3, 272, 264), (600, 3, 133, 261), (4, 1, 2048, 512)):
        counts = [rows] if E == 1 else [rows // 3, rows // 3 - 4, rows // 3 - 6]
        g, x, xs, w, ws, _ = make(rows, E, K, N, 1, counts)
        ct, n = torch.tensor(counts, device="cuda"), sum(counts)
        clean = buf.expert_linear_int8(x, xs, w, ws, ct)
        xs2, ws2 = xs.clone(), ws.clone()
        xs2[3], ws2[0, 7] = float("nan"), float("inf")
        xs2[n:] = float("nan")
        dirty = buf.expert_linear_int8(x, xs2, w, ws2, ct)
        assert torch.isnan(dirty[3]).all() and not torch.isfinite(dirty[:counts[0], 7]).any()
        same = torch.ones((n, N), dtype=torch.bool, device="cuda")
        same[3], same[:counts[0], 7] = False, False
        assert torch.equal(clean[:n][same], dirty[:n][same])


def test_the_most_experts(buf):
    case(buf, 20000, 1024, 528, 256, torch.bfloat16)
    counts = [0] * 1024
    counts[1023] = 300
    case(buf, 300, 1024, 528, 256, torch.float16, "silu", bias=torch.float32, counts=counts)


def test_no_rows(buf):
    w, ws = torch.ones((2, 128, 64), device="cuda", dtype=torch.int8), torch.ones((2, 128), device="cuda")
    x, ct = torch.empty((0, 64), device="cuda", dtype=torch.int8), torch.zeros((2,), dtype=torch.int32, device="cuda")
    assert buf.expert_linear_int8(x, torch.empty((0,), device="cuda"), w, ws, ct).shape == (0, 128)


def test_past_32_bits_of_offset(buf):
    """more than 2^31 bytes of rows, and elements of outputs: the last rows are what they are on their own"""
    for rows, K, N in ((33000, 65536, 64), (280000, 64, 8192)):
        x = torch.empty((rows, K), device="cuda", dtype=torch.int8).random_(-128, 128)
        xs = torch.rand((rows,), device="cuda") / 64
        w = torch.randint(-128, 128, (N, K), device="cuda", dtype=torch.int8)
        ws = torch.rand((N,), device="cuda") / 64
        y = buf.expert_linear_int8(x, xs, w, ws)
        for r in (slice(0, 3), slice(rows - 3, rows)):
            assert torch.equal(y[r], buf.expert_linear_int8(x[r].clone(), xs[r].clone(), w, ws))
        del x, y


def test_past_32_bits_of_offset_with_an_epilogue(buf):
    """bias, residual and outputs of more than 2^31 elements"""
    rows, K, N = 33000, 64, 65536
    g, x, xs, w, ws, _ = make(rows, 1, K, N, 5)
    b, r = torch.randn((N,), device="cuda", generator=g), torch.randn((rows, N), device="cuda", generator=g, dtype=torch.bfloat16)
    y = buf.expert_linear_int8(x, xs, w, ws, bias=b, residual=r, activation="relu")
    for at in (slice(0, 3), slice(rows // 2, rows // 2 + 3), slice(rows - 3, rows)):
        z = product64(x[at], xs[at], w, ws, [3]) + b.double()
        v = torch.relu(z) + r[at].double()
        err = 4 * U * (z - b.double()).abs() + 2 * U * z.abs() + U * v.abs()
        assert ((y[at].double() - v).abs() <= half_step(torch.bfloat16) * (v.abs() + err) + err).all()


@pytest.mark.parametrize("rows,E,K,N", [(4, 1, 4096, 512), (40, 8, 512, 512), (2000, 4, 1024, 520), (500, 1, 8192, 128), (8200, 1, 512, 264), (1000, 1, 1001, 333), (9000, 8, 272, 2048)])
def test_the_same_every_time_and_captured(buf, rows, E, K, N):
    g, x, xs, w, ws, counts = make(rows, E, K, N, 5)
    ct = torch.tensor(counts, dtype=torch.int32, device="cuda")
    x2 = torch.randint(-128, 128, x.shape, device="cuda", dtype=torch.int8)
    xin = x.clone()
    b = torch.randn((E, N), device="cuda")
    step = lambda x: (buf.expert_linear_int8(x, xs, w, ws, ct, b, "silu"), buf.expert_linear_int8(x, xs, w, ws, ct, out_dtype=torch.float32))  # noqa: E731
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


def test_parts_and_copies_give_the_same_bits(buf):
    """without a workspace a product is not split along k, and its rows are not copied; its integers add up to the same"""
    import ctypes
    lib, split = capi.load(), 0
    for rows, K, N, act in ((1087, 5264, 364, 0), (1066, 7744, 226, 5), (337, 6032, 350, 2), (711, 6100, 271, 3), (434, 8196, 568, 5), (2000, 4099, 1003, 2), (1, 3644, 2302, 0)):
        g, x, xs, w, ws, _ = make(rows, 1, K, N, 3)
        cols = N // 2 if act == 5 else N
        d = capi.ExpertLinearInt8(w.data_ptr(), ws.data_ptr(), 1, 0, None, act, capi.DT_FP32, rows, K, N, 1)
        size = lib.zbalhip_expert_linear_int8_workspace(ctypes.byref(d))
        split += size > 0
        ys = []
        for n in (size, 0):
            y = torch.empty((rows, cols), device="cuda")
            part = torch.empty((max(n, 16),), dtype=torch.uint8, device="cuda")
            assert lib.zbalhip_expert_linear_int8(ctypes.byref(d), x.data_ptr(), xs.data_ptr(), None, 0, None, y.data_ptr(), part.data_ptr() if n else None, n,
                                                  torch.cuda.current_stream().cuda_stream) == 0
            ys.append(y)
        assert torch.equal(*ys)
    assert split == 7


@pytest.mark.parametrize("rows,E,K,N,counts,long", [(2000, 1, 4099, 1003, [700], False), (2000, 1, 4099, 1003, [0], True), (1087, 1, 5265, 364, [1086], False),
                                                    (3974, 3, 1651, 1344, [1, 0, 1500], True), (20000, 70, 519, 264, [31] * 70, False),
                                                    (9566, 8, 1670, 320, [900] * 8, False), (9566, 8, 1670, 320, [2000] * 8, True)])
def test_copies_leave_rows_of_nobody_alone(buf, rows, E, K, N, counts, long):
    """rows past the last expert's are neither read nor written, also where unaligned rows are copied to the workspace, x's in front"""
    import ctypes
    lib, wide = capi.load(), (K + 15) // 16 * 16
    g, x, xs, w, ws, _ = make(rows, E, K, N, 6, counts)
    n = min(rows, sum(counts))
    ct = torch.tensor(counts, dtype=torch.int64 if long else torch.int32, device="cuda")
    d = capi.ExpertLinearInt8(w.data_ptr(), ws.data_ptr(), 1, int(long), ct.data_ptr(), 0, capi.DT_FP32, rows, K, N, E)
    size = lib.zbalhip_expert_linear_int8_workspace(ctypes.byref(d))
    assert size >= (rows + E * N) * wide                     # the rule copies these
    part, y = torch.full((size,), 0x5a, dtype=torch.uint8, device="cuda"), torch.full((rows, N), 77.0, device="cuda")
    assert lib.zbalhip_expert_linear_int8(ctypes.byref(d), x.data_ptr(), xs.data_ptr(), None, 0, None, y.data_ptr(), part.data_ptr(), size,
                                          torch.cuda.current_stream().cuda_stream) == 0
    copies = part[:rows * wide].view(rows, wide)
    assert torch.equal(copies[:n, :K].view(torch.int8), x[:n]) and (copies[:n, K:] == 0).all()
    assert (copies[n:] == 0x5a).all()
    want = product64(x, xs, w, ws, counts)
    assert ((y[:n].double() - want).abs() <= 4 * U * want.abs() + 1e-37).all() and (y[n:] == 77.0).all()


def test_residual_in_place(buf):
    g, x, xs, w, ws, _ = make(70, 1, 200, 264, 4)
    r = torch.randn((70, 264), device="cuda").to(torch.bfloat16)
    want = buf.expert_linear_int8(x, xs, w, ws, residual=r)
    assert torch.equal(buf.expert_linear_int8(x, xs, w, ws, residual=r, out=r), want)


@pytest.mark.parametrize("rows,E,K,N,act", [(3, 1, 2048, 512, "none"), (600, 1, 1101, 700, "swiglu"), (2000, 1, 4099, 1003, "silu"), (4100, 3, 256, 2056, "swiglu"),
                                            (4100, 1, 256, 2053, "gelu"), (300, 8, 512, 520, "silu")])
@pytest.mark.parametrize("out", TYPES)
def test_residual_in_place_of_every_tile(buf, rows, E, K, N, act, out):
    """the residual's rows are read ahead of what is stored on them"""
    g, x, xs, w, ws, counts = make(rows, E, K, N, 14)
    ct = torch.tensor(counts, dtype=torch.int32, device="cuda")
    r = torch.randn((rows, N // 2 if act == "swiglu" else N), device="cuda", generator=g).to(out)
    want = buf.expert_linear_int8(x, xs, w, ws, ct, activation=act, residual=r, out_dtype=out)
    for _ in range(3):
        y = r.clone()
        assert torch.equal(buf.expert_linear_int8(x, xs, w, ws, ct, activation=act, residual=y, out_dtype=out, out=y), want)


def test_streams_side_by_side(buf):
    """calls that run side by side share nothing: parts, copies and a gradient's sums lie in workspaces of their own"""
    sets = []
    for rows, K, N in ((1087, 5264, 364), (2000, 4099, 1003), (64, 4096, 512)):
        g, x, xs, w, ws, _ = make(rows, 1, K, N, 15)
        sets.append([(torch.randint(-128, 128, x.shape, device="cuda", generator=g, dtype=torch.int8), xs, w, ws) for _ in range(4)])
    h = [torch.randn((500, 1536), device="cuda") for _ in range(8)]
    norm = lambda i: buf.rms_norm_backward(h[i], h[i + 4])  # noqa: E731
    want = [[buf.expert_linear_int8(*v) for v in s] for s in sets]
    back = [norm(i) for i in range(4)]
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    got, gradients = [], []
    for _ in range(3):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got.append((i, [buf.expert_linear_int8(*s[i]) for s in sets]))
                gradients.append((i, norm(i)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want[k][i]) for i, ys in got for k, a in enumerate(ys))
    assert all(torch.equal(a, b) for i, ys in gradients for a, b in zip(ys, back[i]))


def test_refusals(buf):
    i8 = lambda *s: torch.ones(s, device="cuda", dtype=torch.int8)  # noqa: E731
    f = lambda *s: torch.ones(s, device="cuda")  # noqa: E731
    x, xs, w, ws, ct = i8(8, 64), f(8), i8(2, 32, 64), f(2, 32), torch.tensor([4, 4], device="cuda", dtype=torch.int32)
    call = buf.expert_linear_int8
    for bad in (lambda: call(i8(8, 65), xs, w, ws, ct), lambda: call(x, f(7), w, ws, ct), lambda: call(x, f(8, 1), w, ws, ct), lambda: call(x, xs, w, f(2, 31), ct),
                lambda: call(x, xs, w, ws, ct[:1]), lambda: call(x, xs, w, ws, ct, f(32)), lambda: call(x, xs, w, ws, ct, residual=f(8, 31)), lambda: call(x, xs, i8(64), ws, ct),
                lambda: call(x, xs, w, ws, ct, activation="tanh"), lambda: call(x, xs, w, ws, ct, out_dtype=torch.int8), lambda: call(x, xs, w, ws, ct, out=f(8, 32)),
                lambda: call(i8(8, 128)[:, :64], xs, w, ws, ct), lambda: call(x.cpu(), xs, w, ws, ct)):
        with pytest.raises(ValueError):
            bad()
    for bad, text in ((lambda: call(x.float(), xs, w, ws, ct), "x has type"), (lambda: call(x, xs.half(), w, ws, ct), "xScales"), (lambda: call(x, xs, w.float(), ws, ct), "weight"),
                      (lambda: call(x, xs, w, ws.half(), ct), "weightScales"), (lambda: call(x, xs, w, ws), "tokensPerExpert"), (lambda: call(x, xs, w, ws, ct.float()), "tokensPerExpert"),
                      (lambda: call(x, xs, w, ws, ct, f(2, 32).half()), "bias"), (lambda: call(x, xs, w, ws, ct, residual=f(8, 32)), "residual"),
                      (lambda: call(x, xs, i8(2, 33, 64), f(2, 33), ct, activation="swiglu"), "even"), (lambda: call(x, xs, i8(1025, 1, 64), f(1025, 1), ct.new_zeros(1025)), "experts"),
                      (lambda: call(i8(1, 65552), f(1), i8(1, 65552), f(1)), "out of range"), (lambda: call(i8(9, 63)[1:], xs, i8(2, 32, 63), ws, ct), "aligned")):
        with pytest.raises(capi.ZbalError, match=text):
            bad()
    both = torch.ones((12, 32), device="cuda", dtype=torch.bfloat16)
    with pytest.raises(capi.ZbalError, match="lies on"):
        call(x, xs, w, ws, ct, residual=both[4:], out=both[:8])


def test_a_layer(buf):
    """What a program runs: the norm with its int8 rows for a shared expert, the router, the int8 exchange, the experts' two products with the activation in int8 between
    them, and the weighted sum. Each step against 64 bits, from what the step before it left."""
    T, H, I, E, K = 200, 512, 256, 8, 3
    g = torch.Generator(device="cuda").manual_seed(11)
    rand = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    x, r, w = rand(T, H).to(torch.bfloat16), rand(T, H).to(torch.bfloat16), (1 + 0.1 * rand(H)).to(torch.bfloat16)
    quant = lambda t: ((t / (s := t.abs().amax(-1, keepdim=True) / 127)).round().to(torch.int8), s[..., 0])  # noqa: E731
    w1, s1 = quant(rand(E, 2 * I, H) * H ** -0.5)
    w2, s2 = quant(rand(E, H, I) * I ** -0.5)
    v1, t1 = quant(rand(2 * I, H) * H ** -0.5)
    v2, t2 = quant(rand(H, I) * I ** -0.5)
    gate = (rand(H, E) * H ** -0.5).to(torch.bfloat16)

    y, q, scales, total = buf.rms_norm(x, w, r, quantize=True)
    logits = buf.expert_linear(y, gate, out_dtype=torch.float32)
    idx, weights = buf.group_route(logits, K)
    # the shared expert, on the norm's own int8 rows, added to the residual stream
    a = buf.expert_linear_int8(q, scales, v1, t1, activation="swiglu", out_dtype=torch.float32)
    qa, sa = buf.quantize_rows(a)
    shared = buf.expert_linear_int8(qa, sa, v2, t2, residual=total)
    # the routed experts
    (rows, rs), counts, handle, _, _ = buf.low_latency_dispatch(y, idx, T, E, use_fp8=True)
    assert rows.dtype == torch.int8
    z = buf.expert_linear_int8(rows, rs, w1, s1, counts)
    qz, sz = buf.quantize_rows(z, counts, "swiglu")
    o = buf.expert_linear_int8(qz, sz, w2, s2, counts)
    out = buf.low_latency_combine(o, idx, weights, handle)[0]

    F = torch.nn.functional

    def near(got, want, steps):
        assert ((got.double() - want).abs() <= half_step(got.dtype) * want.abs() + steps * U * want.abs() + 1e-30).all()

    za = product64(q, scales, v1[None], t1[None], [T])
    assert ((a.double() - F.silu(za[:, :I]) * za[:, I:]).abs() <= 32 * U * (F.silu(za[:, :I]).abs() + U * za[:, :I].abs()) * za[:, I:].abs() + 1e-30).all()
    assert ((qa.double() * sa[:, None].double() - a.double()).abs() <= (0.5 + 127 * 4 * U) * sa[:, None].double()).all()
    zs = product64(qa, sa, v2[None], t2[None], [T])
    want = zs + total.double()
    assert ((shared.double() - want).abs() <= half_step(torch.bfloat16) * want.abs() * (1 + 8 * U) + 8 * U * (zs.abs() + want.abs())).all()
    n = counts.tolist()
    near(z, product64(rows, rs, w1, s1, n), 3)
    act = F.silu(z[:, :I].double()) * z[:, I:].double()
    assert ((qz.double() * sz[:, None].double() - act).abs() <= (0.5 + 127 * 40 * U) * sz[:, None].double()).all()
    near(o, product64(qz, sz, w2, s2, n), 3)
    flat = idx.flatten()
    order = torch.sort(flat, stable=True).indices
    at = torch.empty_like(order)
    at[order] = torch.arange(T * K, device="cuda")
    terms = weights[:, :, None].double() * o[at.view(T, K)].double()
    assert ((out.double() - terms.sum(1)).abs() <= half_step(torch.bfloat16) * terms.sum(1).abs() + 8 * U * terms.abs().sum(1)).all()
    # the int8 rows of the exchange are the tokens' own
    assert (rows.double() * rs[:, None].double() - y[order // K].double()).abs().max() <= (0.5 + 1e-3) * rs.max()

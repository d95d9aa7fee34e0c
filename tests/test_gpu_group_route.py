"""Routing by groups of experts and its gradient against plain forms in 64 bits: group shapes that fill a wave's lanes and ones
that do not, ties, experts and whole rows ruled out, NaN and infinities, ids that are no picks or there twice, both id types,
graphs and other streams."""
import math

import pytest
import torch

from memfabric_hybrid_amd import capi
from memfabric_hybrid_amd.buffer import Buffer

pytestmark = pytest.mark.gpu
INF = math.inf


@pytest.fixture(scope="module")
def buf():
    b = Buffer()
    yield b
    torch.cuda.synchronize()
    b.close()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def scores(logits, score):
    l = logits.double()
    return torch.sigmoid(l) if score == "sigmoid" else torch.softmax(l, dim=-1)


def plain(logits, topk, groups=1, kept=1, score="sigmoid", bias=None, group_score="top2", renormalize=True, scale=1.0):
    """One row at a time, with Python's own sorting."""
    s = scores(logits, score)
    c = s if bias is None else s + bias.double()
    T, E = logits.shape
    per = E // groups
    idx, w = torch.full((T, topk), -1, dtype=torch.int64), torch.zeros((T, topk), dtype=torch.float64)
    for t in range(T):
        ok = [e for e in range(E) if logits[t, e].item() > -INF and c[t, e].item() > -INF]
        val = {e: c[t, e].item() for e in ok}
        if groups > 1:
            best = {}
            for g in range(groups):
                v = sorted((val[e] for e in ok if e // per == g), reverse=True)
                if v:
                    best[g] = v[0] + (v[1] if group_score == "top2" and len(v) > 1 else 0.0)
            keep = set(sorted(best, key=lambda g: (-best[g], g))[:kept])
            ok = [e for e in ok if e // per in keep]
        picks = sorted(ok, key=lambda e: (-val[e], e))[:topk]
        total = sum(s[t, e].item() for e in picks)
        for k, e in enumerate(picks):
            idx[t, k] = e
            v = s[t, e].item()
            w[t, k] = (v / total if total > 0 else 0.0) * scale if renormalize else v * scale
    return idx, w


def check(buf, logits, topk, idx_dtype=torch.int64, **kw):
    bias = kw.pop("bias", None)
    idx, w = buf.group_route(logits.cuda(), topk, num_groups=kw.get("groups", 1), topk_groups=kw.get("kept", 1),
                             score=kw.get("score", "sigmoid"), bias=None if bias is None else bias.cuda(),
                             group_score=kw.get("group_score", "top2"), renormalize=kw.get("renormalize", True),
                             scale=kw.get("scale", 1.0), idx_dtype=idx_dtype)
    ridx, rw = plain(logits, topk, bias=bias, **kw)
    assert idx.dtype == idx_dtype and w.dtype == torch.float32
    assert torch.equal(idx.cpu().long(), ridx)
    # a rounding to 32 bits, and a few of 64 before it
    assert torch.allclose(w.cpu().double(), rw, rtol=2.0 ** -24 + 1e-12, atol=1e-44)
    return idx, w


SHAPES = [(1, 1, 1, 1), (5, 1, 1, 5), (64, 1, 1, 8), (65, 1, 1, 8), (256, 8, 4, 8), (256, 8, 8, 32), (102, 6, 2, 7), (384, 16, 3, 9),
          (1000, 40, 7, 32), (1024, 64, 64, 32), (1024, 1, 1, 16), (1024, 2, 1, 16), (64, 64, 5, 5), (96, 3, 2, 6), (62, 31, 9, 10)]


@pytest.mark.parametrize("E,G,kept,K", SHAPES)
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_picks_and_weights(buf, E, G, kept, K, score):
    g = gen(E + G + K)
    logits, bias = torch.randn((37, E), generator=g) * 2, torch.randn((E,), generator=g) * 0.1
    for group_score in ("top2", "max"):
        check(buf, logits, K, groups=G, kept=kept, score=score, group_score=group_score, bias=bias, scale=2.5)
    check(buf, logits, K, groups=G, kept=kept, score=score, renormalize=False, idx_dtype=torch.int32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_half_logits_tie_to_the_lower_index(buf, dtype):
    g = gen(1)
    check(buf, (torch.randn((50, 256), generator=g) * 0.1).to(dtype), 8, groups=8, kept=4)
    check(buf, torch.zeros((3, 96)).to(dtype), 7, groups=8, kept=3, group_score="max")
    check(buf, torch.randint(-2, 3, (40, 100), generator=g).to(dtype), 12, score="softmax")


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E,G,kept,K", [(64, 8, 3, 8), (100, 4, 4, 12), (130, 1, 1, 9)])
def test_ruled_out_experts(buf, E, G, kept, K, score):
    """minus infinity in the logits or in the bias: fewer experts than picks, groups without any, rows without any"""
    g = gen(E + K)
    logits = torch.randn((60, E), generator=g)
    for t in range(60):
        logits[t, torch.randperm(E, generator=g)[: (0, 1, K - 1, K, E // 2, E)[t % 6]:]] = -INF
    logits[7] = -INF
    logits[8, 3:] = -INF
    logits[9, : E // max(G, 2)] = torch.finfo(torch.float32).min
    idx, w = check(buf, logits, K, groups=G, kept=kept, score=score)
    assert (idx[7] == -1).all() and (w[7] == 0).all()
    bias = torch.zeros((E,))
    bias[::3] = -INF
    check(buf, logits, K, groups=G, kept=kept, score=score, bias=bias)


def test_nan_and_infinity(buf):
    logits = torch.randn((6, 70), generator=gen(3))
    logits[0, 5], logits[1, 6], logits[2, :] = math.nan, INF, math.nan
    logits[3, 0], logits[3, 69] = 200.0, -200.0
    idx, w = check(buf, logits, 8)                              # sigmoid: a NaN is no pick, infinity has the score 1
    assert (idx[2] == -1).all() and idx[1, 0] == 6
    bias = torch.zeros((70,))
    bias[0], bias[1], bias[2] = math.nan, INF, -INF
    check(buf, logits, 8, bias=bias)
    idx, w = buf.group_route(logits.cuda(), 8, score="softmax")  # a row whose softmax is no number has no pick
    assert (idx[:3] == -1).all() and (w[:3] == 0).all() and (idx[3:] >= 0).all()


def test_far_logits_keep_their_order(buf):
    """scores that 32 bits cannot tell apart, and ones that vanish there"""
    up = 30.0 + torch.arange(64).float() * 1e-3
    check(buf, torch.stack([up, -5 * up, torch.roll(up, 7) + 60]).contiguous(), 8)


def test_rows_of_infinity_and_of_the_lowest_value(buf):
    logits = torch.randn((8, 256), generator=gen(8))
    logits[0], logits[1, ::2], logits[2, :200] = INF, INF, -INF
    logits[2, 200:] = INF
    logits[3], logits[4, 1::2] = torch.finfo(torch.float32).min, torch.finfo(torch.float32).min
    logits[5, 9:], logits[6, :250] = torch.finfo(torch.float32).min, -1e9
    check(buf, logits, 8)
    check(buf, logits, 8, groups=8, kept=4)
    check(buf, logits, 8, groups=8, kept=4, group_score="max")
    check(buf, logits[3:].contiguous(), 8, score="softmax")
    bias = torch.zeros((256,))
    bias[::2] = INF
    check(buf, logits, 8, bias=bias)
    check(buf, logits, 8, bias=torch.full((256,), INF), groups=8, kept=4)


def test_logits_so_small_that_their_scores_are_equal(buf):
    """ties of 64-bit scores go to the lower index, whatever the logits"""
    logits = torch.zeros((4, 64))
    logits[0, 40:] = 1e-30
    logits[1, 20] = 1e-25
    logits[2] = torch.arange(64) * 1e-35
    logits[3, 8:] = 1e-24
    for group_score in ("top2", "max"):
        check(buf, logits, 8, groups=8, kept=3, group_score=group_score)
        check(buf, logits, 8, groups=8, kept=3, group_score=group_score, score="softmax")
    check(buf, logits, 20)


def picks64(logits, topk, groups, kept, score, bias, group_score):
    """plain()'s picks for many rows at once, with stable sorts"""
    c = scores(logits, score) + bias.double()
    c = torch.where((logits > -INF) & (c > -INF), c, -INF)
    T, E = logits.shape
    v = c.view(T, groups, E // groups).sort(dim=-1, descending=True).values
    of = v[..., 0]
    if group_score == "top2" and E > groups:
        of = of + torch.where(v[..., 1] > -INF, v[..., 1], 0.0)
    keep = torch.zeros((T, groups), dtype=torch.bool).scatter_(1, of.sort(dim=-1, descending=True, stable=True).indices[:, :kept], True)
    c = torch.where(keep.repeat_interleave(E // groups, dim=1), c, -INF)
    value, idx = c.sort(dim=-1, descending=True, stable=True)
    return torch.where(value[:, :topk] > -INF, idx[:, :topk], -1)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("size", [1e2, 1e4, 1e6])
def test_biases_that_cancel_in_a_group(buf, score, size):
    """a group's sum is near one, its two choices are rounded where the bias is: the picks are those of 64 bits all the same"""
    g = gen(int(size))
    for E, groups, kept, K in ((4, 2, 1, 2), (64, 8, 3, 4)):
        T = 1 << 17 if E == 4 else 1 << 14
        logits = torch.randn((T, E), generator=g)
        bias = torch.tensor([size, -size]).repeat(E // 2)
        if E > 4:                                                # one pair in a group is far above its others
            bias = torch.where(torch.arange(E) % 8 < 2, bias, -3 * size)
        for group_score in ("top2", "max"):
            idx = buf.group_route(logits.cuda(), K, groups, kept, score, bias.cuda(), group_score)[0].cpu()
            want = picks64(logits, K, groups, kept, score, bias, group_score)
            assert torch.equal(idx, want), (E, group_score, (idx != want).any(-1).sum().item())


def test_biases_of_the_lowest_value(buf):
    """two of them are minus infinity in 32 bits; a group of theirs still comes before one that is ruled out"""
    low = torch.finfo(torch.float32).min
    logits = torch.randn((40, 8), generator=gen(21))
    logits[:20, :2] = -INF
    for b in ([0, 0, low, low, low, low, 0, 0], [0, 0, low, low, -3.3e38, -3.3e38, 0, 0], [0, 0, 3e38, 3e38, 3.3e38, 3.3e38, 0, 0], [low] * 8):
        for kept in (1, 2, 3):
            for group_score in ("top2", "max"):
                check(buf, logits, 2 * kept, groups=4, kept=kept, bias=torch.tensor(b), group_score=group_score)


def test_an_empty_batch(buf):
    idx, w = buf.group_route(torch.empty((0, 16), device="cuda"), 4)
    assert idx.shape == w.shape == (0, 4)
    gl = buf.group_route_backward(torch.empty((0, 4), device="cuda"), torch.empty((0, 16), device="cuda"), idx)
    assert gl.shape == (0, 16)


# ---- gradient ------------------------------------------------------------------------------------------------------------

def plain_backward(grad, logits, idx, score, renormalize, scale):
    l = logits.double().requires_grad_()
    s = scores(l, score)
    there = (idx >= 0) & (idx < logits.shape[1])
    p = torch.gather(s, 1, torch.where(there, idx, 0)) * there
    if renormalize:
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total > 0, total, 1.0)
    (p * scale * torch.where(there, grad.double(), 0.0)).sum().backward()
    return l.grad


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("E,K", [(1, 1), (7, 3), (64, 8), (65, 32), (256, 8), (1000, 32), (1024, 1)])
def test_gradient(buf, E, K, score, renormalize):
    g = gen(E + K)
    T = 29
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        logits = (torch.randn((T, E), generator=g) * 1.5).to(dtype)
        idx = torch.stack([torch.randperm(E, generator=g)[:K] if E >= K else torch.randint(0, E, (K,), generator=g) for _ in range(T)])
        if T > 5 and K > 1:
            idx[1, 0], idx[2, :], idx[3, -1], idx[4, 1] = -1, -1, E, idx[4, 0]          # none, none at all, none, the same twice
        grad = torch.randn((T, K), generator=g)
        got = buf.group_route_backward(grad.cuda(), logits.cuda(), idx.cuda(), score, renormalize, 2.5).cpu()
        got32 = buf.group_route_backward(grad.cuda(), logits.cuda(), idx.int().cuda(), score, renormalize, 2.5).cpu()
        assert got.dtype == dtype and torch.equal(got, got32)
        want = plain_backward(grad, logits, idx, score, renormalize, 2.5)
        # one rounding of the result; inside, in 32 bits, an exp (2 steps), a sum of E terms and two products of numbers up to |want| + s sum|g s|
        slack = 2.5 * grad.abs().double().sum(-1, keepdim=True) * scores(logits, score) * (8 + E / 16) * 2.0 ** -24
        half = torch.finfo(dtype).eps / 2
        tiny = torch.finfo(dtype).tiny if dtype == torch.float16 else 1e-44
        assert ((got.double() - want).abs() <= half * want.abs() + slack * (1 + half) + tiny).all()


def formula_backward(grad, logits, idx, score, renormalize, scale):
    """The gradient's formula in 64 bits, and the size of the terms that cancel in it. Scores that are no numbers, of a row that is ruled out as
    a whole, are none: such a row has no picks, and no gradient."""
    s = scores(logits, score).nan_to_num(0.0)
    there = (idx >= 0) & (idx < logits.shape[1])
    at = torch.where(there, idx, 0)
    p = torch.gather(s, 1, at) * there
    d = torch.where(there, grad.double(), 0.0) * scale
    mag = d.abs()
    if renormalize:
        total = p.sum(-1, keepdim=True)
        over = torch.where(total > 0, 1 / torch.where(total > 0, total, 1.0), 0.0)
        mag = there * (mag + (mag * p).sum(-1, keepdim=True) * over) * over
        d = there * (d - (d * p).sum(-1, keepdim=True) * over) * over
    D, M = torch.zeros_like(s).scatter_add_(1, at, d), torch.zeros_like(s).scatter_add_(1, at, mag)
    if score == "sigmoid":
        return D * s * (1 - s), M * s
    if renormalize:                                              # the sum is zero
        return D * s, M * s
    return s * (D - (D * s).sum(-1, keepdim=True)), s * (M + (M * s).sum(-1, keepdim=True))


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("E,K", [(7, 3), (64, 8), (65, 17), (256, 8), (1000, 32)])
def test_gradient_of_masked_rows(buf, E, K, score, renormalize):
    """logits of minus infinity: some, all but one, a whole row; picks that the router left out, and ones that are ruled out"""
    g = gen(E + K)
    T = 24
    for dtype in (torch.float32, torch.bfloat16):
        logits = (torch.randn((T, E), generator=g) * 1.5).to(dtype)
        for t in range(T):
            logits[t, torch.randperm(E, generator=g)[: (0, 1, K, E // 2, E)[t % 5]:]] = -INF
        logits[5] = -INF
        idx = buf.group_route(logits.cuda(), K, score=score, renormalize=renormalize)[0].cpu()
        assert (idx[5] == -1).all()
        idx[8::2] = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(8, T, 2)])
        masked = (logits[23] == -INF).nonzero().flatten()
        if masked.numel():                                       # nothing but ruled-out picks
            idx[23] = masked[torch.arange(K) % masked.numel()]
        grad = torch.randn((T, K), generator=g)
        got = buf.group_route_backward(grad.cuda(), logits.cuda(), idx.cuda(), score, renormalize, 2.5).cpu()
        want, mag = formula_backward(grad, logits, idx, score, renormalize, 2.5)
        half, tiny = torch.finfo(dtype).eps / 2, 1e-44
        assert ((got.double() - want).abs() <= half * want.abs() + (8 + E / 16) * 2.0 ** -24 * (1 + half) * mag + tiny).all()
        assert (got[5] == 0).all()


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_gradient_of_rows_without_picks(buf, score, renormalize):
    """whatever their logits: the weights are zeros there, and do not change"""
    logits = torch.randn((6, 96), generator=gen(4))
    logits[0], logits[1, 5], logits[2, 7], logits[3], logits[4, ::2] = -INF, math.nan, INF, math.nan, INF
    idx = torch.full((6, 4), -1)
    got = buf.group_route_backward(torch.ones((6, 4)).cuda(), logits.cuda(), idx.cuda(), score, renormalize, 1.0)
    assert (got == 0).all()


@pytest.mark.parametrize("E,K", [(64, 8), (65, 17), (128, 8), (1024, 32)])
@pytest.mark.parametrize("scale", [1.0, 2.5])
def test_dense_gradient_is_rounded_once(buf, E, K, scale):
    """softmax scores as weights: everything in front of the last rounding is in 64 bits"""
    g = gen(E)
    logits = torch.randn((200, E), generator=g) * 3
    idx = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(200)])
    idx[3, 1], idx[4, 0] = idx[3, 0], -1
    grad = torch.randn((200, K), generator=g)
    got = buf.group_route_backward(grad.cuda(), logits.cuda(), idx.cuda(), "softmax", False, scale).cpu().double()
    want, mag = formula_backward(grad, logits, idx, "softmax", False, scale)
    # exponentials that are good to 2^-31, on both sides of a difference
    assert ((got - want).abs() <= 2.0 ** -24 * want.abs() + 2.0 ** -28 * mag + 1e-44).all()


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_gradient_against_differences(buf, score):
    """the forward call's own weights, at fixed picks"""
    g = gen(5)
    E, K, h = 24, 5, 2.0 ** -8
    logits = torch.randn((1, E), generator=g)
    r = torch.randn((1, K), generator=g)
    idx, _ = buf.group_route(logits.cuda(), K, groups_ := 4, 3, score=score, scale=2.0)
    back = buf.group_route_backward(r.cuda(), logits.cuda(), idx, score, True, 2.0).cpu()[0]
    moved = torch.cat([logits + h * torch.eye(E), logits - h * torch.eye(E)])
    i2, w2 = buf.group_route(moved.cuda(), K, groups_, 3, score=score, scale=2.0)
    same = (i2.cpu().sort(-1).values == idx.cpu().sort(-1).values).all(-1)
    at = torch.zeros((2 * E, E)).scatter_(1, i2.cpu(), w2.cpu())
    loss = (at[:, idx.cpu()[0]].double() * r.double()).sum(-1)
    ok = same[:E] & same[E:]
    assert ok.sum() > E // 2
    diff = (loss[:E] - loss[E:]) / (2 * h)
    # weights of 32 bits over a step of 2^-8, and the third derivative's share
    assert ((diff - back.double()).abs()[ok] <= 4 * r.abs().sum() * (2.0 ** -24 / h + h * h)).all()


# ---- calls ---------------------------------------------------------------------------------------------------------------

def test_captured_and_on_another_stream(buf):
    g = gen(11)
    a, b = (torch.randn((300, 256), generator=g).cuda() for _ in range(2))
    bias = (torch.randn((256,), generator=g) * 0.1).cuda()
    logits = a.clone()
    call = lambda x: buf.group_route(x, 8, 8, 4, bias=bias)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(logits)
        other = call(a)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(other, call(a)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        idx, w = call(logits)
        back = buf.group_route_backward(w, logits, idx)
    for src in (a, b, a, b):
        logits.copy_(src)
        graph.replay()
        eidx, ew = call(src)
        torch.cuda.synchronize()
        assert torch.equal(idx, eidx) and torch.equal(w, ew) and torch.equal(back, buf.group_route_backward(ew, src, eidx))


def test_refusals(buf):
    x = torch.randn((4, 64), device="cuda")
    bad = [dict(num_topk=0), dict(num_topk=33), dict(num_topk=9, num_groups=8), dict(num_topk=2, num_groups=5), dict(num_topk=2, num_groups=8, topk_groups=9),
           dict(num_topk=2, num_groups=0), dict(num_topk=2, num_groups=2, topk_groups=0), dict(num_topk=2, score="tanh"), dict(num_topk=2, group_score="mean"),
           dict(num_topk=2, bias=torch.zeros((63,), device="cuda")), dict(num_topk=2, bias=torch.zeros((64,), device="cuda", dtype=torch.bfloat16)),
           dict(num_topk=2, bias=torch.zeros((64,))), dict(num_topk=2, idx_dtype=torch.int16)]
    for kw in bad:
        with pytest.raises((ValueError, capi.ZbalError)):
            buf.group_route(x, **kw)
    for t in (x.double(), x.t(), x.cpu(), x[0], x.reshape(-1)[1:61].view(4, 15), torch.zeros((2, 1025), device="cuda")):
        with pytest.raises((ValueError, capi.ZbalError)):
            buf.group_route(t, 2)
    idx, w = buf.group_route(x, 2)
    for args in ((w[:3], x, idx), (w, x, idx[:3]), (w.double(), x, idx), (w, x, idx.short()), (w.cpu(), x, idx), (w, x[:3], idx)):
        with pytest.raises((ValueError, KeyError, capi.ZbalError)):
            buf.group_route_backward(*args)

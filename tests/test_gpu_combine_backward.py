"""The gradients of combine and dispatch against plain forms in 64 bits: hidden sizes that a workgroup's lanes do not divide, picks that went
nowhere, tokens without any, more than eight picks, rows that no pick went to, handles older than the last layout."""
import pytest
import torch

from memfabric_hybrid_amd import capi
from memfabric_hybrid_amd.buffer import Buffer

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def buf():
    b = Buffer()
    yield b
    torch.cuda.synchronize()
    b.close()


def exchange(buf, T, H, E, K, dtype, seed, missing=0.2, worst=0):
    """(x, handle, weights, row [T, K] of every pick or -1, rows)"""
    g = torch.Generator().manual_seed(seed)
    idx = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(T)]) if T else torch.empty((0, K), dtype=torch.int64)
    idx[torch.rand((T, K), generator=g) < missing] = -1
    if T > 2:
        idx[T // 2] = -1
    w = torch.randn((T, K), generator=g)
    x = torch.randn((T, H), generator=g).to(dtype)
    row, n = torch.full((T * K,), -1), 0
    flat = idx.flatten()
    for e in range(E):
        at = (flat == e).nonzero().flatten()
        row[at] = torch.arange(n, n + len(at))
        n += len(at)
    d = idx.cuda()
    per_rank, _, per_expert, in_rank, _ = buf.get_dispatch_layout(d, E)
    recv, _, _, _, handle, _ = buf.dispatch(x.cuda(), num_tokens_per_rank=per_rank, is_token_in_rank=in_rank, num_tokens_per_expert=per_expert,
                                            topk_idx=d, topk_weights=w.cuda(), num_worst_tokens=worst)
    return x, recv, handle, w, row.view(T, K), n


@pytest.mark.parametrize("T,H,E,K", [(1, 16, 1, 1), (5, 1040, 16, 3), (61, 2048, 64, 6), (130, 7168, 32, 8), (33, 4096, 40, 9), (7, 8208, 64, 32),
                                     (1100, 512, 8, 2)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients(buf, T, H, E, K, dtype):
    x, recv, handle, w, row, n = exchange(buf, T, H, E, K, dtype, T + H)
    g = torch.Generator().manual_seed(1)
    y = torch.randn((max(n, 1), H), generator=g).to(dtype)
    grad = torch.randn((T, H), generator=g).to(dtype)
    gy, gw = buf.combine_backward(grad.cuda(), y.cuda(), handle)
    gy, gw = gy.cpu().double(), gw.cpu().double()
    there = row >= 0
    yr = y.double()[row.clamp(min=0)]
    prod = yr * grad.double()[:, None, :]
    want = prod.sum(-1) * there
    # a sum of H products in 32 bits, whatever the order
    assert ((gw - want).abs() <= H * 2.0 ** -24 * prod.abs().sum(-1) * there).all()
    rows = row[there]
    wanted = (w.double()[:, :, None] * grad.double()[:, None, :])[there]
    # the product in 32 bits, then rounded to the type
    half = torch.finfo(dtype).eps / 2 + 2.0 ** -23
    assert ((gy[rows] - wanted).abs() <= half * wanted.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_dispatch_gradient(buf, dtype):
    T, H, E, K = 50, 1040, 16, 4
    x, recv, handle, w, row, n = exchange(buf, T, H, E, K, dtype, 3)
    assert torch.equal(recv.cpu()[row[row >= 0]], x[:, None, :].expand(T, K, H)[row >= 0])
    grad = torch.randn((max(n, 1), H), generator=torch.Generator().manual_seed(2)).to(dtype)
    got = buf.dispatch_backward(grad.cuda(), handle).cpu().double()
    parts = grad.double()[row.clamp(min=0)] * (row >= 0)[:, :, None]
    want = parts.sum(1)
    assert ((got - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + K * 2.0 ** -23 * parts.abs().sum(1)).all()


def test_handles_outlive_the_next_layout(buf):
    """two layers run forward before either runs backward"""
    T, H, E, K = 40, 512, 8, 3
    first = exchange(buf, T, H, E, K, torch.bfloat16, 4)
    second = exchange(buf, T, H, E, K, torch.bfloat16, 5)
    for x, recv, handle, w, row, n in (second, first):
        grad = torch.randn((T, H), generator=torch.Generator().manual_seed(n)).to(torch.bfloat16)
        gy, gw = buf.combine_backward(grad.cuda(), recv, handle)
        wanted = (w[:, :, None] * grad.float()[:, None, :])[row >= 0]
        assert torch.equal(gy.cpu()[row[row >= 0]], wanted.to(torch.bfloat16))
        out = buf.combine(recv, handle)[0].cpu().double()
        want = (x.double()[:, None, :] * w.double()[:, :, None] * (row >= 0)[:, :, None])
        assert ((out - want.sum(1)).abs() <= 2.0 ** -8 * want.sum(1).abs() + K * 2.0 ** -22 * want.abs().sum(1)).all()


def test_rows_of_no_pick_are_left_alone(buf):
    T, H, E, K = 9, 256, 8, 3
    x, recv, handle, w, row, n = exchange(buf, T, H, E, K, torch.bfloat16, 6, worst=T * K + 5)
    assert recv.shape[0] == T * K + 5 > n
    grad = torch.randn((T, H), device="cuda").to(torch.bfloat16)
    y = torch.randn((T * K + 5, H), device="cuda").to(torch.bfloat16)
    out, gw = torch.full_like(y, 7.0), torch.empty((T, K), device="cuda")
    in_rank, idx, wt, put_offset, _ = handle
    ids = idx.int()
    lib = capi.load()
    capi.check("combine_backward", lib.zbalhip_combine_backward(
        grad.data_ptr(), y.data_ptr(), y.shape[0], capi.DT_BF16, put_offset.data_ptr(), wt.data_ptr(), ids.data_ptr(), 0,
        handle.send_token_idx.data_ptr(), T, H, K, E, out.data_ptr(), gw.data_ptr(), capi.stream_ptr()))
    assert (out[n:] == 7.0).all()
    # a window that ends early: what it does not hold is neither read nor written
    out2, gw2 = torch.full_like(y, 7.0), torch.empty((T, K), device="cuda")
    capi.check("combine_backward", lib.zbalhip_combine_backward(
        grad.data_ptr(), y.data_ptr(), n // 2, capi.DT_BF16, put_offset.data_ptr(), wt.data_ptr(), ids.data_ptr(), 0,
        handle.send_token_idx.data_ptr(), T, H, K, E, out2.data_ptr(), gw2.data_ptr(), capi.stream_ptr()))
    assert torch.equal(out2[:n // 2], out[:n // 2]) and (out2[n // 2:] == 7.0).all()
    kept = (row < n // 2)
    assert torch.equal(gw2.cpu()[kept], gw.cpu()[kept]) and (gw2.cpu()[~kept] == 0).all()


def test_the_same_every_time_and_captured(buf):
    T, H, E, K = 300, 2048, 16, 4
    x, recv, handle, w, row, n = exchange(buf, T, H, E, K, torch.bfloat16, 8)
    a, b = (torch.randn((T, H), device="cuda").to(torch.bfloat16) for _ in range(2))
    grad = a.clone()
    graph = torch.cuda.CUDAGraph()
    buf.combine_backward(grad, recv, handle)
    with torch.cuda.graph(graph):
        gy, gw = buf.combine_backward(grad, recv, handle)
    for src in (a, b, a):
        grad.copy_(src)
        graph.replay()
        ey, ew = buf.combine_backward(src, recv, handle)
        torch.cuda.synchronize()
        assert torch.equal(gw, ew) and torch.equal(gy[:n], ey[:n])


def test_refusals(buf):
    T, H, E, K = 6, 256, 8, 2
    x, recv, handle, w, row, n = exchange(buf, T, H, E, K, torch.bfloat16, 9, missing=0.0)
    grad = torch.randn((T, H), device="cuda").to(torch.bfloat16)
    for g2, r2 in ((grad.half(), recv), (grad.float(), recv), (grad[:5], recv), (grad[:, :240].contiguous(), recv), (grad.t(), recv), (grad.cpu(), recv),
                   (grad, recv.cpu()), (grad, recv.half())):
        with pytest.raises((ValueError, capi.ZbalError)):
            buf.combine_backward(g2, r2, handle)

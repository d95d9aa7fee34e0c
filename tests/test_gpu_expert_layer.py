"""A mixture-of-experts layer without quantisation, forward and backward, as a training program runs it through Buffer: the router's product,
routing by groups, layout, dispatch, the experts' two products, combine with the shared expert's on top; then every gradient. Against
automatic differentiation of the same layer in 64 bits."""
import pytest
import torch

from memfabric_hybrid_amd.buffer import Buffer

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def buf():
    b = Buffer()
    yield b
    torch.cuda.synchronize()
    b.close()


def parameters(H, E, I, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *s: (torch.randn(s, device="cuda", generator=g) * s[-2] ** -0.5).to(dtype)  # noqa: E731
    return dict(gate=new(H, E), w1=new(E, H, 2 * I), w2=new(E, I, H), s1=new(H, 2 * I), s2=new(I, H)), g


def forward(buf, p, x, K, G, kept, bias):
    E = p["gate"].shape[-1]
    logits = buf.expert_linear(x, p["gate"], out_dtype=torch.float32)
    idx, w = buf.group_route(logits, K, G, kept, bias=bias, scale=2.5)
    per_rank, _, per_expert, in_rank, _ = buf.get_dispatch_layout(idx, E)
    recv, _, _, _, handle, _ = buf.dispatch(x, num_tokens_per_rank=per_rank, is_token_in_rank=in_rank, num_tokens_per_expert=per_expert, topk_idx=idx,
                                            topk_weights=w, num_worst_tokens=idx.numel())
    h, z = buf.expert_linear(recv, p["w1"], per_expert, activation="swiglu", return_preact=True)
    y = buf.expert_linear(h, p["w2"], per_expert)
    routed, _, _ = buf.combine(y, handle)
    sh, sz = buf.expert_linear(x, p["s1"], activation="swiglu", return_preact=True)
    out = buf.expert_linear(sh, p["s2"], residual=routed)
    return out, dict(logits=logits, idx=idx, recv=recv, handle=handle, per_expert=per_expert, h=h, z=z, y=y, sh=sh, sz=sz)


def backward(buf, p, x, s, grad):
    f32, g = torch.float32, {}
    dsh, g["s2"], _, _ = buf.expert_linear_backward(grad, s["sh"], p["s2"], weight_grad_dtype=f32)
    dx_s, g["s1"], _, _ = buf.expert_linear_backward(dsh, x, p["s1"], activation="swiglu", preact=s["sz"], weight_grad_dtype=f32)
    dy, dw = buf.combine_backward(grad, s["y"], s["handle"])
    dh, g["w2"], _, _ = buf.expert_linear_backward(dy, s["h"], p["w2"], s["per_expert"], weight_grad_dtype=f32)
    dr, g["w1"], _, _ = buf.expert_linear_backward(dh, s["recv"], p["w1"], s["per_expert"], "swiglu", s["z"], weight_grad_dtype=f32)
    dx_r = buf.dispatch_backward(dr, s["handle"])
    dl = buf.group_route_backward(dw, s["logits"], s["idx"], scale=2.5)
    dx_g, g["gate"], _, _ = buf.expert_linear_backward(dl, x, p["gate"], weight_grad_dtype=f32)
    g["x"] = dx_s.double() + dx_r.double() + dx_g.double()
    return g


def reference(p, x, K, idx, grad):
    """the same layer in 64 bits with the picks given"""
    q = {k: v.double().requires_grad_() for k, v in p.items()}
    x = x.double().requires_grad_()
    F = torch.nn.functional

    def ffn(v, w1, w2):
        gate, up = (v @ w1).chunk(2, dim=-1)
        return (F.silu(gate) * up) @ w2
    s = torch.sigmoid(x @ q["gate"])
    there = idx >= 0
    w = torch.gather(s, 1, idx.clamp(min=0)) * there
    w = 2.5 * w / w.sum(-1, keepdim=True)
    out = ffn(x, q["s1"], q["s2"])
    for e in range(p["w1"].shape[0]):
        t, k = (idx == e).nonzero(as_tuple=True)
        if len(t):
            out = out.index_add(0, t, ffn(x[t], q["w1"][e], q["w2"][e]) * w[t, k][:, None])
    out.backward(grad.double())
    return out.detach(), dict({k: v.grad for k, v in q.items()}, x=x.grad)


@pytest.mark.parametrize("T,H,E,I,K,G,kept", [(1, 256, 8, 128, 2, 1, 1), (70, 512, 16, 256, 4, 4, 2), (600, 1040, 24, 200, 6, 8, 4)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layer(buf, T, H, E, I, K, G, kept, dtype):
    p, g = parameters(H, E, I, dtype, T)
    x, grad = (torch.randn((T, H), device="cuda", generator=g).to(dtype) for _ in range(2))
    bias = torch.randn((E,), device="cuda", generator=g) * 0.1
    out, s = forward(buf, p, x, K, G, kept, bias)
    got = backward(buf, p, x, s, grad)
    want, grads = reference(p, x, K, s["idx"], grad)
    # In the 2-norm: every tensor between two operators is rounded once (half a step, uniform: 0.58 of it), and at most eight such tensors stand between
    # an input and a gradient, with gains of order one
    half = torch.finfo(dtype).eps / 2
    rel = lambda a, b: ((a.double() - b).norm() / b.norm()).item()  # noqa: E731
    assert rel(out, want) < 4 * half
    for name, v in grads.items():
        assert rel(got[name].view_as(v), v) < 8 * half, name


def test_layer_captured(buf):
    p, g = parameters(512, 16, 128, torch.bfloat16, 3)
    xs = [torch.randn((90, 512), device="cuda", generator=g).to(torch.bfloat16) for _ in range(2)]
    grad = torch.randn((90, 512), device="cuda", generator=g).to(torch.bfloat16)
    bias = torch.zeros((16,), device="cuda")
    x = xs[0].clone()

    def step(x):
        out, s = forward(buf, p, x, 4, 4, 2, bias)
        return [out] + list(backward(buf, p, x, s, grad).values())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x)
    for src in (xs[0], xs[1], xs[0]):
        x.copy_(src)
        graph.replay()
        want = step(src)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("T", [1, 2, 40])
def test_experts_behind_the_low_latency_exchange(buf, T):
    """serving: rows packed by expert and int64 counts, nothing quantised"""
    H, E, I, K = 512, 16, 256, 4
    p, g = parameters(H, E, I, torch.bfloat16, T)
    x = torch.randn((T, H), device="cuda", generator=g).to(torch.bfloat16)
    idx, w = buf.group_route(buf.expert_linear(x, p["gate"], out_dtype=torch.float32), K, 4, 2)
    recv, counts, handle, _, _ = buf.low_latency_dispatch(x, idx, 64, E, use_fp8=False)
    assert counts.dtype == torch.int64
    h = buf.expert_linear(recv, p["w1"], counts, activation="swiglu")
    out, _, _ = buf.low_latency_combine(buf.expert_linear(h, p["w2"], counts), idx, w, handle)
    F = torch.nn.functional
    want = torch.zeros((T, H), dtype=torch.float64, device="cuda")
    for t in range(T):
        for k in range(K):
            e = int(idx[t, k])
            gate, up = (x[t].double() @ p["w1"][e].double()).chunk(2)
            want[t] += w[t, k].double() * ((F.silu(gate) * up) @ p["w2"][e].double())
    # three roundings to bf16, of h, of a pick's row and of the sum; those of h meet I terms of w2's size I^-1/2
    assert (out.double() - want).norm() <= 3 * 2.0 ** -8 * want.norm()

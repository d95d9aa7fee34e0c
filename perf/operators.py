"""The unquantised expert path around the exchange, as cases that can be timed: the router that picks experts by groups, the
experts' own matrix products, and the gradients of all of it.

Three operators, each through the library's public entry points:
  route     Buffer.group_route: logits [tokens, experts] -> the top-k experts of the best groups and their weights;
            Buffer.group_route_backward: the logits' gradient from the weights';
  linear    Buffer.expert_linear: rows sorted by expert times the experts' weights, with bias, activation and residual;
            Buffer.expert_linear_backward: the gradients of the rows, the weights, the bias and the pre-activation;
  combine   Buffer.combine_backward: the gradients of the experts' rows and of the routing weights.

7168 x 2048 with 32 local experts, top-8, is this repository's benchmark layer (the first product of an expert makes gate and up,
2 x 2048 columns); 2048 x 1024 with 64 experts, top-6, is a generic small one.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh", "swiglu")


def _route(name, tokens, experts, topk, groups=1, kept=1, score="sigmoid", group_score="top2", bias=True, renorm=True,
           scale=1.0, dtype="fp32", masked=False, backward=False):
    return {"name": name, "kind": "route", "tokens": tokens, "experts": experts, "topk": topk, "groups": groups, "kept": kept,
            "score": score, "group_score": group_score, "bias": bias, "renorm": renorm, "scale": scale, "dtype": dtype,
            "masked": masked, "backward": backward}


def _linear(name, rows, experts, k, n, activation="none", bias=False, residual=False, dtype="bf16", out="same",
            transposed=False, zipf=False, preact=False, backward=False, grad="same"):
    return {"name": name, "kind": "linear", "rows": rows, "experts": experts, "k": k, "n": n, "activation": activation,
            "bias": bias, "residual": residual, "dtype": dtype, "out": out, "transposed": transposed, "zipf": zipf,
            "preact": preact, "backward": backward, "grad": grad}


def _combine(name, tokens, hidden, experts, topk, dtype="bf16", missing=False):
    return {"name": name, "kind": "combine", "tokens": tokens, "hidden": hidden, "experts": experts, "topk": topk,
            "dtype": dtype, "missing": missing}


def listed():
    return [
        # the router of a decode step of a nearly idle engine: eight groups of 32 experts, four of them kept
        _route("route 7", 7, 256, 8, 8, 4, scale=2.5),
        # the same router on a prefill batch
        _route("route 8192", 8192, 256, 8, 8, 4, scale=2.5),
        # a training batch: the logits' gradient where every expert's score depends on all logits
        _route("route back 16384", 16384, 128, 8, score="softmax", bias=False, renorm=False, backward=True),
        # two tokens being decoded, eight experts each: gate and up of the experts that they reach
        _linear("linear decode 16", 16, 32, 7168, 4096, "swiglu"),
        # one token through a dense second product with its residual, weights as a checkpoint holds them
        _linear("linear 1 residual", 1, 1, 2048, 7168, residual=True, transposed=True),
        # the router's own product for a prefill batch: few columns, a long sum, logits in 32 bits
        _linear("linear gate 4096", 4096, 1, 7168, 256, out="fp32"),
        # gate and up of the benchmark's prefill batch, eight picks of 4096 tokens over 32 experts
        _linear("linear prefill 32768", 32768, 32, 7168, 4096, "swiglu"),
        # sizes that no tile divides, every part of the epilogue
        _linear("linear odd 1021", 1021, 1, 1001, 1531, "gelu", bias=True, residual=True, dtype="fp16"),
        # a training step's second product, weight gradients kept in 32 bits
        _linear("linear back 16384", 16384, 32, 2048, 7168, backward=True, grad="fp32"),
        # a small layer's first product in training: the activation's gradient, the bias's, few rows to an expert
        _linear("linear back 1021", 1021, 64, 2048, 2048, "swiglu", bias=True, backward=True),
        # the exchange's gradient for the benchmark's batch
        _combine("combine back 4096", 4096, 7168, 32, 8),
        # the same for a small layer and a small batch, picks that went nowhere among it
        _combine("combine back 61", 61, 2048, 64, 6, missing=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """A width: mostly a multiple of 64, now and then of 8, now and then anything."""
    v, step = _log_int(rng, lo, hi), rng.choice([64, 64, 64, 8, 1])
    return max(step, v // step * step)


def draw(rng):
    u = rng.random()
    if u < 0.3:
        per, groups = rng.choice([(8, 8), (32, 8), (16, 4), (17, 6), (64, 1), (128, 1), (100, 1), (60, 1), (24, 16)])
        kept = rng.randint(max(1, groups // 4), groups) if groups > 1 else 1
        back = rng.random() < 0.4
        case = _route(None, _log_int(rng, 1, 16384), per * groups, rng.randint(1, min(16, per * kept)), groups, kept,
                      rng.choice(["sigmoid", "softmax"]), rng.choice(["top2", "max"]), rng.random() < 0.6, rng.random() < 0.7,
                      rng.choice([1.0, 2.5]), rng.choice(["fp32", "fp32", "bf16", "fp16"]), rng.random() < 0.25, back)
    elif u < 0.85:
        back = rng.random() < 0.4
        experts = rng.choice([1, 1, 8, 32, 64])
        act = rng.choice(ACTIVATIONS)
        k, n = _size(rng, 256, 7168), _size(rng, 128, 7168)
        if act == "swiglu":
            n += n % 2
        experts = min(experts, int(9e8 / (k * n)))
        zipf = experts > 1 and rng.random() < 0.25
        most = min(32768, (4e11 if back else 1.2e12) / (2 * k * n), 2.4e8 / max(k, n)) / (8 if zipf else 1)
        rows = _log_int(rng, 1, max(2, int(most)))
        case = _linear(None, rows, experts, k, n, act, rng.random() < 0.4, not back and act != "swiglu" and rng.random() < 0.4,
                       rng.choice(["bf16", "bf16", "fp16"]), "fp32" if not back and rng.random() < 0.2 else "same",
                       rng.random() < 0.4, zipf, not back and act != "none" and rng.random() < 0.3,
                       back, "fp32" if act == "none" and rng.random() < 0.5 else "same")
    else:
        hidden, experts, topk = rng.choice([(7168, 32, 8), (4096, 128, 8), (2048, 64, 6), (1040, 16, 3)])
        case = _combine(None, _log_int(rng, 1, 4096), hidden, experts, topk, rng.choice(["bf16", "fp16"]), rng.random() < 0.3)
    del case["name"]
    return case


# ---- what a user's program has in hand before the call ---------------------------------------------------------------

_buffer = None


def buffer():
    """The one Buffer a program keeps."""
    global _buffer
    if _buffer is None:
        from memfabric_hybrid_amd.buffer import Buffer
        _buffer = Buffer()
    return _buffer


def _picks(g, tokens, experts, topk):
    """Distinct experts for every token, uniform."""
    return torch.topk(torch.rand((tokens, experts), device="cuda", generator=g), topk, dim=-1).indices.contiguous()


def _prepare_route(case, g):
    t, e = case["tokens"], case["experts"]
    logits = torch.randn((t, e), device="cuda", generator=g) * 1.5
    if case["masked"]:            # experts that a program has switched off, another choice for every token
        logits.masked_fill_(torch.rand((t, e), device="cuda", generator=g) < 0.3, -math.inf)
    s = dict(case, logits=logits.to(TYPES[case["dtype"]]), bias=None)
    if case["bias"]:
        s["bias"] = torch.randn((e,), device="cuda", generator=g) * 0.05
    if case["backward"]:
        s["idx"] = _picks(g, t, e, case["topk"])
        if case["masked"]:        # a pick that is not there, as the router leaves it
            s["idx"][torch.rand(s["idx"].shape, device="cuda", generator=g) < 0.2] = -1
        s["grad"] = torch.randn((t, case["topk"]), device="cuda", generator=g)
    return s


def _prepare_linear(case, g):
    rows, e, k, n, dt = case["rows"], case["experts"], case["k"], case["n"], TYPES[case["dtype"]]
    out = dt if case["out"] == "same" else TYPES[case["out"]]
    p = 1.0 / torch.arange(1, e + 1, device="cuda") ** (1.2 if case["zipf"] else 0.0)
    picked = torch.multinomial(p, rows, replacement=True, generator=g)
    counts = torch.bincount(picked, minlength=e)
    s = dict(case, dt=dt, out=out, counts=counts.to(torch.int32), cap=int(counts.max()),
             x=torch.randn((rows, k), device="cuda", generator=g).to(dt), residual=None, bias=None)
    shape = (e, n, k) if case["transposed"] else (e, k, n)
    s["w"] = torch.empty(shape, device="cuda", dtype=dt).normal_(generator=g).mul_(k ** -0.5)
    if case["bias"]:
        s["bias"] = torch.randn((e, n), device="cuda", generator=g).to(dt)
    cols = n // 2 if case["activation"] == "swiglu" else n
    if case["residual"]:
        s["residual"] = torch.randn((rows, cols), device="cuda", generator=g).to(out)
    if case["backward"]:
        s["grad_out"] = torch.randn((rows, cols), device="cuda", generator=g).to(dt)
        s["z"] = torch.randn((rows, n), device="cuda", generator=g).to(dt) if case["activation"] != "none" else None
        s["wgrad"] = dt if case["grad"] == "same" else TYPES[case["grad"]]
    return s


def _prepare_combine(case, g):
    t, k, h, e, dt = case["tokens"], case["topk"], case["hidden"], case["experts"], TYPES[case["dtype"]]
    idx = _picks(g, t, e, k)
    if case["missing"]:           # a fifth of the picks, wherever they are
        idx.view(-1)[torch.randperm(t * k, device="cuda", generator=g)[:t * k // 5]] = -1
    flat = idx.flatten()
    # expert by expert, in pick order: where the dispatch puts the pick's row
    order = torch.sort(torch.where(flat < 0, e, flat), stable=True).indices
    row = torch.empty_like(order)
    row[order] = torch.arange(t * k, device="cuda")
    rows = int((flat >= 0).sum())
    w = torch.rand((t, k), device="cuda", generator=g)
    s = dict(case, row=torch.where(flat < 0, rows, row).view(t, k), rows=rows, weights=w,
             x=torch.randn((max(rows, 1), h), device="cuda", generator=g).to(dt),
             grad=torch.randn((t, h), device="cuda", generator=g).to(dt))
    if own:          # the handle that the exchange gave the program in the forward pass
        b = buffer()
        per_rank, _, per_expert, in_rank, _ = b.get_dispatch_layout(idx, e)
        s["handle"] = b.dispatch(s["grad"], num_tokens_per_rank=per_rank, is_token_in_rank=in_rank,
                                 num_tokens_per_expert=per_expert, topk_idx=idx, topk_weights=w)[4]
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"route": _prepare_route, "linear": _prepare_linear, "combine": _prepare_combine}[case["kind"]](case, g)


# ---- the plain forms -------------------------------------------------------------------------------------------------

def _scores(logits, score):
    """In 64 bits: the picks turn on the difference of two scores, however small."""
    l64 = logits.double()
    if score == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-l64))
    e = torch.exp(l64 - l64.max(dim=-1, keepdim=True).values)
    return e / e.sum(dim=-1, keepdim=True)


def _plain_route(s):
    t, e, groups, k = s["tokens"], s["experts"], s["groups"], s["topk"]
    score = _scores(s["logits"], s["score"])
    choice = score if s["bias"] is None else score + s["bias"].double()
    choice = torch.where((s["logits"] > -math.inf) & (choice > -math.inf), choice, -math.inf)
    if groups > 1:
        g = choice.view(t, groups, e // groups)
        best, at = g.max(dim=-1, keepdim=True)
        if s["group_score"] == "top2" and e > groups:
            rest = g.masked_fill(torch.arange(e // groups, device="cuda") == at, -math.inf).max(dim=-1, keepdim=True).values
            best = best + torch.where(rest > -math.inf, rest, 0.0)
        # the groups in falling order, equal ones by their index
        kept = torch.sort(best.squeeze(-1), dim=-1, descending=True, stable=True).indices[:, :s["kept"]]
        mask = torch.zeros((t, groups), dtype=torch.bool, device="cuda").scatter_(1, kept, True)
        choice = torch.where(mask[:, :, None], g, -math.inf).view(t, e)
    value, idx = torch.sort(choice, dim=-1, descending=True, stable=True)
    idx, there = idx[:, :k], value[:, :k] > -math.inf
    w = torch.where(there, torch.gather(score, 1, idx), 0.0)
    if s["renorm"]:
        total = w.sum(dim=-1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    return torch.where(there, idx, -1), (w * s["scale"]).float()


def _plain_route_back(s):
    score = _scores(s["logits"], s["score"])
    there, at = s["idx"] >= 0, s["idx"].clamp(min=0)
    picked = torch.where(there, torch.gather(score, 1, at), 0.0)
    d = torch.where(there, s["grad"].double(), 0.0) * s["scale"]
    if s["renorm"]:
        total = picked.sum(dim=-1, keepdim=True)
        d = torch.where(there & (total > 0), (d - (d * picked).sum(dim=-1, keepdim=True) / total) / total, 0.0)
    dscore = torch.zeros_like(score).scatter_add_(1, at, d)
    if s["score"] == "sigmoid":
        r = dscore * score * (1.0 - score)
    else:
        r = score * (dscore - (dscore * score).sum(dim=-1, keepdim=True))
    return r.to(s["logits"].dtype)


def _activate(z, name):
    if name == "relu":
        return torch.where(z > 0, z, 0.0)
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if name == "swiglu":
        gate, up = z.chunk(2, dim=-1)
        return gate / (1.0 + torch.exp(-gate)) * up
    return z


def _slope(z, name):
    """d activation / dz."""
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "silu":
        p = 1.0 / (1.0 + torch.exp(-z))
        return p * (1.0 + z * (1.0 - p))
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    c = math.sqrt(2.0 / math.pi)
    th = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * (1.0 + th) + 0.5 * z * (1.0 - th * th) * c * (1.0 + 3 * 0.044715 * z * z)


def _plan(s):
    """Row r is row `pos[r]` of expert `eid[r]`; `idx` [experts, cap]: the row there, or one past the last."""
    counts, rows, e = s["counts"].long(), s["rows"], s["experts"]
    start = torch.cumsum(counts, 0) - counts
    at = torch.arange(s["cap"], device="cuda")
    idx = torch.where(at < counts[:, None], start[:, None] + at, rows)
    eid = torch.repeat_interleave(torch.arange(e, device="cuda"), counts, output_size=rows)
    return idx, eid, torch.arange(rows, device="cuda") - start[eid]


def _padded(rows, idx):
    """[experts, cap, width] in 32 bits, zeros where an expert has no such row."""
    return torch.cat([rows.float(), torch.zeros((1, rows.shape[1]), device="cuda")])[idx]


def _weights(s):
    """[experts, k, n] in 32 bits"""
    w = s["w"].float()
    return w.transpose(1, 2).contiguous() if s["transposed"] else w


def _plain_linear(s):
    if s["experts"] == 1:
        z = s["x"].float() @ _weights(s)[0]
        b = s["bias"].float() if s["bias"] is not None else None
    else:
        idx, eid, pos = _plan(s)
        z = torch.bmm(_padded(s["x"], idx), _weights(s))[eid, pos]
        b = s["bias"].float()[eid] if s["bias"] is not None else None
    if b is not None:
        z = z + b
    y = _activate(z, s["activation"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return (y.to(s["out"]), z.to(s["dt"])) if s["preact"] else y.to(s["out"])


def _plain_linear_back(s):
    d, act = s["grad_out"].float(), s["activation"]
    if act == "swiglu":
        gate, up = s["z"].float().chunk(2, dim=-1)
        d = torch.cat([d * up * _slope(gate, "silu"), d * gate / (1.0 + torch.exp(-gate))], dim=-1)
    elif act != "none":
        d = d * _slope(s["z"].float(), act)
    # the pre-activation's gradient is a tensor of the operator's, in the rows' type, and the products take it from there
    d = d.to(s["dt"])
    wt = s["w"].float() if s["transposed"] else s["w"].float().transpose(1, 2).contiguous()
    if s["experts"] == 1:
        dp, xp = d.float()[None], s["x"].float()[None]
        dx = (dp[0] @ wt[0])
    else:
        idx, eid, pos = _plan(s)
        dp, xp = _padded(d, idx), _padded(s["x"], idx)
        dx = torch.bmm(dp, wt)[eid, pos]
    a, b = (dp, xp) if s["transposed"] else (xp, dp)
    dw = torch.bmm(a.transpose(1, 2).contiguous(), b)
    r = {"dx": dx.to(s["dt"]), "dw": dw.to(s["wgrad"])}
    if s["bias"] is not None:
        r["db"] = dp.sum(dim=1).to(s["wgrad"])
    if act != "none":
        r["dz"] = d
    return r


def _plain_combine_back(s):
    row, grad, rows = s["row"], s["grad"].float(), s["rows"]
    x = torch.cat([s["x"][:rows].float(), torch.zeros((1, s["hidden"]), device="cuda")])
    dw = (x[row] * grad[:, None, :]).sum(dim=-1)
    dx = torch.empty((rows + 1, s["hidden"]), device="cuda", dtype=s["x"].dtype)
    dx[row.flatten()] = (s["weights"][:, :, None] * grad[:, None, :]).to(dx.dtype).flatten(0, 1)
    return {"dx": dx[:rows], "dw": dw}


# ---- one pass --------------------------------------------------------------------------------------------------------

def _own(s):
    b, kind = buffer(), s["kind"]
    if kind == "route" and s["backward"]:
        return b.group_route_backward(s["grad"], s["logits"], s["idx"], score=s["score"], renormalize=s["renorm"],
                                      scale=s["scale"])
    if kind == "route":
        return b.group_route(s["logits"], s["topk"], num_groups=s["groups"], topk_groups=s["kept"], score=s["score"],
                             bias=s["bias"], group_score=s["group_score"], renormalize=s["renorm"], scale=s["scale"])
    if kind == "combine":
        dx, dw = b.combine_backward(s["grad"], s["x"], s["handle"])
        return {"dx": dx[:s["rows"]], "dw": dw}
    counts = s["counts"] if s["experts"] > 1 else None
    if s["backward"]:
        dx, dw, db, dz = b.expert_linear_backward(s["grad_out"], s["x"], s["w"], counts, activation=s["activation"],
                                                  preact=s["z"], transposed=s["transposed"], bias=s["bias"] is not None,
                                                  weight_grad_dtype=s["wgrad"])
        r = {"dx": dx, "dw": dw}
        if db is not None:
            r["db"] = db
        if s["activation"] != "none":
            r["dz"] = dz
        return r
    return b.expert_linear(s["x"], s["w"], counts, bias=s["bias"], activation=s["activation"], residual=s["residual"],
                           out_dtype=s["out"], transposed=s["transposed"], return_preact=s["preact"])


def run(state):
    if own:
        return _own(state)
    if state["kind"] == "route":
        return _plain_route_back(state) if state["backward"] else _plain_route(state)
    if state["kind"] == "combine":
        return _plain_combine_back(state)
    return _plain_linear_back(state) if state["backward"] else _plain_linear(state)


# ---- what a pass cannot do without, and how exact it is ---------------------------------------------------------------

def _bytes(name):
    return 4 if name == "fp32" else 2


def work(case):
    if case["kind"] == "route":
        values, picks = case["tokens"] * case["experts"], case["tokens"] * case["topk"]
        if not case["backward"]:
            return {"bytes": values * _bytes(case["dtype"]) + picks * 12, "flops": values * 8}
        # the scores of all experts are needed where each depends on all logits, else those of the picks
        read = values if case["score"] == "softmax" and not case["renorm"] else picks
        return {"bytes": (read + values) * _bytes(case["dtype"]) + picks * 12, "flops": read * 8}
    if case["kind"] == "combine":
        cells = case["tokens"] * case["hidden"]
        rows = case["topk"] * (0.8 if case["missing"] else 1.0)
        return {"bytes": cells * 2 * (1 + 2 * rows) + case["tokens"] * case["topk"] * 20, "flops": 3 * cells * rows}
    rows, e, k, n = case["rows"], case["experts"], case["k"], case["n"]
    cols = n // 2 if case["activation"] == "swiglu" else n
    reached = e if case["zipf"] else e * (1 - (1 - 1 / e) ** rows)
    out = 2 if case["out"] == "same" else 4
    if not case["backward"]:
        return {"bytes": 2 * (rows * k + reached * k * n) + rows * cols * out * (2 if case["residual"] else 1) +
                (rows * n * 2 if case["preact"] else 0) + (reached * n * 2 if case["bias"] else 0), "flops": 2 * rows * k * n}
    grad = 2 if case["grad"] == "same" else 4
    more = 0 if case["activation"] == "none" else 2 * rows * n * 2
    return {"bytes": 2 * (rows * cols + 2 * rows * k + reached * k * n) + e * k * n * grad + more, "flops": 4 * rows * k * n}


def _exact_route(s):
    logits, e, k = s["logits"].double(), s["experts"], s["topk"]
    score = torch.sigmoid(logits) if s["score"] == "sigmoid" else torch.softmax(logits, dim=-1)
    if s["backward"]:
        there = s["idx"] >= 0
        w = logits.clone().requires_grad_()
        p = torch.sigmoid(w) if s["score"] == "sigmoid" else torch.softmax(w, dim=-1)
        p = torch.gather(p, 1, s["idx"].clamp(min=0)) * there
        if s["renorm"]:
            total = p.sum(dim=-1, keepdim=True)
            p = p / torch.where(total > 0, total, 1.0)
        (p * s["scale"] * torch.where(there, s["grad"].double(), 0.0)).sum().backward()
        return w.grad
    choice = score if s["bias"] is None else score + s["bias"].double()
    choice = choice.masked_fill(torch.isinf(logits) | torch.isnan(choice), -math.inf)
    per = e // s["groups"]
    top = torch.topk(choice.view(-1, s["groups"], per), min(2 if s["group_score"] == "top2" else 1, per), dim=-1).values
    of_group = torch.where(top[..., :1] > -math.inf, torch.where(top > -math.inf, top, 0.0).sum(-1, keepdim=True), -math.inf)
    rank = torch.argsort(torch.argsort(of_group[..., 0], dim=-1, descending=True, stable=True), dim=-1)
    choice = choice.masked_fill((rank >= s["kept"]).repeat_interleave(per, dim=-1), -math.inf)
    order = torch.argsort(choice, dim=-1, descending=True, stable=True)[:, :k]
    there = torch.gather(choice, 1, order) > -math.inf
    w = torch.where(there, torch.gather(score, 1, order), 0.0)
    if s["renorm"]:
        w = w / w.sum(dim=-1, keepdim=True).clamp(min=1e-300)
    return order.masked_fill(~there, -1), w * s["scale"]


def _exact_linear(s):
    rows, e, act = s["rows"], s["experts"], s["activation"]
    ends = torch.cumsum(s["counts"], 0).tolist()
    spans = list(zip([0] + ends[:-1], ends))
    f = {"none": lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
         "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh"),
         "swiglu": lambda z: torch.nn.functional.silu(z[:, :z.shape[1] // 2]) * z[:, z.shape[1] // 2:]}[act]
    if not s["backward"]:
        ys, zs = [], []
        for i, (a, b) in enumerate(spans):
            w = s["w"][i].double()
            z = s["x"][a:b].double() @ (w.t() if s["transposed"] else w)
            if s["bias"] is not None:
                z = z + s["bias"][i].double()
            ys.append(f(z))
            zs.append(z if s["preact"] else z[:, :0])
        y = torch.cat(ys)
        if s["residual"] is not None:
            y = y + s["residual"].double()
        return (y, torch.cat(zs)) if s["preact"] else y
    d = s["grad_out"].double()
    if act != "none":
        z = s["z"].double().requires_grad_()
        f(z).backward(d)
        d = z.grad
    dz, d = d, d.to(s["dt"])                        # the tensor that the products take
    dx, dw, db = [], torch.empty(s["w"].shape, device="cuda", dtype=torch.float64), []
    for i, (a, b) in enumerate(spans):
        w, di, xi = s["w"][i].double(), d[a:b].double(), s["x"][a:b].double()
        dx.append(di @ (w if s["transposed"] else w.t()))
        dw[i] = di.t() @ xi if s["transposed"] else xi.t() @ di
        db.append(di.sum(0))
    r = {"dx": torch.cat(dx), "dw": dw}
    if s["bias"] is not None:
        r["db"] = torch.stack(db)
    if act != "none":
        r["dz"] = dz
    return r


def _exact_combine(s):
    row, grad, rows = s["row"], s["grad"].double(), s["rows"]
    dw = torch.zeros(row.shape, device="cuda", dtype=torch.float64)
    dx = torch.zeros((rows + 1, s["hidden"]), device="cuda", dtype=torch.float64)
    for k in range(s["topk"]):
        at = row[:, k]
        there = at < rows
        dw[:, k] = torch.einsum("th,th->t", s["x"][at.clamp(max=max(rows - 1, 0))].double(), grad) * there
        dx[at] = s["weights"][:, k:k + 1].double() * grad
    return {"dx": dx[:rows], "dw": dw}


def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _exact_route, "linear": _exact_linear, "combine": _exact_combine}[case["kind"]](s)

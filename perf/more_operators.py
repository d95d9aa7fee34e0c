"""What stands around the int8 exchange, as cases that can be timed: the norm in front of it, whose rows the router reads and whose int8
rows the products read, the experts' int8 products with a scale for each token and channel, and the activation between two of them.

Three operators, each through the library's public entry points:
  norm      Buffer.rms_norm: rows and the residual -> their sum, its root-mean-square norm, and that in int8 with a scale a row;
            Buffer.rms_norm_backward: the gradients of the rows and of the weight;
  linear8   Buffer.expert_linear_int8: int8 rows sorted by expert times the experts' int8 weights, with the scales of both, bias,
            activation and residual;
  quant     Buffer.quantize_rows: an activation, and its result in int8 with a scale a row.

7168 x 2048 with 32 local experts, top-8, is this repository's benchmark layer (the first product of an expert makes gate and up,
2 x 2048 columns); 2048 x 1024 with 64 experts is a generic small one. What is held in int8 is returned as the values it stands
for, in the type of the rows that it was made from (bf16 for those of 32 bits).
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh", "swiglu")
EPS = 1e-6


def _norm(name, tokens, hidden, residual=True, norm=True, int8=False, weight="same", dtype="bf16", backward=False, grad="same"):
    return {"name": name, "kind": "norm", "tokens": tokens, "hidden": hidden, "residual": residual, "norm": norm, "int8": int8,
            "weight": weight, "dtype": dtype, "backward": backward, "grad": grad}


def _linear8(name, rows, experts, k, n, activation="none", bias=False, residual=False, out="bf16", zipf=False):
    return {"name": name, "kind": "linear8", "rows": rows, "experts": experts, "k": k, "n": n, "activation": activation,
            "bias": bias, "residual": residual, "out": out, "zipf": zipf}


def _quant(name, rows, width, activation="swiglu", dtype="bf16"):
    return {"name": name, "kind": "quant", "rows": rows, "width": width, "activation": activation, "dtype": dtype}


def listed():
    return [
        # one token being decoded, in front of an int8 projection: only the int8 rows and the residual stream are wanted
        _norm("norm decode 1", 1, 7168, norm=False, int8=True),
        # a prefill batch in front of the experts: the router reads the norm, the experts its int8 rows
        _norm("norm prefill 4096", 4096, 7168, int8=True),
        # the first norm of a stack, which has no residual yet: a size that nothing divides, in 32 bits
        _norm("norm odd 1021", 1021, 1531, residual=False, dtype="fp32"),
        # a training batch: the gradient that comes down the residual stream joins in, weight gradient kept in 32 bits
        _norm("norm back 16384", 16384, 2048, backward=True, grad="fp32"),
        # a short sequence of wide rows
        _norm("norm back 61", 61, 7168, residual=False, backward=True, dtype="fp16"),
        # two tokens being decoded, eight experts each: gate and up of the experts that they reach
        _linear8("int8 decode 16", 16, 32, 7168, 4096, "swiglu"),
        # one token through a dense second product with its residual
        _linear8("int8 1 residual", 1, 1, 2048, 7168, residual=True),
        # gate and up of the benchmark's prefill batch, eight picks of 4096 tokens over 32 experts
        _linear8("int8 prefill 32768", 32768, 32, 7168, 4096, "swiglu"),
        # sizes that no tile divides, every part of the epilogue
        _linear8("int8 odd 1021", 1021, 1, 1001, 1531, "gelu", bias=True, residual=True, out="fp16"),
        # a small layer's second product, a few rows to an expert, kept in 32 bits for the weighted sum
        _linear8("int8 small 1021", 1021, 64, 1024, 2048, out="fp32"),
        # between the two products of the benchmark's prefill batch
        _quant("swiglu rows 32768", 32768, 4096),
        # and of a decode step
        _quant("swiglu rows 16", 16, 4096),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """A width: mostly a multiple of 64, now and then of 8, now and then anything."""
    v, step = _log_int(rng, lo, hi), rng.choice([64, 64, 64, 8, 1])
    return max(step, v // step * step)


def draw(rng):
    u = rng.random()
    if u < 0.4:
        hidden, dtype, back = _size(rng, 64, 8192), rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.random() < 0.4
        tokens = _log_int(rng, 1, min(16384, int(2.9e7 / hidden)))
        int8 = not back and rng.random() < 0.5
        case = _norm(None, tokens, hidden, rng.random() < 0.7, not int8 or rng.random() < 0.5, int8, rng.choice(["same", "fp32"]),
                     dtype, back, rng.choice(["same", "fp32"]) if back else "same")
    elif u < 0.8:
        experts, act = rng.choice([1, 1, 8, 32, 64]), rng.choice(ACTIVATIONS)
        k, n = _size(rng, 128, 7168), _size(rng, 128, 7168)
        if act == "swiglu":
            n += n % 2
        experts = min(experts, int(9e8 / (k * n)))
        zipf = experts > 1 and rng.random() < 0.25
        most = min(32768, 1.2e12 / (2 * k * n), 2.4e8 / max(k, n)) / (8 if zipf else 1)
        case = _linear8(None, _log_int(rng, 1, max(2, int(most))), experts, k, n, act, rng.random() < 0.4,
                        act != "swiglu" and rng.random() < 0.4, rng.choice(["bf16", "bf16", "fp16", "fp32"]), zipf)
    else:
        act = rng.choice(("none", "swiglu", "swiglu", "silu", "relu", "gelu", "gelu_tanh"))
        width = _size(rng, 64, 8192)
        width += width % 2
        case = _quant(None, _log_int(rng, 1, min(32768, int(1.3e8 / width))), width, act, rng.choice(["bf16", "bf16", "fp16", "fp32"]))
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


def _prepare_norm(case, g):
    t, h, dt = case["tokens"], case["hidden"], TYPES[case["dtype"]]
    # a residual stream has tokens of different sizes, and some channels that are larger than others
    size = torch.exp(torch.randn((t, 1), device="cuda", generator=g) * 0.5)
    channel = torch.exp(torch.randn((h,), device="cuda", generator=g) * 0.3)
    s = dict(case, dt=dt, x=(torch.randn((t, h), device="cuda", generator=g) * size * channel).to(dt), res=None, gtotal=None)
    s["w"] = (1.0 + 0.2 * torch.randn((h,), device="cuda", generator=g)).to(dt if case["weight"] == "same" else torch.float32)
    if case["backward"]:
        s["grad_out"] = torch.randn((t, h), device="cuda", generator=g).to(dt)
        s["wgrad"] = s["w"].dtype if case["grad"] == "same" else torch.float32
        if case["residual"]:
            s["gtotal"] = torch.randn((t, h), device="cuda", generator=g).to(dt)
    elif case["residual"]:
        s["res"] = (torch.randn((t, h), device="cuda", generator=g) * size).to(dt)
    return s


def _int8(shape, g):
    """Rows of normally distributed values, scaled so that four standard deviations reach the end of the range."""
    return (torch.randn(shape, device="cuda", generator=g) * 32.0).round_().clamp_(-127, 127).to(torch.int8)


def _prepare_linear8(case, g):
    rows, e, k, n, out = case["rows"], case["experts"], case["k"], case["n"], TYPES[case["out"]]
    p = 1.0 / torch.arange(1, e + 1, device="cuda") ** (1.2 if case["zipf"] else 0.0)
    picked = torch.multinomial(p, rows, replacement=True, generator=g)
    counts = torch.bincount(picked, minlength=e)
    s = dict(case, dt=out, counts=counts.to(torch.int32), cap=int(counts.max()), x=_int8((rows, k), g), residual=None, bias=None)
    s["xs"] = torch.exp(torch.randn((rows,), device="cuda", generator=g) * 0.5) / 32.0
    s["w"] = torch.empty((e, n, k), device="cuda", dtype=torch.int8)
    for i in range(e):
        s["w"][i] = _int8((n, k), g)
    s["ws"] = torch.exp(torch.randn((e, n), device="cuda", generator=g) * 0.3) * (k ** -0.5 / 32.0)
    if case["bias"]:
        s["bias"] = torch.randn((e, n), device="cuda", generator=g)
    if case["residual"]:
        s["residual"] = torch.randn((rows, n // 2 if case["activation"] == "swiglu" else n), device="cuda", generator=g).to(out)
    return s


def _prepare_quant(case, g):
    x = torch.randn((case["rows"], case["width"]), device="cuda", generator=g).to(TYPES[case["dtype"]])
    return dict(case, x=x)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"norm": _prepare_norm, "linear8": _prepare_linear8, "quant": _prepare_quant}[case["kind"]](case, g)


def _of_values(s):
    """The type of the values that int8 rows stand for."""
    return torch.bfloat16 if s["dtype"] == "fp32" else TYPES[s["dtype"]]


# ---- the plain forms -------------------------------------------------------------------------------------------------

def _quantize(y):
    """int8 rows and their scales: the largest of a row becomes 127; a row of zeros has the scale 0."""
    amax = y.abs().max(dim=-1, keepdim=True).values
    q = torch.round(y * torch.where(amax > 0, 127.0 / amax, 0.0))
    return q, (amax / 127.0)[:, 0]


def _plain_norm(s):
    h = s["x"].float()
    if s["res"] is not None:
        h = h + s["res"].float()
    y = h * (1.0 / torch.sqrt((h * h).mean(dim=-1, keepdim=True) + EPS)) * s["w"].float()
    r = {}
    if s["res"] is not None:
        r["total"] = h.to(s["dt"])
    if s["norm"]:
        r["y"] = y.to(s["dt"])
    if s["int8"]:
        q, r["scales"] = _quantize(y)
        r["values"] = (q * r["scales"][:, None]).to(_of_values(s))
    return r


def _plain_norm_back(s):
    h, g = s["x"].float(), s["grad_out"].float()
    r = 1.0 / torch.sqrt((h * h).mean(dim=-1, keepdim=True) + EPS)
    n, d = h * r, g * s["w"].float()
    dx = r * (d - n * (d * n).mean(dim=-1, keepdim=True))
    if s["gtotal"] is not None:
        dx = dx + s["gtotal"].float()
    return {"dx": dx.to(s["dt"]), "dw": (g * n).sum(dim=0).to(s["wgrad"])}


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


def _plain_linear8(s):
    rows, e, w = s["rows"], s["experts"], s["w"].float()
    if e == 1:
        z, eid = s["x"].float() @ w[0].t(), torch.zeros((1,), dtype=torch.int64, device="cuda")
    else:
        # row r is row `pos[r]` of expert `eid[r]`; `idx` [experts, cap]: the row there, or one past the last
        counts = s["counts"].long()
        start = torch.cumsum(counts, 0) - counts
        at = torch.arange(s["cap"], device="cuda")
        idx = torch.where(at < counts[:, None], start[:, None] + at, rows)
        eid = torch.repeat_interleave(torch.arange(e, device="cuda"), counts, output_size=rows)
        pos = torch.arange(rows, device="cuda") - start[eid]
        x = torch.cat([s["x"].float(), torch.zeros((1, s["k"]), device="cuda")])[idx]
        z = torch.bmm(w, x.transpose(1, 2).contiguous()).transpose(1, 2)[eid, pos]
    z = z * s["ws"][eid] * s["xs"][:, None]
    if s["bias"] is not None:
        z = z + s["bias"][eid]
    y = _activate(z, s["activation"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["dt"])


def _plain_quant(s):
    q, scales = _quantize(_activate(s["x"].float(), s["activation"]))
    return {"values": (q * scales[:, None]).to(_of_values(s)), "scales": scales}


# ---- one pass --------------------------------------------------------------------------------------------------------

def _values(q, scales, s):
    return torch.mul(q, scales[:, None], out=torch.empty(q.shape, dtype=_of_values(s), device="cuda"))


def _own(s):
    b, kind = buffer(), s["kind"]
    if kind == "norm" and s["backward"]:
        dx, dw = b.rms_norm_backward(s["grad_out"], s["x"], s["w"], grad_total=s["gtotal"], eps=EPS, weight_grad_dtype=s["wgrad"])
        return {"dx": dx, "dw": dw}
    if kind == "norm":
        y, q, scales, total = b.rms_norm(s["x"], s["w"], residual=s["res"], eps=EPS, need_norm=s["norm"], quantize=s["int8"])
        r = {"total": total, "y": y}
        if s["int8"]:
            r["scales"], r["values"] = scales, _values(q, scales, s)
        return {name: v for name, v in r.items() if v is not None}
    if kind == "quant":
        q, scales = b.quantize_rows(s["x"], activation=s["activation"])
        return {"values": _values(q, scales, s), "scales": scales}
    return b.expert_linear_int8(s["x"], s["xs"], s["w"], s["ws"], s["counts"] if s["experts"] > 1 else None, bias=s["bias"],
                                activation=s["activation"], residual=s["residual"], out_dtype=s["dt"])


def run(state):
    if own:
        return _own(state)
    if state["kind"] == "norm":
        return _plain_norm_back(state) if state["backward"] else _plain_norm(state)
    return _plain_quant(state) if state["kind"] == "quant" else _plain_linear8(state)


# ---- what a pass cannot do without, and how exact it is ---------------------------------------------------------------

def _bytes(name):
    return 4 if name == "fp32" else 2


def work(case):
    if case["kind"] == "norm":
        t, cells, b = case["tokens"], case["tokens"] * case["hidden"], _bytes(case["dtype"])
        if case["backward"]:
            return {"bytes": cells * b * (4 if case["residual"] else 3) + case["hidden"] * 4, "flops": cells * 10}
        return {"bytes": cells * (b * (1 + 2 * case["residual"] + case["norm"]) + case["int8"]) + case["hidden"] * b +
                t * 4 * case["int8"], "flops": cells * 6}
    if case["kind"] == "quant":
        cols = case["width"] // 2 if case["activation"] == "swiglu" else case["width"]
        return {"bytes": case["rows"] * (case["width"] * _bytes(case["dtype"]) + cols + 4), "flops": case["rows"] * cols * 8}
    rows, e, k, n, b = case["rows"], case["experts"], case["k"], case["n"], _bytes(case["out"])
    cols = n // 2 if case["activation"] == "swiglu" else n
    reached = e if case["zipf"] else e * (1 - (1 - 1 / e) ** rows)
    return {"bytes": rows * (k + 4) + reached * n * (k + 4 + 4 * case["bias"]) + rows * cols * b * (1 + case["residual"]),
            "flops": 2 * rows * k * n}


def _exact_int8(y):
    scales = y.abs().amax(dim=-1) / 127
    q = torch.round(y / torch.where(scales > 0, scales, 1.0)[:, None])
    return q * scales[:, None], scales


def _exact_norm(s):
    h = s["x"].double()
    if s["backward"]:
        h, w = h.requires_grad_(), s["w"].double().requires_grad_()
        y = h * torch.rsqrt(h.pow(2).mean(dim=-1, keepdim=True) + EPS) * w
        y.backward(s["grad_out"].double())
        return {"dx": h.grad if s["gtotal"] is None else h.grad + s["gtotal"].double(), "dw": w.grad}
    r = {}
    if s["res"] is not None:
        h = r["total"] = h + s["res"].double()
    y = h * torch.rsqrt(h.pow(2).mean(dim=-1, keepdim=True) + EPS) * s["w"].double()
    if s["norm"]:
        r["y"] = y
    if s["int8"]:
        r["values"], r["scales"] = _exact_int8(y)
    return r


def _act64(z, name):
    f = torch.nn.functional
    return {"none": lambda: z, "relu": lambda: torch.relu(z), "silu": lambda: f.silu(z), "gelu": lambda: f.gelu(z),
            "gelu_tanh": lambda: f.gelu(z, approximate="tanh"),
            "swiglu": lambda: f.silu(z[:, :z.shape[1] // 2]) * z[:, z.shape[1] // 2:]}[name]()


def _exact_linear8(s):
    ends = torch.cumsum(s["counts"], 0).tolist()
    ys = []
    for i, (a, b) in enumerate(zip([0] + ends[:-1], ends)):
        z = (s["x"][a:b].double() @ s["w"][i].double().t()) * s["xs"][a:b, None].double() * s["ws"][i].double()
        if s["bias"] is not None:
            z = z + s["bias"][i].double()
        ys.append(_act64(z, s["activation"]))
    y = torch.cat(ys)
    return y if s["residual"] is None else y + s["residual"].double()


def _exact_quant(s):
    values, scales = _exact_int8(_act64(s["x"].double(), s["activation"]))
    return {"values": values, "scales": scales}


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "linear8": _exact_linear8, "quant": _exact_quant}[case["kind"]](s)

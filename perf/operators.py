"""Measured cases of the dense operators: ``linear``, ``segment_matmul`` and ``layer_norm``.

``run`` makes one pass through an operator.  With ``own`` true it calls the package as a program would; with ``own``
false it computes the same in elementary torch operations in 32 bits, rounded once at the end.  ``exact`` computes it
in 64 bits.

Sizes are those of graphs the package is tested and benchmarked on (a 2,449,029-node product graph with 128 features,
a 232,965-node graph with 602 raw features and 4 x 64 = 256 hidden ones, 1 M nodes with 64 features, small test graphs
of 5,000 nodes) and plain powers of two.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ---- cases -----------------------------------------------------------------------------------------------------------
def _linear(name, dtype, m, k, n, act="none", bias=True, residual=False, train=False):
    case = dict(op="linear", dtype=dtype, m=m, k=k, n=n, act=act, bias=bias, residual=residual, train=train)
    return dict(case, name=name) if name else case


def _segment(name, dtype, m, k, n, groups, skew, bias=False, train=False):
    case = dict(op="segment_matmul", dtype=dtype, m=m, k=k, n=n, groups=groups, skew=skew, bias=bias, train=train)
    return dict(case, name=name) if name else case


def _norm(name, dtype, m, d, train=False):
    case = dict(op="layer_norm", dtype=dtype, m=m, d=d, train=train)
    return dict(case, name=name) if name else case


def listed():
    return [
        # the feature transform of a small test graph: launch and host latency
        _linear("linear-small", "f32", 5000, 16, 32),
        # one node answered online (a serving step's single row): the weight is all there is to read
        _linear("linear-one-row", "bf16", 1, 4096, 4096, act="silu"),
        # first layer over raw features of odd width (602: rows off every 16-byte grid), inference
        _linear("linear-raw-features", "bf16", 232_965, 602, 256, act="relu"),
        # a hidden layer of full-batch training on the product graph
        _linear("linear-products-train", "bf16", 2_449_029, 128, 256, act="gelu", train=True),
        # a skip-connected layer of full-batch training in single precision
        _linear("linear-skip-train", "f32", 1_000_000, 64, 64, act="silu", residual=True, train=True),
        # a wide feed-forward product over a batch of rows: bound by arithmetic
        _linear("linear-wide", "f16", 8192, 4096, 4096, act="gelu", residual=True),
        # relations of a small heterogeneous graph, some of them without rows: latency
        _segment("segments-small", "f32", 3001, 64, 64, 8, 1.0),
        # typed edge messages, 40 relations of very unequal size
        _segment("segments-typed-edges", "bf16", 1_000_003, 128, 128, 40, 1.0, bias=True),
        # rows routed to 64 experts, training
        _segment("segments-experts-train", "f16", 32_768, 1024, 2048, 64, 0.5, train=True),
        # typed node transforms in single precision, training
        _segment("segments-typed-train", "f32", 300_007, 64, 128, 12, 1.0, bias=True, train=True),
        # normalisation of the product graph's hidden rows, training
        _norm("norm-products-train", "bf16", 2_449_029, 128, train=True),
        # wide rows in single precision, inference
        _norm("norm-wide", "f32", 16_384, 4096),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    """One more case of the same ranges, at most as large as the largest listed one."""
    while True:
        op = rng.choice(["linear", "segment_matmul", "layer_norm"])
        dtype = rng.choice(["f32", "f16", "bf16"])
        train = rng.random() < 0.5
        m = _log_int(rng, 1, 2_449_029)
        if op == "layer_norm":
            case = _norm(None, dtype, m, _log_int(rng, 16, 8192), train=train)
        else:
            k, n = _log_int(rng, 16, 4096), _log_int(rng, 16, 4096)
            if rng.random() < 0.6:          # (most layers' widths are whole vectors; the rest stays as drawn, odd ones among them)
                k, n = (k + 7) // 8 * 8, (n + 7) // 8 * 8
            if op == "linear":
                # (no drawn gradient of relu: its step at 0 turns the last bit of a sum into a whole gradient)
                act = rng.choice(["none", "gelu", "silu"] if train else ["none", "relu", "gelu", "silu"])
                case = _linear(None, dtype, m, k, n, act=act, bias=rng.random() < 0.7, residual=rng.random() < 0.4, train=train)
            else:
                case = _segment(None, dtype, m, k, n, _log_int(rng, 1, 256), rng.choice([0.0, 0.5, 1.0]), bias=rng.random() < 0.4,
                                train=train)
        cost = work(case)
        if cost["bytes"] <= 6.5e9 and cost["flops"] <= (2.8e11 if dtype != "f32" else 7e10):
            return case


def work(case):
    e, m = BYTES[case["dtype"]], case["m"]
    if case["op"] == "layer_norm":
        d = case["d"]
        bytes_, flops = 2 * m * d * e + 2 * d * e, 8 * m * d
        if case["train"]:                       # x and dy read, dx written, dw and db written
            bytes_, flops = bytes_ + 2 * m * d * e + 2 * d * e, flops + 16 * m * d
        return {"bytes": bytes_, "flops": flops}
    k, n = case["k"], case["n"]
    groups = case.get("groups", 1)
    weights = groups * k * n * e + (groups * n * e if case["bias"] else 0)
    bytes_, flops = m * k * e + weights + m * n * e, 2 * m * n * k
    if case.get("residual"):
        bytes_ += m * n * e
    if case["train"]:                           # dy read, dx, dW, db written
        bytes_, flops = bytes_ + m * n * e + m * k * e + weights, 3 * flops
    return {"bytes": bytes_, "flops": flops}


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _group_rows(case, seed):
    """Rows of every group: unequal by a power law of the group's rank, the smallest groups often empty."""
    g, m = case["groups"], case["m"]
    gen = torch.Generator().manual_seed(seed * 2 + 1)
    weight = torch.arange(1, g + 1, dtype=torch.float64) ** -case["skew"]
    weight = weight[torch.randperm(g, generator=gen)] * (0.5 + torch.rand(g, generator=gen, dtype=torch.float64))
    if g > 2:
        weight[torch.randint(0, g, (max(1, g // 8),), generator=gen)] = 0
    if float(weight.sum()) == 0:
        weight[0] = 1
    edge = (torch.cumsum(weight, 0) / weight.sum() * m).round().to(torch.int64)
    edge[-1] = m
    return [0] + edge.tolist()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0):
        t = torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)
        return t.mul_(scale).add_(shift) if shift else t.mul_(scale)

    state = {"case": case}
    m = case["m"]
    if case["op"] == "layer_norm":
        d = case["d"]
        state["x"] = normal(m, d, scale=1.5, shift=0.25)
        state["weight"], state["bias"] = normal(d, scale=0.25, shift=1.0), normal(d, scale=0.25)
        out = (m, d)
    elif case["op"] == "linear":
        k, n = case["k"], case["n"]
        state["x"], state["weight"] = normal(m, k), normal(n, k, scale=k ** -0.5)
        state["bias"] = normal(n, scale=0.25) if case["bias"] else None
        state["residual"] = normal(m, n) if case["residual"] else None
        out = (m, n)
    else:
        k, n = case["k"], case["n"]
        state["x"], state["weight"] = normal(m, k), normal(case["groups"], k, n, scale=k ** -0.5)
        state["bias"] = normal(case["groups"], n, scale=0.25) if case["bias"] else None
        state["rows"] = _group_rows(case, seed)
        state["ptr"] = torch.tensor(state["rows"], dtype=torch.int64, device="cuda")
        out = (m, n)
    if case["train"]:
        state["grad"] = normal(*out)
        state["leaves"] = [state[key] for key in ("x", "weight", "bias", "residual") if state.get(key) is not None]
        for leaf in state["leaves"]:
            leaf.requires_grad_(True)
    return state


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"linear": _plain_linear, "segment_matmul": _plain_segment, "layer_norm": _plain_norm}[state["case"]["op"]](state)


def _run_own(state):
    import geot_amd as geot
    case = state["case"]
    if case["op"] == "linear":
        y = geot.linear(state["x"], state["weight"], state["bias"], residual=state["residual"], activation=case["act"])
    elif case["op"] == "segment_matmul":
        y = geot.segment_matmul(state["x"], state["ptr"], state["weight"], state["bias"])
    else:
        y = geot.layer_norm(state["x"], state["weight"], state["bias"])
    if not case["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, state["leaves"], state["grad"])]


def _activate(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * math.sqrt(0.5 / math.pi)
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def _plain_linear(state):
    case, dtype = state["case"], state["x"].dtype
    x, w = state["x"].float(), state["weight"].float()
    z = x @ w.t()
    if state["bias"] is not None:
        z += state["bias"].float()
    y = _activate(z, case["act"])
    if state["residual"] is not None:
        y = y + state["residual"].float()
    if not case["train"]:
        return [y.to(dtype)]
    dz = state["grad"].float()
    if case["act"] != "none":
        dz = dz * _slope(z, case["act"])
    out = [y.to(dtype), (dz @ w).to(dtype), (dz.t() @ x).to(dtype)]
    if state["bias"] is not None:
        out.append(dz.sum(0).to(dtype))
    if state["residual"] is not None:
        out.append(state["grad"])
    return out


def _plain_segment(state):
    case, dtype, rows = state["case"], state["x"].dtype, state["rows"]
    train = case["train"]
    y = torch.empty(case["m"], case["n"], dtype=dtype, device="cuda")
    if train:
        dx, dw = torch.empty_like(state["x"]), torch.zeros_like(state["weight"])
        db = torch.zeros_like(state["bias"]) if state["bias"] is not None else None
    for g in range(case["groups"]):
        a, b = rows[g], rows[g + 1]
        if a == b:
            continue
        x, w = state["x"][a:b].float(), state["weight"][g].float()
        z = x @ w
        if state["bias"] is not None:
            z += state["bias"][g].float()
        y[a:b] = z
        if train:
            dz = state["grad"][a:b].float()
            dx[a:b] = dz @ w.t()
            dw[g] = x.t() @ dz
            if db is not None:
                db[g] = dz.sum(0)
    if not train:
        return [y]
    return [y, dx, dw] + ([db] if db is not None else [])


def _plain_norm(state):
    dtype = state["x"].dtype
    x, w, b = state["x"].float(), state["weight"].float(), state["bias"].float()
    x = x - x.mean(-1, keepdim=True)
    s = (x.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    h = x * s
    y = (h * w + b).to(dtype)
    if not state["case"]["train"]:
        return [y]
    dy = state["grad"].float()
    g = dy * w
    dx = s * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    return [y, dx.to(dtype), (dy * h).sum(0).to(dtype), dy.sum(0).to(dtype)]


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        get = {key: (t.detach().double() if torch.is_tensor(t) and t.is_floating_point() else None) for key, t in state.items()
               if key in ("x", "weight", "bias", "residual", "grad")}
        for key in ("bias", "residual", "grad"):
            get.setdefault(key, None)
        if case["op"] == "linear":
            return _exact_linear(case, **get)
        if case["op"] == "segment_matmul":
            return _exact_segment(case, state["rows"], get["x"], get["weight"], get["bias"], get["grad"])
        return _exact_norm(case, get["x"], get["weight"], get["bias"], get["grad"])


def _exact_linear(case, x, weight, bias, residual, grad):
    act = case["act"]
    z = torch.mm(x, weight.T.contiguous())
    z = z if bias is None else z.add_(bias)
    normal_cdf = torch.special.ndtr(z) if act == "gelu" else None
    logistic = torch.sigmoid(z) if act == "silu" else None
    y = {"none": lambda: z.clone(), "relu": lambda: torch.where(z > 0, z, torch.zeros_like(z)), "gelu": lambda: z * normal_cdf,
         "silu": lambda: z * logistic}[act]()
    if residual is not None:
        y += residual
    if not case["train"]:
        return [y]
    if act == "relu":
        grad_z = torch.where(z > 0, grad, torch.zeros_like(grad))
    elif act == "gelu":
        density = torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
        grad_z = grad * (normal_cdf + z * density)
    elif act == "silu":
        grad_z = grad * (logistic + z * logistic * (1 - logistic))
    else:
        grad_z = grad
    result = [y, torch.mm(grad_z, weight), torch.mm(grad_z.T.contiguous(), x)]
    if bias is not None:
        result.append(torch.sum(grad_z, dim=0))
    if residual is not None:
        result.append(grad)
    return result


def _exact_segment(case, rows, x, weight, bias, grad):
    pieces = [slice(lo, hi) for lo, hi in zip(rows[:-1], rows[1:])]
    y = torch.cat([torch.mm(x[p], weight[g]) + (0 if bias is None else bias[g]) for g, p in enumerate(pieces)])
    if not case["train"]:
        return [y]
    dx = torch.cat([torch.mm(grad[p], weight[g].T.contiguous()) for g, p in enumerate(pieces)])
    dw = torch.stack([torch.mm(x[p].T.contiguous(), grad[p]) for p in pieces])
    return [y, dx, dw] + ([] if bias is None else [torch.stack([torch.sum(grad[p], dim=0) for p in pieces])])


def _exact_norm(case, x, weight, bias, grad):
    variance, mean = torch.var_mean(x, dim=-1, unbiased=False, keepdim=True)
    scale = 1 / torch.sqrt(variance + 1e-5)
    unit = (x - mean) * scale
    y = unit * weight + bias
    if not case["train"]:
        return [y]
    inner = grad * weight
    along = torch.sum(inner * unit, dim=-1, keepdim=True) / x.shape[-1]
    dx = (inner - torch.mean(inner, dim=-1, keepdim=True) - unit * along) * scale
    return [y, dx, torch.sum(grad * unit, dim=0), torch.sum(grad, dim=0)]

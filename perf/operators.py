"""Cases of the matrix products around a transformer block: products with a bias, an activation and a residual in their
epilogue, products grouped by expert, their backward forms, and the orthogonalisation of an update.

``run`` computes the plain form with elementary torch operations in 32 bits; with ``own`` set it makes the calls of the
library. Every case is a single call on inputs that are at hand, so each output is rounded once.
"""
import math

import torch

own = False

TYPES = {"half": torch.float16, "bfloat16": torch.bfloat16, "single": torch.float32}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPSILON = 1e-7


def listed():
    return [
        # one token of a chat: one row against a square weight
        dict(name="linear_token", kind="linear", type="half", c_type="half", rows=1, n=4096, k=4096, bias=True,
             act="silu", residual=False, keep=False),
        # a served batch: few rows, the projection back into the residual stream
        dict(name="linear_decode", kind="linear", type="bfloat16", c_type="bfloat16", rows=48, n=4096, k=8192, bias=True,
             act="identity", residual=True, keep=False),
        # sizes that are multiples of nothing, and leading dimensions that follow them
        dict(name="linear_odd", kind="linear", type="half", c_type="half", rows=777, n=1501, k=1003, bias=True,
             act="gelu", residual=True, keep=True),
        # the first product of a feed-forward block in training: keeps what the backward pass needs
        dict(name="linear_train", kind="linear", type="bfloat16", c_type="bfloat16", rows=8192, n=8192, k=2048,
             bias=True, act="gelu", residual=False, keep=True),
        # single precision throughout
        dict(name="linear_single", kind="linear", type="single", c_type="single", rows=2048, n=2048, k=2048, bias=True,
             act="relu", residual=True, keep=False),
        # backward through the second product and the activation, with the bias gradient
        dict(name="linear_backward", kind="linear_grad", type="bfloat16", rows=8192, n=8192, k=2048, act="gelu_tanh",
             residual=False),
        # experts while tokens are generated: most experts see a row or none
        dict(name="experts_decode", kind="experts", type="bfloat16", c_type="bfloat16", rows=64, groups=32, n=2048,
             k=2048, bias=False, act="silu", residual=False, keep=False),
        # experts over a prompt
        dict(name="experts_prompt", kind="experts", type="bfloat16", c_type="bfloat16", rows=16384, groups=32, n=4096,
             k=2048, bias=True, act="gelu_tanh", residual=False, keep=False),
        # backward through the experts' second product and the activation
        dict(name="experts_backward", kind="experts_grad", type="half", rows=8192, groups=16, n=4096, k=1024,
             act="silu", residual=False),
        # the experts' weight gradients, summed in single precision
        dict(name="experts_weight", kind="experts_weight", type="bfloat16", c_type="single", rows=16384, groups=32,
             n=2048, k=2048),
        # the update of one square weight
        dict(name="update_square", kind="update", type="bfloat16", rows=4096, n=4096, batch=1),
        # the updates of several small weights at once, in single precision
        dict(name="update_single", kind="update", type="single", rows=512, n=1000, batch=4),
    ]


def _spread(rng, low, high, step):
    """A size spread over the logarithm of the range; half of them multiples of `step`, half as they come."""
    size = math.exp(rng.uniform(math.log(low), math.log(high)))
    size = round(size / step) * step if rng.random() < 0.5 else round(size)
    return int(min(high, max(low, size)))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear_grad", "experts", "experts_grad", "experts_weight", "update"])
    act = rng.choice(["identity", "relu", "gelu", "gelu_tanh", "silu"])
    half = rng.choice(["half", "bfloat16"])
    yes = lambda: rng.random() < 0.5
    if kind == "linear":
        t = rng.choice(["half", "bfloat16", "half", "bfloat16", "single"])
        most = 2048 if t == "single" else 8192
        rows = _spread(rng, 1, most, 64)
        return dict(kind=kind, type=t, c_type="single" if t == "single" or rng.random() < 0.2 else t, rows=rows,
                    n=_spread(rng, 256, most, 128), k=_spread(rng, 256, 8192 if rows <= 64 else 2048, 64),
                    bias=yes(), act=act, residual=yes(), keep=yes())
    if kind == "linear_grad":
        return dict(kind=kind, type=half, rows=_spread(rng, 16, 8192, 64), n=_spread(rng, 256, 8192, 128),
                    k=_spread(rng, 256, 2048, 64), act=act, residual=yes())
    if kind == "experts":
        return dict(kind=kind, type=half, c_type=half, rows=_spread(rng, 1, 16384, 64), groups=_spread(rng, 2, 64, 8),
                    n=_spread(rng, 256, 4096, 128), k=_spread(rng, 256, 2048, 64), bias=yes(), act=act, residual=yes(),
                    keep=yes())
    if kind == "experts_grad":
        return dict(kind=kind, type=half, rows=_spread(rng, 16, 8192, 64), groups=_spread(rng, 2, 32, 8),
                    n=_spread(rng, 256, 4096, 128), k=_spread(rng, 256, 1024, 64), act=act, residual=yes())
    if kind == "experts_weight":
        return dict(kind=kind, type=half, c_type=rng.choice(["single", half]), rows=_spread(rng, 16, 16384, 64),
                    groups=_spread(rng, 2, 32, 8), n=_spread(rng, 256, 2048, 128), k=_spread(rng, 256, 2048, 64))
    t = rng.choice(["bfloat16", "bfloat16", "single"])
    most = 1024 if t == "single" else 2048
    return dict(kind=kind, type=t, rows=_spread(rng, 128, most, 64), n=_spread(rng, 128, most, 64),
                batch=rng.choice([1, 1, 2, 3, 4]))


def _normal(generator, shape, scale, dtype):
    return torch.empty(shape, device="cuda", dtype=torch.float32).normal_(generator=generator).mul_(scale).to(dtype)


def _sizes(rows, groups, seed):
    """Rows of each expert as a router leaves them: a few popular experts, some with no row at all."""
    g = torch.Generator().manual_seed(seed)
    popular = torch.empty(groups).exponential_(generator=g) + 0.3
    popular[torch.rand(groups, generator=g) < 0.1] = 0
    popular[int(torch.randint(groups, (1,), generator=g))] += 1.0
    picks = torch.multinomial(popular, rows, replacement=True, generator=g)
    return torch.bincount(picks, minlength=groups)


def prepare(case, seed):
    s = dict(case)
    dtype = TYPES[case["type"]]
    c_dtype = TYPES[case.get("c_type", case["type"])]
    kind, rows, n = case["kind"], case["rows"], case["n"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    s["stream"] = torch.cuda.current_stream()
    new = lambda shape, t=dtype: torch.empty(shape, device="cuda", dtype=t)
    if kind == "update":
        # a gradient: a few strong directions over noise
        shape, rank = (case["batch"], rows, n), 8
        strong = _normal(g, (case["batch"], rows, rank), 1.0, torch.float32) @ _normal(g, (case["batch"], rank, n), 1.0,
                                                                                       torch.float32)
        s["g"] = (1e-3 * (_normal(g, shape, 1.0, torch.float32) + 0.3 * strong)).to(dtype)
        s["c"] = new(shape)
        s["scale"] = math.sqrt(max(1.0, rows / n))
        return s
    k = case["k"]
    groups = case.get("groups", 0)
    if groups:
        sizes = _sizes(rows, groups, seed)
        s["sizes"] = sizes.tolist()
        s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), sizes.cumsum(0)]).cuda()
    if kind == "experts_weight":
        s["x"] = _normal(g, (rows, k), 1.0, dtype)
        s["y"] = _normal(g, (rows, n), 1e-2, dtype)
        s["c"] = new((groups, k, n), c_dtype)
        return s
    s["x"] = _normal(g, (rows, k), 1.0, dtype)
    s["c"] = new((rows, n), c_dtype)
    s["z"] = s["d"] = s["bias"] = None
    if kind in ("linear", "experts"):
        # weights as rows of outputs, [n, k]
        s["w"] = _normal(g, (groups, n, k) if groups else (n, k), k ** -0.5, dtype)
        if case["bias"]:
            s["bias"] = _normal(g, (groups, n) if groups else (n,), 0.2, dtype)
        if case["keep"]:
            s["z"] = new((rows, n))
    else:
        # the backward product reads the next layer's weights the other way round, [k, n]
        s["w"] = _normal(g, (groups, k, n) if groups else (k, n), k ** -0.5, dtype)
        s["z"] = _normal(g, (rows, n), 1.0, dtype)
        s["bias_grad"] = new((groups, n) if groups else (n,))
    if case["residual"]:
        s["d"] = _normal(g, (rows, n), 1.0, c_dtype)
    return s


# ---- the library's calls ---------------------------------------------------------------------------------------------

def _precision(cb, name):
    return {"half": cb.Precision.kHalf, "bfloat16": cb.Precision.kBFloat16, "single": cb.Precision.kSingle}[name]


def _activation(cb, name):
    return {"identity": cb.Activation.kIdentity, "relu": cb.Activation.kRelu, "gelu": cb.Activation.kGelu,
            "gelu_tanh": cb.Activation.kGeluTanh, "silu": cb.Activation.kSilu}[name]


def _calls(s):
    import clblast_b200 as cb
    row, no, yes = cb.Layout.kRowMajor, cb.Transpose.kNo, cb.Transpose.kYes
    kind, rows, n, stream = s["kind"], s["rows"], s["n"], s["stream"]
    if kind == "update":
        st = cb.NewtonSchulz(row, rows, n, s["scale"], s["g"], 0, n, rows * n, s["c"], 0, n, rows * n, s["batch"],
                             steps=STEPS, coefficients=COEFFICIENTS, epsilon=EPSILON, stream=stream)
        out = [s["c"]]
    elif kind == "experts_weight":
        st = cb.GemmGroupedWeight(s["groups"], rows, s["k"], n, 1.0, s["x"], 0, s["k"], s["y"], 0, n, s["offsets"], 0.0,
                                  s["c"], 0, n, s["k"] * n, stream=stream)
        out = [s["c"]]
    else:
        k, act = s["k"], _activation(cb, s["act"])
        beta = 1.0 if s["d"] is not None else 0.0
        if kind == "linear":
            st = cb.GemmEpilogue(row, no, yes, rows, n, k, 1.0, s["x"], 0, k, s["w"], 0, k, s["bias"], 0, act, s["z"], 0,
                                 n, beta, s["d"], 0, n, s["c"], 0, n, stream=stream)
        elif kind == "linear_grad":
            st = cb.GemmEpilogueGrad(row, no, no, rows, n, k, 1.0, s["x"], 0, k, s["w"], 0, n, beta, s["d"], 0, n, act,
                                     s["z"], 0, n, s["c"], 0, n, s["bias_grad"], 0, stream=stream)
        elif kind == "experts":
            st = cb.GemmGrouped(yes, s["groups"], rows, n, k, 1.0, s["x"], 0, k, s["w"], 0, k, n * k, s["offsets"],
                                s["bias"], 0, n, act, s["z"], 0, n, beta, s["d"], 0, n, s["c"], 0, n, stream=stream)
        else:
            st = cb.GemmGroupedGrad(no, s["groups"], rows, n, k, 1.0, s["x"], 0, k, s["w"], 0, n, n * k, s["offsets"],
                                    beta, s["d"], 0, n, act, s["z"], 0, n, s["c"], 0, n, s["bias_grad"], 0, n,
                                    stream=stream)
        if kind.endswith("grad"):
            out = [s["c"], s["bias_grad"]]
        else:
            out = [s["c"], s["z"]] if s["z"] is not None else [s["c"]]
    assert st == cb.StatusCode.kSuccess, st
    return out


# ---- the plain form --------------------------------------------------------------------------------------------------

def _act(z, name):
    if name == "relu":
        return z * (z > 0)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(z, name):
    if name == "relu":
        return (z > 0).float()
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


def _places(s):
    """Where each row goes in a [groups, longest] table of rows."""
    longest = max(s["sizes"])
    rows = torch.arange(s["rows"], device="cuda")
    group = torch.searchsorted(s["offsets"], rows, right=True) - 1
    return group, group * longest + rows - s["offsets"][group], longest


def _padded(x, place, groups, longest):
    table = torch.zeros(groups * longest, x.shape[1], device="cuda")
    return table.index_copy(0, place, x.float()).view(groups, longest, -1)


def _product(s):
    """x w in 32 bits, by expert where there are experts; w is [n, k] in the forward kinds."""
    w = s["w"].float()
    if s["kind"] in ("linear", "experts"):
        w = w.mT
    if "groups" not in s:
        return s["x"].float() @ w, None
    group, place, longest = _places(s)
    p = torch.bmm(_padded(s["x"], place, s["groups"], longest), w)
    return p.view(s["groups"] * longest, -1)[place], group


def _plain(s):
    kind, dtype = s["kind"], TYPES[s["type"]]
    c_dtype = TYPES[s.get("c_type", s["type"])]
    if kind == "update":
        a, b, c = COEFFICIENTS
        x = s["g"].float()
        x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + EPSILON)
        tall = s["rows"] > s["n"]
        x = x.mT if tall else x
        for _ in range(STEPS):
            m = x @ x.mT
            x = a * x + (b * m + c * (m @ m)) @ x
        return [(s["scale"] * (x.mT if tall else x)).to(dtype).contiguous()]
    if kind == "experts_weight":
        _, place, longest = _places(s)
        x, y = (_padded(s[v], place, s["groups"], longest) for v in ("x", "y"))
        return [torch.bmm(x.mT, y).to(c_dtype)]
    p, group = _product(s)
    if kind in ("linear", "experts"):
        if s["bias"] is not None:
            p = p + (s["bias"].float() if group is None else s["bias"].float()[group])
        c = _act(p, s["act"])
        c = c + s["d"].float() if s["d"] is not None else c
        return [c.to(c_dtype)] + ([p.to(dtype)] if s["z"] is not None else [])
    p = p + s["d"].float() if s["d"] is not None else p
    p = p * _slope(s["z"].float(), s["act"])
    if group is None:
        total = p.sum(0)
    else:
        total = torch.zeros(s["groups"], s["n"], device="cuda").index_add(0, group, p)
    return [p.to(dtype), total.to(dtype)]


def run(state):
    return _calls(state) if own else _plain(state)


# ---- 64 bits ---------------------------------------------------------------------------------------------------------

def _cdf64(z):
    return 0.5 * torch.special.erfc(-z / math.sqrt(2.0))


def _value64(z, name):
    if name == "relu":
        return torch.clamp(z, min=0.0)
    if name == "gelu":
        return z * _cdf64(z)
    if name == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z * torch.sigmoid(z) if name == "silu" else z


def _slope64(z, name):
    if name == "relu":
        return torch.where(z > 0, 1.0, 0.0).double()
    if name == "gelu":
        return _cdf64(z) + z * torch.exp(-z ** 2 / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        u = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
        p = torch.sigmoid(u)
        return p + z * p * (1 - p) * 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * z ** 2)
    if name == "silu":
        p = torch.sigmoid(z)
        return p + z * p * (1 - p)
    return torch.ones_like(z)


def exact(case, seed):
    s = prepare(case, seed)
    kind, rows = case["kind"], case["rows"]
    if kind == "update":
        result = []
        for m in s["g"].double():
            # the polynomial acts on the singular values alone: on the Gram matrix of the shorter side
            side = m if m.shape[0] <= m.shape[1] else m.T
            x = side / (torch.linalg.norm(side) + EPSILON)
            one = torch.eye(x.shape[0], device="cuda", dtype=torch.float64)
            for _ in range(STEPS):
                gram = x @ x.T
                x = (COEFFICIENTS[0] * one + gram @ (COEFFICIENTS[1] * one + COEFFICIENTS[2] * gram)) @ x
            result.append(s["scale"] * (x if m.shape[0] <= m.shape[1] else x.T))
        return [torch.stack(result)]
    if "groups" in case:
        ends = torch.tensor(s["sizes"]).cumsum(0).tolist()
        spans = list(zip([0] + ends[:-1], ends))
    else:
        spans = [(0, rows)]
    if kind == "experts_weight":
        return [torch.stack([s["x"][i:j].double().T @ s["y"][i:j].double() for i, j in spans])]
    parts, totals, kept = [], [], []
    for g, (i, j) in enumerate(spans):
        w = (s["w"][g] if "groups" in case else s["w"]).double()
        p = s["x"][i:j].double() @ (w.T if kind in ("linear", "experts") else w)
        if kind in ("linear", "experts"):
            if s["bias"] is not None:
                p += (s["bias"][g] if "groups" in case else s["bias"]).double()
            kept.append(p)
            p = _value64(p, case["act"])
            parts.append(p if s["d"] is None else p + s["d"][i:j].double())
        else:
            p = p if s["d"] is None else p + s["d"][i:j].double()
            p = p * _slope64(s["z"][i:j].double(), case["act"])
            parts.append(p)
            totals.append(p.sum(0))
    if kind in ("linear", "experts"):
        return [torch.cat(parts)] + ([torch.cat(kept)] if case["keep"] else [])
    return [torch.cat(parts), torch.stack(totals) if "groups" in case else totals[0]]


def work(case):
    size = {"half": 2, "bfloat16": 2, "single": 4}
    t, c = size[case["type"]], size[case.get("c_type", case["type"])]
    kind, rows, n = case["kind"], case["rows"], case["n"]
    if kind == "update":
        short, long = min(rows, n), max(rows, n)
        # the Gram matrix and its square are symmetric: half of each
        flops = STEPS * case["batch"] * (short * short * long + short ** 3 + 2 * short * short * long)
        return {"bytes": 2 * t * rows * n * case["batch"], "flops": flops}
    k, groups = case["k"], case.get("groups", 1)
    if kind == "experts_weight":
        return {"bytes": t * rows * (k + n) + c * groups * k * n, "flops": 2 * rows * n * k}
    bytes_ = t * (rows * k + min(groups, rows) * n * k) + c * rows * n
    if case["residual"]:
        bytes_ += c * rows * n
    if kind in ("linear", "experts"):
        bytes_ += t * min(groups, rows) * n if case["bias"] else 0
        bytes_ += t * rows * n if case["keep"] else 0
    else:
        bytes_ += t * rows * n + t * groups * n
    return {"bytes": bytes_, "flops": 2 * rows * n * k}

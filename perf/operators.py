"""Measured cases of the operators built on the matrix product: the product with bias, activation and
residual in its epilogue, products grouped by expert, and softmax cross entropy over a large vocabulary.

``run`` computes a case in its plain form, or, where ``own`` is true, through the framework's entry points
(``NativeMatmul.prepare_epilogue`` and its neighbours).  Matrices are row-major; ``precision`` names the input
format as in the rest of the framework: bf16 and fp16 tensors, or FP32 tensors whose products take operands
rounded to TF32 (nearest even).
"""

import math
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "tf32": torch.float32}
IGNORE = -100
_context = []


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # The up projection of a feed-forward block over a prompt or a training batch; z is kept for the backward pass.
        {"name": "up projection, batch", "op": "epilogue", "precision": "bf16", "m": 4096, "k": 4096, "n": 14336,
         "activation": "gelu", "bias": True, "residual": False, "preact": True, "out": "input"},
        # The down projection while 16 sequences decode: HBM-bound on the weight.
        {"name": "down projection, decode", "op": "epilogue", "precision": "bf16", "m": 16, "k": 8192, "n": 8192,
         "activation": "none", "bias": False, "residual": True, "preact": False, "out": "input"},
        # One token of one sequence.
        {"name": "up projection, one token", "op": "epilogue", "precision": "fp16", "m": 1, "k": 4096, "n": 14336,
         "activation": "silu", "bias": True, "residual": False, "preact": False, "out": "input"},
        # A small head on odd sizes, FP32 tensors in and out: latency, and rows that no 16-byte copy can address.
        {"name": "small head, odd sizes", "op": "epilogue", "precision": "tf32", "m": 511, "k": 257, "n": 129,
         "activation": "relu", "bias": True, "residual": True, "preact": False, "out": "fp32"},
        # The backward pass of the first case.
        {"name": "up projection, backward", "op": "epilogue_backward", "precision": "bf16", "m": 4096, "k": 4096,
         "n": 14336, "activation": "gelu", "out": "input"},
        # A backward pass on odd sizes.
        {"name": "odd projection, backward", "op": "epilogue_backward", "precision": "fp16", "m": 777, "k": 1500,
         "n": 1100, "activation": "silu", "out": "input"},
        # Experts over a prompt or a training batch.
        {"name": "experts, batch", "op": "grouped", "precision": "bf16", "rows": 16384, "groups": 64, "k": 2048,
         "n": 2816, "out": "input"},
        # Experts while a few sequences decode: one to a few rows each, some experts without any.
        {"name": "experts, decode", "op": "grouped", "precision": "bf16", "rows": 64, "groups": 32, "k": 4096, "n": 2048,
         "out": "input"},
        # The backward pass of experts of uneven load.
        {"name": "experts, backward", "op": "grouped_backward", "precision": "bf16", "rows": 8192, "groups": 32,
         "k": 2048, "n": 1408, "out": "input"},
        # The training loss of a language model's head, with both gradients.
        {"name": "loss and gradients", "op": "cross_entropy_step", "precision": "bf16", "m": 4096, "k": 4096,
         "v": 128000, "out": "input"},
        # The same on a short ragged batch and a vocabulary of odd size.
        {"name": "loss and gradients, odd", "op": "cross_entropy_step", "precision": "bf16", "m": 200, "k": 768,
         "v": 32001, "out": "input"},
        # Scoring text: the loss alone.
        {"name": "loss, scoring", "op": "cross_entropy", "precision": "bf16", "m": 1000, "k": 1024, "v": 50257},
    ]


def _spread(rng, low, high):
    """A size spread over the logarithm of [low, high]; half of them multiples of 64 where that fits, the others any number."""
    size = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5 and size >= 64:
        size = size // 64 * 64
    return max(low, min(high, size))


def draw(rng):
    while True:
        op = rng.choice(("epilogue", "epilogue", "epilogue_backward", "grouped", "grouped_backward",
                         "cross_entropy_step", "cross_entropy"))
        precision = rng.choice(("bf16", "bf16", "fp16", "tf32"))
        out = rng.choice(("input", "fp32"))
        if op == "epilogue":
            case = {"op": op, "precision": precision, "m": _spread(rng, 1, 8192), "k": _spread(rng, 32, 14336),
                    "n": _spread(rng, 32, 28672), "activation": rng.choice(("none", "relu", "gelu", "gelu_tanh", "silu")),
                    "bias": rng.random() < 0.6, "residual": rng.random() < 0.4, "preact": rng.random() < 0.3, "out": out}
        elif op == "epilogue_backward":
            case = {"op": op, "precision": rng.choice(("bf16", "fp16")), "m": _spread(rng, 1, 8192),
                    "k": _spread(rng, 32, 8192), "n": _spread(rng, 32, 14336),
                    "activation": rng.choice(("relu", "gelu", "gelu_tanh", "silu")), "out": "input"}
        elif op in ("grouped", "grouped_backward"):
            case = {"op": op, "precision": precision, "rows": _spread(rng, 1, 16384), "groups": _spread(rng, 2, 128),
                    "k": _spread(rng, 32, 4096), "n": _spread(rng, 32, 4096), "out": out}
        elif op == "cross_entropy_step":
            case = {"op": op, "precision": "bf16", "m": _spread(rng, 1, 4096), "k": _spread(rng, 64, 4096),
                    "v": _spread(rng, 1000, 128000), "out": "input"}
        else:
            case = {"op": op, "precision": precision, "m": _spread(rng, 1, 8192), "k": _spread(rng, 64, 4096),
                    "v": _spread(rng, 1000, 128000)}
        if work(case)["flops"] <= 4e12 and work(case)["bytes"] <= 4e9:
            return case


def _element(case):
    return 4 if case["precision"] == "tf32" else 2


def _out_element(case):
    return 4 if case["out"] == "fp32" else _element(case)


def _out_dtype(case):
    return torch.float32 if case["out"] == "fp32" else DTYPES[case["precision"]]


def work(case):
    e, op = _element(case), case["op"]
    if op in ("epilogue", "epilogue_backward"):
        m, k, n = case["m"], case["k"], case["n"]
        eo = _out_element(case)
        if op == "epilogue":
            outs = 1 + int(case["residual"]) + int(case["preact"])
            return {"bytes": e * (m * k + k * n) + eo * outs * m * n + e * n * int(case["bias"]), "flops": 2 * m * k * n}
        return {"bytes": e * (2 * m * n + m * k + k * n) + eo * (m * k + k * n) + 4 * n, "flops": 4 * m * k * n}
    if op in ("grouped", "grouped_backward"):
        m, g, k, n = case["rows"], case["groups"], case["k"], case["n"]
        eo, used = _out_element(case), min(case["groups"], case["rows"])
        if op == "grouped":
            return {"bytes": e * (m * k + used * k * n) + eo * m * n, "flops": 2 * m * k * n}
        return {"bytes": e * (m * k + m * n + used * k * n) + eo * (m * k + g * k * n), "flops": 4 * m * k * n}
    m, k, v = case["m"], case["k"], case["v"]
    if op == "cross_entropy":
        return {"bytes": e * (m * k + k * v) + 16 * m, "flops": 2 * m * k * v}
    return {"bytes": e * (m * k + k * v) + _out_element(case) * (m * k + k * v) + 20 * m, "flops": 8 * m * k * v}


# ------------------------------------------------------------------------------------------ inputs
def _normal(shape, dtype, gen, scale=1.0):
    x = torch.randn(shape, generator=gen, device="cuda")
    return (x * scale).to(dtype) if scale != 1.0 else x.to(dtype)


def _offsets(rows, groups, gen):
    """Row offsets of uneven groups: about one in eight is empty, the largest has two to four times the mean; a few rows at the end belong to none."""
    load = torch.rand(groups, generator=gen, device="cuda") + 0.5
    load = load * (torch.rand(groups, generator=gen, device="cuda") > 0.125)
    load[groups // 2] = 1.0
    ends = torch.cumsum(load / load.sum(), 0) * rows
    offsets = torch.zeros(groups + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = ends.round().to(torch.int32)
    return offsets.clamp_(max=rows - rows // 50)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype, op = DTYPES[case["precision"]], case["op"]
    s = {"case": dict(case), "launch": None}
    if op in ("epilogue", "epilogue_backward"):
        m, k, n = case["m"], case["k"], case["n"]
        odtype = _out_dtype(case)
        s["a"] = _normal((m, k), dtype, gen)
        s["b"] = _normal((k, n), dtype, gen, k ** -0.5)
        if op == "epilogue":
            s["bias"] = _normal((n,), dtype, gen, 0.5) if case["bias"] else None
            s["residual"] = _normal((m, n), odtype, gen) if case["residual"] else None
            s["out"] = torch.zeros((m, n), dtype=odtype, device="cuda")
            s["preact"] = torch.zeros((m, n), dtype=odtype, device="cuda") if case["preact"] else None
        else:
            s["preact"] = _normal((m, n), dtype, gen)
            s["dout"] = _normal((m, n), dtype, gen)
            s["da"] = torch.zeros((m, k), dtype=odtype, device="cuda")
            s["db"] = torch.zeros((k, n), dtype=odtype, device="cuda")
            s["dbias"] = torch.zeros((n,), dtype=torch.float32, device="cuda")
    elif op in ("grouped", "grouped_backward"):
        m, g, k, n = case["rows"], case["groups"], case["k"], case["n"]
        odtype = _out_dtype(case)
        s["a"] = _normal((m, k), dtype, gen)
        s["b"] = _normal((g, k, n), dtype, gen, k ** -0.5)
        s["offsets"] = _offsets(m, g, gen)
        s["capacity"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())
        s["assigned"] = int(s["offsets"][-1])
        if op == "grouped":
            s["out"] = torch.zeros((m, n), dtype=odtype, device="cuda")
        else:
            s["dout"] = _normal((m, n), dtype, gen)
            s["da"] = torch.zeros((m, k), dtype=odtype, device="cuda")
            s["db"] = torch.zeros((g, k, n), dtype=odtype, device="cuda")
    else:
        m, k, v = case["m"], case["k"], case["v"]
        s["hidden"] = _normal((m, k), dtype, gen)
        s["weight"] = _normal((k, v), dtype, gen, 2.0 * k ** -0.5)
        labels = torch.randint(0, v, (m,), generator=gen, device="cuda")
        ignored = torch.rand((m,), generator=gen, device="cuda") < 0.1
        s["labels"] = torch.where(ignored, torch.full_like(labels, IGNORE), labels)
        s["loss"] = torch.zeros((m,), dtype=torch.float32, device="cuda")
        s["lse"] = torch.zeros((m,), dtype=torch.float32, device="cuda")
        if op == "cross_entropy_step":
            odtype = _out_dtype(case)
            s["grad"] = torch.rand((m,), generator=gen, device="cuda") * (2.0 / m)
            s["dhidden"] = torch.zeros((m, k), dtype=odtype, device="cuda")
            s["dweight"] = torch.zeros((k, v), dtype=odtype, device="cuda")
    return s


# ------------------------------------------------------------------------------------------ the framework's calls
def _native():
    if not _context:
        if "matrix-multiplication_b200" not in sys.path:
            sys.path.insert(0, "matrix-multiplication_b200")
        from gpumat import NativeMatmul

        _context.append(NativeMatmul(device=torch.cuda.current_device()))
    return _context[0]


def _launches(s):
    """The prepared launches of a case, as a program keeps them."""
    case, native = s["case"], _native()
    op, precision = case["op"], case["precision"]
    if op == "epilogue":
        return (native.prepare_epilogue(s["a"], s["b"], s["out"], precision=precision, bias=s["bias"],
                                        activation=case["activation"], residual=s["residual"], preact=s["preact"]),)
    if op == "epilogue_backward":
        return (native.prepare_epilogue_backward(s["dout"], s["a"], s["b"], precision=precision,
                                                 activation=case["activation"], preact=s["preact"], da=s["da"],
                                                 db=s["db"], dbias=s["dbias"]),)
    if op == "grouped":
        return (native.prepare_grouped(s["a"], s["b"], s["offsets"], s["out"], precision=precision),)
    if op == "grouped_backward":
        return (native.prepare_grouped_backward(s["dout"], s["a"], s["b"], s["offsets"], precision=precision,
                                                da=s["da"], db=s["db"]),)
    loss = native.prepare_cross_entropy(s["hidden"], s["weight"], s["labels"], s["loss"], s["lse"],
                                        precision=precision, ignore_index=IGNORE)
    if op == "cross_entropy":
        return (loss,)
    return (loss, native.prepare_cross_entropy_backward(s["grad"], s["hidden"], s["weight"], s["labels"], s["lse"],
                                                        precision=precision, dhidden=s["dhidden"],
                                                        dweight=s["dweight"], ignore_index=IGNORE))


def _outputs(s):
    op = s["case"]["op"]
    if op == "epilogue":
        return {"out": s["out"], "preact": s["preact"]}
    if op == "epilogue_backward":
        return {"da": s["da"], "db": s["db"], "dbias": s["dbias"]}
    if op == "grouped":
        return {"out": s["out"]}
    if op == "grouped_backward":
        return {"da": s["da"], "db": s["db"]}
    if op == "cross_entropy":
        return {"loss": s["loss"], "lse": s["lse"]}
    return {"loss": s["loss"], "lse": s["lse"], "dhidden": s["dhidden"], "dweight": s["dweight"]}


# ------------------------------------------------------------------------------------------ plain forms
def _operand(x, precision):
    """A product's operand in 32 bits: exact for bf16 and fp16; FP32 words rounded to TF32, nearest even."""
    if precision != "tf32":
        return x.float()
    bits = x.contiguous().view(torch.int32)
    return ((bits + 0xFFF + ((bits >> 13) & 1)) & -0x2000).view(torch.float32)


def _activation(z, name):
    if name == "relu":
        return torch.clamp(z, min=0.0)
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * 0.7071067811865476))
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(0.7978845608028654 * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _activation_slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * 0.7071067811865476)) + z * 0.3989422804014327 * torch.exp(-0.5 * z * z)
    if name == "gelu_tanh":
        t = torch.tanh(0.7978845608028654 * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * 0.7978845608028654 * (1.0 + 0.134145 * z * z)
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    return torch.ones_like(z)


def _places(s):
    """For each row its group and its place in it; rows of no group are left out."""
    offsets = s["offsets"].long()
    row = torch.arange(s["assigned"], device="cuda")
    group = torch.bucketize(row, offsets[1:], right=True)
    return row, group, row - offsets[group]


def _padded(x, s, places):
    row, group, place = places
    full = torch.zeros((s["case"]["groups"], s["capacity"], x.shape[1]), dtype=x.dtype, device="cuda")
    full[group, place] = x[row]
    return full


def _plain_grouped(s):
    case = s["case"]
    precision, odtype = case["precision"], _out_dtype(case)
    places = _places(s)
    row, group, place = places
    a, b = _padded(_operand(s["a"], precision), s, places), _operand(s["b"], precision)
    if case["op"] == "grouped":
        out = s["out"].clone()
        out[row] = torch.bmm(a, b)[group, place].to(odtype)
        return {"out": out}
    dout = _padded(_operand(s["dout"], precision), s, places)
    da = s["da"].clone()
    da[row] = torch.bmm(dout, b.transpose(1, 2))[group, place].to(odtype)
    return {"da": da, "db": torch.bmm(a.transpose(1, 2), dout).to(odtype)}


def _plain_cross_entropy(s):
    case = s["case"]
    precision, labels = case["precision"], s["labels"]
    h, w = _operand(s["hidden"], precision), _operand(s["weight"], precision)
    z = h @ w
    top = z.amax(1, keepdim=True)
    lse = top[:, 0] + torch.log(torch.exp(z - top).sum(1))
    kept = labels != IGNORE
    index = torch.where(kept, labels, torch.zeros_like(labels))
    picked = z.gather(1, index[:, None])[:, 0]
    loss = torch.where(kept, lse - picked, torch.zeros_like(lse))
    if case["op"] == "cross_entropy":
        return {"loss": loss, "lse": lse}
    scale = torch.where(kept, s["grad"], torch.zeros_like(s["grad"]))
    dz = torch.exp(z - lse[:, None]) * scale[:, None]
    del z
    dz[torch.arange(case["m"], device="cuda"), index] -= scale
    odtype = _out_dtype(case)
    return {"loss": loss, "lse": lse, "dhidden": (dz @ w.t()).to(odtype), "dweight": (h.t() @ dz).to(odtype)}


def run(state):
    if own:
        if state["launch"] is None:
            state["launch"] = _launches(state)
        for launch in state["launch"]:
            launch()
        return _outputs(state)
    case = state["case"]
    op, precision = case["op"], case["precision"]
    if op == "epilogue":
        odtype = _out_dtype(case)
        z = _operand(state["a"], precision) @ _operand(state["b"], precision)
        if state["bias"] is not None:
            z = z + state["bias"].float()
        out = _activation(z, case["activation"])
        if state["residual"] is not None:
            out = out + state["residual"].float()
        return {"out": out.to(odtype), "preact": z.to(odtype) if case["preact"] else None}
    if op == "epilogue_backward":
        odtype = _out_dtype(case)
        dz = state["dout"].float() * _activation_slope(state["preact"].float(), case["activation"])
        return {"da": (dz @ _operand(state["b"], precision).t()).to(odtype),
                "db": (_operand(state["a"], precision).t() @ dz).to(odtype), "dbias": dz.sum(0)}
    if op in ("grouped", "grouped_backward"):
        return _plain_grouped(state)
    return _plain_cross_entropy(state)


# ------------------------------------------------------------------------------------------ 64 bits
def _tf32_64(x):
    """FP32 words rounded to 10 fraction bits, ties to even, by scaling each to an integer of 11 bits."""
    mantissa, exponent = torch.frexp(x.double())
    return torch.ldexp(torch.round(torch.ldexp(mantissa, torch.tensor(11, device="cuda"))), exponent - 11)


def _value(x, case):
    return _tf32_64(x) if case["precision"] == "tf32" else x.double()


def _normal_cdf(z):
    return 0.5 * torch.special.erfc(-z / math.sqrt(2.0))


def _exact_activation(z, name):
    """(act(z), act'(z)) in 64 bits."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        on = (z > 0).double()
        return z * on, on
    if name == "gelu":
        cdf = _normal_cdf(z)
        return z * cdf, cdf + z * torch.exp(-z * z / 2.0) / math.sqrt(2.0 * math.pi)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * torch.sigmoid(-z)
    c = math.sqrt(2.0 / math.pi)
    # 0.5 (1 + tanh u) is the logistic function of 2 u.
    s = torch.sigmoid(2.0 * c * (z + 0.044715 * z ** 3))
    return z * s, s + z * s * (1.0 - s) * 2.0 * c * (1.0 + 3.0 * 0.044715 * z ** 2)


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "epilogue":
        z = _value(s["a"], case) @ _value(s["b"], case)
        if s["bias"] is not None:
            z = z + s["bias"].double()
        out, _ = _exact_activation(z, case["activation"])
        if s["residual"] is not None:
            out = out + s["residual"].double()
        return {"out": out, "preact": z if case["preact"] else None}
    if op == "epilogue_backward":
        _, slope = _exact_activation(s["preact"].double(), case["activation"])
        dz = s["dout"].double() * slope
        return {"da": dz @ _value(s["b"], case).T, "db": _value(s["a"], case).T @ dz, "dbias": dz.sum(0)}
    if op in ("grouped", "grouped_backward"):
        a, b, offsets = _value(s["a"], case), s["b"], s["offsets"].tolist()
        result = {"out": s["out"].double()} if op == "grouped" else {"da": s["da"].double(), "db": s["db"].double()}
        for g in range(case["groups"]):
            lo, hi = offsets[g], offsets[g + 1]
            if lo == hi:
                continue
            if op == "grouped":
                result["out"][lo:hi] = a[lo:hi] @ _value(b[g], case)
            else:
                dout = _value(s["dout"][lo:hi], case)
                result["da"][lo:hi] = dout @ _value(b[g], case).T
                result["db"][g] = a[lo:hi].T @ dout
        return result
    h, w, labels = _value(s["hidden"], case), _value(s["weight"], case), s["labels"]
    z = h @ w
    lse = torch.logsumexp(z, 1)
    kept = (labels != IGNORE).double()
    index = labels.clamp(min=0)
    rows = torch.arange(case["m"], device="cuda")
    result = {"loss": (lse - z[rows, index]) * kept, "lse": lse}
    if op == "cross_entropy":
        return result
    z -= lse[:, None]
    p = z.exp_()
    p[rows, index] -= 1.0
    p *= (s["grad"].double() * kept)[:, None]
    return {**result, "dhidden": p @ w.T, "dweight": h.T @ p}

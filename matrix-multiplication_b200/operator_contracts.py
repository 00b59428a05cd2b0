"""Operand contracts of the operators next to the matrix product (``NativeMatmul.prepare_epilogue`` and its
neighbours), in the manner of ``precision.validate_operands``: TypeError for a wrong type or dtype, ValueError
for a wrong rank, device, layout, shape, size or an output that overlaps another operand.  The reference has no
such operators.
"""

from __future__ import annotations

from precision import INPUT_DTYPES, PRECISIONS

ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu")
ACTIVATION_IDS = {name: index for index, name in enumerate(ACTIVATIONS)}
OPERATOR_PRECISIONS = ("tf32", "fp16", "bf16")
SIZE_MAX = 2**31 - 1024     # a tile past the end still has coordinates of 32 bits
GROUPS_MAX = 2**28          # sums over all groups' tiles have 32 bits


def _input_dtype(precision: str):
    import torch

    if precision not in PRECISIONS:
        raise ValueError(f"Unknown precision: {precision}")
    if precision not in OPERATOR_PRECISIONS:
        raise ValueError(f"the operators run on the tensor cores in {', '.join(OPERATOR_PRECISIONS)}, not {precision}")
    return getattr(torch, INPUT_DTYPES[precision])


def _check(name: str, tensor, dtypes: tuple, ndim: int, device: int) -> None:
    import torch

    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if tensor.ndim != ndim:
        raise ValueError(f"{name} must have {ndim} dimension{'s' if ndim > 1 else ''}")
    if tensor.dtype not in dtypes:
        raise TypeError(f"{name} must have dtype {' or '.join(str(d) for d in dict.fromkeys(dtypes))}")
    if tensor.device.type != "cuda" or tensor.device.index != device:
        raise ValueError(f"{name} must be on cuda:{device}")
    if not tensor.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _shape(name: str, tensor, shape: tuple) -> None:
    if tuple(tensor.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, not {tuple(tensor.shape)}")


def _sizes(*sizes: int) -> None:
    if any(size <= 0 or size > SIZE_MAX for size in sizes):
        raise ValueError(f"matrix dimensions must be positive and at most {SIZE_MAX}")


def _range(tensor) -> tuple[int, int]:
    begin = tensor.data_ptr()
    return begin, begin + tensor.numel() * tensor.element_size()


def _no_overlap(outputs: dict, inputs: dict) -> None:
    """No output shares memory with an input or another output."""
    written = [(name, *_range(t)) for name, t in outputs.items() if t is not None]
    read = [(name, *_range(t)) for name, t in inputs.items() if t is not None]
    for index, (name, begin, end) in enumerate(written):
        for other, lo, hi in written[index + 1:] + read:
            if begin < hi and lo < end:
                raise ValueError(f"{name} must not overlap {other}")


def _activation(activation) -> None:
    if not isinstance(activation, str) or activation not in ACTIVATION_IDS:
        raise ValueError(f"unknown activation: {activation!r} (one of {', '.join(ACTIVATIONS)})")


def validate_epilogue(a, b, out, precision: str, device: int, bias=None, activation: str = "none", residual=None,
                      preact=None) -> tuple[int, int, int]:
    import torch

    dtype = _input_dtype(precision)
    either = (torch.float32, dtype)
    _activation(activation)
    _check("a", a, (dtype,), 2, device)
    _check("b", b, (dtype,), 2, device)
    _check("out", out, either, 2, device)
    m, k = a.shape
    n = b.shape[1]
    _sizes(m, k, n)
    _shape("b", b, (k, n))
    _shape("out", out, (m, n))
    if bias is not None:
        _check("bias", bias, either, 1, device)
        _shape("bias", bias, (n,))
    if residual is not None:
        _check("residual", residual, (out.dtype,), 2, device)
        _shape("residual", residual, (m, n))
    if preact is not None:
        _check("preact", preact, either, 2, device)
        _shape("preact", preact, (m, n))
    inputs = {"a": a, "b": b, "bias": bias}
    if residual is not None and residual.data_ptr() != out.data_ptr():
        inputs["residual"] = residual       # out itself may be the residual: each element is read before it is written
    _no_overlap({"out": out, "preact": preact}, inputs)
    return m, k, n


def validate_epilogue_backward(dout, a, b, precision: str, device: int, activation: str = "none", preact=None, da=None,
                               db=None, dbias=None) -> tuple[int, int, int]:
    import torch

    dtype = _input_dtype(precision)
    either = (torch.float32, dtype)
    _activation(activation)
    if da is None and db is None and dbias is None:
        raise ValueError("no gradient is asked for: pass da, db or dbias")
    _check("dout", dout, (dtype,), 2, device)
    m, n = dout.shape
    k = 1
    if da is not None:
        _check("b", b, (dtype,), 2, device)
        _check("da", da, either, 2, device)
        k = b.shape[0]
        _shape("b", b, (k, n))
        _shape("da", da, (m, k))
    if db is not None:
        _check("a", a, (dtype,), 2, device)
        _check("db", db, either, 2, device)
        if da is not None and a.shape[1] != k:
            raise ValueError("expected dout=(m, n), a=(m, k) and b=(k, n)")
        k = a.shape[1]
        _shape("a", a, (m, k))
        _shape("db", db, (k, n))
    if dbias is not None:
        _check("dbias", dbias, either, 1, device)
        _shape("dbias", dbias, (n,))
    if activation != "none":
        _check("preact", preact, either, 2, device)
        _shape("preact", preact, (m, n))
    _sizes(m, k, n)
    _no_overlap({"da": da, "db": db, "dbias": dbias},
                {"dout": dout, "a": a if db is not None else None, "b": b if da is not None else None,
                 "preact": preact if activation != "none" else None})
    return m, k, n


def _check_offsets(offsets, groups: int, device: int) -> None:
    import torch

    if groups > GROUPS_MAX:
        raise ValueError(f"groups must be at most {GROUPS_MAX}")
    _check("offsets", offsets, (torch.int32, torch.int64), 1, device)
    _shape("offsets", offsets, (groups + 1,))


def validate_grouped(a, b, offsets, out, precision: str, device: int) -> tuple[int, int, int, int]:
    import torch

    dtype = _input_dtype(precision)
    _check("a", a, (dtype,), 2, device)
    _check("b", b, (dtype,), 3, device)
    _check("out", out, (torch.float32, dtype), 2, device)
    rows, k = a.shape
    groups, _, n = b.shape
    _sizes(rows, groups, k, n)
    _shape("b", b, (groups, k, n))
    _shape("out", out, (rows, n))
    _check_offsets(offsets, groups, device)
    _no_overlap({"out": out}, {"a": a, "b": b, "offsets": offsets})
    return rows, groups, k, n


def validate_grouped_backward(dout, a, b, offsets, precision: str, device: int, da=None,
                              db=None) -> tuple[int, int, int, int]:
    import torch

    dtype = _input_dtype(precision)
    either = (torch.float32, dtype)
    if da is None and db is None:
        raise ValueError("no gradient is asked for: pass da or db")
    _check("dout", dout, (dtype,), 2, device)
    rows, n = dout.shape
    groups = k = 0
    if da is not None:
        _check("b", b, (dtype,), 3, device)
        _check("da", da, either, 2, device)
        groups, k, _ = b.shape
        _shape("b", b, (groups, k, n))
        _shape("da", da, (rows, k))
    if db is not None:
        _check("a", a, (dtype,), 2, device)
        _check("db", db, either, 3, device)
        if da is not None and (db.shape[0] != groups or a.shape[1] != k):
            raise ValueError("expected dout=(rows, n), a=(rows, k), b=(groups, k, n) and db=(groups, k, n)")
        groups, k = db.shape[0], a.shape[1]
        _shape("a", a, (rows, k))
        _shape("db", db, (groups, k, n))
    _sizes(rows, groups, k, n)
    _check_offsets(offsets, groups, device)
    _no_overlap({"da": da, "db": db},
                {"dout": dout, "a": a if db is not None else None, "b": b if da is not None else None,
                 "offsets": offsets})
    return rows, groups, k, n


def _check_loss(hidden, weight, labels, lse, dtype, device: int, ignore_index) -> tuple[int, int, int]:
    import torch

    if isinstance(ignore_index, bool) or not isinstance(ignore_index, int) or not -2**63 <= ignore_index < 2**63:
        raise ValueError("ignore_index must be an int of 64 bits")
    _check("hidden", hidden, (dtype,), 2, device)
    _check("weight", weight, (dtype,), 2, device)
    _check("labels", labels, (torch.int32, torch.int64), 1, device)
    _check("lse", lse, (torch.float32,), 1, device)
    m, k = hidden.shape
    v = weight.shape[1]
    _sizes(m, k, v)
    _shape("weight", weight, (k, v))
    _shape("labels", labels, (m,))
    _shape("lse", lse, (m,))
    return m, k, v


def validate_cross_entropy(hidden, weight, labels, loss, lse, precision: str, device: int,
                           ignore_index: int = -100) -> tuple[int, int, int]:
    import torch

    dtype = _input_dtype(precision)
    m, k, v = _check_loss(hidden, weight, labels, lse, dtype, device, ignore_index)
    _check("loss", loss, (torch.float32,), 1, device)
    _shape("loss", loss, (m,))
    _no_overlap({"loss": loss, "lse": lse}, {"hidden": hidden, "weight": weight, "labels": labels})
    return m, k, v


def validate_cross_entropy_backward(grad, hidden, weight, labels, lse, precision: str, device: int, dhidden=None,
                                    dweight=None, ignore_index: int = -100) -> tuple[int, int, int]:
    import torch

    dtype = _input_dtype(precision)
    if precision == "fp16":
        raise ValueError("the gradient of each logit is held in the input format, and fp16 cannot hold the small ones; "
                         "use bf16 or tf32")
    either = (torch.float32, dtype)
    if dhidden is None and dweight is None:
        raise ValueError("no gradient is asked for: pass dhidden or dweight")
    m, k, v = _check_loss(hidden, weight, labels, lse, dtype, device, ignore_index)
    _check("grad", grad, (torch.float32,), 1, device)
    _shape("grad", grad, (m,))
    if dhidden is not None:
        _check("dhidden", dhidden, either, 2, device)
        _shape("dhidden", dhidden, (m, k))
    if dweight is not None:
        _check("dweight", dweight, either, 2, device)
        _shape("dweight", dweight, (k, v))
    _no_overlap({"dhidden": dhidden, "dweight": dweight},
                {"grad": grad, "hidden": hidden, "weight": weight, "labels": labels, "lse": lse})
    return m, k, v

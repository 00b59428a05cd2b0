"""Refusals of the operators next to the matrix product, without a GPU: operand contracts in Python and the C-ABI's
own argument checks, which come before any device work."""

from __future__ import annotations

import ctypes

import pytest
import torch

import operator_contracts as ops
from operator_contracts import (ACTIVATION_IDS, ACTIVATIONS, validate_cross_entropy, validate_cross_entropy_backward,
                       validate_epilogue, validate_epilogue_backward, validate_grouped, validate_grouped_backward)

BF16, FP32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def cpu_tensors_pass_as_device_tensors(monkeypatch):
    """The checks but for the device, which cannot be met here (it has its own test)."""
    def check(name, tensor, dtypes, ndim, device):
        if not isinstance(tensor, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if tensor.ndim != ndim:
            raise ValueError(f"{name} must have {ndim} dimensions")
        if tensor.dtype not in dtypes:
            raise TypeError(f"{name} must have dtype {dtypes}")
        if not tensor.is_contiguous():
            raise ValueError(f"{name} must be contiguous")

    request_device = ops._check
    monkeypatch.setattr(ops, "_check", check)
    yield request_device


def mats():
    return (torch.ones((4, 8), dtype=BF16), torch.ones((8, 16), dtype=BF16), torch.ones((4, 16), dtype=FP32))


def test_activation_ids_match_the_header():
    assert ACTIVATIONS == ("none", "relu", "gelu", "gelu_tanh", "silu")
    assert ACTIVATION_IDS == {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


def test_epilogue_accepts_its_contract():
    a, b, out = mats()
    assert validate_epilogue(a, b, out, "bf16", 0) == (4, 8, 16)
    assert validate_epilogue(a, b, out.to(BF16), "bf16", 0, torch.ones(16), "gelu", torch.ones((4, 16), dtype=BF16),
                             torch.ones((4, 16), dtype=BF16)) == (4, 8, 16)
    assert validate_epilogue(a, b, out, "bf16", 0, residual=out) == (4, 8, 16)     # in place


@pytest.mark.parametrize("change,error", [
    ({"a": None}, TypeError), ({"a": torch.ones(8, dtype=BF16)}, ValueError),
    ({"a": torch.ones((4, 8))}, TypeError), ({"b": torch.ones((8, 16), dtype=torch.float16)}, TypeError),
    ({"b": torch.ones((16, 8), dtype=BF16).t()}, ValueError), ({"b": torch.ones((9, 16), dtype=BF16)}, ValueError),
    ({"out": torch.ones((4, 16), dtype=torch.float16)}, TypeError), ({"out": torch.ones((5, 16))}, ValueError),
    ({"a": torch.ones((0, 8), dtype=BF16), "out": torch.ones((0, 16))}, ValueError),
    ({"precision": "fp32"}, ValueError), ({"precision": "int8"}, ValueError),
    ({"activation": "tanh"}, ValueError), ({"activation": None}, ValueError), ({"activation": 2}, ValueError),
    ({"bias": torch.ones(15)}, ValueError), ({"bias": torch.ones((1, 16))}, ValueError),
    ({"bias": torch.ones(16, dtype=torch.float64)}, TypeError),
    ({"residual": torch.ones((4, 16), dtype=BF16)}, TypeError), ({"residual": torch.ones((16,))}, ValueError),
    ({"preact": torch.ones((4, 15))}, ValueError), ({"preact": torch.ones((4, 16), dtype=torch.int32)}, TypeError),
])
def test_epilogue_refuses(change, error):
    a, b, out = mats()
    args = {"a": a, "b": b, "out": out, "precision": "bf16", "device": 0} | change
    with pytest.raises(error):
        validate_epilogue(**args)


def test_outputs_must_not_overlap():
    store = torch.zeros(4096, dtype=BF16)
    a, b = store[:32].view(4, 8), torch.ones((8, 16), dtype=BF16)
    with pytest.raises(ValueError, match="out must not overlap a"):
        validate_epilogue(a, b, store[16:80].view(4, 16), "bf16", 0)
    a = torch.ones((4, 8), dtype=BF16)
    out, shifted = store[:64].view(4, 16), store[16:80].view(4, 16)
    with pytest.raises(ValueError, match="residual"):
        validate_epilogue(a, b, out, "bf16", 0, residual=shifted)
    with pytest.raises(ValueError, match="preact"):
        validate_epilogue(a, b, out, "bf16", 0, preact=out)
    with pytest.raises(ValueError, match="da must not overlap"):
        dout = torch.ones((4, 16), dtype=BF16)
        both = torch.zeros(1024, dtype=BF16)
        validate_epilogue_backward(dout, a, b, "bf16", 0, da=both[:32].view(4, 8), db=both[16:144].view(8, 16))


def test_device_is_checked(cpu_tensors_pass_as_device_tensors, monkeypatch):
    monkeypatch.setattr(ops, "_check", cpu_tensors_pass_as_device_tensors)
    a, b, out = mats()
    with pytest.raises(ValueError, match="cuda:0"):
        validate_epilogue(a, b, out, "bf16", 0)


def backward_args():
    a, b, _ = mats()
    return {"dout": torch.ones((4, 16), dtype=BF16), "a": a, "b": b, "precision": "bf16", "device": 0,
            "activation": "gelu", "preact": torch.ones((4, 16), dtype=BF16), "da": torch.ones((4, 8)),
            "db": torch.ones((8, 16)), "dbias": torch.ones(16)}


def test_epilogue_backward_accepts_any_subset():
    args = backward_args()
    assert validate_epilogue_backward(**args) == (4, 8, 16)
    assert validate_epilogue_backward(**(args | {"a": None, "db": None})) == (4, 8, 16)
    assert validate_epilogue_backward(**(args | {"b": None, "da": None})) == (4, 8, 16)
    assert validate_epilogue_backward(**(args | {"a": None, "b": None, "da": None, "db": None})) == (4, 1, 16)
    assert validate_epilogue_backward(**(args | {"activation": "none", "preact": None})) == (4, 8, 16)


@pytest.mark.parametrize("change,error", [
    ({"da": None, "db": None, "dbias": None}, ValueError), ({"preact": None}, TypeError), ({"a": None}, TypeError),
    ({"b": None}, TypeError), ({"dout": torch.ones((4, 16))}, TypeError),
    ({"a": torch.ones((5, 8), dtype=BF16)}, ValueError), ({"a": torch.ones((4, 9), dtype=BF16)}, ValueError),
    ({"b": torch.ones((8, 15), dtype=BF16)}, ValueError), ({"da": torch.ones((8, 4))}, ValueError),
    ({"db": torch.ones((16, 8))}, ValueError), ({"dbias": torch.ones(8)}, ValueError),
    ({"preact": torch.ones((4, 8))}, ValueError), ({"activation": "swish"}, ValueError),
])
def test_epilogue_backward_refuses(change, error):
    with pytest.raises(error):
        validate_epilogue_backward(**(backward_args() | change))


def grouped_args():
    return {"a": torch.ones((6, 8), dtype=BF16), "b": torch.ones((3, 8, 16), dtype=BF16),
            "offsets": torch.zeros(4, dtype=torch.int32), "precision": "bf16", "device": 0}


@pytest.mark.parametrize("change,error", [
    ({"a": torch.ones((6, 9), dtype=BF16)}, ValueError), ({"b": torch.ones((8, 16), dtype=BF16)}, ValueError),
    ({"offsets": torch.zeros(3, dtype=torch.int32)}, ValueError), ({"offsets": torch.zeros(4)}, TypeError),
    ({"offsets": [0, 1, 2, 6]}, TypeError), ({"out": torch.ones((6, 8))}, ValueError),
    ({"a": torch.ones((0, 8), dtype=BF16), "out": torch.ones((0, 16))}, ValueError), ({"precision": "fp32"}, ValueError),
])
def test_grouped_refuses(change, error):
    args = grouped_args() | {"out": torch.ones((6, 16))}
    assert validate_grouped(**args) == (6, 3, 8, 16)
    with pytest.raises(error):
        validate_grouped(**(args | change))


@pytest.mark.parametrize("change,error", [
    ({"da": None, "db": None}, ValueError), ({"a": None}, TypeError), ({"b": None}, TypeError),
    ({"db": torch.ones((2, 8, 16))}, ValueError), ({"da": torch.ones((6, 16))}, ValueError),
    ({"dout": torch.ones((5, 16), dtype=BF16)}, ValueError), ({"offsets": None}, TypeError),
    ({"offsets": torch.zeros(5, dtype=torch.int64)}, ValueError),
])
def test_grouped_backward_refuses(change, error):
    args = grouped_args() | {"dout": torch.ones((6, 16), dtype=BF16), "da": torch.ones((6, 8)),
                             "db": torch.ones((3, 8, 16))}
    assert validate_grouped_backward(**args) == (6, 3, 8, 16)
    assert validate_grouped_backward(**(args | {"da": None, "b": None})) == (6, 3, 8, 16)
    assert validate_grouped_backward(**(args | {"db": None, "a": None})) == (6, 3, 8, 16)
    with pytest.raises(error):
        validate_grouped_backward(**(args | change))


def loss_args():
    return {"hidden": torch.ones((5, 8), dtype=BF16), "weight": torch.ones((8, 30), dtype=BF16),
            "labels": torch.zeros(5, dtype=torch.int64), "lse": torch.zeros(5), "precision": "bf16", "device": 0}


@pytest.mark.parametrize("change,error", [
    ({"weight": torch.ones((9, 30), dtype=BF16)}, ValueError), ({"labels": torch.zeros(4, dtype=torch.int64)}, ValueError),
    ({"labels": torch.zeros(5)}, TypeError), ({"loss": torch.zeros(5, dtype=BF16)}, TypeError),
    ({"lse": torch.zeros(6)}, ValueError), ({"ignore_index": True}, ValueError), ({"ignore_index": 1.5}, ValueError),
    ({"ignore_index": 2 ** 63}, ValueError), ({"precision": "fp32"}, ValueError),
])
def test_cross_entropy_refuses(change, error):
    args = loss_args() | {"loss": torch.zeros(5)}
    assert validate_cross_entropy(**args) == (5, 8, 30)
    with pytest.raises(error):
        validate_cross_entropy(**(args | change))
    with pytest.raises(ValueError, match="overlap"):
        validate_cross_entropy(**(args | {"loss": args["lse"]}))


@pytest.mark.parametrize("change,error", [
    ({"dhidden": None, "dweight": None}, ValueError), ({"grad": torch.zeros(5, dtype=BF16)}, TypeError),
    ({"grad": torch.zeros(4)}, ValueError), ({"dhidden": torch.ones((8, 5))}, ValueError),
    ({"dweight": torch.ones((30, 8))}, ValueError),
])
def test_cross_entropy_backward_refuses(change, error):
    args = loss_args() | {"grad": torch.zeros(5), "dhidden": torch.ones((5, 8)), "dweight": torch.ones((8, 30))}
    assert validate_cross_entropy_backward(**args) == (5, 8, 30)
    with pytest.raises(error):
        validate_cross_entropy_backward(**(args | change))


def test_cross_entropy_backward_refuses_fp16():
    args = loss_args() | {"grad": torch.zeros(5), "dhidden": torch.ones((5, 8)), "precision": "fp16"}
    with pytest.raises(ValueError, match="fp16"):
        validate_cross_entropy_backward(**args)


# ---------------------------------------------------------------- the C entry points' own checks
@pytest.fixture(scope="module")
def lib(library_path):
    from gpumat import load_library

    return load_library(library_path)


def _call(lib, name, *args):
    error = ctypes.create_string_buffer(512)
    rc = getattr(lib, name)(*args, error, len(error))
    return rc, error.value.decode()


CALLS = {
    "matmul_epilogue": lambda ctx, prec, m=4: (ctx, prec, 16, 16, None, 0, 0, None, 16, 0, None, 0, m, 8, 8, None),
    "matmul_epilogue_backward": lambda ctx, prec, m=4: (ctx, prec, 16, 16, 16, None, 0, 0, 16, 0, 16, 0, None, 0, m, 8, 8,
                                                        None),
    "matmul_grouped": lambda ctx, prec, m=4: (ctx, prec, 16, 16, 16, 0, 2, 16, 0, m, 8, 8, None),
    "matmul_grouped_backward": lambda ctx, prec, m=4: (ctx, prec, 16, 16, 16, 16, 0, 2, 16, 0, 16, 0, m, 8, 8, None),
    "matmul_cross_entropy": lambda ctx, prec, m=4: (ctx, prec, 16, 16, 16, 1, -100, 16, 16, m, 8, 8, None),
    "matmul_cross_entropy_backward": lambda ctx, prec, m=4: (ctx, prec, 16, 16, 16, 16, 1, -100, 16, 16, 0, 16, 0, m, 8, 8,
                                                             None),
}


@pytest.mark.parametrize("name", CALLS)
def test_entry_points_refuse_before_any_device_work(lib, name):
    """Checked on a context-sized block of zeros: these refusals come before anything of it is read."""
    block = ctypes.create_string_buffer(4096)
    ctx = ctypes.addressof(block)
    assert _call(lib, name, *CALLS[name](None, 3)) == (1, f"{name}: context is null")
    for precision in (0, 4, -1):
        rc, text = _call(lib, name, *CALLS[name](ctx, precision))
        assert rc == 1 and text.startswith(f"{name}: the precision must be")
    rc, text = _call(lib, name, *CALLS[name](ctx, 3, m=0))
    assert (rc, text) == (1, f"{name}: dimensions must be positive")
    rc, text = _call(lib, name, *CALLS[name](ctx, 3, m=2**31 - 1023))
    assert (rc, text) == (1, f"{name}: dimensions must be at most 2147482624")
    null = list(CALLS[name](ctx, 3))
    null[2] = None
    rc, text = _call(lib, name, *null)
    assert rc == 1 and "null" in text
    odd = list(CALLS[name](ctx, 3))
    odd[3] = 17
    rc, text = _call(lib, name, *odd)
    assert (rc, text) == (1, f"{name}: a pointer is not aligned to its element size")
    assert getattr(lib, name)(*CALLS[name](None, 3), None, 0) == 1      # the error buffer may be null


def test_entry_points_refuse_more(lib):
    block = ctypes.create_string_buffer(4096)
    ctx = ctypes.addressof(block)
    args = list(CALLS["matmul_epilogue"](ctx, 3))
    args[6] = 5
    assert _call(lib, "matmul_epilogue", *args) == (1, "matmul_epilogue: unknown activation")
    args = list(CALLS["matmul_epilogue_backward"](ctx, 3))
    args[8] = args[10] = None
    assert "no gradient" in _call(lib, "matmul_epilogue_backward", *args)[1]
    args = list(CALLS["matmul_epilogue_backward"](ctx, 3))
    args[7] = 2                                                        # an activation without preact
    assert "null" in _call(lib, "matmul_epilogue_backward", *args)[1]
    args = list(CALLS["matmul_grouped"](ctx, 3))
    args[6] = 0
    assert "positive" in _call(lib, "matmul_grouped", *args)[1]
    assert "fp16" in _call(lib, "matmul_cross_entropy_backward", *CALLS["matmul_cross_entropy_backward"](ctx, 2))[1]


def test_sizes_whose_tiles_would_leave_32_bits_are_refused():
    ops._sizes(1, ops.SIZE_MAX)
    for size in (0, -1, ops.SIZE_MAX + 1, 2**31 - 1, 2**40):
        with pytest.raises(ValueError, match="must be positive and at most 2147482624"):
            ops._sizes(4, size)

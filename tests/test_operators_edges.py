"""Edges of the operators next to the matrix product that need no GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

import operator_contracts as ops
from gpumat import load_library


def _call(library, name, *args):
    error = ctypes.create_string_buffer(512)
    return getattr(library, name)(*args, error, len(error)), error.value.decode()


@pytest.mark.parametrize("groups", (2**28 + 1, 2**31 - 1024))
def test_more_groups_than_a_plan_counts_are_refused(library_path, monkeypatch, groups):
    """A group weighs at least six K blocks in the plan of the weight gradient: from 2^31 / 6 groups on their sum
    passed 32 bits, and tiles were looked up outside the table.  Refused before any device work."""
    library = load_library(library_path)
    block = ctypes.create_string_buffer(4096)
    ctx = ctypes.addressof(block)
    assert _call(library, "matmul_grouped", ctx, 3, 16, 16, 16, 0, groups, 16, 0, 4, 8, 8, None) == \
        (1, "matmul_grouped: groups must be at most 268435456")
    assert _call(library, "matmul_grouped_backward", ctx, 3, 16, 16, 16, 16, 0, groups, 16, 0, 16, 0, 4, 8, 8, None) == \
        (1, "matmul_grouped_backward: groups must be at most 268435456")

    monkeypatch.setattr(ops, "_check", lambda *args: None)
    bf16 = dict(dtype=torch.bfloat16, device="meta")
    b, offsets = torch.empty((groups, 8, 8), **bf16), torch.empty(groups + 1, dtype=torch.int32, device="meta")
    rows = torch.empty((4, 8), **bf16)
    with pytest.raises(ValueError, match="groups must be at most 268435456"):
        ops.validate_grouped(rows, b, offsets, rows, "bf16", 0)
    with pytest.raises(ValueError, match="groups must be at most 268435456"):
        ops.validate_grouped_backward(rows, rows, None, offsets, "bf16", 0, db=b)

"""Edges of the operators next to the matrix product that need no GPU."""

from __future__ import annotations

import ctypes
from pathlib import Path

import pytest
import torch

import operator_contracts as ops
from gpumat import NativeMatmul, load_library


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


def test_operands_that_no_gradient_reads_may_be_anything(monkeypatch):
    """They are not checked, so they do not reach the library either: a tensor on another device could not be recorded
    on the stream, and what is no tensor has no pointer."""
    monkeypatch.setattr(ops, "_check", lambda *args: None)
    taken = []
    native = object.__new__(NativeMatmul)
    native._device = 0
    monkeypatch.setattr(NativeMatmul, "_operator_precision", lambda self, precision: 3)
    monkeypatch.setattr(NativeMatmul, "_operator",
                        lambda self, name, arguments, tensors, outputs: taken.append([t for t in tensors if t is not None]))
    a, b, dout = torch.ones((4, 8)), torch.ones((8, 16)), torch.ones((4, 16))
    da, db, dbias = torch.empty((4, 8)), torch.empty((8, 16)), torch.empty(16)
    for unread in (torch.ones(3), "no tensor", 7):
        native.prepare_epilogue_backward(dout, a, unread, precision="bf16", preact=unread, db=db)
        native.prepare_epilogue_backward(dout, unread, b, precision="bf16", preact=unread, da=da)
        native.prepare_epilogue_backward(dout, unread, unread, precision="bf16", preact=unread, dbias=dbias)
        experts, offsets = torch.ones((2, 8, 16)), torch.zeros(3, dtype=torch.int32)
        native.prepare_grouped_backward(dout, a, unread, offsets, precision="bf16", db=torch.empty((2, 8, 16)))
        native.prepare_grouped_backward(dout, unread, experts, offsets, precision="bf16", da=da)
        assert len(taken) == 5 and not any(t is unread for tensors in taken for t in tensors)
        taken.clear()


def test_every_command_of_the_build_is_sm100a_only(monkeypatch, tmp_path):
    """The commands that build() runs, and no others: each source compiled once, all objects linked, for one
    architecture."""
    import build

    ran = []

    def run(cmd):
        ran.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).touch()
        return ""

    monkeypatch.setattr(build, "_run", run)
    output = build.build(force=True, output=tmp_path / "library.so")
    assert output.exists() and len(ran) == len(build.SOURCES) + 1
    compiles, link = ran[:-1], ran[-1]
    assert sorted(cmd[-1] for cmd in compiles) == sorted(map(str, build.SOURCES)) and all("-c" in cmd for cmd in compiles)
    assert sorted(link[link.index("-o") + 2:]) == sorted(cmd[cmd.index("-o") + 1] for cmd in compiles) and "-shared" in link
    for cmd in (*ran, build.command()):
        assert cmd.count("-gencode") == 1 and cmd[cmd.index("-gencode") + 1] == "arch=compute_100a,code=sm_100a"
        assert not any(flag.startswith(("-arch", "--gpu", "-code", "--generate-code", "-gencode=")) for flag in cmd)

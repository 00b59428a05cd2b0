"""Edges of the operators next to the matrix product (needs a B200): logits at the ends of FP32's range, the
activations' ends, first calls, and waits that run out."""

from __future__ import annotations

import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import operator_reference as ref
from operator_contracts import SIZE_MAX
from operator_reference import DTYPES, assert_within
from test_operators_gpu import guarded, loss_inputs, randn, sizes_to_offsets
from test_operators_use_gpu import odd_weight

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32
LOAD, MMA, EPILOGUE, DRAIN = 1, 2, 4, 8
LOWEST = float(torch.finfo(torch.bfloat16).min)     # also a TF32 value


# ---------------------------------------------------------------- logits at the ends of FP32's range
# Rows on every tile kind, a vocabulary that TMA addresses and one that it does not (read in place for few
# rows, copied for more).
@pytest.mark.parametrize("precision", ("bf16", "tf32"))
@pytest.mark.parametrize("shape", [(3, 40, 2000), (64, 64, 20001), (200, 33, 1001), (300, 64, 50048), (1100, 24, 33024)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("masked", ("first", "last", "middle", "all but one"))
def test_loss_of_columns_masked_with_the_lowest_value(native, precision, shape, masked):
    """A weight row of 0 and the lowest value masks columns for the rows of `hidden` that have a 1 there.

    Masked columns add nothing to a sum: lse is that of the other columns, to the allowance of a product of the other
    k terms (a masked column's own sum may be off by any amount below its size).
    """
    m, k, v = shape
    hidden, weight, labels, grad = loss_inputs(m, k, v, precision)
    mask = torch.zeros(v, dtype=torch.bool, device="cuda")
    if masked == "first":
        mask[:v // 3] = True
    elif masked == "last":
        mask[-(v // 3):] = True
    elif masked == "middle":
        mask[70:v - 90] = True
    else:
        mask[:] = True
        mask[v // 2] = False
    kept = (~mask).nonzero()[:, 0]
    labels = torch.where(labels == -100, labels, kept[labels % len(kept)])
    hidden[:, 0], weight[0] = 1.0, torch.where(mask, LOWEST, 0.0)
    place = torch.zeros(v, dtype=torch.int64, device="cuda")
    place[kept] = torch.arange(len(kept), device="cuda")
    seen = torch.where(labels == -100, labels, place[labels.clamp(min=0)])
    expected = ref.cross_entropy(hidden[:, 1:], weight[1:, kept], seen, precision)
    # Chains and roundings are those of all v columns and k terms.
    slack = (v / 128.0) * ref.U + 2 * ref.U * (hidden[:, 1:].double().abs() @ weight[1:, kept].double().abs()).amax(1)
    (loss, ul), (lse, us) = guarded((m,), FP32), guarded((m,), FP32)
    native.prepare_cross_entropy(hidden, weight, labels, loss, lse, precision=precision)()
    assert_within(lse, expected["lse"][0], expected["lse"][1] + slack, "lse")
    assert_within(loss, expected["loss"][0], expected["loss"][1] + 2 * slack, "loss")
    ul(), us()
    # The gradients of masked columns are exactly zero.
    dhidden, dweight = torch.full((m, k), 7.0, device="cuda"), torch.full((k, v), 7.0, device="cuda")
    native.prepare_cross_entropy_backward(grad, hidden, weight, labels, lse, precision=precision, dhidden=dhidden,
                                          dweight=dweight)()
    assert not dweight[:, mask].any() and not dhidden[:, 0].any()
    assert torch.isfinite(dweight).all() and torch.isfinite(dhidden).all()


@pytest.mark.parametrize("precision", ("bf16", "tf32"))
@pytest.mark.parametrize("m,v", [(5, 3000), (64, 20001), (300, 50048), (1100, 33024)])
def test_loss_of_rows_without_a_column_left(native, precision, m, v):
    """Every column of some rows masked: all logits are the lowest value, so lse is it (half a step of it is far above
    log v) and the loss log v; of one row alone in the tile as of all.  Its logarithm and the sum of v ones, in chains
    of at most 256 + v / 256 terms, are off by (600 + v / 128) 2^-23 at most."""
    dtype = DTYPES[precision]
    hidden, weight = torch.zeros((m, 16), dtype=dtype, device="cuda"), torch.zeros((16, v), dtype=dtype, device="cuda")
    weight[0] = LOWEST
    hidden[1::3, 0] = 1.0
    weight[1], hidden[2::3, 1] = -LOWEST, 1.0      # and rows at the highest value
    labels = torch.arange(m, device="cuda") % v
    loss, lse = torch.empty(m, device="cuda"), torch.empty(m, device="cuda")
    native.prepare_cross_entropy(hidden, weight, labels, loss, lse, precision=precision)()
    log_v = torch.full((m,), float(v), dtype=torch.float64, device="cuda").log()
    tol = torch.full_like(log_v, (600.0 + v / 128.0) * ref.U) + 4 * ref.U * log_v
    assert_within(loss, log_v, tol, "loss")
    expected = log_v.clone()
    expected[1::3], expected[2::3] = LOWEST, -LOWEST
    assert_within(lse, expected, tol, "lse")


def test_loss_between_the_ends_of_the_range(native):
    """One logit of the highest value among the lowest: lse is it, the other labels' losses pass FP32's range."""
    m, v = 9, 4096
    for where in (0, 31, 32, 2049, v - 1):
        hidden, weight = torch.ones((m, 8), dtype=torch.bfloat16, device="cuda"), torch.zeros((8, v), dtype=torch.bfloat16, device="cuda")
        weight[0] = LOWEST
        weight[0, where] = -LOWEST
        labels = torch.full((m,), where, device="cuda")
        labels[3] = (where + 1) % v
        loss, lse = torch.empty(m, device="cuda"), torch.empty(m, device="cuda")
        native.prepare_cross_entropy(hidden, weight, labels, loss, lse, precision="bf16")()
        assert bool((lse == -LOWEST).all())
        assert float(loss[3]) == float("inf") and float(loss.nan_to_num(posinf=0.0).abs().sum()) == 0.0


@pytest.mark.parametrize("m,k,v", [(1, 16, 11), (5, 98, 222), (24, 267, 2408), (56, 109, 5175), (200, 64, 33000), (90, 64, 20001)])
def test_loss_of_a_row_depends_on_its_own_logits_alone(native, m, k, v):
    """Bit by bit the same after other calls, which leave other values in the memory behind the last row, and beside rows
    whose logits are at the ends of FP32's range."""
    hidden, weight, labels, _ = loss_inputs(m, k, v, "bf16")
    other = torch.full((200, k), 3e38, dtype=BF16, device="cuda")
    big = torch.full((k, v), 1.0, dtype=BF16, device="cuda")
    junk = torch.empty((200, v), dtype=BF16, device="cuda")
    loss, lse = torch.empty(m, device="cuda"), torch.empty(m, device="cuda")
    run = native.prepare_cross_entropy(hidden, weight, labels, loss, lse, precision="bf16")
    dirty = native.prepare_epilogue(other, big, junk, precision="bf16")
    run()
    first = loss.clone(), lse.clone()
    for _ in range(20):
        loss.zero_(), lse.zero_()
        torch.cuda.synchronize()
        dirty()
        run()
        assert torch.equal(loss, first[0]) and torch.equal(lse, first[1])
    if m > 2:
        hidden[m // 2] = 1e38
        run()
        rows = torch.arange(m, device="cuda") != m // 2
        assert torch.equal(loss[rows], first[0][rows]) and torch.equal(lse[rows], first[1][rows])


# ---------------------------------------------------------------- the activations' ends
@pytest.mark.parametrize("m", (1, 70, 300))
def test_gelu_keeps_its_relative_precision_in_the_tails(native, m):
    """gelu(z) = z Phi(z) and its slope Phi(z) + z phi(z) in FP32, at every z in [-12, 12].

    With u = 2^-23 the kernel's Phi(-|z|) is off by at most (12 + z^2 / 2) u of itself: 1.3 u the fit, 0.9 u the
    coefficients' roundings, 3.5 u those of Horner's seven steps, 2 u those of t (reciprocal 1 ulp), 2 u the hardware's
    exponential, 1.5 u the products, and z^2 / 2 u the two roundings of the exponent z^2 / 2 log2 e.  phi(z) is within
    those bounds too.  1 - Phi and each last operation add half a step of their result.
    """
    n = 4096
    gen = torch.Generator(device="cuda").manual_seed(m)
    z = torch.empty(n, device="cuda").uniform_(-12.0, 12.0, generator=gen)
    z[:3] = torch.tensor([0.0, -3.0, -5.0])
    zd = z.double()
    tail = 0.5 * torch.special.erfc(zd.abs() / math.sqrt(2.0))
    cdf = 0.5 * torch.special.erfc(-zd / math.sqrt(2.0))
    peak = torch.exp(-zd * zd / 2.0) / math.sqrt(2.0 * math.pi)
    bound = (12.0 + zd * zd / 2.0) * ref.U
    for precision in ("bf16", "tf32"):
        dtype = DTYPES[precision]
        a, b = torch.zeros((m, 8), dtype=dtype, device="cuda"), torch.zeros((8, n), dtype=dtype, device="cuda")
        out = torch.empty((m, n), device="cuda")
        native.prepare_epilogue(a, b, out, precision=precision, bias=z, activation="gelu")()
        assert_within(out, (zd * cdf).expand(m, n), (zd.abs() * (bound * tail + ref.U * cdf)).expand(m, n), "gelu")
        dbias = torch.empty(n, device="cuda")
        native.prepare_epilogue_backward(torch.ones((1, n), dtype=dtype, device="cuda"), precision=precision,
                                         activation="gelu", preact=z.view(1, n), dbias=dbias)()
        assert_within(dbias, cdf + zd * peak, bound * (tail + zd.abs() * peak) + ref.U * cdf, "slope")


@pytest.mark.parametrize("act", ("relu", "gelu", "gelu_tanh", "silu"))
def test_slopes_of_large_values(native, act):
    """Where an activation is z or 0 to all 24 bits its slope is 1 or 0 exactly, up to the largest finite z; NaN stays
    NaN (relu has slope 0 there, as the comparison z > 0 says)."""
    z = torch.tensor([1e2, 1e4, 6e4, 1e10, 1e19, 1.8e19, 1.9e19, 1e20, 1e30, 3.3e38], device="cuda")
    z = torch.cat([z, -z, torch.tensor([float("nan"), 0.5], device="cuda")])
    want = torch.cat([torch.ones(10), torch.zeros(10)]).cuda()
    dbias = torch.empty(22, device="cuda")
    for dtype, precision in ((BF16, "bf16"), (FP32, "tf32")):
        native.prepare_epilogue_backward(torch.ones((1, 22), dtype=dtype, device="cuda"), precision=precision,
                                         activation=act, preact=z.view(1, 22), dbias=dbias)()
        assert torch.equal(dbias[:20], want), f"{act}: {dbias.tolist()}"
        assert bool(torch.isnan(dbias[20])) == (act != "relu") and float(dbias[21]) > 0.5


# ---------------------------------------------------------------- first calls
FIRST_CALLS = """
import sys, threading
sys.path[:0] = [{package!r}, {tests!r}]
import torch
import operator_reference as ref
from gpumat import NativeMatmul

torch.manual_seed(1)
def randn(*shape, dtype=torch.bfloat16):
    return torch.randn(shape, device="cuda").to(dtype)

native = NativeMatmul()
stream = torch.cuda.Stream()
def case(dtype):
    name = {{torch.bfloat16: "bf16", torch.float16: "fp16", torch.float32: "tf32"}}[dtype]
    a, b, d, z = (randn(*s, dtype=dtype) for s in ((150, 130), (130, 264), (150, 264), (150, 264)))
    out, da, db = torch.zeros_like(d), torch.zeros_like(a), torch.zeros_like(b)
    runs = (native.prepare_epilogue(a, b, out, precision=name, activation="silu"),
            native.prepare_epilogue_backward(d, a, b, precision=name, activation="silu", preact=z, da=da, db=db))
    def check():
        back = ref.epilogue_backward(d, a, b, name, z, "silu")
        for got, key in ((da, "da"), (db, "db")):
            ref.assert_within(got, *back[key], f"{{name}} {{key}}")
        ref.assert_within(out, *ref.epilogue(a, b, name, None, "silu")["out"], name)
    return runs, check

# The first operator call of the process, in a capture.
with torch.cuda.stream(stream):
    runs, check = case(torch.bfloat16)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=stream):
    for run in runs:
        run()
graph.replay()
torch.cuda.synchronize()
check()
# The first calls in a format, from four threads at once.
checks, errors, gate = [], [], threading.Barrier(4)
def work(dtype):
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            runs, check = case(dtype)
            torch.cuda.current_stream().synchronize()
            gate.wait()
            for run in runs:
                run()
            torch.cuda.current_stream().synchronize()
        checks.append(check)
    except BaseException as error:
        errors.append(error)
        gate.abort()
threads = [threading.Thread(target=work, args=(d,)) for d in (torch.float16, torch.float16, torch.float32, torch.float32)]
for t in threads: t.start()
for t in threads: t.join()
assert not errors and len(checks) == 4, errors
for check in checks: check()
assert native.device_status() == 0
print("first calls hold")
"""


def test_first_calls_of_a_process(gpu_ready, library_path):
    """Kernels get their attributes by a format's first call: in a graph capture, and by four threads at once."""
    root = Path(__file__).resolve().parents[1]
    script = FIRST_CALLS.format(package=str(root / "matrix-multiplication_b200"), tests=str(root / "tests"))
    result = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True, timeout=300)
    assert result.returncode == 0 and "first calls hold" in result.stdout, result.stdout + result.stderr


# ---------------------------------------------------------------- waits that run out
def _limited_cases(native):
    """(name, launch, outputs, what the outputs hold before the call) for every kind of tile, epilogue and layout."""
    def filled(*shape, dtype=BF16):
        return torch.empty(shape, dtype=dtype, device="cuda")

    for m, k, n in ((16, 4096, 512), (16, 512, 16384), (100, 4096, 4096), (128, 64, 40000), (120, 64, 40001), (260, 320, 1000)):
        a, b = randn((m, k), BF16, 1), randn((k, n), BF16, 2, k ** -0.5)
        out, z = filled(m, n), filled(m, n, dtype=FP32)
        yield f"epilogue {m}x{k}x{n}", native.prepare_epilogue(a, b, out, precision="bf16", preact=z), (out, z), None
        dout, da, db, dbias = randn((m, n), BF16, 3), filled(m, k), filled(k, n), filled(n, dtype=FP32)
        yield (f"backward {m}x{k}x{n}",
               native.prepare_epilogue_backward(dout, a, b, precision="bf16", activation="silu", preact=dout, da=da, db=db,
                                                dbias=dbias), (da, db, dbias), None)
    for m, k, n in ((128, 64, 40000), (120, 64, 40001), (3000, 64, 8192), (3000, 64, 8190)):
        a, b = randn((m, k), BF16, 1), randn((k, n), BF16, 2, k ** -0.5)
        for dtype in (BF16, FP32):
            residual, place = randn((m, n), dtype, 4), filled(m, n, dtype=dtype)
            if m < 1000:
                out = filled(m, n, dtype=dtype)
                yield (f"residual {m}x{k}x{n} {dtype}",
                       native.prepare_epilogue(a, b, out, precision="bf16", activation="relu", residual=residual), (out,), None)
            yield (f"residual in place {m}x{k}x{n} {dtype}",
                   native.prepare_epilogue(a, b, place, precision="bf16", residual=place), (place,), residual)
    b, dout, da = randn((256, 20352), BF16, 2), randn((30, 20352), BF16, 3), filled(30, 256)
    yield "chunks of a long sum", native.prepare_epilogue_backward(dout, b=b, precision="bf16", da=da), (da,), None
    for sizes in ((10, 6), (500, 0, 600), (3, 1000, 1, 40)):
        ends, offsets = sizes_to_offsets(sizes)
        a, w = randn((ends[-1], 1024), BF16, 5), randn((len(sizes), 1024, 512), BF16, 6, 0.03)
        out, dout = filled(ends[-1], 512), randn((ends[-1], 512), BF16, 7)
        yield f"grouped {sizes}", native.prepare_grouped(a, w, offsets, out, precision="bf16"), (out,), None
        da, dw = filled(ends[-1], 1024), filled(len(sizes), 1024, 512)
        yield (f"grouped backward {sizes}",
               native.prepare_grouped_backward(dout, a, w, offsets, precision="bf16", da=da, db=dw), (da, dw), None)
    for m, k, v in ((100, 512, 20000), (100, 1024, 30001), (700, 64, 70000)):
        hidden, weight, labels, grad = loss_inputs(m, k, v, "bf16")
        loss, lse = filled(m, dtype=FP32), filled(m, dtype=FP32)
        yield f"loss {m}x{k}x{v}", native.prepare_cross_entropy(hidden, weight, labels, loss, lse, precision="bf16"), (loss, lse), None
        known = torch.logsumexp(hidden.float() @ weight.float(), 1)
        dh, dw = filled(m, k), filled(k, v)
        yield (f"loss backward {m}x{k}x{v}",
               native.prepare_cross_entropy_backward(grad, hidden, weight, labels, known, precision="bf16", dhidden=dh,
                                                     dweight=dw), (dh, dw), None)
    a, b, out = randn((16, 2048), BF16, 1), odd_weight(2048, 20001, BF16, 1), filled(16, 20001)
    yield "weight read in place", native.prepare_epilogue(a, b, out, precision="bf16"), (out,), None


def check_limited(native, limits):
    """For each limit and case: every element is NaN or what it is without a limit, NaN comes with a status, and the
    next call is right.  Returns the status words met."""
    reached = set()
    for name, run, outs, before in _limited_cases(native):
        def prepare():
            for t in outs:
                t.fill_(-12345.0) if before is None else t.copy_(before)
            torch.cuda.synchronize()

        prepare()
        run()
        torch.cuda.synchronize()
        good = [t.clone() for t in outs]
        assert native.device_status() == 0 and not any(bool(torch.isnan(t).any()) for t in good), name
        for limit in limits:
            prepare()
            native.set_wait_limit(limit)
            try:
                run()
                status = native.device_status()
            finally:
                native.set_wait_limit(0)
            reached.add(status)
            assert not status & DRAIN, f"{name}, {limit} ns: a drain wait ran out ({status:#x})"
            lost = 0
            for t, want in zip(outs, good):
                nan = torch.isnan(t)
                stale = ~nan & (t != want)
                assert not bool(stale.any()), f"{name}, {limit} ns: {int(stale.sum())} of {t.numel()} elements are neither"
                lost += int(nan.sum())
            assert lost == 0 or status, f"{name}, {limit} ns: NaN without a status"
        prepare()
        run()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(good, outs)) and native.device_status() == 0, name
    return reached


def test_every_element_that_a_short_wait_left_unfinished_is_nan(native):
    """From one poll to a few microseconds (a pair of CTAs that gave up waits two seconds for copies under way)."""
    assert any(status & (LOAD | MMA | EPILOGUE) for status in check_limited(native, (1, 2500)))


def test_a_tile_whose_sum_takes_seconds(native):
    """Sums of the largest length that are not split over CTAs: one tile runs 2^25 K blocks, longer than the limit of
    waits for progress.  Exact in FP32."""
    k, v = SIZE_MAX, 8
    at = torch.tensor([0, 63, 64, 12345, 1 << 30, k - 1], device="cuda")
    tall, row = torch.ones((k, v), dtype=BF16, device="cuda"), torch.zeros((1, k), dtype=BF16, device="cuda")
    row[0, at] = 1.0
    tall[at] = torch.arange(48, device="cuda").to(BF16).view(6, 8) / 16
    want = tall[at].sum(0, dtype=FP32)
    loss, lse = torch.empty(1, device="cuda"), torch.empty(1, device="cuda")
    native.prepare_cross_entropy(row, tall, torch.tensor([2], device="cuda"), loss, lse, precision="bf16")()
    assert native.device_status() == 0
    assert_within(lse, torch.logsumexp(want.double(), 0)[None], torch.full((1,), 600 * ref.U, device="cuda").double(), "lse")
    offsets = torch.tensor([0, 1], device="cuda")
    out = torch.zeros((1, v), device="cuda")
    native.prepare_grouped(row, tall.view(1, k, v), offsets, out, precision="bf16")()
    assert native.device_status() == 0 and torch.equal(out[0], want)
    column, db = row.view(k, 1).expand(k, 8).contiguous(), torch.zeros((1, 8, v), device="cuda")
    del row
    offsets[1] = k
    native.prepare_grouped_backward(tall, column, None, offsets, precision="bf16", db=db)()
    assert native.device_status() == 0 and torch.equal(db[0], want.expand(8, v))


# ---------------------------------------------------------------- uneven groups
@pytest.mark.parametrize("precision", ("bf16", "tf32"))
@pytest.mark.parametrize("groups,rows,hot", [(400, 3001, 2900), (300, 700, 690), (64, 2048, 1024), (513, 20000, 19480)])
def test_one_group_with_most_of_the_rows(native, precision, groups, rows, hot):
    """Tiles follow the mean group; a group of many times the mean is cut into as many of them as it takes, in both
    directions, wherever it stands."""
    k, n, dtype = 136, 200, DTYPES[precision]
    a, b, dout = randn((rows, k), dtype, 1), randn((groups, k, n), dtype, 2, k ** -0.5), randn((rows, n), dtype, 3)
    for where in (0, groups // 2, groups - 1):
        gen = torch.Generator().manual_seed(where)
        sizes = torch.bincount(torch.randint(0, groups, (rows - hot,), generator=gen), minlength=groups)
        sizes[where] += hot
        ends, offsets = sizes_to_offsets(sizes.tolist())
        (out, uo), (da, ua), (db, ub) = guarded((rows, n), FP32), guarded((rows, k), FP32), guarded((groups, k, n), FP32)
        native.prepare_grouped(a, b, offsets, out, precision=precision)()
        native.prepare_grouped_backward(dout, a, b, offsets, precision=precision, da=da, db=db)()
        assert_within(out, *ref.grouped(a, b, ends, precision, out), "out")
        (eda, tda), (edb, tdb) = ref.grouped_backward(dout, a, b, ends, precision, da)
        assert_within(da, eda, tda, "da")
        assert_within(db, edb, tdb, "db")
        uo(), ua(), ub()


# ---------------------------------------------------------------- bias of whole and half tiles
@pytest.mark.parametrize("precision", ("bf16", "fp16", "tf32"))
@pytest.mark.parametrize("m,k,n", [(2304, 2048, 384), (4352, 1024, 384), (2304, 2048, 640), (2100, 600, 1400)])
def test_bias_where_half_tiles_follow_whole_ones(native, precision, m, k, n):
    """Eight pairs of CTAs, whose last round runs as halves of tiles in other columns than the tiles before them.  A
    warpgroup without columns in the last whole tile is at its half tile while the other still adds the whole
    tile's bias: each reads its own."""
    dtype = DTYPES[precision]
    a, b, bias = randn((m, k), dtype, 1), randn((k, n), dtype, 2, k ** -0.5), randn((n,), FP32, 3, 5.0)
    native.set_sm_limit(16)
    try:
        for act, out_dtype, has_preact in (("gelu", dtype, True), ("none", dtype, False), ("silu", FP32, False)):
            out = torch.empty((m, n), dtype=out_dtype, device="cuda")
            preact = torch.empty((m, n), device="cuda") if has_preact else None
            run = native.prepare_epilogue(a, b, out, precision=precision, bias=bias, activation=act, preact=preact)
            run()
            expected = ref.epilogue(a, b, precision, bias, act)
            assert_within(out, *expected["out"], f"out {act}")
            first = out.clone()
            for _ in range(40):
                out.zero_()
                run()
                assert torch.equal(out, first)
            if has_preact:
                assert_within(preact, *expected["preact"], "preact")
    finally:
        native.set_sm_limit(0)

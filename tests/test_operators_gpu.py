"""The operators next to the matrix product against plain 64-bit forms (needs a B200): the product with bias,
activation and residual in its epilogue, products grouped by expert, and cross entropy over a vocabulary, each with
its gradients.  Sizes from one row up, odd ones, every tile and layout, empty groups, ignored rows, special values."""

from __future__ import annotations

import pytest
import torch

import operator_reference as ref
from operator_contracts import ACTIVATIONS
from operator_reference import DTYPES, assert_within

pytestmark = pytest.mark.gpu

PRECISIONS = ("bf16", "fp16", "tf32")


def randn(shape, dtype, seed, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def offset_copy(x):
    """The same matrix one element past an allocation: no 16-byte alignment."""
    flat = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:]
    return flat.view(x.shape).copy_(x)


def guarded(shape, dtype, fill=7.0):
    """An output inside a larger allocation, and a check that nothing around it was written."""
    count = 1
    for s in shape:
        count *= s
    whole = torch.full((count + 512,), fill, dtype=dtype, device="cuda")
    out = whole[256:256 + count].view(shape)

    def untouched():
        assert bool((whole[:256] == fill).all()) and bool((whole[256 + count:] == fill).all())

    return out, untouched


# ---------------------------------------------------------------- product with epilogue
EPILOGUE_SHAPES = [
    # one row up to the widest transposed tile; odd sizes; every regular tile
    (1, 1, 1), (1, 4096, 1000), (2, 33, 65), (16, 512, 777), (17, 129, 256), (33, 64, 130), (64, 1000, 264),
    (65, 64, 64), (127, 257, 129), (129, 65, 257), (513, 129, 577), (300, 512, 72), (1000, 1024, 1000),
    (1024, 320, 2048), (2049, 72, 4104),
]


@pytest.mark.parametrize("precision", PRECISIONS)
@pytest.mark.parametrize("shape", EPILOGUE_SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_epilogue_every_size(native, precision, shape):
    m, k, n = shape
    dtype = DTYPES[precision]
    act = ACTIVATIONS[(m + n) % len(ACTIVATIONS)]
    a, b = randn((m, k), dtype, m + k), randn((k, n), dtype, n, k ** -0.5)
    bias = randn((n,), dtype, 3)
    for out_dtype in dict.fromkeys((dtype, torch.float32)):
        residual = randn((m, n), out_dtype, 4)
        out, untouched = guarded((m, n), out_dtype)
        preact, preact_untouched = guarded((m, n), out_dtype)
        run = native.prepare_epilogue(a, b, out, precision=precision, bias=bias, activation=act, residual=residual,
                                      preact=preact)
        assert run() is out
        expected = ref.epilogue(a, b, precision, bias, act, residual)
        assert_within(out, *expected["out"], f"out {act}")
        assert_within(preact, *expected["preact"], "preact")
        untouched()
        preact_untouched()
        first = out.clone()
        run()
        assert torch.equal(first, out)


@pytest.mark.parametrize("m", (5, 200))
@pytest.mark.parametrize("act", ACTIVATIONS)
def test_epilogue_every_activation_and_combination(native, act, m):
    k, n = 192, 264
    a, b = randn((m, k), torch.bfloat16, 1), randn((k, n), torch.bfloat16, 2, 3 * k ** -0.5)
    for bias_dtype in (None, torch.float32, torch.bfloat16):
        for has_residual in (False, True):
            for out_dtype, preact_dtype in ((torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32),
                                            (torch.float32, None)):
                bias = None if bias_dtype is None else randn((n,), bias_dtype, 3)
                residual = randn((m, n), out_dtype, 4) if has_residual else None
                out = torch.empty((m, n), dtype=out_dtype, device="cuda")
                preact = None if preact_dtype is None else torch.empty((m, n), dtype=preact_dtype, device="cuda")
                native.prepare_epilogue(a, b, out, precision="bf16", bias=bias, activation=act, residual=residual,
                                        preact=preact)()
                expected = ref.epilogue(a, b, "bf16", bias, act, residual)
                assert_within(out, *expected["out"], f"{act} {bias_dtype} {has_residual}")
                if preact is not None:
                    assert_within(preact, *expected["preact"], "preact")


@pytest.mark.parametrize("precision", PRECISIONS)
@pytest.mark.parametrize("shape", [(3, 40, 72), (140, 136, 264)], ids=str)
def test_epilogue_unaligned_everything(native, precision, shape):
    m, k, n = shape
    dtype = DTYPES[precision]
    a, b = offset_copy(randn((m, k), dtype, 1)), offset_copy(randn((k, n), dtype, 2))
    bias, residual = offset_copy(randn((n,), dtype, 3)), offset_copy(randn((m, n), dtype, 4))
    out, preact = (offset_copy(torch.zeros((m, n), dtype=dtype, device="cuda")) for _ in range(2))
    native.prepare_epilogue(a, b, out, precision=precision, bias=bias, activation="silu", residual=residual,
                            preact=preact)()
    expected = ref.epilogue(a, b, precision, bias, "silu", residual)
    assert_within(out, *expected["out"], "out")
    assert_within(preact, *expected["preact"], "preact")


@pytest.mark.parametrize("m", (9, 150, 400))
def test_epilogue_residual_in_place(native, m):
    k, n = 128, 520
    a, b = randn((m, k), torch.bfloat16, 1), randn((k, n), torch.bfloat16, 2, k ** -0.5)
    for dtype in (torch.bfloat16, torch.float32):
        out = randn((m, n), dtype, 3)
        expected = ref.epilogue(a, b, "bf16", None, "gelu", out)
        native.prepare_epilogue(a, b, out, precision="bf16", activation="gelu", residual=out)()
        assert_within(out, *expected["out"], "in place")


def test_epilogue_carries_special_values(native):
    """NaN and infinities pass through the activations as in torch; one bad row stays one bad row."""
    k, n = 64, 128
    for m in (8, 136):
        a, b = randn((m, k), torch.bfloat16, 1), randn((k, n), torch.bfloat16, 2)
        a[3] = float("nan")
        a[5] = 0.0
        a[5, 0] = float("inf")
        for act in ACTIVATIONS:
            out = torch.empty((m, n), dtype=torch.float32, device="cuda")
            native.prepare_epilogue(a, b, out, precision="bf16", activation=act)()
            assert bool(torch.isnan(out[3]).all())
            z = a[5].double() @ b.double()
            expected, _ = ref.activation(z, act)
            plus = z == float("inf")
            assert bool((out[5][plus] == float("inf")).all())
            if act == "relu":
                assert bool((out[5][z == -float("inf")] == 0).all())
            keep = [i for i in range(m) if i not in (3, 5)]
            assert bool(torch.isfinite(out[keep]).all())


@pytest.mark.parametrize("precision", ("fp16", "bf16"))
def test_epilogue_ties_round_to_even(native, precision):
    """An identity product: the one rounding of out is to nearest even."""
    dtype = DTYPES[precision]
    step = torch.finfo(dtype).eps
    for m in (4, 128):
        a = torch.eye(m, 64, dtype=dtype, device="cuda")
        b = torch.ones((64, 64), dtype=dtype, device="cuda")
        bias = torch.tensor([step / 2, 3 * step / 2] * 32, dtype=torch.float32, device="cuda")
        out = torch.empty((m, 64), dtype=dtype, device="cuda")
        native.prepare_epilogue(a[:, :64].contiguous(), b, out, precision=precision, bias=bias)()
        expected = torch.tensor([1.0, 1.0 + 2 * step] * 32, dtype=torch.float64, device="cuda")
        assert torch.equal(out[:min(m, 64)].double(), expected.expand(min(m, 64), 64))


BACKWARD_SHAPES = [(1, 8, 8), (1, 300, 77), (7, 64, 1000), (64, 256, 256), (129, 65, 257), (513, 129, 577),
                   (777, 300, 220), (1024, 512, 1536), (2048, 1024, 640)]


@pytest.mark.parametrize("precision", PRECISIONS)
@pytest.mark.parametrize("shape", BACKWARD_SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_epilogue_backward_every_size(native, precision, shape):
    m, k, n = shape
    dtype = DTYPES[precision]
    act = ACTIVATIONS[(m + k + n) % len(ACTIVATIONS)]
    dout, a, b = randn((m, n), dtype, 1), randn((m, k), dtype, 2), randn((k, n), dtype, 3, k ** -0.5)
    preact = randn((m, n), dtype, 4, 2.0)
    for grad_dtype in dict.fromkeys((dtype, torch.float32)):
        (da, ua), (db, ub), (dbias, uc) = (guarded(s, grad_dtype) for s in ((m, k), (k, n), (n,)))
        run = native.prepare_epilogue_backward(dout, a, b, precision=precision, activation=act, preact=preact, da=da,
                                               db=db, dbias=dbias)
        run()
        expected = ref.epilogue_backward(dout, a, b, precision, preact, act)
        for name, got in (("da", da), ("db", db), ("dbias", dbias)):
            assert_within(got, *expected[name], f"{name} {act}")
        ua(), ub(), uc()
        first = [t.clone() for t in (da, db, dbias)]
        run()
        assert all(torch.equal(x, y) for x, y in zip(first, (da, db, dbias)))


@pytest.mark.parametrize("act", ACTIVATIONS)
def test_epilogue_backward_each_gradient_alone(native, act):
    m, k, n = 200, 136, 264
    dout, a, b = (randn(s, torch.bfloat16, i) for i, s in enumerate(((m, n), (m, k), (k, n))))
    preact = None if act == "none" else randn((m, n), torch.float32, 9, 2.0)
    expected = ref.epilogue_backward(dout, a, b, "bf16", preact, act)
    da = torch.empty((m, k), dtype=torch.float32, device="cuda")
    native.prepare_epilogue_backward(dout, b=b, precision="bf16", activation=act, preact=preact, da=da)()
    assert_within(da, *expected["da"], "da")
    db = torch.empty((k, n), dtype=torch.float32, device="cuda")
    native.prepare_epilogue_backward(dout, a, precision="bf16", activation=act, preact=preact, db=db)()
    assert_within(db, *expected["db"], "db")
    dbias = torch.empty((n,), dtype=torch.float32, device="cuda")
    native.prepare_epilogue_backward(dout, precision="bf16", activation=act, preact=preact, dbias=dbias)()
    assert_within(dbias, *expected["dbias"], "dbias")


@pytest.mark.parametrize("act", ("gelu", "gelu_tanh", "silu"))
def test_epilogue_gradients_against_differences(native, act):
    """The gradients against central differences of the 64-bit form of the whole expression."""
    m, k, n = 24, 40, 48
    a, b = randn((m, k), torch.bfloat16, 1), randn((k, n), torch.bfloat16, 2, k ** -0.5)
    bias, dout = randn((n,), torch.float32, 3), randn((m, n), torch.bfloat16, 4)
    preact = torch.empty((m, n), dtype=torch.float32, device="cuda")
    out = torch.empty_like(preact)
    native.prepare_epilogue(a, b, out, precision="bf16", bias=bias, activation=act, preact=preact)()
    da = torch.empty((m, k), dtype=torch.float32, device="cuda")
    db = torch.empty((k, n), dtype=torch.float32, device="cuda")
    dbias = torch.empty((n,), dtype=torch.float32, device="cuda")
    native.prepare_epilogue_backward(dout, a, b, precision="bf16", activation=act, preact=preact, da=da, db=db,
                                     dbias=dbias)()

    def total(a64, b64, bias64):
        return (ref.activation(a64 @ b64 + bias64, act)[0] * dout.double()).sum()

    h = 1e-4
    expected = ref.epilogue_backward(dout, a, b, "bf16", preact, act)
    for which, got, name in ((0, da, "da"), (1, db, "db"), (2, dbias, "dbias")):
        for index in (0, got.numel() // 2, got.numel() - 1):
            sides = []
            for sign in (1, -1):
                args = [a.double(), b.double(), bias.double()]
                args[which] = args[which].clone()
                args[which].view(-1)[index] += sign * h
                sides.append(total(*args))
            difference = float(sides[0] - sides[1]) / (2 * h)
            # Differences: h^2 / 6 times a third derivative, below 10 per term on these sizes' 24-48 terms.
            slack = float(expected[name][1].reshape(-1)[index]) + h * h * 10 * 48 + 1e-6
            assert abs(float(got.reshape(-1)[index]) - difference) <= slack + 2.0 ** -24 * abs(difference)


# ---------------------------------------------------------------- grouped products
def sizes_to_offsets(sizes, dtype=torch.int32, first=0):
    ends = [first]
    for s in sizes:
        ends.append(ends[-1] + s)
    return ends, torch.tensor(ends, dtype=dtype, device="cuda")


GROUPED = [
    # (sizes, rows past the last group, k, n)
    ((1,), 0, 1, 1),
    ((1, 0, 3), 2, 64, 128),
    ((0, 0), 5, 40, 24),
    ((5, 17, 0, 1, 30, 16, 2), 3, 100, 200),
    ((20, 40, 33), 0, 72, 264),
    ((64, 1, 100), 7, 129, 65),
    ((100, 130, 90), 0, 256, 512),
    ((300, 0, 513, 129), 11, 200, 1000),
    ((1000, 24, 600), 0, 1024, 256),
    (tuple(range(0, 40)), 9, 64, 72),
]


@pytest.mark.parametrize("precision", PRECISIONS)
@pytest.mark.parametrize("case", GROUPED, ids=lambda c: f"{len(c[0])}g{sum(c[0])}r{c[2]}x{c[3]}")
def test_grouped_forward_and_backward(native, precision, case):
    sizes, tail, k, n = case
    dtype = DTYPES[precision]
    ends, offsets = sizes_to_offsets(sizes)
    rows, groups = ends[-1] + tail, len(sizes)
    a, b = randn((rows, k), dtype, 1), randn((groups, k, n), dtype, 2, k ** -0.5)
    dout = randn((rows, n), dtype, 3)
    # Rows of no group may hold anything and must reach no sum.
    a[ends[-1]:], dout[ends[-1]:] = float("nan"), float("nan")
    for out_dtype in dict.fromkeys((dtype, torch.float32)):
        out, untouched = guarded((rows, n), out_dtype)
        expected, tol = ref.grouped(a[:ends[-1]].nan_to_num(), b, ends, precision, out[:ends[-1]])
        run = native.prepare_grouped(a, b, offsets, out, precision=precision)
        run()
        assert_within(out[:ends[-1]], expected, tol, "out") if ends[-1] else None
        assert bool((out[ends[-1]:] == 7.0).all())
        untouched()
        da, ua = guarded((rows, k), out_dtype)
        db, ub = guarded((groups, k, n), out_dtype)
        back = native.prepare_grouped_backward(dout, a, b, offsets, precision=precision, da=da, db=db)
        back()
        (eda, tda), (edb, tdb) = ref.grouped_backward(dout[:ends[-1]], a[:ends[-1]], b, ends, precision, da[:ends[-1]])
        assert_within(da[:ends[-1]], eda, tda, "da") if ends[-1] else None
        assert bool((da[ends[-1]:] == 7.0).all())
        assert_within(db, edb, tdb, "db")
        ua(), ub()
        first = (out.clone(), da.clone(), db.clone())
        run(), back()
        assert all(torch.equal(x, y) for x, y in zip(first, (out, da, db)))


def test_grouped_keeps_values_of_neighbours_out(native):
    """NaN in one expert's weight, and in one group's rows, stay in that group's results."""
    for sizes in ((6, 9, 4), (70, 90, 150), (200, 333, 140)):
        for k, n in ((72, 136), (100, 200)):
            ends, offsets = sizes_to_offsets(sizes, torch.int64)
            rows = ends[-1]
            a, b, dout = (randn(s, torch.bfloat16, i) for i, s in enumerate(((rows, k), (3, k, n), (rows, n))))
            b[1] = float("nan")
            out = torch.empty((rows, n), dtype=torch.bfloat16, device="cuda")
            native.prepare_grouped(a, b, offsets, out, precision="bf16")()
            finite = torch.isfinite(out).all(1)
            assert bool(finite[:ends[1]].all()) and bool(finite[ends[2]:].all()) and not bool(finite[ends[1]:ends[2]].any())
            dout[ends[1]:ends[2]] = float("inf")
            a[ends[1]:ends[2]] = float("nan")
            da = torch.empty((rows, k), dtype=torch.bfloat16, device="cuda")
            db = torch.empty((3, k, n), dtype=torch.float32, device="cuda")
            native.prepare_grouped_backward(dout, a, b, offsets, precision="bf16", da=da, db=db)()
            finite = torch.isfinite(da).all(1)
            assert bool(finite[:ends[1]].all()) and bool(finite[ends[2]:].all())
            assert bool(torch.isfinite(db[0]).all()) and bool(torch.isfinite(db[2]).all())


def test_grouped_clips_offsets(native):
    """Offsets out of range or out of order read and write nothing outside the matrices."""
    rows, k, n = 300, 64, 128
    a, b = randn((rows, k), torch.bfloat16, 1), randn((4, k, n), torch.bfloat16, 2)
    bad = torch.tensor([-5, 40, 30, 2 ** 40, 100], dtype=torch.int64, device="cuda")
    ends = [0, 40, 40, rows, rows]
    out, untouched = guarded((rows, n), torch.float32)
    native.prepare_grouped(a, b, bad, out, precision="bf16")()
    expected, tol = ref.grouped(a, b, ends, "bf16", out)
    assert_within(out, expected, tol, "clipped offsets")
    untouched()


def test_grouped_reads_offsets_when_it_runs(native):
    rows, k, n = 64, 64, 64
    a, b = randn((rows, k), torch.bfloat16, 1), randn((2, k, n), torch.bfloat16, 2)
    offsets = torch.tensor([0, 10, 64], dtype=torch.int32, device="cuda")
    out = torch.empty((rows, n), dtype=torch.float32, device="cuda")
    run = native.prepare_grouped(a, b, offsets, out, precision="bf16")
    for ends in ([0, 10, 64], [0, 50, 64], [0, 0, 64]):
        offsets.copy_(torch.tensor(ends, dtype=torch.int32))
        run()
        assert_within(out, *ref.grouped(a, b, ends, "bf16", out), str(ends))


def test_grouped_many_groups(native):
    """More groups than one pass of the plan's block takes."""
    sizes = [i % 3 for i in range(2500)]
    ends, offsets = sizes_to_offsets(sizes)
    k, n = 64, 64
    a, b = randn((ends[-1], k), torch.bfloat16, 1), randn((2500, k, n), torch.bfloat16, 2)
    dout = randn((ends[-1], n), torch.bfloat16, 3)
    out = torch.empty((ends[-1], n), dtype=torch.float32, device="cuda")
    native.prepare_grouped(a, b, offsets, out, precision="bf16")()
    assert_within(out, *ref.grouped(a, b, ends, "bf16", out), "out")
    da, db = torch.empty_like(a), torch.empty_like(b)
    native.prepare_grouped_backward(dout, a, b, offsets, precision="bf16", da=da, db=db)()
    (eda, tda), (edb, tdb) = ref.grouped_backward(dout, a, b, ends, "bf16", da)
    assert_within(da, eda, tda, "da")
    assert_within(db, edb, tdb, "db")


# ---------------------------------------------------------------- cross entropy
LOSS_SHAPES = [(1, 64, 1), (1, 8, 7), (3, 65, 300), (33, 128, 1000), (130, 72, 513), (200, 768, 3201), (300, 256, 4096),
               (1024, 128, 9001), (257, 64, 40000)]


def loss_inputs(m, k, v, precision, label_dtype=torch.int64):
    dtype = DTYPES[precision]
    hidden, weight = randn((m, k), dtype, 1), randn((k, v), dtype, 2, 3.0 * k ** -0.5)
    gen = torch.Generator(device="cuda").manual_seed(5)
    labels = torch.randint(0, v, (m,), generator=gen, device="cuda").to(label_dtype)
    if m > 2:
        labels[1::7] = -100
        labels[0], labels[2] = v - 1, 0
    grad = torch.rand((m,), generator=gen, device="cuda") - 0.3
    return hidden, weight, labels, grad


@pytest.mark.parametrize("precision", PRECISIONS)
@pytest.mark.parametrize("shape", LOSS_SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_cross_entropy_every_size(native, precision, shape):
    m, k, v = shape
    hidden, weight, labels, grad = loss_inputs(m, k, v, precision, torch.int32 if v % 2 else torch.int64)
    (loss, ul), (lse, us) = guarded((m,), torch.float32), guarded((m,), torch.float32)
    run = native.prepare_cross_entropy(hidden, weight, labels, loss, lse, precision=precision)
    run()
    expected = ref.cross_entropy(hidden, weight, labels, precision)
    assert_within(loss, *expected["loss"], "loss")
    assert_within(lse, *expected["lse"], "lse")
    ul(), us()
    first = (loss.clone(), lse.clone())
    run()
    assert torch.equal(first[0], loss) and torch.equal(first[1], lse)
    if precision == "fp16":
        return
    expected = ref.cross_entropy_backward(grad, hidden, weight, labels, precision)
    for dtype in dict.fromkeys((DTYPES[precision], torch.float32)):
        (dh, uh), (dw, uw) = guarded((m, k), dtype), guarded((k, v), dtype)
        back = native.prepare_cross_entropy_backward(grad, hidden, weight, labels, lse, precision=precision, dhidden=dh,
                                                     dweight=dw)
        back()
        assert_within(dh, *expected["dhidden"], "dhidden")
        assert_within(dw, *expected["dweight"], "dweight")
        uh(), uw()
        first = (dh.clone(), dw.clone())
        back()
        assert torch.equal(first[0], dh) and torch.equal(first[1], dw)
        ignored = labels == -100
        assert bool((dh[ignored] == 0).all())


def test_cross_entropy_in_several_pieces(native):
    """More rows than one 64 MB piece holds: dH is added up over pieces, each gradient alone and both."""
    m, k, v = 8200, 64, 9000
    hidden, weight, labels, grad = loss_inputs(m, k, v, "bf16")
    loss, lse = (torch.empty((m,), dtype=torch.float32, device="cuda") for _ in range(2))
    native.prepare_cross_entropy(hidden, weight, labels, loss, lse, precision="bf16")()
    expected = ref.cross_entropy_backward(grad, hidden, weight, labels, "bf16")
    for dtype in (torch.bfloat16, torch.float32):
        dh = torch.full((m, k), 7.0, dtype=dtype, device="cuda")
        dw = torch.full((k, v), 7.0, dtype=dtype, device="cuda")
        for args in ({"dhidden": dh}, {"dweight": dw}, {"dhidden": dh, "dweight": dw}):
            native.prepare_cross_entropy_backward(grad, hidden, weight, labels, lse, precision="bf16", **args)()
            for name, got in args.items():
                assert_within(got, *expected[name], name)
                got.fill_(7.0) if len(args) == 1 else None


def test_cross_entropy_far_logits(native):
    """Logits of several hundred, where exp alone would overflow; a row of equal logits; one certain row."""
    m, k, v = 140, 64, 2000
    hidden, weight, labels, grad = loss_inputs(m, k, v, "bf16")
    hidden = (hidden.float() * 30).to(torch.bfloat16)
    hidden[4] = 0.0
    loss, lse = (torch.empty((m,), dtype=torch.float32, device="cuda") for _ in range(2))
    native.prepare_cross_entropy(hidden, weight, labels, loss, lse, precision="bf16")()
    expected = ref.cross_entropy(hidden, weight, labels, "bf16")
    assert_within(loss, *expected["loss"], "loss")
    assert_within(lse, *expected["lse"], "lse")
    dh, dw = torch.empty_like(hidden), torch.empty_like(weight)
    native.prepare_cross_entropy_backward(grad, hidden, weight, labels, lse, precision="bf16", dhidden=dh, dweight=dw)()
    expected = ref.cross_entropy_backward(grad, hidden, weight, labels, "bf16")
    assert_within(dh, *expected["dhidden"], "dhidden")
    assert_within(dw, *expected["dweight"], "dweight")


def test_cross_entropy_marks_bad_labels_and_keeps_rows_apart(native):
    m, k, v = 150, 64, 1000
    hidden, weight, labels, grad = loss_inputs(m, k, v, "bf16")
    labels[10], labels[11], labels[12] = v, -1, 2 ** 40
    hidden[20] = float("nan")
    labels[21] = -100
    loss, lse = (torch.empty((m,), dtype=torch.float32, device="cuda") for _ in range(2))
    native.prepare_cross_entropy(hidden, weight, labels, loss, lse, precision="bf16")()
    bad = torch.zeros(m, dtype=torch.bool, device="cuda")
    bad[10:13] = True
    bad[20] = labels[20] != -100
    assert torch.equal(torch.isnan(loss), bad)
    assert bool(torch.isnan(lse[20]))
    assert float(loss[21]) == 0.0
    dh = torch.empty_like(hidden)
    native.prepare_cross_entropy_backward(grad, hidden, weight, labels, lse, precision="bf16", dhidden=dh)()
    rows = torch.isnan(dh).any(1)
    assert bool(rows[10:13].all()) and int(rows.sum()) == 3 + int(bad[20])


@pytest.mark.parametrize("m", (3, 300))
def test_cross_entropy_with_logits_of_minus_infinity(native, m):
    """Whole stretches of -infinity before, between and after logits near -1000: they add nothing, the rest is exact;
    a row of nothing but -infinity has lse -infinity."""
    k, v = 64, 2000
    hidden = randn((m, k), torch.bfloat16, 1).abs() + 0.5
    weight = randn((k, v), torch.bfloat16, 2, 0.3) - 15.0
    weight[:, :700] = float("-inf")
    weight[:, 900:1300] = float("-inf")
    weight[:, 1999] = float("-inf")
    labels = torch.full((m,), 800, device="cuda")
    loss, lse = (torch.empty((m,), dtype=torch.float32, device="cuda") for _ in range(2))
    native.prepare_cross_entropy(hidden, weight, labels, loss, lse, precision="bf16")()
    live = torch.cat([torch.arange(700, 900), torch.arange(1300, 1999)]).cuda()
    expected = ref.cross_entropy(hidden, weight[:, live].contiguous(), torch.full_like(labels, 100), "bf16")
    assert_within(lse, *expected["lse"], "lse")
    assert_within(loss, *expected["loss"], "loss")
    weight.fill_(float("-inf"))
    native.prepare_cross_entropy(hidden, weight, labels, loss, lse, precision="bf16")()
    assert bool((lse == float("-inf")).all())


def test_cross_entropy_every_row_ignored(native):
    m, k, v = 40, 64, 500
    hidden, weight, labels, grad = loss_inputs(m, k, v, "bf16")
    labels.fill_(5)
    loss, lse = (torch.empty((m,), dtype=torch.float32, device="cuda") for _ in range(2))
    native.prepare_cross_entropy(hidden, weight, labels, loss, lse, precision="bf16", ignore_index=5)()
    dh, dw = torch.ones_like(hidden), torch.ones_like(weight)
    native.prepare_cross_entropy_backward(grad, hidden, weight, labels, lse, precision="bf16", dhidden=dh, dweight=dw,
                                          ignore_index=5)()
    assert not bool(loss.any()) and not bool(dh.any()) and not bool(dw.any())


def test_cross_entropy_gradients_against_differences(native):
    m, k, v = 12, 16, 300
    hidden, weight, labels, grad = loss_inputs(m, k, v, "bf16")
    loss, lse = (torch.empty((m,), dtype=torch.float32, device="cuda") for _ in range(2))
    native.prepare_cross_entropy(hidden, weight, labels, loss, lse, precision="bf16")()
    dh = torch.empty((m, k), dtype=torch.float32, device="cuda")
    dw = torch.empty((k, v), dtype=torch.float32, device="cuda")
    native.prepare_cross_entropy_backward(grad, hidden, weight, labels, lse, precision="bf16", dhidden=dh, dweight=dw)()
    kept = (labels != -100).double()

    def total(h, w):
        z = h @ w
        picked = z.gather(1, labels.clamp(min=0).long()[:, None])[:, 0]
        return ((torch.logsumexp(z, 1) - picked) * kept * grad.double()).sum()

    h = 1e-4
    expected = ref.cross_entropy_backward(grad, hidden, weight, labels, "bf16")
    for which, got, name in ((0, dh, "dhidden"), (1, dw, "dweight")):
        for index in (0, 5, got.numel() // 2, got.numel() - 1):
            sides = []
            for sign in (1, -1):
                args = [hidden.double(), weight.double()]
                args[which] = args[which].clone()
                args[which].view(-1)[index] += sign * h
                sides.append(total(*args))
            difference = float(sides[0] - sides[1]) / (2 * h)
            slack = float(expected[name][1].reshape(-1)[index]) + h * h * 10 * 48 + 1e-6
            assert abs(float(got.reshape(-1)[index]) - difference) <= slack + 2.0 ** -24 * abs(difference)

"""The operators as a program uses them (needs a B200): together in one training step, on other streams, in CUDA
graphs, after a wait that ran out, on a part of the SMs, with outputs of every alignment and past 32-bit offsets."""

from __future__ import annotations

import threading

import pytest
import torch

import operator_reference as ref
from operator_contracts import SIZE_MAX
from operator_reference import DTYPES, assert_within
from test_operators_gpu import guarded, loss_inputs, offset_copy, randn, sizes_to_offsets

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32
LOAD, MMA, EPILOGUE, DRAIN = 1, 2, 4, 8


def test_training_step_of_a_small_model(native):
    """Up and down projections with a residual, experts, the loss, and every gradient back to the input; each stage
    against the 64-bit form of that stage on the values it was given."""
    m, d, f, groups, v = 333, 192, 520, 4, 3001
    x = randn((m, d), BF16, 1)
    up, down = randn((d, f), BF16, 2, d ** -0.5), randn((f, d), BF16, 3, f ** -0.5)
    bias = randn((f,), BF16, 4, 0.1)
    experts = randn((groups, d, d), BF16, 5, d ** -0.5)
    ends, offsets = sizes_to_offsets((100, 0, 133, 100))
    head = randn((d, v), BF16, 6, 2 * d ** -0.5)
    labels = torch.randint(0, v, (m,), generator=torch.Generator(device="cuda").manual_seed(7), device="cuda")
    labels[::9] = -100
    empty = lambda *s, dtype=BF16: torch.empty(s, dtype=dtype, device="cuda")
    h, z, y, e = empty(m, f), empty(m, f), empty(m, d), empty(m, d)
    loss, lse = empty(m, dtype=FP32), empty(m, dtype=FP32)
    grad = torch.full((m,), 1.0 / m, device="cuda")
    de, dhead, dy, dexperts = empty(m, d), empty(d, v), empty(m, d), empty(groups, d, d)
    dh, ddown, dx, dup, dbias = empty(m, f), empty(f, d), empty(m, d), empty(d, f), empty(f, dtype=FP32)
    step = [
        native.prepare_epilogue(x, up, h, precision="bf16", bias=bias, activation="gelu", preact=z),
        native.prepare_epilogue(h, down, y, precision="bf16", residual=x),
        native.prepare_grouped(y, experts, offsets, e, precision="bf16"),
        native.prepare_cross_entropy(e, head, labels, loss, lse, precision="bf16"),
        native.prepare_cross_entropy_backward(grad, e, head, labels, lse, precision="bf16", dhidden=de, dweight=dhead),
        native.prepare_grouped_backward(de, y, experts, offsets, precision="bf16", da=dy, db=dexperts),
        native.prepare_epilogue_backward(dy, h, down, precision="bf16", da=dh, db=ddown),
        native.prepare_epilogue_backward(dh, x, up, precision="bf16", activation="gelu", preact=z, da=dx, db=dup,
                                         dbias=dbias),
    ]
    for launch in step:
        launch()
    torch.cuda.synchronize()
    first = ref.epilogue(x, up, "bf16", bias, "gelu")
    assert_within(h, *first["out"], "h")
    assert_within(z, *first["preact"], "z")
    assert_within(y, *ref.epilogue(h, down, "bf16", None, "none", x)["out"], "y")
    assert_within(e, *ref.grouped(y, experts, ends, "bf16", e), "e")
    forward = ref.cross_entropy(e, head, labels, "bf16")
    assert_within(loss, *forward["loss"], "loss")
    assert_within(lse, *forward["lse"], "lse")
    back = ref.cross_entropy_backward(grad, e, head, labels, "bf16")
    assert_within(de, *back["dhidden"], "de")
    assert_within(dhead, *back["dweight"], "dhead")
    (edy, tdy), (edx, tdx) = ref.grouped_backward(de, y, experts, ends, "bf16", dy)
    assert_within(dy, edy, tdy, "dy")
    assert_within(dexperts, edx, tdx, "dexperts")
    back = ref.epilogue_backward(dy, h, down, "bf16")
    assert_within(dh, *back["da"], "dh")
    assert_within(ddown, *back["db"], "ddown")
    back = ref.epilogue_backward(dh, x, up, "bf16", z, "gelu")
    for name, got in (("da", dx), ("db", dup), ("dbias", dbias)):
        assert_within(got, *back[name], name)
    # The same step captured into a graph gives the same bits, twice.
    outs = (h, y, e, loss, de, dhead, dy, dexperts, dh, ddown, dx, dup, dbias)
    eager = [t.clone() for t in outs]
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step = [
            native.prepare_epilogue(x, up, h, precision="bf16", bias=bias, activation="gelu", preact=z),
            native.prepare_epilogue(h, down, y, precision="bf16", residual=x),
            native.prepare_grouped(y, experts, offsets, e, precision="bf16"),
            native.prepare_cross_entropy(e, head, labels, loss, lse, precision="bf16"),
            native.prepare_cross_entropy_backward(grad, e, head, labels, lse, precision="bf16", dhidden=de,
                                                  dweight=dhead),
            native.prepare_grouped_backward(de, y, experts, offsets, precision="bf16", da=dy, db=dexperts),
            native.prepare_epilogue_backward(dy, h, down, precision="bf16", da=dh, db=ddown),
            native.prepare_epilogue_backward(dh, x, up, precision="bf16", activation="gelu", preact=z, da=dx, db=dup,
                                             dbias=dbias),
        ]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for launch in step:
            launch()
    for _ in range(2):
        for t in outs:
            t.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, outs))
    del graph


def _unaligned_cases(native):
    """One call of each operator whose scratch holds copies, plans or sums: (launch, its outputs)."""
    a, b = offset_copy(randn((200, 129), BF16, 1)), randn((129, 77), BF16, 2)
    out = torch.zeros((200, 77), dtype=BF16, device="cuda")
    yield native.prepare_epilogue(a, b, out, precision="bf16", activation="silu"), (out,)
    dout, z = randn((200, 77), BF16, 3), randn((200, 77), BF16, 4)
    da, db, dbias = torch.zeros_like(a), torch.zeros_like(b), torch.zeros(77, device="cuda")
    yield native.prepare_epilogue_backward(dout, a, b, precision="bf16", activation="gelu", preact=z, da=da, db=db,
                                           dbias=dbias), (da, db, dbias)
    ends, offsets = sizes_to_offsets((90, 0, 110))
    w = randn((3, 129, 77), BF16, 5)
    go, gda, gdb = torch.zeros_like(out), torch.zeros_like(a), torch.zeros_like(w)
    yield native.prepare_grouped(a, w, offsets, go, precision="bf16"), (go,)
    yield native.prepare_grouped_backward(dout, a, w, offsets, precision="bf16", da=gda, db=gdb), (gda, gdb)
    hidden, weight, labels, grad = loss_inputs(200, 129, 1001, "bf16")
    loss, lse = torch.zeros(200, device="cuda"), torch.zeros(200, device="cuda")
    yield native.prepare_cross_entropy(hidden, weight, labels, loss, lse, precision="bf16"), (loss, lse)
    dh, dw = torch.zeros_like(hidden), torch.zeros_like(weight)
    yield native.prepare_cross_entropy_backward(grad, hidden, weight, labels, lse, precision="bf16", dhidden=dh,
                                                dweight=dw), (dh, dw)


def test_two_graphs_and_eager_calls_share_no_scratch(native):
    """Two captured graphs replayed on two streams beside each other and beside eager calls on a third."""
    eager = list(_unaligned_cases(native))
    for launch, _ in eager:
        launch()
    torch.cuda.synchronize()
    expected = [[t.clone() for t in outs] for _, outs in eager]
    sides = []
    for _ in range(2):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            cases = list(_unaligned_cases(native))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            for launch, _ in cases:
                launch()
        sides.append((stream, graph, cases))
    for _ in range(5):
        for stream, graph, cases in sides:
            with torch.cuda.stream(stream):
                for _, outs in cases:
                    for t in outs:
                        t.fill_(3.0)
                graph.replay()
        for launch, outs in eager:
            for t in outs:
                t.fill_(3.0)
        for launch, _ in eager:
            launch()
        torch.cuda.synchronize()
        for cases in (eager, sides[0][2], sides[1][2]):
            for (_, outs), want in zip(cases, expected):
                assert all(torch.equal(x, y) for x, y in zip(outs, want))
    del sides


def test_a_prepared_call_keeps_its_stream_and_its_tensors(native):
    stream = torch.cuda.Stream()
    a, b = randn((300, 256), BF16, 1), randn((256, 512), BF16, 2)
    out = torch.zeros((300, 512), dtype=FP32, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        run = native.prepare_epilogue(a, b, out, precision="bf16")
    expected = ref.epilogue(a, b, "bf16")["out"]
    del a, b
    torch.cuda.empty_cache()
    run()                                     # from another current stream: runs on the stream it was prepared on
    stream.synchronize()
    assert_within(out, *expected, "other stream")
    before = torch.cuda.current_device()
    run()
    assert torch.cuda.current_device() == before
    torch.cuda.synchronize()


def test_calls_fail_after_close(native, library_path):
    from gpumat import NativeMatmul

    other = NativeMatmul(library_path)
    a, b = randn((64, 64), BF16, 1), randn((64, 64), BF16, 2)
    out = torch.zeros((64, 64), dtype=FP32, device="cuda")
    run = other.prepare_epilogue(a, b, out, precision="bf16")
    other.close()
    with pytest.raises(RuntimeError, match="closed"):
        run()
    with pytest.raises(RuntimeError, match="closed"):
        other.prepare_grouped(a, b.view(1, 64, 64), torch.tensor([0, 64], dtype=torch.int32, device="cuda"), out,
                              precision="bf16")


def test_refusals_reach_the_caller(native):
    a, b = randn((64, 64), BF16, 1), randn((64, 64), BF16, 2)
    out = torch.zeros((64, 64), dtype=FP32, device="cuda")
    with pytest.raises(ValueError, match="not fp32"):
        native.prepare_epilogue(a.float(), b.float(), out, precision="fp32")
    with pytest.raises(ValueError, match="cuda:0"):
        native.prepare_epilogue(a.cpu(), b, out, precision="bf16")
    with pytest.raises(ValueError, match="contiguous"):
        native.prepare_epilogue(a, b.t(), out, precision="bf16")
    with pytest.raises(ValueError, match="activation"):
        native.prepare_epilogue(a, b, out, precision="bf16", activation="swish")


@pytest.mark.parametrize("n", (1028, 1032, 1037))
@pytest.mark.parametrize("m", (70, 300, 2100))
def test_outputs_and_pre_activations_of_other_alignments(native, m, n):
    """n % 8 == 4: TMA writes FP32 rows and not 16-bit ones, so one kernel stores both ways; odd rows leave
    in aligned chunks of 16 bytes."""
    k = 136
    a, b, bias = randn((m, k), BF16, 1), randn((k, n), BF16, 2, k ** -0.5), randn((n,), FP32, 3)
    for out_dtype, preact_dtype in ((BF16, FP32), (FP32, BF16), (BF16, BF16), (FP32, FP32)):
        for residual in (None, randn((m, n), out_dtype, 4)):
            (out, ua), (preact, ub) = guarded((m, n), out_dtype), guarded((m, n), preact_dtype)
            native.prepare_epilogue(a, b, out, precision="bf16", bias=bias, activation="gelu_tanh", residual=residual,
                                    preact=preact)()
            expected = ref.epilogue(a, b, "bf16", bias, "gelu_tanh", residual)
            assert_within(out, *expected["out"], f"out {out_dtype} {residual is not None}")
            assert_within(preact, *expected["preact"], f"preact {preact_dtype}")
            ua(), ub()


@pytest.mark.parametrize("precision", ("bf16", "tf32"))
def test_large_odd_gradients(native, precision):
    """Large gradients with odd rows, at any base alignment."""
    dtype = DTYPES[precision]
    m, k, n = 1500, 1501, 1403
    dout, a, b = randn((m, n), dtype, 1), randn((m, k), dtype, 2), randn((k, n), dtype, 3, k ** -0.5)
    for offset in (0, 1):
        whole = [torch.full((r * c + 64,), 7.0, dtype=dtype, device="cuda") for r, c in ((m, k), (k, n))]
        da, db = (t[16 + offset:16 + offset + r * c].view(r, c) for t, (r, c) in zip(whole, ((m, k), (k, n))))
        native.prepare_epilogue_backward(dout, a, b, precision=precision, da=da, db=db)()
        expected = ref.epilogue_backward(dout, a, b, precision)
        assert_within(da, *expected["da"], "da")
        assert_within(db, *expected["db"], "db")
        for t, count in zip(whole, (m * k, k * n)):
            assert bool((t[:16 + offset] == 7.0).all()) and bool((t[16 + offset + count:] == 7.0).all())


def test_large_odd_grouped_and_vocabulary_gradients(native):
    ends, offsets = sizes_to_offsets((300, 0, 257, 100))
    rows, k, n = ends[-1], 1001, 703
    a, b, dout = randn((rows, k), BF16, 1), randn((4, k, n), BF16, 2), randn((rows, n), BF16, 3)
    db, untouched = guarded((4, k, n), BF16)
    native.prepare_grouped_backward(dout, a, b, offsets, precision="bf16", db=db)()
    _, (edb, tdb) = ref.grouped_backward(dout, a, b, ends, "bf16", a)
    assert_within(db, edb, tdb, "db")
    untouched()
    m, k, v = 4300, 301, 9001                # two pieces of the vocabulary
    hidden, weight, labels, grad = loss_inputs(m, k, v, "bf16")
    loss, lse = torch.zeros(m, device="cuda"), torch.zeros(m, device="cuda")
    native.prepare_cross_entropy(hidden, weight, labels, loss, lse, precision="bf16")()
    (dh, ua), (dw, ub) = guarded((m, k), BF16), guarded((k, v), BF16)
    native.prepare_cross_entropy_backward(grad, hidden, weight, labels, lse, precision="bf16", dhidden=dh, dweight=dw)()
    expected = ref.cross_entropy_backward(grad, hidden, weight, labels, "bf16")
    assert_within(dh, *expected["dhidden"], "dhidden")
    assert_within(dw, *expected["dweight"], "dweight")
    ua(), ub()


DEEP = [(1, 3, 70001), (20, 130, 9001), (130, 20, 30000), (302, 264, 20352), (9000, 40, 24), (20011, 33, 65),
        (40000, 200, 3)]


@pytest.mark.parametrize("precision", ("bf16", "fp16", "tf32"))
@pytest.mark.parametrize("shape", DEEP, ids=lambda s: "x".join(map(str, s)))
def test_few_gradients_from_long_sums(native, precision, shape):
    """A small da summed over many columns, or a small db over many rows, is added up from chunks of the sum."""
    m, k, n = shape
    dtype = DTYPES[precision]
    dout, a, b = randn((m, n), dtype, 1), randn((m, k), dtype, 2), randn((k, n), dtype, 3)
    expected = ref.epilogue_backward(dout, a, b, precision)
    for grad_dtype in dict.fromkeys((dtype, FP32)):
        (da, ua), (db, ub) = guarded((m, k), grad_dtype), guarded((k, n), grad_dtype)
        run = native.prepare_epilogue_backward(dout, a, b, precision=precision, da=da, db=db)
        run()
        assert_within(da, *expected["da"], "da")
        assert_within(db, *expected["db"], "db")
        ua(), ub()
        first = da.clone(), db.clone()
        run()
        assert torch.equal(first[0], da) and torch.equal(first[1], db)


@pytest.mark.parametrize("precision", ("bf16", "tf32"))
@pytest.mark.parametrize("shape", [(3, 65, 40001), (50, 264, 30000), (2100, 40, 18001), (20000, 24, 40)],
                         ids=lambda s: "x".join(map(str, s)))
def test_vocabulary_gradients_from_long_sums(native, precision, shape):
    """The same of the loss: one piece of the vocabulary and several, the last one short."""
    m, k, v = shape
    dtype = DTYPES[precision]
    hidden, weight, labels, grad = loss_inputs(m, k, v, precision)
    loss, lse = torch.zeros(m, device="cuda"), torch.zeros(m, device="cuda")
    native.prepare_cross_entropy(hidden, weight, labels, loss, lse, precision=precision)()
    expected = ref.cross_entropy_backward(grad, hidden, weight, labels, precision)
    for grad_dtype in dict.fromkeys((dtype, FP32)):
        (dh, ua), (dw, ub) = guarded((m, k), grad_dtype), guarded((k, v), grad_dtype)
        native.prepare_cross_entropy_backward(grad, hidden, weight, labels, lse, precision=precision, dhidden=dh,
                                              dweight=dw)()
        assert_within(dh, *expected["dhidden"], "dhidden")
        assert_within(dw, *expected["dweight"], "dweight")
        ua(), ub()


def test_on_some_of_the_sms(native):
    a, b = randn((1000, 512), BF16, 1), randn((512, 2048), BF16, 2, 0.05)
    w = randn((3, 512, 256), BF16, 3)
    ends, offsets = sizes_to_offsets((400, 100, 500))
    out, go = torch.zeros((1000, 2048), device="cuda"), torch.zeros((1000, 256), device="cuda")
    dw = torch.zeros((3, 512, 256), device="cuda")
    try:
        for sms in (2, 16, 0):
            native.set_sm_limit(sms)
            out.zero_(), go.zero_(), dw.zero_()
            native.prepare_epilogue(a, b, out, precision="bf16")()
            native.prepare_grouped(a, w, offsets, go, precision="bf16")()
            native.prepare_grouped_backward(go.to(BF16), a, w, offsets, precision="bf16", db=dw)()
            assert_within(out, *ref.epilogue(a, b, "bf16")["out"], f"{sms} SMs")
            assert_within(go, *ref.grouped(a, w, ends, "bf16", go), f"grouped, {sms} SMs")
            _, (edb, tdb) = ref.grouped_backward(go.to(BF16), a, w, ends, "bf16", a)
            assert_within(dw, edb, tdb, f"grouped gradient, {sms} SMs")
    finally:
        native.set_sm_limit(0)


def _timeout_cases(native):
    """One call of every kind of tile and epilogue, deep enough that its waits are not already complete."""
    for m, k, n in ((16, 4096, 512), (16, 512, 16384), (100, 4096, 4096), (600, 2048, 2048), (4096, 512, 2048)):
        a, b = randn((m, k), BF16, 1), randn((k, n), BF16, 2, k ** -0.5)
        out, z = torch.zeros((m, n), dtype=BF16, device="cuda"), torch.zeros((m, n), device="cuda")
        yield f"epilogue {m}x{k}x{n}", native.prepare_epilogue(a, b, out, precision="bf16", preact=z), (out, z)
        res = randn((m, n), BF16, 4)
        yield f"residual {m}x{k}x{n}", native.prepare_epilogue(a, b, out, precision="bf16", residual=res), (out,)
        dout, da, db = randn((m, n), BF16, 3), torch.zeros_like(a), torch.zeros_like(b)
        yield f"backward {m}x{k}x{n}", native.prepare_epilogue_backward(dout, a, b, precision="bf16", da=da, db=db), (da,)
    for sizes in ((10, 6), (500, 0, 600)):
        ends, offsets = sizes_to_offsets(sizes)
        a, w = randn((ends[-1], 1024), BF16, 5), randn((len(sizes), 1024, 512), BF16, 6, 0.03)
        out = torch.zeros((ends[-1], 512), dtype=BF16, device="cuda")
        yield f"grouped {sizes}", native.prepare_grouped(a, w, offsets, out, precision="bf16"), (out,)
    hidden, weight, labels, _ = loss_inputs(300, 1024, 20000, "bf16")
    loss, lse = torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda")
    yield "loss", native.prepare_cross_entropy(hidden, weight, labels, loss, lse, precision="bf16"), (lse,)


def test_waits_that_run_out_leave_nan_and_a_usable_context(native):
    for name, run, outs in _timeout_cases(native):
        run()
        torch.cuda.synchronize()
        good = [t.clone() for t in outs]
        assert native.device_status() == 0
        native.set_wait_limit(1)
        try:
            for t in outs:
                t.zero_()
            run()
            status = native.device_status()
        finally:
            native.set_wait_limit(0)
        assert status & (LOAD | MMA | EPILOGUE), f"{name}: status {status:#x}"
        assert not status & DRAIN, f"{name}: a drain wait ran out ({status:#x})"
        assert all(bool(torch.isnan(t).any()) for t in outs), f"{name}: no NaN after a timeout"
        run()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(good, outs)), f"{name}: wrong after a timeout"
        assert native.device_status() == 0


def test_offsets_past_32_bits(native):
    """Outputs, weights and logits' matrices of more than 2^31 elements: their ends against the 64-bit form."""
    m, k, n = 65600, 64, 32768
    a, b = randn((m, k), BF16, 1), randn((k, n), BF16, 2)
    out = torch.empty((m, n), dtype=BF16, device="cuda")
    native.prepare_epilogue(a, b, out, precision="bf16", activation="relu")()
    rows = torch.tensor([0, 1, 40000, m - 2, m - 1], device="cuda")
    assert_within(out[rows], *ref.epilogue(a[rows], b, "bf16", None, "relu")["out"], "rows at both ends")
    dbias = torch.empty((n,), device="cuda")
    native.prepare_epilogue_backward(out, precision="bf16", dbias=dbias)()
    expected = out[:, -8:].double().sum(0)
    assert_within(dbias[-8:], expected, (m + 2) * ref.U * out[:, -8:].double().abs().sum(0), "bias gradient")
    del out
    groups, k, n = 300, 2048, 4096
    sizes = [2] * groups
    ends, offsets = sizes_to_offsets(sizes, torch.int64)
    a, w = randn((ends[-1], k), BF16, 3), torch.empty((groups, k, n), dtype=BF16, device="cuda")
    for g in range(groups):
        w[g] = randn((k, n), BF16, 100 + g, 0.02)
    go = torch.empty((ends[-1], n), dtype=BF16, device="cuda")
    native.prepare_grouped(a, w, offsets, go, precision="bf16")()
    for g in (0, 150, groups - 1):
        assert_within(go[2 * g:2 * g + 2], *ref.product(a[2 * g:2 * g + 2].double(), w[g].double()), f"group {g}")
    db = torch.empty_like(w)
    native.prepare_grouped_backward(go, a, w, offsets, precision="bf16", db=db)()
    for g in (0, groups - 1):
        rows = slice(2 * g, 2 * g + 2)
        assert_within(db[g], *ref.product(a[rows].double().T, go[rows].double()), f"gradient of group {g}")
    del w, db
    k, v, m = 16400, 131072, 8
    weight = torch.empty((k, v), dtype=BF16, device="cuda")
    for r in range(0, k, 1025):
        weight[r:r + 1025] = randn((min(1025, k - r), v), BF16, r, 0.01)
    hidden = randn((m, k), BF16, 4)
    labels = torch.tensor([0, 1, v - 1, v // 2, 5, v - 2, -100, 7], device="cuda")
    loss, lse = torch.empty(m, device="cuda"), torch.empty(m, device="cuda")
    native.prepare_cross_entropy(hidden, weight, labels, loss, lse, precision="bf16")()
    z = torch.cat([hidden.double() @ weight[:, c:c + 16384].double() for c in range(0, v, 16384)], 1)
    # Allowance as in operator_reference.cross_entropy, with |A||B| bounded by its largest column.
    size = torch.stack([(hidden.double().abs() @ weight[:, c:c + 16384].double().abs()).amax(1)
                        for c in range(0, v, 16384)]).amax(0)
    tz = (k + 2) * ref.U * size
    tlse = tz + (600.0 + v / 128.0 + 16.0 * z.abs().amax(1)) * ref.U
    exact = torch.logsumexp(z, 1)
    assert_within(lse, exact, tlse, "lse")
    picked = z.gather(1, labels.clamp(min=0)[:, None])[:, 0]
    expected = torch.where(labels == -100, torch.zeros_like(exact), exact - picked)
    assert_within(loss, expected, 2 * tlse + ref.U * exact.abs(), "loss")


def test_the_longest_rows(native):
    """The largest size a call takes, as columns and as the length of a sum; exact in FP32."""
    n = SIZE_MAX
    b = torch.arange(n, dtype=torch.int32, device="cuda").remainder_(251).to(BF16).view(1, n)
    a = torch.full((1, 1), 2.0, dtype=BF16, device="cuda")
    out = torch.empty((1, n), dtype=BF16, device="cuda")
    native.prepare_epilogue(a, b, out, precision="bf16")()
    for c in range(0, n, 1 << 28):
        assert torch.equal(out[:, c:c + (1 << 28)], 2.0 * b[:, c:c + (1 << 28)])
    out.zero_()
    native.prepare_epilogue_backward(b, precision="bf16", dbias=out.view(n))()
    assert torch.equal(out, b)
    out.zero_()
    out[0, ::1 << 20] = 3.0
    da = torch.empty((1, 1), device="cuda")
    b[0, ::1 << 20] = 5.0
    native.prepare_epilogue_backward(out, b=b, precision="bf16", da=da)()
    assert float(da) == 15.0 * len(range(0, n, 1 << 20))


def test_threads_share_a_context(native):
    """Four threads prepare and enqueue on their own streams at once."""
    eager = list(_unaligned_cases(native))
    for launch, _ in eager:
        launch()
    torch.cuda.synchronize()
    wrong = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            cases = list(_unaligned_cases(native))
            for _ in range(20):
                for launch, _ in cases:
                    launch()
            torch.cuda.current_stream().synchronize()
            wrong.extend(1 for (_, outs), (_, want) in zip(cases, eager)
                         if not all(torch.equal(x, y) for x, y in zip(outs, want)))
            done.append(1)

    done = []
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(done) == 4 and not wrong


def odd_weight(k, n, dtype, offset):
    """A weight whose rows no 16-byte copy can address, `offset` elements into memory that NaN surrounds."""
    whole = torch.full((k * n + 64,), float("nan"), dtype=dtype, device="cuda")
    return whole[16 + offset:16 + offset + k * n].view(k, n).copy_(randn((k, n), dtype, 2, 3.0 * k ** -0.5))


@pytest.mark.parametrize("dtype", (BF16, torch.float16), ids=("bf16", "fp16"))
@pytest.mark.parametrize("shape", [(1, 1024, 20001), (3, 64, 113301), (16, 770, 32003), (17, 128, 40009), (33, 1000, 20007),
                                   (64, 130, 100002), (64, 2048, 18949), (2, 1, 200001), (5, 3, 150001)], ids=lambda s: "x".join(map(str, s)))
def test_few_rows_by_an_unaligned_weight(native, dtype, shape):
    """Products that read such a weight in place, at both ends of its memory; with a residual in place."""
    m, k, n = shape
    precision = "bf16" if dtype == BF16 else "fp16"
    for offset in (0, 1, 7):
        a, b = randn((m, k), dtype, 1), odd_weight(k, n, dtype, offset)
        (out, ua), (preact, ub) = guarded((m, n), dtype), guarded((m, n), FP32)
        bias = randn((n,), FP32, 3)
        run = native.prepare_epilogue(a, b, out, precision=precision, bias=bias, activation="gelu", preact=preact)
        run()
        expected = ref.epilogue(a, b, precision, bias, "gelu")
        assert_within(out, *expected["out"], "out")
        assert_within(preact, *expected["preact"], "preact")
        ua(), ub()
        first = out.clone()
        run()
        assert torch.equal(first, out)
        residual = randn((m, n), dtype, 4)
        out.copy_(residual)
        native.prepare_epilogue(a, b, out, precision=precision, residual=out)()
        assert_within(out, *ref.epilogue(a, b, precision, None, "none", residual)["out"], "residual in place")


@pytest.mark.parametrize("dtype", (BF16, torch.float16), ids=("bf16", "fp16"))
@pytest.mark.parametrize("shape", [(1, 1024, 50257), (2, 64, 60001), (40, 200, 50003), (100, 768, 32001), (128, 65, 70002)],
                         ids=lambda s: "x".join(map(str, s)))
def test_loss_of_few_rows_by_an_unaligned_weight(native, dtype, shape):
    m, k, v = shape
    precision = "bf16" if dtype == BF16 else "fp16"
    hidden, _, labels, _ = loss_inputs(m, k, v, precision)
    for offset in (0, 1):
        weight = odd_weight(k, v, dtype, offset)
        (loss, ul), (lse, us) = guarded((m,), FP32), guarded((m,), FP32)
        run = native.prepare_cross_entropy(hidden, weight, labels, loss, lse, precision=precision)
        run()
        expected = ref.cross_entropy(hidden, weight, labels, precision)
        assert_within(loss, *expected["loss"], "loss")
        assert_within(lse, *expected["lse"], "lse")
        ul(), us()
        first = loss.clone(), lse.clone()
        run()
        assert torch.equal(first[0], loss) and torch.equal(first[1], lse)


def test_unaligned_weights_in_a_graph_and_after_waits_that_ran_out(native):
    a, b = randn((16, 2048), BF16, 1), odd_weight(2048, 20001, BF16, 1)
    hidden, _, labels, _ = loss_inputs(100, 1024, 30001, "bf16")
    weight = odd_weight(1024, 30001, BF16, 1)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        out = torch.zeros((16, 20001), dtype=BF16, device="cuda")
        loss, lse = torch.zeros(100, device="cuda"), torch.zeros(100, device="cuda")
        runs = [(native.prepare_epilogue(a, b, out, precision="bf16"), (out,)),
                (native.prepare_cross_entropy(hidden, weight, labels, loss, lse, precision="bf16"), (lse,))]
    torch.cuda.synchronize()
    good = []
    for run, outs in runs:
        run()
        torch.cuda.synchronize()
        good.append([t.clone() for t in outs])
        assert native.device_status() == 0
        native.set_wait_limit(1)
        try:
            run()
            status = native.device_status()
        finally:
            native.set_wait_limit(0)
        assert status & (LOAD | MMA | EPILOGUE) and not status & DRAIN, f"status {status:#x}"
        assert all(bool(torch.isnan(t).any()) for t in outs)
        run()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(good[-1], outs)) and native.device_status() == 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for run, _ in runs:
            run()
    for _ in range(3):
        for _, outs in runs:
            for t in outs:
                t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for (_, outs), want in zip(runs, good):
            assert all(torch.equal(x, y) for x, y in zip(outs, want))
    del graph


@pytest.mark.parametrize("precision", ("bf16", "fp16", "tf32"))
@pytest.mark.parametrize("shape", [(300, 64, 1037), (1000, 300, 515), (2100, 72, 1026), (130, 2000, 33)],
                         ids=lambda s: "x".join(map(str, s)))
def test_unaligned_residuals_apart_and_in_place(native, precision, shape):
    m, k, n = shape
    dtype = DTYPES[precision]
    a, b = randn((m, k), dtype, 1), randn((k, n), dtype, 2, k ** -0.5)
    for out_dtype in dict.fromkeys((dtype, FP32)):
        residual = randn((m, n), out_dtype, 4)
        expected = ref.epilogue(a, b, precision, None, "silu", residual)
        for given in (residual, offset_copy(residual), None):
            (out, untouched), (preact, ub) = guarded((m, n), out_dtype), guarded((m, n), FP32)
            if given is None:
                out.copy_(residual)
            native.prepare_epilogue(a, b, out, precision=precision, activation="silu", preact=preact,
                                    residual=out if given is None else given)()
            assert_within(out, *expected["out"], "out")
            assert_within(preact, *expected["preact"], "preact")
            untouched(), ub()

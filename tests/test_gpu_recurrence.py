"""The gated linear recurrence and its gradients against the plain form in f64 (tests/layers_reference.py)."""
import itertools

import numpy as np
import pytest

from homura_b200.host import BF16, DTYPE_NAMES, F16, F32, F64, FLOATS, BackendError, CudaBackend
from layers_reference import raw, recurrence, recurrence_backward, rounded, value, within

pytestmark = pytest.mark.gpu

state_dtype = lambda dtype: F64 if dtype == F64 else F32
# batch, time, channels: one step, ends inside a lane's rows, a round, a cluster's round; odd and even channels; few and
# many channels; more items than lanes of a warp, and a time axis that several blocks share
SIZES = [(1, 1, 1), (3, 1, 257), (2, 2, 64), (1, 7, 33), (2, 8, 64), (1, 9, 2), (1, 63, 31), (1, 64, 128), (3, 65, 66),
         (1, 129, 5), (1, 511, 32), (2, 513, 34), (1, 1500, 7), (1, 4097, 1), (40, 33, 130), (300, 17, 520), (5, 40, 1000)]


def make(rng, b, t, c, dtype, sigmoid):
    gate = rng.normal(1.0, 2.0, (b, t, c)) if sigmoid else rng.uniform(-1.0, 1.0, (b, t, c)) ** 3
    if not sigmoid:
        gate[rng.random((b, t, c)) < 0.02] = 0.0
        gate[rng.random((b, t, c)) < 0.02] = 1.0
    return raw(gate, dtype), raw(rng.normal(size=(b, t, c)), dtype)


def window(be, stored, dtype, kind):
    """An upload of `stored` ([batch, time, channels]) in some layout: the same elements, other strides."""
    b, t, c = stored.shape
    if kind == "contiguous":
        return be.upload(stored, dtype)
    if kind == "half":      # the second half of a wider buffer: odd offsets for odd channel counts
        wide = np.zeros((b, t, 2 * c), stored.dtype)
        wide[..., c:] = stored
        return be.upload(wide, dtype).narrow(2, c, c)
    if kind == "time first":
        return be.upload(np.ascontiguousarray(stored.transpose(1, 0, 2)), dtype).transpose(0, 1)
    assert kind == "time last"
    return be.upload(np.ascontiguousarray(stored.transpose(0, 2, 1)), dtype).transpose(1, 2)


def forward(be, gate, x, initial, dtype, want_last=True, layout="contiguous", **flags):
    b, t, c = gate.shape
    out = window(be, np.zeros_like(gate), dtype, layout)
    sd = state_dtype(dtype)
    h0 = None if initial is None else be.upload(raw(initial, sd), sd)
    last = be.empty((b, c), sd) if want_last else None
    be.linear_recurrence(out, window(be, gate, dtype, layout), window(be, x, dtype, layout), h0, last, **flags)
    return be.download(out), (be.download(last) if want_last else None)


def check_forward(be, rng, size, dtype, state, layout="contiguous", **flags):
    b, t, c = size
    gate, x = make(rng, b, t, c, dtype, flags.get("sigmoid", False))
    initial = raw(rng.normal(size=(b, c)), state_dtype(dtype)).astype(np.float64) if state else None
    got, last = forward(be, gate, x, initial, dtype, layout=layout, **flags)
    h, e, want_last, el = recurrence(value(gate, dtype), value(x, dtype), initial, dtype, **flags)
    what = f"{DTYPE_NAMES[dtype]} {size} {layout} {flags}"
    within(value(got, dtype), h, rounded(e, h, dtype), "out " + what)
    within(last, want_last, rounded(el, want_last, state_dtype(dtype)), "last " + what)


@pytest.mark.parametrize("dtype", FLOATS, ids=[DTYPE_NAMES[d] for d in FLOATS])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_forward(cuda, dtype, size):
    rng = np.random.default_rng(sum(size) + dtype)
    for sigmoid, complement in itertools.product((False, True), repeat=2):
        check_forward(cuda, rng, size, dtype, state=sigmoid != complement, sigmoid=sigmoid, complement=complement,
                      reverse=bool(rng.integers(2)))


@pytest.mark.parametrize("layout", ["half", "time first", "time last"])
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_layouts(cuda, dtype, layout):
    rng = np.random.default_rng(5)
    for size in ((2, 70, 66), (3, 33, 31), (1, 600, 64)):
        for reverse in (False, True):
            check_forward(cuda, rng, size, dtype, True, layout, sigmoid=True, complement=True, reverse=reverse)
            check_backward(cuda, rng, size, dtype, True, layout, sigmoid=True, complement=True, reverse=reverse)


def check_backward(be, rng, size, dtype, state, layout="contiguous", **flags):
    b, t, c = size
    sd = state_dtype(dtype)
    gate, x = make(rng, b, t, c, dtype, flags.get("sigmoid", False))
    out, dout = raw(rng.normal(size=size), dtype), raw(rng.normal(size=size), dtype)
    vec = lambda: raw(rng.normal(size=(b, c)), sd).astype(np.float64)
    initial, dlast = (vec(), vec()) if state else (None, None)
    dgate, dx = (window(be, np.zeros_like(gate), dtype, layout) for _ in range(2))
    dinitial = be.empty((b, c), sd)
    w = lambda v: window(be, v, dtype, layout)
    up = lambda v: None if v is None else be.upload(raw(v, sd), sd)
    complement = flags.get("complement", False)
    be.linear_recurrence_backward(dgate, dx, w(gate), w(x) if complement else None, w(out), w(dout), up(initial), up(dlast), dinitial, **flags)
    want = recurrence_backward(value(gate, dtype), value(x, dtype), value(out, dtype), initial, value(dout, dtype), dlast, dtype, **flags)
    what = f"{DTYPE_NAMES[dtype]} {size} {layout} {flags}"
    within(value(be.download(dgate), dtype), want[0], rounded(want[1], want[0], dtype), "dgate " + what)
    within(value(be.download(dx), dtype), want[2], rounded(want[3], want[2], dtype), "dx " + what)
    within(be.download(dinitial), want[4], rounded(want[5], want[4], sd), "dinitial " + what)


@pytest.mark.parametrize("dtype", FLOATS, ids=[DTYPE_NAMES[d] for d in FLOATS])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_backward(cuda, dtype, size):
    rng = np.random.default_rng(sum(size) + 31 * dtype)
    for sigmoid, complement in itertools.product((False, True), repeat=2):
        check_backward(cuda, rng, size, dtype, state=sigmoid == complement, sigmoid=sigmoid, complement=complement,
                       reverse=bool(rng.integers(2)))


def test_gradients_are_the_differences(cuda):
    """The gradients of sum(out * weight) + sum(last * weight), against central differences of the kernel itself in f64."""
    rng = np.random.default_rng(2)
    b, t, c, step = 2, 70, 3, 1e-6
    for sigmoid, complement, reverse in itertools.product((False, True), repeat=3):
        flags = {"sigmoid": sigmoid, "complement": complement, "reverse": reverse}
        gate, x = make(rng, b, t, c, F64, sigmoid)
        initial, wl = rng.normal(size=(b, c)), rng.normal(size=(b, c))
        w = rng.normal(size=(b, t, c))

        def loss(gate, x, initial):
            out, last = forward(cuda, gate, x, initial, F64, **flags)
            return float((out * w).sum() + (last * wl).sum())

        up = lambda v: cuda.upload(v, F64)
        out = cuda.upload(forward(cuda, gate, x, initial, F64, **flags)[0], F64)
        dgate, dx, di = cuda.empty((b, t, c), F64), cuda.empty((b, t, c), F64), cuda.empty((b, c), F64)
        cuda.linear_recurrence_backward(dgate, dx, up(gate), up(x), out, up(w), up(initial), up(wl), di, **flags)
        for name, arr, grad in (("gate", gate, dgate), ("x", x, dx), ("initial", initial, di)):
            got = cuda.download(grad).reshape(-1)
            for k in rng.choice(arr.size, 6, replace=False):
                d = np.zeros(arr.size)
                d[k] = step
                d = d.reshape(arr.shape)
                vary = lambda s: loss(*(v + s * d if v is arr else v for v in (gate, x, initial)))
                diff = (vary(1) - vary(-1)) / (2 * step)
                # second-order truncation (|f'''| of some hundred) step^2 and cancellation of |f| ~ 1e2 in 1e-16 / step
                assert abs(diff - got[k]) <= 1e-7 * (1 + abs(diff)), (name, flags, diff, got[k])


def test_no_steps_and_nothing(cuda):
    initial = np.arange(10, dtype=np.float32).reshape(2, 5)
    z = cuda.empty((2, 0, 5), BF16)
    h0, last = cuda.upload(initial, F32), cuda.empty((2, 5), F32)
    cuda.linear_recurrence(z, z, z, h0, last)
    assert (cuda.download(last) == initial).all()
    cuda.linear_recurrence(z, z, z, None, last, sigmoid=True)
    assert (cuda.download(last) == 0).all()
    cuda.linear_recurrence_backward(z, z, z, None, z, z, None, h0, last)
    assert (cuda.download(last) == initial).all()
    cuda.linear_recurrence_backward(z, z, z, z, z, z, None, None, last, complement=True)
    assert (cuda.download(last) == 0).all()
    for shape in ((0, 3, 5), (2, 3, 0), (0, 0, 0)):
        e = cuda.empty(shape, F32)
        s = cuda.empty((shape[0], shape[2]), F32)
        cuda.linear_recurrence(e, e, e, s, s)
        cuda.linear_recurrence_backward(e, e, e, e, e, e, s, s, s)


@pytest.mark.parametrize("t", [1, 5, 700])
def test_state_in_place_and_in_pieces(cuda, t):
    """`last` may be `initial`, `out` may be x or gate; a sequence in pieces gives the states of the whole one."""
    rng = np.random.default_rng(t)
    b, c = 3, 70
    for dtype in (BF16, F32):
        gate, x = make(rng, b, 2 * t, c, dtype, True)
        initial = rng.normal(size=(b, c)).astype(np.float32)
        state = cuda.upload(initial, F32)
        pieces = []
        for k in range(2):
            g, v = cuda.upload(gate[:, k * t:(k + 1) * t], dtype), cuda.upload(x[:, k * t:(k + 1) * t], dtype)
            target = v if k else g
            cuda.linear_recurrence(target, g, v, state, state, sigmoid=True, complement=True)
            pieces.append(cuda.download(target))
        h, e, last, el = recurrence(value(gate, dtype), value(x, dtype), initial.astype(np.float64), dtype, True, True)
        within(value(np.concatenate(pieces, 1), dtype), h, rounded(e, h, dtype), f"pieces of {t}")
        # (the state between the pieces is stored unrounded but for f32's half step, which the bound's steps cover)
        within(cuda.download(state), last, rounded(el, last, F32) + 2.0**-23 * np.abs(initial).max(), f"state after pieces of {t}")


def test_resets_saturated_gates_and_values_that_are_no_numbers(cuda):
    rng = np.random.default_rng(11)
    b, t, c = 1, 300, 40
    gate, x = rng.uniform(0.5, 1, (b, t, c)), rng.normal(size=(b, t, c))
    gate[0, 100] = 0.0                      # forgets everything
    x[0, 50, 3], x[0, 60, 4], x[0, 70, 5] = np.inf, -np.inf, np.nan
    x[0, 150, 6] = np.inf
    gate[0, 20, 7] = np.nan
    x[0, 299, 8] = np.nan                   # the last step
    x[0, 0, 9] = np.inf                     # the first
    initial = rng.normal(size=(b, c))
    initial[0, 10] = np.inf
    gate, x, initial = raw(gate, F32), raw(x, F32), raw(initial, F32)
    got, last = forward(cuda, gate, x, initial, F32)
    with np.errstate(invalid="ignore"):
        h, e, wl, el = recurrence(value(gate, F32), value(x, F32), initial.astype(np.float64), F32)
        e, el = np.nan_to_num(e, nan=0.0, posinf=0.0), np.nan_to_num(el, nan=0.0, posinf=0.0)
    within(got, h, rounded(e, np.nan_to_num(h, posinf=0, neginf=0), F32), "values that are no numbers")
    within(last, wl, rounded(el, np.nan_to_num(wl, posinf=0, neginf=0), F32), "last of them")
    # a reset leaves the bits of a sequence that begins there
    clean = raw(rng.normal(size=(b, t, c)), F32)
    whole, _ = forward(cuda, gate[:, :, 11:], clean[:, :, 11:], None, F32)
    tail, _ = forward(cuda, np.ascontiguousarray(gate[:, 100:, 11:]), np.ascontiguousarray(clean[:, 100:, 11:]), None, F32)
    hw = recurrence(value(gate[:, 100:, 11:], F32), value(clean[:, 100:, 11:], F32), None, F32)
    within(whole[:, 100:], hw[0], rounded(hw[1], hw[0], F32), "behind a reset")
    within(tail, hw[0], rounded(hw[1], hw[0], F32), "from a reset on")
    # products of gates that overflow f32 multiply states of zero here: they stay zero
    for t in (40, 300, 5000):
        big, zero = np.full((1, t, 33), 30.0, np.float32), np.zeros((1, t, 33), np.float32)
        got, last = forward(cuda, big, zero, None, F32)
        assert (got == 0).all() and (last == 0).all()
    # logits far out: a is 0 or 1 to the last bit, 1 - a keeps its relative precision
    logits = np.array([-200.0, -90.0, -30.0, -1.0, 0.0, 1.0, 30.0, 90.0, 200.0, np.inf, -np.inf], np.float32)
    for dtype in FLOATS:
        gate = raw(np.broadcast_to(logits[:, None, None], (11, 3, 34)).astype(np.float64), dtype)
        x = raw(rng.normal(size=(11, 3, 34)), dtype)
        got, _ = forward(cuda, gate, x, None, dtype, sigmoid=True, complement=True)
        h, e, _, _ = recurrence(np.clip(value(gate, dtype), -700, 700), value(x, dtype), None, dtype, True, True)
        # (f32 exponentials below 2^-126 are flushed: 3 steps of at most 2^-126 |x|)
        within(value(got, dtype), h, rounded(e + 2.0**-124, h, dtype), f"saturated {DTYPE_NAMES[dtype]}")


def test_results_repeat_and_do_not_depend_on_the_neighbours(cuda):
    """Twice the same bits; a channel's result has the same bits whatever stands beside it in the tensor's other channels."""
    rng = np.random.default_rng(3)
    gate, x = make(rng, 2, 3000, 96, F32, True)
    one, _ = forward(cuda, gate, x, None, F32, sigmoid=True)
    two, _ = forward(cuda, gate, x, None, F32, sigmoid=True)
    assert (one.view(np.uint32) == two.view(np.uint32)).all()
    other = x.copy()
    other[:, :, 1::2] = np.nan
    mixed, _ = forward(cuda, gate, other, None, F32, sigmoid=True)
    assert (mixed[:, :, ::2].view(np.uint32) == one[:, :, ::2].view(np.uint32)).all()


def test_broadcast_operands(cuda):
    """Inputs may broadcast by strides of 0: one decay per channel for all steps and batches."""
    rng = np.random.default_rng(4)
    b, t, c = 2, 200, 66
    decay, x = raw(rng.uniform(0.9, 1.0, (1, 1, c)), F32), raw(rng.normal(size=(b, t, c)), F32)
    out = cuda.empty((b, t, c), F32)
    cuda.linear_recurrence(out, cuda.upload(decay, F32).expand(b, t, c), cuda.upload(x, F32))
    h, e, _, _ = recurrence(np.broadcast_to(value(decay, F32), (b, t, c)), value(x, F32), None, F32)
    within(cuda.download(out), h, rounded(e, h, F32), "one decay for all steps")


def test_two_backends_at_once_and_refused_states(cuda):
    """Two contexts (streams) of one device work on their own tensors at the same time."""
    other = CudaBackend(0)
    try:
        rng = np.random.default_rng(8)
        gate, x = make(rng, 1, 4096, 64, F32, True)
        want, _ = forward(cuda, gate, x, None, F32, sigmoid=True)
        outs = []
        for be in (cuda, other) * 4:
            out = be.empty(gate.shape, F32)
            g, v = be.upload(gate, F32), be.upload(x, F32)
            be.linear_recurrence(out, g, v, sigmoid=True)
            outs.append((be, out, g, v))
        for be, out, _, _ in outs:
            assert (be.download(out).view(np.uint32) == want.view(np.uint32)).all()
    finally:
        other.close()
    t = cuda.empty((2, 3, 4), BF16)
    with pytest.raises(BackendError, match="initial state has the wrong dtype"):
        cuda.linear_recurrence(t, t, t, cuda.empty((2, 4), BF16))

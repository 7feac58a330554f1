"""Where the trainable operators of include/homura_cuda_layers.h could go wrong by more than rounding: groups of one value, signs
at an activation's kink, long sums, logits and values at the ends of their types. Expected values are exact or follow from
the definition; a tolerance counts the roundings on a value's way."""
import math
import threading

import numpy as np
import pytest

from homura_b200.host import BF16, DTYPE_NAMES, F16, F32, F64, FLOATS, BackendError, CudaBackend, Generator
from layers_reference import dropout, group_norm, group_norm_backward, raw, rounded, value, within
from test_gpu_recurrence import check_backward, check_forward

pytestmark = pytest.mark.gpu

stat_dtype = lambda dtype: F64 if dtype == F64 else F32


def norm(be, x, dtype, groups, weight=None, bias=None, kind=None, eps=1e-5):
    """Forward with F32 (F64) parameters: out, mean and rstd as stored."""
    out = be.empty(x.shape, dtype)
    stats = [be.empty((x.shape[0], groups), stat_dtype(dtype)) for _ in range(2)]
    up = lambda v: None if v is None else be.upload(raw(v, stat_dtype(dtype)), stat_dtype(dtype))
    be.group_norm(out, be.upload(x, dtype), groups, up(weight), up(bias), *stats, eps=eps, activation=kind)
    return be.download(out), be.download(stats[0]), be.download(stats[1])


# rows in registers, a cluster's shared memory (with and without whole vectors) and pieces; groups whose size is a power of two
# and groups whose reciprocal size is not a number of the computation type
CONSTANT = [(3, 1, 64, 4), (3, 1, 60, 6), (3, 1, 4998, 3), (2, 200, 64, 4), (2, 77, 320, 32), (2, 390, 58, 2), (1, 3000, 16, 1), (2, 33, 257, 1),
            (1, 60000, 64, 2)]


@pytest.mark.parametrize("dtype", FLOATS, ids=[DTYPE_NAMES[d] for d in FLOATS])
@pytest.mark.parametrize("size", CONSTANT, ids=str)
def test_a_constant_group_becomes_its_bias(cuda, dtype, size):
    """Sums of these values and their quotient by the size are exact, so the mean is the value, every deviation is 0 and the
    output the bias, whatever the weight."""
    n, s, c, groups = size
    rng = np.random.default_rng(sum(size))
    w, b = rng.normal(1, 0.3, c), rng.normal(0, 0.3, c)
    for level in (0.0, 3.25, -1000.0, 30000.0):
        x = raw(np.full((n, s, c), level), dtype)
        got, mean, rstd = norm(cuda, x, dtype, groups, w, b)
        want = raw(np.broadcast_to(raw(b, stat_dtype(dtype)).astype(np.float64), x.shape), dtype)
        assert (mean == value(x, dtype)[0, 0, 0]).all(), (level, mean)
        # 1 / sqrt(eps), eps rounded to the computation type, by a function good to two units in the last place
        assert (np.abs(rstd * np.sqrt(1e-5) - 1) <= (4 * 2.0**-52 if dtype == F64 else 4 * 2.0**-23)).all(), (level, rstd)
        assert (value(got, dtype) == value(want, dtype)).all(), (level, np.abs(value(got, dtype) - value(want, dtype)).max())


@pytest.mark.parametrize("dtype", FLOATS, ids=[DTYPE_NAMES[d] for d in FLOATS])
@pytest.mark.parametrize("size", [(1, 512, 4), (200, 64, 4), (77, 320, 32), (390, 58, 2), (33, 257, 1), (60000, 64, 2)], ids=str)
def test_relu_passes_gradients_exactly_where_it_passed_values(cuda, dtype, size):
    """The bias puts the value in the middle of each channel on relu's kink: forward and backward have to take it for the same
    side. With a gradient of 1 everywhere dbias counts the elements that the backward pass took for positive."""
    s, c, groups = size
    rng = np.random.default_rng(sum(size))
    sd = stat_dtype(dtype)
    real = np.float64 if dtype == F64 else np.float32
    # some hundred above a spread of a few: steps of the half types are 1 and 1/4 there
    x = raw((192 + rng.integers(-8, 9, (1, s, c))).astype(np.float64), dtype)
    _, mean, rstd = norm(cuda, x, dtype, groups)
    wide = lambda v: np.repeat(v, c // groups, 1)[0]
    w = rng.uniform(0.5, 2, c).astype(real)
    middle = value(x, dtype)[0, s // 2].astype(real)
    b = -((middle - wide(mean)) * wide(rstd) * w)
    out, mean2, rstd2 = norm(cuda, x, dtype, groups, w, b, "relu")
    assert (mean == mean2).all() and (rstd == rstd2).all()
    out = value(out, dtype)[0]
    assert (out[s // 2] == 0).all()
    up = lambda v: cuda.upload(np.ascontiguousarray(v), sd)
    dx, dw, db = cuda.empty(x.shape, dtype), cuda.empty((c,), sd), cuda.empty((c,), sd)
    cuda.group_norm_backward(dx, cuda.upload(x, dtype), cuda.upload(raw(np.ones(x.shape), dtype), dtype), up(mean), up(rstd), groups,
                             up(w), up(b), dw, db, activation="relu")
    assert (cuda.download(db) == (out > 0).sum(0)).all(), np.abs(cuda.download(db) - (out > 0).sum(0)).max()


def one_large_many_small(be, large, s, c, n, dtype, groups):
    """dbias and dweight where dout is 2048 in the rows `large` and 2^-13 in all others, half a unit of f32 at 2048, so that an f32
    sum that has 2048 in it loses every addition; x = 1, mean = 0, rstd = 1. Samples are one sample, by a stride of 0."""
    d = np.full((1, s, c), 2.0**-13)
    d[0, large] = 2048.0
    src = be.upload(raw(np.ones((1, s, c)), dtype), dtype).expand(n, s, c)
    dout = be.upload(raw(d, dtype), dtype).expand(n, s, c)
    stat = lambda v: be.upload(np.full((1, groups), v, np.float32), F32).expand(n, groups)
    dx, dw, db = be.empty((n, s, c), dtype), be.empty((c,), F32), be.empty((c,), F32)
    be.group_norm_backward(dx, src, dout, stat(0), stat(1), groups, None, None, dw, db)
    return be.download(dw), be.download(db), n * d[0, :, 0].sum()


def test_sums_over_long_runs_of_rows(cuda):
    """As many strips as blocks, so a run is every position, one row at a time: at most 64 are added in f32, then in f64."""
    dw, db, want = one_large_many_small(cuda, [0], 2000, 129, 600, F16, 1)
    for got in (dw, db):
        # 64 roundings of the f32 sum, one of the product with the weight, half a step of the result
        assert (np.abs(got - want) <= (65 * 2.0**-24 + 2.0**-24) * want).all(), (got, want)


def test_sums_over_long_runs_of_whole_vectors(cuda):
    """The same with 16-byte vectors, whose runs are shorter instead: 15 rows at a time, 267 a thread."""
    dw, db, want = one_large_many_small(cuda, list(range(15)), 4000, 136, 600, F16, 1)
    for got in (dw, db):
        assert (np.abs(got - want) <= (65 * 2.0**-24 + 2.0**-24) * want).all(), (got, want)


def test_sums_over_a_clusters_rows(cuda):
    """Words in a cluster's shared memory, 98 rows a thread, the first of each thread large."""
    rows = [r for r in range(6272) if r % 784 < 8]
    dw, db, want = one_large_many_small(cuda, rows, 6272, 58, 1, F16, 2)
    for got in (dw, db):
        assert (np.abs(got - want) <= (65 * 2.0**-24 + 2.0**-24) * want).all(), (got, want)


@pytest.mark.parametrize("dtype", [BF16, F32, F64], ids=["bf16", "f32", "f64"])
@pytest.mark.parametrize("size", [(2, 1, 64, 2), (2, 90, 64, 4), (1, 33, 257, 1)], ids=str)
def test_gradients_far_out_on_an_activation(cuda, dtype, size):
    """Where an activation's slope is 0 or 1 to the last bit the gradient is 0 or dout, however large the value, in the types that
    hold such values; mean = 0 and rstd = 1, so the activation sees the input."""
    n, s, c, groups = size
    rng = np.random.default_rng(sum(size))
    sd = stat_dtype(dtype)
    up = lambda v, dt: cuda.upload(raw(v, dt), dt)
    for far in (200.0, 1e10, 1e14, 1e18, 1e20, 3e38) + ((1e60, 1e120, 1e300) if dtype == F64 else ()):
        sign = rng.integers(0, 2, (n, s, c)) * 2.0 - 1
        d = value(raw(rng.normal(size=(n, s, c)), dtype), dtype)
        for kind in ("relu", "silu", "gelu", "gelu_tanh"):
            dx, db = cuda.empty((n, s, c), dtype), cuda.empty((c,), sd)
            cuda.group_norm_backward(dx, up(sign * far, dtype), up(d, dtype), up(np.zeros((n, groups)), sd), up(np.ones((n, groups)), sd),
                                     groups, None, None, None, db, activation=kind)
            got, want, size_of = cuda.download(db), np.where(sign > 0, d, 0.0).sum((0, 1)), np.abs(d).sum((0, 1))
            # a slope of 1 within the 32 units of 1 + |z| at z = 200 of tests/layers_reference.py, at most n s additions
            u = 2.0**-53 if dtype == F64 else 2.0**-24
            assert (np.abs(got - want) <= (40 + n * s) * u * size_of).all(), (kind, far, got, want)


@pytest.mark.parametrize("dtype", FLOATS, ids=[DTYPE_NAMES[d] for d in FLOATS])
@pytest.mark.parametrize("channels", [64, 7, 300])
def test_a_logit_of_minus_infinity_forgets(cuda, dtype, channels):
    """sigmoid(-inf) is 0: nothing of the state before is left, however large that is, in the outputs, the state and the
    gradients."""
    rng = np.random.default_rng(channels)
    sd = stat_dtype(dtype)
    large = 60000.0 if dtype == F16 else 1e37
    for t in (1, 2, 9, 300):
        gate, x = rng.normal(size=(2, t, channels)), rng.normal(size=(2, t, channels))
        k = t // 2
        gate[:, k] = -np.inf
        x[:, k] = 0.0
        x[:, :k] = large
        gate[:, :k] = -20.0
        up = lambda v: cuda.upload(raw(v, dtype), dtype)
        out, last = cuda.empty((2, t, channels), dtype), cuda.empty((2, channels), sd)
        first = cuda.upload(raw(np.full((2, channels), large), sd), sd)
        cuda.linear_recurrence(out, up(gate), up(x), first, last, sigmoid=True)
        got = value(cuda.download(out), dtype)
        assert (got[:, k] == 0).all(), np.abs(got[:, k]).max()
        if k == t - 1:
            assert (cuda.download(last) == 0).all()
        # dinitial is the product of all gates, dgate has the factor a
        dgate, dx, di = cuda.empty((2, t, channels), dtype), cuda.empty((2, t, channels), dtype), cuda.empty((2, channels), sd)
        dlast = cuda.upload(raw(np.full((2, channels), 0.1), sd), sd)
        cuda.linear_recurrence_backward(dgate, dx, up(gate), None, out, up(np.full((2, t, channels), 0.1)), first, dlast, di, sigmoid=True)
        if k == 0:
            assert (cuda.download(di) == 0).all()
        assert (value(cuda.download(dgate), dtype)[:, k] == 0).all()


def test_products_of_gates_beyond_the_range_show(cuda):
    """Gates whose product leaves f32 within a piece, with states that stay in it (the header asks for gates whose products stay
    in range): a result is right or no finite number, never a finite wrong one, and a state of zero stays zero."""
    for t in (60, 300, 5000):
        apart, within_a_lane = np.full(t, 0.5), np.full(t, 0.5)
        apart[:50] = 30.0        # 1e-38 becomes 7e35, the product of 50 gates is 7e73, those of 16 are in range
        apart[50] = 0.0          # and infinity times 0 would be no number where the reset leaves x
        within_a_lane[:8] = 1e6  # 1e-38 becomes 1e10, the product of 8 gates is 1e48
        for gates in (apart, within_a_lane):
            for start in (0.0, 1e-38):
                x = np.zeros(t)
                x[50] = 1.0
                want, h = np.zeros(t), start
                for k in range(t):
                    h = gates[k] * h + x[k]
                    want[k] = h
                row = lambda v: cuda.upload(v.astype(np.float32), F32)
                out = cuda.empty((1, t, 33), F32)
                cuda.linear_recurrence(out, row(gates[None, :, None]).expand(1, t, 33), row(x[None, :, None]).expand(1, t, 33), row(np.full((1, 33), start)))
                got = cuda.download(out)[0].astype(np.float64)
                # three roundings a step, and as many again where a piece is folded first; subnormals are rounded absolutely
                right = np.abs(got - want[:, None]) <= 6 * t * 2.0**-24 * np.abs(want[:, None]) + 2.0**-126
                assert (right | ((start != 0.0) & ~np.isfinite(got))).all(), (t, start, got[~right][:4])


@pytest.mark.parametrize("dtype,size,kind", [(F32, (1300003, 1, 8, 1), "silu"), (BF16, (200001, 1, 64, 1), "gelu"), (F16, (30011, 3, 8, 2), None),
                                             (F64, (20011, 1, 12, 3), "relu"), (BF16, (3001, 20, 16, 2), "silu")], ids=str)
def test_many_samples(cuda, dtype, size, kind):
    """Hundreds of row blocks, runs of more than eight samples a team, and their partials for dweight and dbias."""
    n, s, c, groups = size
    rng = np.random.default_rng(n)
    sd = stat_dtype(dtype)
    x, d = raw(rng.normal(size=(n, s, c)), dtype), raw(rng.normal(0.3, 1, size=(n, s, c)), dtype)
    w, b = raw(rng.normal(1, 0.3, c), sd), raw(rng.normal(0, 0.3, c), sd)
    forward = group_norm(value(x, dtype), value(w, sd), value(b, sd), groups, 1e-5, kind, dtype)
    y, mean, rstd = norm(cuda, x, dtype, groups, w, b, kind)
    within(value(y, dtype), forward[0], rounded(forward[1], forward[0], dtype), "out")
    within(mean, forward[2], rounded(forward[3], forward[2], sd), "mean")
    within(rstd, forward[4], rounded(forward[5], forward[4], sd), "rstd")
    up = lambda v, dt: cuda.upload(v, dt)
    dx, dw, db = cuda.empty(x.shape, dtype), cuda.empty((c,), sd), cuda.empty((c,), sd)
    cuda.group_norm_backward(dx, up(x, dtype), up(d, dtype), up(mean, sd), up(rstd, sd), groups, up(w, sd), up(b, sd), dw, db, activation=kind)
    want = group_norm_backward(value(x, dtype), value(d, dtype), mean.astype(np.float64), rstd.astype(np.float64), value(w, sd), value(b, sd),
                               groups, kind, dtype)
    within(value(cuda.download(dx), dtype), want[0], rounded(want[1], want[0], dtype), "dsrc")
    within(cuda.download(dw), want[2], rounded(want[3], want[2], sd), "dweight")
    within(cuda.download(db), want[4], rounded(want[5], want[4], sd), "dbias")


@pytest.mark.parametrize("dtype", [BF16, F32, F64], ids=["bf16", "f32", "f64"])
def test_a_wait_that_runs_out_is_reported_and_leaves_the_context_usable(dtype):
    """The blocks of a cluster wait for one another's sums with a limit. With a limit of 0 all give up at once, every peer alive: the
    kernel ends, the next synchronisation says so once, and the following calls give the same bits as before."""
    rng = np.random.default_rng(1)
    be, sd = CudaBackend(0), stat_dtype(dtype)
    try:
        up = lambda v: be.upload(raw(v, dtype), dtype)
        for t in (300, 5000):
            gate, x, d = (up(rng.normal(size=(2, t, 34))) for _ in range(3))
            out, last = be.empty((2, t, 34), dtype), be.empty((2, 34), sd)
            dgate, dx, di = be.empty((2, t, 34), dtype), be.empty((2, t, 34), dtype), be.empty((2, 34), sd)
            forward = lambda: be.linear_recurrence(out, gate, x, None, last, sigmoid=True)
            backward = lambda: be.linear_recurrence_backward(dgate, dx, gate, None, out, d, None, None, di, sigmoid=True)
            forward(), backward()
            be.synchronize()
            want = [be.download(v) for v in (out, last, dgate, dx, di)]
            for call in (forward, backward):
                be.lib.hmc_test_wait_limit(0)
                try:
                    call()
                finally:
                    be.lib.hmc_test_wait_limit(-1)
                with pytest.raises(BackendError, match="gave up a bounded wait"):
                    be.synchronize()
                be.synchronize()
            forward(), backward()
            be.synchronize()
            for a, v in zip(want, [be.download(v) for v in (out, last, dgate, dx, di)]):
                assert (a == v).all()
    finally:
        be.close()


def test_threads_that_call_for_the_first_time_at_once(cuda):
    """Eight threads with a context each: kernels that need more shared memory than a launch gets unasked."""
    rng = np.random.default_rng(4)
    x, gate = rng.normal(size=(2, 700, 72)), rng.normal(size=(2, 700, 72))
    ready, results = threading.Barrier(8), [None] * 8

    def work(k):
        be = CudaBackend(0)
        try:
            found = []
            ready.wait(60)
            for dtype in (BF16, F16, F32, F64):
                up = lambda v: be.upload(raw(v, dtype), dtype)
                h, y, z = (be.empty(x.shape, dtype) for _ in range(3))
                stats = [be.empty((2, 6), stat_dtype(dtype)) for _ in range(2)]
                be.linear_recurrence(h, up(gate), up(x), sigmoid=True)
                be.group_norm(y, h, 6, None, None, *stats, activation="silu")
                be.dropout(z, y, Generator(3), 0.25, residual=h)
                grads = [be.empty(x.shape, dtype) for _ in range(3)]
                be.group_norm_backward(grads[0], h, z, *stats, 6, activation="silu")
                be.linear_recurrence_backward(grads[1], grads[2], up(gate), None, h, grads[0], sigmoid=True)
                found += [be.download(v) for v in (h, y, z, *grads)]
            results[k] = found
        finally:
            be.close()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert all(r is not None for r in results)
    for r in results[1:]:
        assert all((a.view(np.uint8) == v.view(np.uint8)).all() for a, v in zip(results[0], r))


@pytest.mark.parametrize("dtype", [F32, F64], ids=["f32", "f64"])
@pytest.mark.parametrize("s", [1, 200, 40000])
def test_activations_keep_their_relative_precision_in_the_tails(cuda, dtype, s):
    """A weight of 0 leaves the bias as the activation's argument. Relative bounds in units of the computation type, with the
    rounding of the exponential's argument as its leading term: u = 2^-24 (2^-53); ex2.approx 4, rcp.approx 2, the fit of erfc 2
    and its polynomial 4, sums and products 1 each."""
    z = np.concatenate([-np.geomspace(1e-6, 13.0, 250), np.geomspace(1e-6, 30.0, 246), [-20.0, -40.0, -80.0, 0.0]])
    z = raw(z, dtype)
    c = z.size
    x = raw(np.where(np.arange(s * c).reshape(1, s, c) % 2, 1.0, -1.0), dtype)
    u, least = (2.0**-53, 2.0**-1022) if dtype == F64 else (2.0**-24, 2.0**-126)
    z64 = value(z, dtype)
    inner = np.sqrt(8 / np.pi) * (z64 + 0.044715 * z64**3)
    sigmoid = lambda v: np.exp(np.minimum(v, 0)) / (1 + np.exp(-np.abs(v)))
    # gelu: -z^2 / 2 is rounded in x = |z| / sqrt(2) (twice, squared), in the fused sum and in the product with log2(e) (twice)
    wants = {"silu": (z64 * sigmoid(z64), 2 * np.abs(z64) + 12),
             "gelu": (z64 * np.array([0.5 * math.erfc(-v / math.sqrt(2)) for v in z64]), 3 * z64**2 + 20),
             "gelu_tanh": (z64 * sigmoid(inner), 6 * np.abs(inner) + 14)}
    for kind, (want, units) in wants.items():
        got, _, _ = norm(cuda, x, dtype, 4, np.zeros(c), z64, kind)
        off = np.abs(value(got, dtype)[0] - want)
        # (results below the smallest normal number, times |z|, are flushed)
        assert (off <= (units + 1) * u * np.abs(want) + 2 * np.abs(z64) * least).all(), (kind, z64[(off / np.abs(want + least)).argmax()], (off / np.abs(want + least)).max() / u)


@pytest.mark.parametrize("layout", ["half", "time first", "time last"])
@pytest.mark.parametrize("dtype", [F16, F64], ids=["f16", "f64"])
def test_layouts_of_the_other_types(cuda, dtype, layout):
    rng = np.random.default_rng(6)
    for size in ((2, 70, 66), (3, 33, 31), (1, 600, 64)):
        for reverse in (False, True):
            check_forward(cuda, rng, size, dtype, True, layout, sigmoid=True, complement=True, reverse=reverse)
            check_backward(cuda, rng, size, dtype, True, layout, sigmoid=True, complement=True, reverse=reverse)


@pytest.mark.parametrize("dtype", [F16, F64], ids=["f16", "f64"])
def test_dropout_of_strided_operands_in_the_other_types(cuda, dtype):
    """The mask goes by logical positions; the residual is broadcast along the first dimension."""
    rng = np.random.default_rng(7)
    x, r = raw(rng.normal(size=(5, 33, 18)), dtype), raw(rng.normal(size=(1, 33, 18)), dtype)
    turned = cuda.upload(np.ascontiguousarray(x.transpose(2, 0, 1)), dtype).transpose(0, 1).transpose(1, 2)
    for p in (0.0, 0.3, 1.0):
        out, gen = cuda.empty(x.shape, dtype), Generator(11)
        seed, offset = cuda.dropout(out, turned, gen, p, residual=cuda.upload(r, dtype).expand(5, 33, 18))
        want, bound, _ = dropout(value(x, dtype), value(r, dtype), p, seed, offset, dtype)
        within(value(cuda.download(out), dtype), want, rounded(bound, want, dtype), f"p {p}")

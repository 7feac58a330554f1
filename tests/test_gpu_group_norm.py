"""Group norm with an activation, channels last, and its gradients against the plain form in f64 (tests/layers_reference.py)."""
import numpy as np
import pytest

from homura_b200.host import ACTIVATIONS, BF16, DTYPE_NAMES, F16, F32, F64, FLOATS, CudaBackend
from layers_reference import group_norm, group_norm_backward, raw, rounded, value, within

pytestmark = pytest.mark.gpu

stat_dtype = lambda dtype: F64 if dtype == F64 else F32
# samples, positions, channels, groups: a group of one value, per token, odd widths, a group per channel, one group of
# all, groups that straddle vectors (10, 6, 3 channels), many positions, a group wider than a tile, many samples
SIZES = [(1, 1, 1, 1), (2, 1, 8, 8), (5, 1, 128, 1), (70, 1, 256, 2), (3, 1, 4096, 32), (2, 1, 5000, 1), (3, 1, 5001, 3),
         (2, 3, 12, 4), (2, 7, 30, 10), (1, 33, 320, 32), (4, 100, 40, 4), (2, 65, 96, 16), (2, 500, 7, 7), (1, 1000, 33, 3),
         (1, 4099, 16, 2), (2, 50, 3000, 2), (1, 9, 6007, 1), (600, 2, 24, 3), (300, 5, 64, 4), (2, 1200, 640, 32)]
KINDS = list(ACTIVATIONS)


def make(rng, n, s, c, dtype):
    return raw(rng.normal(size=(n, s, c)) * rng.uniform(0.5, 2, c) + rng.normal(0.5, 0.5, c), dtype)


def forward(be, x, w, b, groups, kind, dtype, pdtype, eps=1e-5, pad=0):
    n, s, c = x.shape
    stats = [be.empty((n, groups), stat_dtype(dtype)) for _ in range(2)]
    if pad:   # rows of a wider buffer, beginning at an odd place
        wide = np.full((n, s, c + 2 * pad), 77, x.dtype)
        wide[..., pad:pad + c] = x
        src, out = be.upload(wide, dtype).narrow(2, pad, c), be.upload(wide, dtype).narrow(2, pad, c)
    else:
        src, out = be.upload(x, dtype), be.empty(x.shape, dtype)
    up = lambda v: None if v is None else be.upload(v, pdtype)
    be.group_norm(out, src, groups, up(w), up(b), stats[0], stats[1], eps=eps, activation=kind)
    if pad:
        whole = be.download_storage(out).reshape(n, s, c + 2 * pad)
        edge = np.concatenate([whole[..., :pad], whole[..., pad + c:]], -1)
        assert (edge == np.full(1, 77, x.dtype)).all(), "wrote beside its channels"
    return be.download(out), be.download(stats[0]), be.download(stats[1])


def check_forward(be, rng, size, dtype, kind, affine, pdtype=None, pad=0):
    n, s, c, groups = size
    pdtype = dtype if pdtype is None else pdtype
    x = make(rng, n, s, c, dtype)
    w, b = (raw(rng.normal(1, 0.3, c), pdtype), raw(rng.normal(0, 0.3, c), pdtype)) if affine else (None, None)
    y, mean, rstd = forward(be, x, w, b, groups, kind, dtype, pdtype, pad=pad)
    wide = lambda v: None if v is None else value(v, pdtype)
    want = group_norm(value(x, dtype), wide(w), wide(b), groups, 1e-5, kind, dtype)
    what = f"{DTYPE_NAMES[dtype]} {size} {kind}"
    within(mean, want[2], rounded(want[3], want[2], stat_dtype(dtype)), "mean " + what)
    within(rstd, want[4], rounded(want[5], want[4], stat_dtype(dtype)), "rstd " + what)
    within(value(y, dtype), want[0], rounded(want[1], want[0], dtype), "out " + what)


def check_backward(be, rng, size, dtype, kind, affine, pdtype=None, pad=0, in_place=False):
    n, s, c, groups = size
    pdtype = dtype if pdtype is None else pdtype
    sd = stat_dtype(dtype)
    x, dout = make(rng, n, s, c, dtype), raw(rng.normal(size=(n, s, c)), dtype)
    w, b = (raw(rng.normal(1, 0.3, c), pdtype), raw(rng.normal(0, 0.3, c), pdtype)) if affine else (None, None)
    wide = lambda v: None if v is None else value(v, pdtype)
    moments = group_norm(value(x, dtype), wide(w), wide(b), groups, 1e-5, kind, dtype)
    mean, rstd = raw(moments[2], sd), raw(moments[4], sd)
    if pad:
        place = lambda v: be.upload(np.pad(v, ((0, 0), (0, 0), (pad, pad))), dtype).narrow(2, pad, c)
    else:
        place = lambda v: be.upload(v, dtype)
    src, d = place(x), place(dout)
    dsrc = d if in_place else place(np.zeros_like(x))
    dw, db = be.empty((c,), pdtype), be.empty((c,), pdtype)
    up = lambda v: None if v is None else be.upload(v, pdtype)
    be.group_norm_backward(dsrc, src, d, be.upload(mean, sd), be.upload(rstd, sd), groups, up(w), up(b), dw, db, activation=kind)
    want = group_norm_backward(value(x, dtype), value(dout, dtype), mean.astype(np.float64), rstd.astype(np.float64), wide(w), wide(b),
                               groups, kind, dtype)
    what = f"{DTYPE_NAMES[dtype]} {size} {kind}"
    within(value(be.download(dsrc), dtype), want[0], rounded(want[1], want[0], dtype), "dsrc " + what)
    within(value(be.download(dw), pdtype), want[2], rounded(want[3], want[2], pdtype), "dweight " + what)
    within(value(be.download(db), pdtype), want[4], rounded(want[5], want[4], pdtype), "dbias " + what)


@pytest.mark.parametrize("dtype", FLOATS, ids=[DTYPE_NAMES[d] for d in FLOATS])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_forward(cuda, dtype, size):
    rng = np.random.default_rng(sum(size) + dtype)
    for k, kind in enumerate(KINDS):
        check_forward(cuda, rng, size, dtype, kind, affine=k != 2)


@pytest.mark.parametrize("dtype", FLOATS, ids=[DTYPE_NAMES[d] for d in FLOATS])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_backward(cuda, dtype, size):
    rng = np.random.default_rng(sum(size) + 17 * dtype)
    for k, kind in enumerate(KINDS):
        check_backward(cuda, rng, size, dtype, kind, affine=k != 2)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_parameters_in_f32_and_rows_of_a_wider_buffer(cuda, dtype):
    rng = np.random.default_rng(7)
    for size in ((3, 1, 256, 4), (2, 65, 40, 4), (2, 600, 96, 8)):
        for pad in (0, 1, 4, 8):
            check_forward(cuda, rng, size, dtype, "silu", True, F32, pad)
            check_backward(cuda, rng, size, dtype, "silu", True, F32, pad)
            check_backward(cuda, rng, size, dtype, "gelu", True, F32, pad, in_place=True)


def test_in_place_and_strided_positions(cuda):
    rng = np.random.default_rng(9)
    n, s, c, groups = 3, 40, 24, 3
    x = make(rng, n, s, c, F32)
    want = group_norm(value(x, F32), None, None, groups, 1e-5, "relu", F32)
    t = cuda.upload(x, F32)
    cuda.group_norm(t, t, groups, activation="relu")
    within(cuda.download(t), want[0], rounded(want[1], want[0], F32), "in place")
    # positions first, samples second in memory; four dimensions with evenly spaced positions
    t = cuda.upload(np.ascontiguousarray(x.transpose(1, 0, 2)), F32).transpose(0, 1)
    out = cuda.empty((n, s, c), F32)
    cuda.group_norm(out, t, groups, activation="relu")
    within(cuda.download(out), want[0], rounded(want[1], want[0], F32), "positions first")
    out = cuda.empty((n, 5, 8, c), F32)
    cuda.group_norm(out, cuda.upload(x.reshape(n, 5, 8, c), F32), groups, activation="relu")
    within(cuda.download(out).reshape(n, s, c), want[0], rounded(want[1], want[0], F32), "maps")
    # one parameter for all channels, by a stride of 0
    w = cuda.upload(np.array([1.5], np.float32), F32).expand(c)
    b = cuda.upload(np.array([0.25], np.float32), F32).expand(c)
    want = group_norm(value(x, F32), np.full(c, 1.5), np.full(c, 0.25), groups, 1e-5, None, F32)
    out = cuda.empty((n, s, c), F32)
    cuda.group_norm(out, cuda.upload(x, F32), groups, w, b)
    within(cuda.download(out), want[0], rounded(want[1], want[0], F32), "broadcast parameters")


@pytest.mark.parametrize("s", [1, 200])
def test_hard_values(cuda, s):
    """Constant groups, means far above the spread, an outlier at the front, NaN and infinity staying in their group."""
    rng = np.random.default_rng(21)
    n, c, groups = 4, 64, 4
    x = rng.normal(size=(n, s, c))
    x[0, :, :16] = 3.25                     # constant: rstd = 1 / sqrt(eps)
    x[1] += 1000.0
    x[2, 0, 0] = 30000.0                    # where a shift by the first value would lose everything
    x[3, s // 2, 20] = np.nan
    x[3, s - 1, 40] = np.inf
    for dtype in (F32, BF16, F64):
        stored = raw(x, dtype)
        y, mean, rstd = forward(cuda, stored, None, None, groups, None, dtype, dtype)
        want = group_norm(value(stored, dtype), None, None, groups, 1e-5, None, dtype)
        wide = lambda v: v.reshape(n, s, groups, -1)
        clean = np.ones((n, groups), bool)
        clean[3, 1] = clean[3, 2] = False
        pick = lambda v: wide(v).transpose(0, 2, 1, 3)[clean]
        within(pick(value(y, dtype)), pick(want[0]), rounded(pick(want[1]), pick(want[0]), dtype), f"hard values {DTYPE_NAMES[dtype]}")
        within(mean[clean], want[2][clean], rounded(want[3], want[2], stat_dtype(dtype))[clean], "means")
        within(rstd[clean], want[4][clean], rounded(want[5], want[4], stat_dtype(dtype))[clean], "rstds")
        assert np.isnan(wide(value(y, dtype)).transpose(0, 2, 1, 3)[~clean]).all()


def test_gradients_are_the_differences(cuda):
    rng = np.random.default_rng(3)
    n, s, c, groups, step = 2, 9, 12, 3, 1e-6
    for kind in KINDS:
        x, w, b, d = rng.normal(size=(n, s, c)), rng.normal(1, 0.3, c), rng.normal(0, 0.3, c), rng.normal(size=(n, s, c))
        up = lambda v: cuda.upload(v, F64)

        def loss(x, w, b):
            return float((forward(cuda, x, w, b, groups, kind, F64, F64)[0] * d).sum())

        _, mean, rstd = forward(cuda, x, w, b, groups, kind, F64, F64)
        dx, dw, db = cuda.empty(x.shape, F64), cuda.empty((c,), F64), cuda.empty((c,), F64)
        cuda.group_norm_backward(dx, up(x), up(d), up(mean), up(rstd), groups, up(w), up(b), dw, db, activation=kind)
        for name, arr, grad in (("x", x, dx), ("weight", w, dw), ("bias", b, db)):
            got = cuda.download(grad).reshape(-1)
            for k in rng.choice(arr.size, 8, replace=False):
                e = np.zeros(arr.size)
                e[k] = step
                e = e.reshape(arr.shape)
                vary = lambda sign: loss(*(v + sign * e if v is arr else v for v in (x, w, b)))
                diff = (vary(1) - vary(-1)) / (2 * step)
                # truncation of some tens times step^2 and cancellation of |loss| ~ 30 in 1e-16 * 216 / step; relu's kink
                # would show only for |z| < step
                assert abs(diff - got[k]) <= 2e-7 * (1 + abs(diff)), (kind, name, diff, got[k])


def test_empty_tensors(cuda):
    for shape in ((0, 3, 8), (2, 0, 8), (2, 3, 0)):
        t = cuda.empty(shape, F32)
        cuda.group_norm(t, t, 4, activation="silu")
        mean = cuda.empty((shape[0], 4), F32)
        dw, db = cuda.upload(np.full(shape[2], 5, np.float32), F32), cuda.upload(np.full(shape[2], 5, np.float32), F32)
        cuda.group_norm_backward(t, t, t, mean, mean, 4, None, None, dw, db)
        assert (cuda.download(dw) == 0).all() and (cuda.download(db) == 0).all()


def test_only_what_is_asked_for(cuda):
    rng = np.random.default_rng(5)
    n, s, c, groups = 2, 90, 40, 5
    x, d = make(rng, n, s, c, F32), raw(rng.normal(size=(n, s, c)), F32)
    m = group_norm(value(x, F32), None, None, groups, 1e-5, "silu", F32)
    mean, rstd = raw(m[2], F32), raw(m[4], F32)
    want = group_norm_backward(value(x, F32), value(d, F32), mean.astype(np.float64), rstd.astype(np.float64), None, None, groups, "silu", F32)
    up = lambda v: cuda.upload(v, F32)
    for with_w, with_b in ((False, False), (True, False), (False, True)):
        dx, dw, db = cuda.empty(x.shape, F32), cuda.empty((c,), F32), cuda.empty((c,), F32)
        cuda.group_norm_backward(dx, up(x), up(d), up(mean), up(rstd), groups, None, None, dw if with_w else None, db if with_b else None,
                                 activation="silu")
        within(cuda.download(dx), want[0], rounded(want[1], want[0], F32), "dsrc")
        if with_w:
            within(cuda.download(dw), want[2], rounded(want[3], want[2], F32), "dweight")
        if with_b:
            within(cuda.download(db), want[4], rounded(want[5], want[4], F32), "dbias")


def test_results_repeat(cuda):
    rng = np.random.default_rng(6)
    x = make(rng, 3, 1500, 320, BF16)
    w, b = raw(rng.normal(1, 0.3, 320), BF16), raw(rng.normal(0, 0.3, 320), BF16)
    runs = [forward(cuda, x, w, b, 32, "silu", BF16, BF16) for _ in range(3)]
    for r in runs[1:]:
        for a, v in zip(runs[0], r):
            assert (a.view(np.uint8) == v.view(np.uint8)).all()
    grads = []
    for _ in range(3):
        dx, dw, db = cuda.empty(x.shape, BF16), cuda.empty((320,), BF16), cuda.empty((320,), BF16)
        cuda.group_norm_backward(dx, cuda.upload(x, BF16), cuda.upload(runs[0][0], BF16), cuda.upload(runs[0][1], F32),
                                 cuda.upload(runs[0][2], F32), 32, cuda.upload(w, BF16), cuda.upload(b, BF16), dw, db, activation="silu")
        grads.append([cuda.download(v) for v in (dx, dw, db)])
    for g in grads[1:]:
        assert all((a == v).all() for a, v in zip(grads[0], g))


def test_two_backends_at_once(cuda):
    other = CudaBackend(0)
    try:
        rng = np.random.default_rng(8)
        x = make(rng, 2, 2000, 64, F32)
        want, _, _ = forward(cuda, x, None, None, 4, "gelu", F32, F32)
        outs = []
        for be in (cuda, other) * 4:
            out, src = be.empty(x.shape, F32), be.upload(x, F32)
            be.group_norm(out, src, 4, activation="gelu")
            outs.append((be, out, src))
        for be, out, _ in outs:
            assert (be.download(out) == want).all()
    finally:
        other.close()


@pytest.mark.parametrize("dtype,size", [(F32, (1, 60000, 64, 2)), (BF16, (1, 9000, 532, 2)), (F16, (2, 9001, 531, 1)), (F32, (1, 30001, 33, 1)),
                                        (BF16, (3, 20000, 256, 1))],
                         ids=["f32 lines", "bf16 words", "f16 odd", "f32 words", "bf16 lines"])
def test_groups_beyond_a_cluster(cuda, dtype, size):
    """Groups whose rows no cluster's shared memory holds: pieces that a second kernel merges."""
    rng = np.random.default_rng(sum(size))
    check_forward(cuda, rng, size, dtype, "silu", True)
    check_backward(cuda, rng, size, dtype, "silu", True)
    check_backward(cuda, rng, size, dtype, "relu", False, F32 if dtype != F32 else None)

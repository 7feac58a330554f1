"""Dropout from the counter-based generator against the plain form in f64 (tests/layers_reference.py): the mask word for
word, the values within their rounding."""
import numpy as np
import pytest

from homura_b200.host import BF16, DTYPE_NAMES, F16, F32, F64, FLOATS, BackendError, Generator
from layers_reference import dropout, philox_words, raw, rounded, value, within

pytestmark = pytest.mark.gpu


def check(be, rng, shape, dtype, p, residual, layout=None):
    x, r = raw(rng.normal(size=shape), dtype), raw(rng.normal(size=shape), dtype)
    gen = Generator(int(rng.integers(2**63)))
    gen.offset = int(rng.integers(2**40))
    place = layout or (lambda v: be.upload(v, dtype))
    out, src = place(np.zeros_like(x)), place(x)
    offset = gen.offset
    state = be.dropout(out, src, gen, p, place(r) if residual else None)
    assert state == (gen.seed, offset) and gen.offset == offset + -(-x.size // 4)
    want, e, kept = dropout(value(x, dtype), value(r, dtype) if residual else None, p, *state, dtype)
    got = value(be.download(out), dtype).reshape(shape)
    within(got, want, rounded(e, want, dtype), f"{DTYPE_NAMES[dtype]} {shape} p={p}")
    base = value(r, dtype) if residual else np.zeros(shape)
    assert (got[~kept] == base[~kept]).all(), "a dropped element left something"
    # the gradient regenerates the mask
    d = raw(rng.normal(size=shape), dtype)
    dsrc = place(np.zeros_like(x))
    be.dropout_backward(dsrc, place(d), p, state)
    want, e, _ = dropout(value(d, dtype), None, p, *state, dtype)
    within(value(be.download(dsrc), dtype).reshape(shape), want, rounded(e, want, dtype), "gradient")


@pytest.mark.parametrize("dtype", FLOATS, ids=[DTYPE_NAMES[d] for d in FLOATS])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 9, 31, 2047, 2048, 2049, 100003, (1 << 20) + 5])
def test_sizes(cuda, dtype, n):
    rng = np.random.default_rng(n)
    for p in (0.0, 0.1, 0.5, 0.9):
        check(cuda, rng, (n,), dtype, p, residual=p in (0.1, 0.9))


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_layouts(cuda, dtype):
    """The mask goes by the logical position: transposed, narrowed and misaligned views give the same elements."""
    rng = np.random.default_rng(2)
    up = lambda v: cuda.upload(v, dtype)
    for residual in (False, True):
        check(cuda, rng, (33, 70), dtype, 0.3, residual, lambda v: up(np.ascontiguousarray(v.T)).t())
        check(cuda, rng, (5, 9, 14), dtype, 0.3, residual, lambda v: up(np.ascontiguousarray(v.transpose(2, 0, 1))).permute(1, 2, 0))
        check(cuda, rng, (33, 70), dtype, 0.3, residual, lambda v: up(np.pad(v, ((0, 0), (3, 5)))).narrow(1, 3, 70))
        check(cuda, rng, (4001,), dtype, 0.3, residual, lambda v: up(np.pad(v, (1, 2))).narrow(0, 1, 4001))
        check(cuda, rng, (), dtype, 0.3, residual)


def test_in_place_and_no_numbers(cuda):
    rng = np.random.default_rng(3)
    for residual in (False, True):
        for target in ("src", "residual")[:1 + residual]:
            x, r = rng.normal(size=5000).astype(np.float32), rng.normal(size=5000).astype(np.float32)
            x[::7], x[3::11] = np.nan, np.inf
            s, t = cuda.upload(x, F32), cuda.upload(r, F32)
            gen = Generator(5)
            state = cuda.dropout(s if target == "src" else t, s, gen, 0.5, t if residual else None)
            want, e, _ = dropout(x.astype(np.float64), r.astype(np.float64) if residual else None, 0.5, *state, F32)
            within(cuda.download(s if target == "src" else t), want, rounded(e, np.nan_to_num(want, posinf=0, neginf=0), F32), "in place")


def test_ends_of_the_probabilities(cuda):
    x = np.arange(1, 100001, dtype=np.float32)
    s, out = cuda.upload(x, F32), cuda.empty((100000,), F32)
    cuda.dropout(out, s, Generator(1), 0.0)
    assert (cuda.download(out) == x).all()
    cuda.dropout(out, s, Generator(1), 1.0)
    assert (cuda.download(out) == 0).all()
    cuda.dropout(out, s, Generator(1), 1.0, s)
    assert (cuda.download(out) == x).all()
    cuda.dropout(out, s, Generator(1), 1.0 - 2.0**-40)   # rounds to every word
    assert (cuda.download(out) == 0).all()
    for p in (0.01, 0.3, 0.99):
        gen = Generator(77)
        cuda.dropout(out, s, gen, p)
        dropped = (cuda.download(out) == 0).mean()
        assert abs(dropped - p) < 6 * (p * (1 - p) / 100000) ** 0.5
    empty = cuda.empty((0, 5), F32)
    gen = Generator(1)
    assert cuda.dropout(empty, empty, gen, 0.5) == (1, 0) and gen.offset == 0
    with pytest.raises(BackendError, match="between 0 and 1"):
        cuda.dropout(out, s, gen, 1.5)


def test_the_words_are_the_uniform_samplers(cuda):
    """The mask of p = 1/2 is the top bit of the words hmc_random_uniform turns into samples."""
    n = 4097
    u = cuda.empty((n,), F32)
    cuda.random_uniform(u, Generator(12345), 0.0, 1.0)
    out = cuda.empty((n,), F32)
    cuda.dropout(out, cuda.upload(np.ones(n, np.float32), F32), Generator(12345), 0.5)
    assert ((cuda.download(out) != 0) == (cuda.download(u) >= 0.5)).all()
    assert ((philox_words(n, 12345, 0) >= 2**31) == (cuda.download(u) >= 0.5)).all()


def test_block_numbers_pass_32_and_64_bits(cuda):
    x = cuda.upload(np.ones(1000, np.float32), F32)
    out = cuda.empty((1000,), F32)
    for offset in (2**32 - 100, 2**64 - 100):
        gen = Generator(9)
        gen.offset = offset
        state = cuda.dropout(out, x, gen, 0.5)
        kept = dropout(np.ones(1000), None, 0.5, *state, F32)[2]
        assert ((cuda.download(out) != 0) == kept).all()

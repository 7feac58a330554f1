"""The operators of include/homura_cuda_layers.h together, as a training step of a recurrent block uses them: gates and
inputs from one projection, the recurrence, group norm with silu over heads, dropout on the residual stream, a squared
loss, all gradients back to the projection, and an AdamW step of the parameters by the optimizer that was there before.
The same run is captured into a CUDA graph and replayed, and continued token by token."""
import ctypes

import numpy as np
import pytest

from homura_b200 import ffi
from homura_b200.host import BF16, F16, F32, F64, I64, BackendError, CudaBackend, Generator
from layers_reference import (activation, dropout, gates, group_norm, group_norm_backward, raw, recurrence, recurrence_backward,
                              rounded, value, within)

pytestmark = pytest.mark.gpu


class Block:
    """One block on the device: [batch, time, channels], `groups` heads."""

    def __init__(self, be, b, t, c, groups, dtype, seed, p=0.2):
        rng = np.random.default_rng(seed)
        self.be, self.shape, self.groups, self.dtype, self.p, self.seed = be, (b, t, c), groups, dtype, p, seed
        sd = F64 if dtype == F64 else F32
        self.projection = raw(rng.normal(size=(b, t, 2 * c)) + np.repeat([1.5, 0.0], c), dtype)
        self.residual = raw(rng.normal(size=(b, t, c)), dtype)
        self.target = raw(rng.normal(size=(b, t, c)), dtype)
        self.weight, self.bias = raw(rng.normal(1, 0.2, c), sd), raw(rng.normal(0, 0.2, c), sd)
        up = lambda v, d=dtype: be.upload(v, d)
        proj = up(self.projection)
        self.gate, self.x = proj.narrow(2, 0, c), proj.narrow(2, c, c)
        self.d_residual, self.d_target = up(self.residual), up(self.target)
        self.w, self.b = up(self.weight, sd), up(self.bias, sd)
        self.h, self.y, self.z = (be.empty((b, t, c), dtype) for _ in range(3))
        # every token is a sample of its own: a group per head
        self.mean, self.rstd = be.empty((b * t, groups), sd), be.empty((b * t, groups), sd)
        self.last = be.empty((b, c), sd)
        dproj = be.empty((b, t, 2 * c), dtype)
        self.dproj, self.dgate, self.dx = dproj, dproj.narrow(2, 0, c), dproj.narrow(2, c, c)
        self.dz, self.dy, self.dh = (be.empty((b, t, c), dtype) for _ in range(3))
        self.dw, self.db = be.empty((c,), sd), be.empty((c,), sd)

    def tokens(self, v):
        b, t, c = self.shape
        return v.reshape(b * t, 1, c)

    def step(self):
        be = self.be
        gen = Generator(self.seed)
        be.linear_recurrence(self.h, self.gate, self.x, last=self.last, sigmoid=True, complement=True)
        be.group_norm(self.tokens(self.y), self.tokens(self.h), self.groups, self.w, self.b, self.mean, self.rstd, activation="silu")
        state = be.dropout(self.z, self.y, gen, self.p, self.d_residual)
        be.binary(ffi.HMC_BINARY_SUB, self.dz, self.z, self.d_target)  # the gradient of half the squared distance
        be.dropout_backward(self.dy, self.dz, self.p, state)
        be.group_norm_backward(self.tokens(self.dh), self.tokens(self.h), self.tokens(self.dy), self.mean, self.rstd, self.groups, self.w,
                               self.b, self.dw, self.db, activation="silu")
        be.linear_recurrence_backward(self.dgate, self.dx, self.gate, self.x, self.h, self.dh, sigmoid=True, complement=True)
        return state

    def results(self):
        return {k: self.be.download(getattr(self, k)) for k in ("h", "last", "y", "mean", "rstd", "z", "dz", "dy", "dh", "dw", "db", "dproj")}


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("size", [(2, 130, 96, 3), (1, 700, 40, 4), (3, 1, 64, 2)], ids=str)
def test_a_training_step(cuda, dtype, size):
    b, t, c, groups = size
    block = Block(cuda, *size, dtype, seed=sum(size))
    state = block.step()
    r = block.results()
    v = lambda k: value(r[k], dtype)
    gate, x = value(block.projection[..., :c], dtype), value(block.projection[..., c:], dtype)
    flat = lambda a: a.reshape(b * t, 1, c)
    # each stage against the plain form on what the stage before really left
    h, e, last, el = recurrence(gate, x, None, dtype, True, True)
    within(v("h"), h, rounded(e, h, dtype), "h")
    within(r["last"], last, rounded(el, last, F32), "last")
    w, bias = block.weight.astype(np.float64), block.bias.astype(np.float64)
    y, ey, mean, em, rstd, er = group_norm(flat(v("h")), w, bias, groups, 1e-5, "silu", dtype)
    within(flat(v("y")), y, rounded(ey, y, dtype), "y")
    within(r["mean"], mean, rounded(em, mean, F32), "mean")
    z, ez, _ = dropout(v("y"), value(block.residual, dtype), 0.2, *state, dtype)
    within(v("z"), z, rounded(ez, z, dtype), "z")
    dy, edy, _ = dropout(v("dz"), None, 0.2, *state, dtype)
    within(v("dy"), dy, rounded(edy, dy, dtype), "dy")
    dh, edh, dw, edw, db, edb = group_norm_backward(flat(v("h")), flat(v("dy")), r["mean"].astype(np.float64), r["rstd"].astype(np.float64),
                                                    w, bias, groups, "silu", dtype)
    within(flat(v("dh")), dh, rounded(edh, dh, dtype), "dh")
    within(r["dw"], dw, rounded(edw, dw, F32), "dw")
    within(r["db"], db, rounded(edb, db, F32), "db")
    dgate, eg, dx, ex, _, _ = recurrence_backward(gate, x, v("h"), None, v("dh"), None, dtype, True, True)
    within(v("dproj")[..., :c], dgate, rounded(eg, dgate, dtype), "dgate")
    within(v("dproj")[..., c:], dx, rounded(ex, dx, dtype), "dx")
    # the optimizer takes the parameters from here
    for param, grad in ((block.w, block.dw), (block.b, block.db)):
        before = cuda.download(param)
        m, s = cuda.upload(np.zeros(c, np.float32), F32), cuda.upload(np.zeros(c, np.float32), F32)
        cuda.adamw_step(param, grad, m, s, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, step=1.0)
        g = cuda.download(grad)
        moved = cuda.download(param) - before
        ok = np.abs(g) > 1e-6
        assert np.allclose(moved[ok], -1e-3 * np.sign(g[ok]), atol=1e-5)


def test_the_whole_gradient_is_the_difference(cuda):
    """The step's gradient with respect to the projection against central differences of its own forward pass in f64."""
    b, t, c, groups = 2, 37, 24, 3
    block = Block(cuda, b, t, c, groups, F64, seed=5)
    block.step()
    grad = block.results()["dproj"].reshape(-1)
    rng = np.random.default_rng(1)

    def loss(projection):
        probe = Block(cuda, b, t, c, groups, F64, seed=5)
        probe_in = cuda.upload(projection, F64)
        probe.gate, probe.x = probe_in.narrow(2, 0, c), probe_in.narrow(2, c, c)
        probe.step()
        return 0.5 * float((cuda.download(probe.dz) ** 2).sum())

    step = 1e-6
    for k in rng.choice(grad.size, 10, replace=False):
        d = np.zeros(grad.size)
        d[k] = step
        d = d.reshape(b, t, 2 * c)
        diff = (loss(block.projection + d) - loss(block.projection - d)) / (2 * step)
        # truncation of some tens times step^2, cancellation of |loss| ~ 2e3 in 1e-16 * 2e3 / step
        assert abs(diff - grad[k]) <= 2e-6 * (1 + abs(diff)), (k, diff, grad[k])


def test_token_by_token_follows_the_whole_sequence(cuda):
    """The forward pass of 40 steps against 40 calls of one step that hand the state on in place."""
    b, t, c, groups = 2, 40, 64, 4
    for dtype in (BF16, F32):
        block = Block(cuda, b, t, c, groups, dtype, seed=9)
        block.step()
        whole = block.results()
        state = cuda.upload(np.zeros((b, c), np.float32), F32)
        h, y = cuda.empty((b, 1, c), dtype), cuda.empty((b, 1, c), dtype)
        got_h, got_y = [], []
        for k in range(t):
            cuda.linear_recurrence(h, block.gate.narrow(1, k, 1), block.x.narrow(1, k, 1), state, state, sigmoid=True, complement=True)
            cuda.group_norm(y.reshape(b, 1, c), h, groups, block.w, block.b, activation="silu")
            got_h.append(cuda.download(h))
            got_y.append(cuda.download(y))
        gate, x = value(block.projection[..., :c], dtype), value(block.projection[..., c:], dtype)
        want, e, last, el = recurrence(gate, x, None, dtype, True, True)
        within(value(np.concatenate(got_h, 1), dtype), want, rounded(e, want, dtype), "states token by token")
        within(cuda.download(state), last, rounded(el, last, F32) + 40 * 2.0**-24 * np.abs(want).max(), "the state handed on")
        a, b_ = value(np.concatenate(got_y, 1), dtype), value(whole["y"], dtype)
        # (h agrees to its dtype's step, which the norm may scale by rstd of the smallest spread)
        assert np.median(np.abs(a - b_)) <= {BF16: 2.0**-7, F32: 2.0**-20}[dtype]


def _runtime():
    for name in ("libcudart.so.12", "libcudart.so"):
        try:
            return ctypes.CDLL(name)
        except OSError:
            continue
    from pathlib import Path
    for line in Path("/proc/self/maps").read_text().splitlines():
        if "libcudart" in line:
            return ctypes.CDLL(line.split()[-1])
    raise OSError("the CUDA runtime is not loaded")


def test_a_captured_step_replays(cuda):
    """The step queued once in a stream capture and replayed on new inputs gives the bits of the eager calls, two graphs of
    two blocks in turn among them."""
    rt = _runtime()
    for fn in ("cudaStreamBeginCapture", "cudaStreamEndCapture", "cudaGraphInstantiate", "cudaGraphLaunch", "cudaGraphExecDestroy",
               "cudaGraphDestroy"):
        getattr(rt, fn).restype = ctypes.c_int
    be = CudaBackend(0)
    try:
        blocks = [Block(be, 2, 300, 96, 3, BF16, seed=11), Block(be, 1, 2000, 64, 2, BF16, seed=12)]
        want = []
        for blk in blocks:
            blk.step()        # (loads the kernels, fills the allocator)
            want.append(blk.results())
        stream = ctypes.c_void_p()
        be._check(be.lib.hmc_context_stream(be.ctx, ctypes.byref(stream)))
        graphs = []
        for blk in blocks:
            # workspaces of a captured call have to outlive the capture: none is given back while it runs
            held, allocate = [], be.storage
            be.storage = lambda n: held.append(allocate(n)) or held[-1]
            graph, run = ctypes.c_void_p(), ctypes.c_void_p()
            assert rt.cudaStreamBeginCapture(stream, 2) == 0
            try:
                blk.step()
            finally:
                assert rt.cudaStreamEndCapture(stream, ctypes.byref(graph)) == 0
                be.storage = allocate
            assert rt.cudaGraphInstantiate(ctypes.byref(run), graph, 0) == 0
            graphs.append((graph, run, held))
        for blk in blocks:    # nothing of the eager results is left
            for k in ("h", "y", "z", "dz", "dy", "dh", "dproj"):
                be.fill(getattr(blk, k), 0.0)
            be.fill(blk.dw, 0.0)
        for _ in range(2):
            for _, run, _ in graphs:
                assert rt.cudaGraphLaunch(run, stream) == 0
        for blk, w in zip(blocks, want):
            got = blk.results()
            for k in w:
                assert (got[k].view(np.uint8) == w[k].view(np.uint8)).all(), k
        for graph, run, _ in graphs:
            assert rt.cudaGraphExecDestroy(run) == 0 and rt.cudaGraphDestroy(graph) == 0
    finally:
        be.close()

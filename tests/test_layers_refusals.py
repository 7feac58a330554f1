"""What the operators of include/homura_cuda_layers.h refuse, without a GPU: arguments are checked before the context is
looked at, so a call with none reports its first bad argument, and one whose arguments are sound reports the context."""
import ctypes

import numpy as np
import pytest

import homura_b200
from homura_b200 import ffi
from homura_b200.host import (BF16, F16, F32, F64, I32, ACTIVATIONS, BackendError, CudaBackend, Generator, Storage, TensorData, activation_code,
                              channels_last_desc, check_positions, contiguous_strides, plain_desc, recurrence_flags)

HOST = np.zeros(1 << 16, dtype=np.uint8)  # an address that is not null; no call here gets as far as using it


def desc(sizes, dtype=F32, strides=None, offset=0, data=True):
    d = ffi.hmc_tensor_desc()
    d.data, d.offset, d.dtype, d.ndim = HOST.ctypes.data if data else None, offset, dtype, len(sizes)
    st = contiguous_strides(sizes) if strides is None else strides
    for k, (n, s) in enumerate(zip(sizes, st)):
        d.sizes[k], d.strides[k] = n, s
    return d


def refused(status, piece):
    message = homura_b200.load().hmc_last_error().decode()
    assert status == ffi.HMC_INVALID and piece in message, (status, message)


def recur(out=None, gate=None, x=None, initial=None, last=None, flags=0):
    three = lambda d: desc([2, 3, 4]) if d is None else d
    return homura_b200.load().hmc_linear_recurrence(None, three(out), three(gate), three(x), initial, last, flags)


def test_recurrence_refusals():
    refused(recur(), "null context")
    refused(recur(initial=desc([2, 4]), last=desc([2, 4]), flags=7), "null context")
    refused(recur(gate=desc([2, 3, 4], I32)), "floating point")
    refused(recur(gate=desc([2, 12])), "3 dimensions")
    refused(recur(x=desc([2, 3, 5])), "x has the wrong sizes")
    refused(recur(x=desc([2, 3, 4], BF16)), "x has the wrong dtype")
    refused(recur(x=desc([2, 3, 4], data=False)), "null data pointer")
    refused(recur(out=desc([2, 3, 4], strides=[12, 0, 1])), "not distinct")
    refused(recur(out=desc([2, 3, 4], strides=[12, -4, 1])), "negative stride")
    refused(recur(x=desc([2, 3, 4], strides=[2**62, 4, 1])), "beyond 63 bits")
    refused(recur(x=desc([2, 3, 4], offset=-1)), "negative offset")
    refused(recur(flags=8), "unknown flags")
    refused(recur(initial=desc([2, 4], BF16)), "the initial state has the wrong dtype")
    refused(recur(initial=desc([4, 2])), "the initial state has the wrong sizes")
    refused(recur(last=desc([2, 4], F64)), "the last state has the wrong dtype")
    refused(recur(last=desc([2, 4], strides=[0, 1])), "not distinct")
    half, double = desc([2, 3, 4], F16), desc([2, 3, 4], F64)
    refused(recur(half, half, half, desc([2, 4], F16)), "the initial state has the wrong dtype")
    refused(recur(half, half, half, desc([2, 4])), "null context")
    refused(recur(double, double, double, desc([2, 4])), "the initial state has the wrong dtype")
    refused(recur(double, double, double, desc([2, 4], F64)), "null context")
    refused(homura_b200.load().hmc_linear_recurrence(None, desc([2, 3, 4]), None, desc([2, 3, 4]), None, None, 0), "null description")
    # an empty tensor needs no memory
    empty = desc([2, 0, 4], data=False)
    refused(recur(empty, empty, empty), "null context")
    big = desc([2**40, 3, 2**40], strides=[0, 0, 0])
    refused(recur(big, big, big), "overflows")


def test_recurrence_backward_refusals():
    lib = homura_b200.load()
    t = desc([2, 3, 4])

    def call(dgate=t, dx=t, dinitial=None, gate=t, x=t, out=t, initial=None, dout=t, dlast=None, flags=0):
        return lib.hmc_linear_recurrence_backward(None, dgate, dx, dinitial, gate, x, out, initial, dout, dlast, flags)

    refused(call(), "null context")
    refused(call(x=None), "null context")
    refused(call(x=None, flags=ffi.HMC_RECURRENCE_COMPLEMENT), "null description of x")
    refused(call(out=desc([2, 3, 5])), "the forward output has the wrong sizes")
    refused(call(dout=desc([2, 3, 4], F16)), "the output's gradient has the wrong dtype")
    refused(call(dgate=None), "null description of the gate's gradient")
    refused(call(dgate=desc([2, 3, 4], strides=[0, 4, 1])), "not distinct")
    refused(call(dx=desc([2, 3, 4], strides=[12, 4, 0])), "not distinct")
    refused(call(dlast=desc([2, 3])), "the last state's gradient has the wrong sizes")
    refused(call(dinitial=desc([2, 4], strides=[4, 0])), "not distinct")
    refused(call(flags=-1), "unknown flags")


def test_group_norm_refusals():
    lib = homura_b200.load()
    t, stat, par = desc([2, 3, 8]), desc([2, 4]), desc([8])
    long = desc([2, 3000000, 8])  # a group that no cluster holds: its pieces' moments need a workspace
    nbytes = ctypes.c_int64(-1)
    assert lib.hmc_group_norm_workspace(t, 4, 0, ctypes.byref(nbytes)) == ffi.HMC_OK and nbytes.value >= 0
    assert lib.hmc_group_norm_workspace(long, 4, 0, ctypes.byref(nbytes)) == ffi.HMC_OK and nbytes.value > 0
    need = nbytes.value
    ws = (HOST.ctypes.data + 15) // 16 * 16

    def call(out=t, src=t, weight=None, bias=None, mean=None, rstd=None, groups=4, eps=1e-5, act=ffi.HMC_ACTIVATION_NONE, ws=ws, n=1 << 15):
        return lib.hmc_group_norm(None, out, src, weight, bias, mean, rstd, groups, eps, act, ws, n)

    refused(call(), "null context")
    refused(call(out=long, src=long, n=need), "null context")
    refused(call(out=long, src=long, n=need - 1), f"group norm needs {need}")
    refused(call(out=long, src=long, ws=None), f"group norm needs {need}")
    refused(call(out=long, src=long, ws=ws + 4, n=need), "16-byte aligned")
    refused(call(groups=3), "do not divide")
    refused(call(groups=0), "do not divide")
    refused(call(groups=-4), "do not divide")
    refused(call(src=desc([2, 3, 8], I32)), "floating point")
    refused(call(src=desc([2, 24])), "3 dimensions")
    refused(call(src=desc([2, 3, 8], strides=[24, 1, 3])), "not channels last")
    refused(call(out=desc([2, 3, 8], strides=[24, 1, 3])), "not channels last")
    refused(call(out=desc([2, 3, 8], strides=[0, 8, 1])), "not distinct")
    refused(call(out=desc([2, 3, 8], F16)), "the output has the wrong dtype")
    refused(call(weight=par), "both weight and bias")
    refused(call(mean=stat), "both mean and rstd")
    refused(call(weight=desc([8], F16), bias=desc([8], F16)), "neither the input's dtype nor F32")
    refused(call(weight=par, bias=desc([8], F16)), "the bias has the wrong dtype")
    refused(call(weight=desc([4]), bias=desc([4])), "the weight has the wrong sizes")
    refused(call(mean=desc([2, 8]), rstd=desc([2, 8])), "the mean has the wrong sizes")
    refused(call(mean=stat, rstd=desc([2, 4], F64)), "the rstd has the wrong dtype")
    refused(call(eps=-1.0), "eps of at least 0")
    refused(call(eps=float("nan")), "eps of at least 0")
    refused(call(act=ffi.HMC_UNARY_EXP), "activation")
    empty = desc([2, 0, 8])
    refused(call(out=empty, src=empty, ws=None, n=0), "null context")
    refused(call(out=empty, src=empty, mean=stat, rstd=stat), "moments of empty groups")
    assert lib.hmc_group_norm_workspace(t, 4, 0, None) == ffi.HMC_INVALID
    refused(lib.hmc_group_norm_workspace(desc([2**30, 2**20, 2**10], strides=[0, 0, 1]), 4, 0, ctypes.byref(nbytes)), "too many elements")
    assert lib.hmc_group_norm_workspace(None, 4, 0, ctypes.byref(nbytes)) == ffi.HMC_INVALID
    assert lib.hmc_group_norm_workspace(t, 5, 0, ctypes.byref(nbytes)) == ffi.HMC_INVALID
    # sizes alone decide: a description without memory is enough
    assert lib.hmc_group_norm_workspace(desc([2, 3000000, 8], data=False), 4, 0, ctypes.byref(nbytes)) == ffi.HMC_OK and nbytes.value == need


def test_group_norm_backward_refusals():
    lib = homura_b200.load()
    t, stat, par = desc([2, 3, 8]), desc([2, 4]), desc([8])
    ws = (HOST.ctypes.data + 15) // 16 * 16

    def call(dsrc=t, dweight=None, dbias=None, src=t, dout=t, mean=stat, rstd=stat, weight=None, bias=None, groups=4,
             act=ffi.HMC_ACTIVATION_NONE, ws=ws, n=1 << 15):
        return lib.hmc_group_norm_backward(None, dsrc, dweight, dbias, src, dout, mean, rstd, weight, bias, groups, act, ws, n)

    refused(call(), "null context")
    refused(call(dweight=par, dbias=par, weight=par, bias=par), "null context")
    refused(call(dweight=par), "null context")
    refused(call(mean=None), "need mean and rstd")
    refused(call(dout=desc([2, 3, 8], strides=[24, 1, 3])), "not channels last")
    refused(call(dout=desc([2, 4, 8])), "the output's gradient has the wrong sizes")
    refused(call(dsrc=None), "null description")
    refused(call(dweight=desc([8], F16)), "neither the input's dtype nor F32")
    refused(call(dweight=desc([8], F64), weight=par, bias=par), "the weight's gradient has the wrong dtype")
    refused(call(dbias=desc([8], strides=[0])), "not distinct")
    refused(call(n=0), "group norm needs")
    refused(call(act=99), "activation")


def test_dropout_refusals():
    lib = homura_b200.load()
    t = desc([24])

    def call(out=t, src=t, residual=None, p=0.5, seed=1, offset=0):
        return lib.hmc_dropout(None, out, src, residual, p, seed, offset)

    refused(call(), "null context")
    refused(call(residual=t), "null context")
    for p in (-0.1, 1.1, float("nan"), float("inf")):
        refused(call(p=p), "between 0 and 1")
    refused(call(src=desc([24], I32)), "floating point")
    refused(call(out=desc([23])), "the output has the wrong sizes")
    refused(call(out=desc([24], BF16)), "the output has the wrong dtype")
    refused(call(out=desc([24], strides=[0])), "not distinct")
    refused(call(residual=desc([2, 12])), "the residual needs 1 dimensions")
    refused(call(src=None), "null description")
    refused(call(src=desc([24], data=False)), "null data pointer")
    wide = desc([2] * 25)
    wide.ndim = 26
    refused(call(src=wide, out=wide), "26 dimensions")


def test_the_glue_refuses_what_it_cannot_describe():
    fake = lambda shape, strides=None: TensorData(Storage(16, array=HOST), F32, tuple(shape), tuple(strides or contiguous_strides(shape)))
    d = channels_last_desc("group_norm", fake([2, 3, 4, 8]))
    assert d.ndim == 3 and list(d.sizes[:3]) == [2, 12, 8] and list(d.strides[:3]) == [96, 8, 1]
    d = channels_last_desc("group_norm", fake([5, 8]))
    assert d.ndim == 3 and list(d.sizes[:3]) == [5, 1, 8] and d.strides[0] == 8
    d = channels_last_desc("group_norm", fake([2, 1, 1, 8]))
    assert list(d.sizes[:3]) == [2, 1, 8]
    d = channels_last_desc("group_norm", fake([2, 0, 4, 8]))
    assert list(d.sizes[:3]) == [2, 0, 8]
    with pytest.raises(BackendError, match="not evenly spaced"):
        channels_last_desc("group_norm", fake([2, 3, 4, 8], [1000, 100, 8, 1]))
    with pytest.raises(BackendError, match="needs"):
        channels_last_desc("group_norm", fake([8]))
    assert plain_desc("x", None) is None
    assert [activation_code(a) for a in ACTIVATIONS] == [-1, 3, 15, 16, 17]
    with pytest.raises(BackendError, match="activation"):
        activation_code("tanh")
    assert recurrence_flags(True, False, True) == 5 and recurrence_flags(False, True, False) == 2


def test_every_declared_symbol_of_the_layers_is_exported():
    import re
    from pathlib import Path
    text = (Path(__file__).resolve().parent.parent / "include" / "homura_cuda_layers.h").read_text()
    names = sorted(set(re.findall(r"\b(hmc_\w+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S))))
    assert names == ["hmc_dropout", "hmc_group_norm", "hmc_group_norm_backward", "hmc_group_norm_workspace",
                     "hmc_linear_recurrence", "hmc_linear_recurrence_backward"]
    for n in names:
        assert hasattr(homura_b200.load(), n) and n in ffi.FUNCTIONS


def test_positions_in_another_order_are_refused():
    """[2, 4, 6, 8] and [2, 6, 4, 8] both have 24 positions; they are not the same ones. The positions in one dimension, or with
    dimensions of 1 between them, are."""
    fake = lambda *shape: TensorData(Storage(16, array=HOST), F32, shape, contiguous_strides(shape))
    maps, turned = fake(2, 4, 6, 8), fake(2, 6, 4, 8)
    be, stats = object.__new__(CudaBackend), fake(2, 4)  # (refused before the backend is looked at)
    with pytest.raises(BackendError, match="shapes"):
        be.group_norm(turned, maps, 4)
    with pytest.raises(BackendError, match="shapes"):
        be.group_norm_backward(turned, maps, maps, stats, stats, 4)
    with pytest.raises(BackendError, match="shapes"):
        be.group_norm_backward(maps, maps, turned, stats, stats, 4)
    check_positions("group_norm", maps, maps, fake(2, 24, 8), fake(2, 4, 1, 6, 8))
    check_positions("group_norm", fake(2, 8), fake(2, 1, 8))


def test_a_refused_dropout_leaves_the_generator_where_it_was():
    """Nothing was drawn, so the next call's mask is the one it would have had."""
    fake = lambda shape, dtype=F32: TensorData(Storage(16, array=HOST), dtype, shape, contiguous_strides(shape))
    be = object.__new__(CudaBackend)  # (a context that is null: the library refuses every call)
    be.lib, be.ctx = homura_b200.load(), None
    gen = Generator(7)
    gen.reserve(5)
    for shape, p in (((3, 5), 0.5), ((3, 5), 2.0), ((0,), 0.5)):
        with pytest.raises(BackendError):
            be.dropout(fake(shape), fake(shape), gen, p)
        assert gen.offset == 5
    with pytest.raises(BackendError, match="wrong sizes"):
        be.dropout(fake((4,)), fake((5,)), gen, 0.5)
    assert gen.offset == 5
    first = gen.reserve(3)
    gen.reserve(1)
    gen.give_back(first, 3)  # another call has drawn since: what it drew stays its own
    assert gen.offset == 9

"""What is measured of the sequence block's operators: the gated linear recurrence, group norm with an activation
(channels last) and dropout from the counter-based generator, each in its forward and its backward direction.

``run`` computes a case in its plain form (elementary torch operations in f32, sums in f64) or, with ``own``, through
:class:`homura_b200.host.CudaBackend`; ``exact`` computes it in f64 by another route (the recurrence step by step, the
moments by their definition, the generator in 16-bit limbs).
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-5
_backend = None


def listed():
    return [
        # one token of 64 sequences that are being generated: the state goes in and comes out, latency counts
        {"name": "recurrence token", "op": "recurrence", "backward": False, "dtype": "bf16", "b": 64, "t": 1, "d": 4096,
         "sigmoid": True, "complement": True, "state": True, "packed": True},
        # a training batch: gate logits and inputs are the two halves of one projection
        {"name": "recurrence batch", "op": "recurrence", "backward": False, "dtype": "bf16", "b": 8, "t": 2048, "d": 4096,
         "sigmoid": True, "complement": True, "state": False, "packed": True},
        # one long sequence of odd sizes, continued from a state: little parallel work but along the time axis
        {"name": "recurrence long", "op": "recurrence", "backward": False, "dtype": "f32", "b": 1, "t": 65521, "d": 1000,
         "sigmoid": False, "complement": False, "state": True, "packed": False},
        # gradients of the training batch
        {"name": "recurrence backward", "op": "recurrence", "backward": True, "dtype": "bf16", "b": 4, "t": 4096, "d": 2048,
         "sigmoid": True, "complement": True, "state": False, "packed": True},
        # gradients at sizes that no vector divides
        {"name": "recurrence backward odd", "op": "recurrence", "backward": True, "dtype": "f32", "b": 3, "t": 5003, "d": 1001,
         "sigmoid": False, "complement": False, "state": True, "packed": False},
        # feature maps of an image model, 64 x 64 positions, ten channels a group
        {"name": "group norm maps", "op": "group_norm", "backward": False, "dtype": "f16", "n": 16, "s": 4096, "c": 320, "g": 32,
         "activation": "silu", "affine": True},
        # gradients of a deeper layer's maps
        {"name": "group norm maps backward", "op": "group_norm", "backward": True, "dtype": "bf16", "n": 16, "s": 1024, "c": 640,
         "g": 32, "activation": "silu", "affine": True},
        # every token of a sequence model by itself, a group per head of 128 channels
        {"name": "group norm tokens", "op": "group_norm", "backward": False, "dtype": "bf16", "n": 32768, "s": 1, "c": 4096,
         "g": 32, "activation": "none", "affine": True},
        # gradients of the same in f32
        {"name": "group norm tokens backward", "op": "group_norm", "backward": True, "dtype": "f32", "n": 16384, "s": 1, "c": 4096,
         "g": 16, "activation": "gelu", "affine": True},
        # the last layer of a small classifier
        {"name": "dropout small", "op": "dropout", "backward": False, "dtype": "f32", "rows": 32, "cols": 1001, "p": 0.5,
         "residual": False},
        # the residual sum behind a block, training batch
        {"name": "dropout residual", "op": "dropout", "backward": False, "dtype": "bf16", "rows": 16384, "cols": 4096, "p": 0.1,
         "residual": True},
        # its gradient at odd sizes
        {"name": "dropout backward odd", "op": "dropout", "backward": True, "dtype": "f16", "rows": 8191, "cols": 8193, "p": 0.25,
         "residual": False},
    ]


def _log_int(rng, low, high):
    """An integer of [low, high], spread over the logarithm; every third a multiple of 8 where there is one."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))
    if rng.random() < 0.33 and v >= 8:
        v -= v % 8
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(["recurrence", "group_norm", "dropout"])
    dtype = rng.choice(["f16", "bf16", "f32"])
    backward = rng.random() < 0.5
    most = 32_000_000  # elements of a tensor: no more bytes than the largest listed case
    if op == "recurrence":
        t = _log_int(rng, 1, 65536)
        d = _log_int(rng, 1, min(8192, most // t))
        b = _log_int(rng, 1, max(1, min(64, most // (t * d))))
        sigmoid = rng.random() < 0.6
        return {"op": op, "backward": backward, "dtype": dtype, "b": b, "t": t, "d": d, "sigmoid": sigmoid,
                "complement": rng.random() < 0.5, "state": rng.random() < 0.5, "packed": rng.random() < 0.5}
    if op == "group_norm":
        g = rng.choice([1, 2, 3, 4, 6, 8, 16, 32, 64])
        c = g * _log_int(rng, 1, 8192 // g)
        s = 1 if rng.random() < 0.35 else _log_int(rng, 2, min(16384, most // c))
        n = _log_int(rng, 1, max(1, min(32768, most // (s * c))))
        return {"op": op, "backward": backward, "dtype": dtype, "n": n, "s": s, "c": c, "g": g,
                "activation": rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]), "affine": rng.random() < 0.8}
    cols = _log_int(rng, 1, 16384)
    rows = _log_int(rng, 1, max(1, most // cols))
    return {"op": op, "backward": backward, "dtype": dtype, "rows": rows, "cols": cols, "p": round(rng.uniform(0.0, 0.9), 3),
            "residual": (not backward) and rng.random() < 0.5}


# ---- inputs ----

def _normal(gen, shape, dtype, mean=0.0, std=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(std).add_(mean).to(dtype)


def _uniform(gen, shape, low, high):
    return torch.rand(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(high - low).add_(low)


def _two(case, shape, dtype, make_first, make_second):
    """Two tensors of `shape`, as the halves of one buffer's last dimension where the case packs them."""
    first, second = make_first().to(dtype), make_second().to(dtype)
    if not case["packed"]:
        return first, second
    both = torch.cat([first, second], -1)
    return both[..., :shape[-1]], both[..., shape[-1]:]


def _empty_two(case, shape, dtype):
    if not case["packed"]:
        return torch.empty(shape, dtype=dtype, device="cuda"), torch.empty(shape, dtype=dtype, device="cuda")
    both = torch.empty(shape[:-1] + (2 * shape[-1],), dtype=dtype, device="cuda")
    return both[..., :shape[-1]], both[..., shape[-1]:]


def _prepare_recurrence(case, gen, s):
    dtype, shape = DTYPES[case["dtype"]], (case["b"], case["t"], case["d"])
    if case["sigmoid"]:   # logits of gates that forget over one to some hundred steps
        gates = lambda: _normal(gen, shape, torch.float32, 2.0, 1.5)
    else:                 # decays in (0, 1), now and then a reset
        gates = lambda: _uniform(gen, shape, 0.6, 1.0) * (_uniform(gen, shape, 0.0, 1.0) > 0.002)
    s["gate"], s["x"] = _two(case, shape, dtype, gates, lambda: _normal(gen, shape, torch.float32))
    if case["state"]:
        s["initial"] = _normal(gen, (shape[0], shape[2]), torch.float32)
    if case["backward"]:
        s["out"] = _plain_recurrence(case, s)[0]
        s["dout"] = _normal(gen, shape, dtype)
        if case["state"]:
            s["dlast"] = _normal(gen, (shape[0], shape[2]), torch.float32)
    if own:
        if case["backward"]:
            s["to_dgate"], s["to_dx"] = _empty_two(case, shape, dtype)
        else:
            s["to_out"] = torch.empty(shape, dtype=dtype, device="cuda")
        if case["state"]:
            s["to_state"] = torch.empty((shape[0], shape[2]), dtype=torch.float32, device="cuda")


def _prepare_group_norm(case, gen, s):
    dtype, shape, c = DTYPES[case["dtype"]], (case["n"], case["s"], case["c"]), case["c"]
    # activations whose channels have offsets and spreads of their own
    s["src"] = (_normal(gen, shape, torch.float32) * _uniform(gen, (c,), 0.5, 2.0) + _normal(gen, (c,), torch.float32, 0.5, 0.5)).to(dtype)
    if case["affine"]:
        s["weight"] = _normal(gen, (c,), dtype, 1.0, 0.2)
        s["bias"] = _normal(gen, (c,), dtype, 0.0, 0.2)
    if case["backward"]:
        s["mean"], s["rstd"] = (v.float() for v in _plain_moments(case, s))
        s["dout"] = _normal(gen, shape, dtype)
    if own:
        s["to_" + ("dsrc" if case["backward"] else "out")] = torch.empty(shape, dtype=dtype, device="cuda")
        if case["backward"] and case["affine"]:
            s["to_dweight"], s["to_dbias"] = (torch.empty((c,), dtype=dtype, device="cuda") for _ in range(2))
        if not case["backward"]:
            s["to_mean"], s["to_rstd"] = (torch.empty((case["n"], case["g"]), dtype=torch.float32, device="cuda") for _ in range(2))


def _prepare_dropout(case, gen, s, seed):
    dtype, shape = DTYPES[case["dtype"]], (case["rows"], case["cols"])
    s["src"] = _normal(gen, shape, dtype)
    if case["residual"]:
        s["residual"] = _normal(gen, shape, dtype)
    # the generator's seed and the blocks it has handed out before this call
    s["seed"], s["offset"] = (seed * 0x9E3779B97F4A7C15 + 11) % 2**64, (seed * 977) % 2**40
    if own:
        s["to_out"] = torch.empty(shape, dtype=dtype, device="cuda")


def prepare(case, seed):
    global _backend
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {}
    if case["op"] == "recurrence":
        _prepare_recurrence(case, gen, s)
    elif case["op"] == "group_norm":
        _prepare_group_norm(case, gen, s)
    else:
        _prepare_dropout(case, gen, s, seed)
    state = {"case": case, "torch": s}
    if own:
        from homura_b200 import host
        if _backend is None:
            _backend = host.CudaBackend(torch.cuda.current_device())
        codes = {torch.float16: host.F16, torch.bfloat16: host.BF16, torch.float32: host.F32}
        state["own"] = {k: host.TensorData(host.Storage(v.untyped_storage().nbytes(), ptr=v.untyped_storage().data_ptr(),
                                                        device=_backend.device, owner=v),
                                           codes[v.dtype], tuple(v.shape), tuple(v.stride()), v.storage_offset())
                        for k, v in s.items() if isinstance(v, torch.Tensor)}
        if case["op"] == "dropout":
            generator = host.Generator(s["seed"])
            generator.offset = s["offset"]
            state["generator"] = generator
        torch.cuda.synchronize()  # the backend works on a stream of its own
    return state


# ---- the framework's calls ----

def _own_recurrence(case, state):
    t, s = state["own"], state["torch"]
    flags = {"sigmoid": case["sigmoid"], "complement": case["complement"]}
    if case["backward"]:
        _backend.linear_recurrence_backward(t["to_dgate"], t["to_dx"], t["gate"], t["x"], t["out"], t["dout"],
                                            initial=t.get("initial"), dlast=t.get("dlast"), dinitial=t.get("to_state"), **flags)
        outputs = [s["to_dgate"], s["to_dx"]]
    else:
        _backend.linear_recurrence(t["to_out"], t["gate"], t["x"], initial=t.get("initial"), last=t.get("to_state"), **flags)
        outputs = [s["to_out"]]
    return outputs + ([s["to_state"]] if case["state"] else [])


def _own_group_norm(case, state):
    t, s = state["own"], state["torch"]
    activation = None if case["activation"] == "none" else case["activation"]
    if case["backward"]:
        _backend.group_norm_backward(t["to_dsrc"], t["src"], t["dout"], t["mean"], t["rstd"], case["g"], weight=t.get("weight"),
                                     bias=t.get("bias"), dweight=t.get("to_dweight"), dbias=t.get("to_dbias"), activation=activation)
        return [s["to_dsrc"]] + ([s["to_dweight"], s["to_dbias"]] if case["affine"] else [])
    _backend.group_norm(t["to_out"], t["src"], case["g"], weight=t.get("weight"), bias=t.get("bias"), mean=t["to_mean"],
                        rstd=t["to_rstd"], eps=EPS, activation=activation)
    return [s["to_out"], s["to_mean"], s["to_rstd"]]


def _own_dropout(case, state):
    t, s, generator = state["own"], state["torch"], state["generator"]
    if case["backward"]:
        _backend.dropout_backward(t["to_out"], t["src"], case["p"], (s["seed"], s["offset"]))
    else:
        generator.offset = s["offset"]
        _backend.dropout(t["to_out"], t["src"], generator, case["p"], residual=t.get("residual"))
    return [s["to_out"]]


# ---- plain forms ----

def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 1, by doubling."""
    step, t = 1, a.shape[1]
    while step < t:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


def _plain_gates(case, s):
    gate, x = s["gate"].float(), s["x"].float()
    if not case["sigmoid"]:
        return gate, (1.0 - gate if case["complement"] else None), x
    e = torch.exp(-gate.abs())
    small, large = e / (1.0 + e), 1.0 / (1.0 + e)
    a, rest = torch.where(gate > 0, large, small), torch.where(gate > 0, small, large)
    return a, rest, x


def _plain_recurrence(case, s):
    a, rest, x = _plain_gates(case, s)
    u = rest * x if case["complement"] else x
    if case["state"]:
        u = torch.cat([u[:, :1] + a[:, :1] * s["initial"][:, None], u[:, 1:]], 1)
    h = _scan(a, u)
    return [h.to(s["gate"].dtype)] + ([h[:, -1]] if case["state"] else [])


def _plain_recurrence_backward(case, s):
    a, rest, x = _plain_gates(case, s)
    dout, out = s["dout"].float(), s["out"].float()
    if case["state"]:
        dout = torch.cat([dout[:, :-1], dout[:, -1:] + s["dlast"][:, None]], 1)
    first = s["initial"][:, None] if case["state"] else torch.zeros_like(out[:, :1])
    before = torch.cat([first, out[:, :-1]], 1)
    following = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    g = _scan(following.flip(1), dout.flip(1)).flip(1)
    dgate = g * (before - x) if case["complement"] else g * before
    if case["sigmoid"]:
        dgate = dgate * a * rest
    dx = g * rest if case["complement"] else g
    return [dgate.to(s["gate"].dtype), dx.to(s["gate"].dtype)] + ([a[:, 0] * g[:, 0]] if case["state"] else [])


def _plain_moments(case, s):
    x = s["src"].view(case["n"], case["s"], case["g"], -1).double()
    mean = x.mean((1, 3), keepdim=True)
    var = (x - mean).square().mean((1, 3))
    return mean[:, 0, :, 0], 1.0 / torch.sqrt(var + EPS)


def _plain_activation(kind, z):
    """(activation, its derivative) of z."""
    if kind == "relu":
        return z.clamp_min(0.0), (z > 0).to(z.dtype)
    if kind == "silu":
        sig = 1.0 / (1.0 + torch.exp(-z))
        return z * sig, sig * (1.0 + z * (1.0 - sig))
    if kind == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if kind == "gelu_tanh":
        k = math.sqrt(2.0 / math.pi)
        t = torch.tanh(k * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * k * (1.0 + 3 * 0.044715 * z * z)
    return z, torch.ones_like(z)


def _plain_normalised(case, s, mean, rstd):
    x = s["src"].view(case["n"], case["s"], case["g"], -1).float()
    xhat = ((x - mean[:, None, :, None]) * rstd[:, None, :, None]).view(case["n"], case["s"], -1)
    return xhat, (xhat * s["weight"].float() + s["bias"].float() if case["affine"] else xhat)


def _plain_group_norm(case, s):
    mean, rstd = (v.float() for v in _plain_moments(case, s))
    z = _plain_normalised(case, s, mean, rstd)[1]
    return [_plain_activation(case["activation"], z)[0].to(s["src"].dtype), mean, rstd]


def _plain_group_norm_backward(case, s):
    xhat, z = _plain_normalised(case, s, s["mean"], s["rstd"])
    dz = s["dout"].float() * _plain_activation(case["activation"], z)[1]
    p = dz * s["weight"].float() if case["affine"] else dz
    p, x = (v.view(case["n"], case["s"], case["g"], -1) for v in (p, xhat))
    m1 = p.mean((1, 3), keepdim=True, dtype=torch.float64).float()
    m2 = (p * x).mean((1, 3), keepdim=True, dtype=torch.float64).float()
    dsrc = (s["rstd"][:, None, :, None] * (p - m1 - x * m2)).view(s["src"].shape)
    out = [dsrc.to(s["src"].dtype)]
    if case["affine"]:
        out += [(dz * xhat).sum((0, 1), dtype=torch.float64).to(s["weight"].dtype), dz.sum((0, 1), dtype=torch.float64).to(s["bias"].dtype)]
    return out


def _plain_words(n, seed, offset):
    """The first n 32-bit words of the Philox4x32-10 blocks from `offset` on under `seed`, as int64."""
    low = 0xFFFFFFFF
    block = torch.arange(-(-n // 4), dtype=torch.int64, device="cuda") + offset
    c0, c1 = block & low, (block >> 32) & low
    c2, c3 = torch.zeros_like(c0), torch.zeros_like(c0)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # the low 64 bits, whatever their sign
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], 1).view(-1)[:n]


def _plain_dropout(case, s):
    x = s["src"].float()
    keep = (_plain_words(x.numel(), s["seed"], s["offset"]) >= round(case["p"] * 2.0**32)).view(x.shape)
    y = torch.where(keep, x * (1.0 / (1.0 - case["p"])), 0.0)
    if case["residual"]:
        y = s["residual"].float() + y
    return [y.to(s["src"].dtype)]


def run(state):
    case, s = state["case"], state["torch"]
    if own:
        if case["op"] == "recurrence":
            return _own_recurrence(case, state)
        if case["op"] == "group_norm":
            return _own_group_norm(case, state)
        return _own_dropout(case, state)
    if case["op"] == "recurrence":
        return _plain_recurrence_backward(case, s) if case["backward"] else _plain_recurrence(case, s)
    if case["op"] == "group_norm":
        return _plain_group_norm_backward(case, s) if case["backward"] else _plain_group_norm(case, s)
    return _plain_dropout(case, s)


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "recurrence":
        n, states = case["b"] * case["t"] * case["d"], 4 * case["b"] * case["d"] if case["state"] else 0
        if case["backward"]:  # gate, out, dout (and x) in, dgate and dx out; initial, dlast, dinitial
            return {"bytes": (6 if case["complement"] else 5) * n * es + 3 * states,
                    "flops": n * (4 + 5 * case["sigmoid"] + 3 * case["complement"])}
        return {"bytes": 3 * n * es + 2 * states, "flops": n * (2 + 3 * case["sigmoid"] + 2 * case["complement"])}
    if case["op"] == "group_norm":
        n, c, stats = case["n"] * case["s"] * case["c"], case["c"] * es * 2 * case["affine"], 8 * case["n"] * case["g"]
        act = 0 if case["activation"] == "none" else 5
        if case["backward"]:
            return {"bytes": 3 * n * es + 2 * c + stats, "flops": n * (16 + 2 * act)}
        return {"bytes": 2 * n * es + c + stats, "flops": n * (9 + act)}
    n = case["rows"] * case["cols"]
    return {"bytes": (3 if case["residual"] else 2) * n * es, "flops": 2 * n}


# ---- the definitions in 64 bits ----

def _exact_recurrence(case, s):
    gate, x = s["gate"].double(), s["x"].double()
    a = torch.sigmoid(gate) if case["sigmoid"] else gate
    rest = torch.sigmoid(-gate) if case["sigmoid"] else 1.0 - gate
    t = case["t"]
    start = s["initial"].double() if case["state"] else torch.zeros_like(x[:, 0])
    if not case["backward"]:
        u = (rest * x if case["complement"] else x).transpose(0, 1).contiguous()
        at = a.transpose(0, 1).contiguous()
        out, h = torch.empty_like(u), start
        for k in range(t):
            h = torch.addcmul(u[k], at[k], h, out=out[k])
        return [out.transpose(0, 1)] + ([h.clone()] if case["state"] else [])
    at, up = a.transpose(0, 1).contiguous(), s["dout"].double().transpose(0, 1).contiguous()
    if case["state"]:
        up[t - 1] += s["dlast"].double()
    for k in range(t - 2, -1, -1):
        up[k].addcmul_(at[k + 1], up[k + 1])
    g = up.transpose(0, 1)
    da = torch.empty_like(a)
    da[:, 0] = g[:, 0] * start
    da[:, 1:] = g[:, 1:] * s["out"][:, :-1].double()
    du = g
    if case["complement"]:
        da, du = da - g * x, g * rest
    if case["sigmoid"]:
        da = da * (a * rest)
    return [da, du] + ([a[:, 0] * g[:, 0]] if case["state"] else [])


def _exact_group_norm(case, s):
    shape = (case["n"], case["s"], case["g"], case["c"] // case["g"])
    n = shape[1] * shape[3]
    x = s["src"].double().view(shape)
    w = s["weight"].double() if case["affine"] else torch.ones(case["c"], dtype=torch.float64, device=x.device)
    b = s["bias"].double() if case["affine"] else torch.zeros_like(w)
    w, b = w.view(shape[2:]), b.view(shape[2:])
    if case["backward"]:
        mean, rstd = s["mean"].double(), s["rstd"].double()
    else:
        mean = x.sum(3).sum(1) / n
        rstd = ((x - mean[:, None, :, None]).pow(2).sum(3).sum(1) / n + EPS).rsqrt()
    xhat = (x - mean[:, None, :, None]) * rstd[:, None, :, None]
    z = xhat * w + b
    kind = case["activation"]
    if not case["backward"]:
        if kind == "relu":
            z = torch.relu(z)
        elif kind != "none":
            z = torch.nn.functional.silu(z) if kind == "silu" else torch.nn.functional.gelu(z, approximate="tanh" if kind == "gelu_tanh" else "none")
        return [z.reshape(s["src"].shape), mean, rstd]
    dz = s["dout"].double().view(shape)
    if kind == "relu":
        dz = dz * (z > 0)
    elif kind != "none":
        with torch.enable_grad():
            leaf = z.detach().requires_grad_()
            y = torch.nn.functional.silu(leaf) if kind == "silu" else torch.nn.functional.gelu(leaf, approximate="tanh" if kind == "gelu_tanh" else "none")
            dz, = torch.autograd.grad(y, leaf, dz)
    p = dz * w
    s1, s2 = p.sum(3).sum(1) / n, (p * xhat).sum(3).sum(1) / n
    dsrc = rstd[:, None, :, None] * (p - s1[:, None, :, None] - xhat * s2[:, None, :, None])
    return [dsrc.reshape(s["src"].shape)] + ([(dz * xhat).sum(1).sum(0).reshape(-1), dz.sum(1).sum(0).reshape(-1)] if case["affine"] else [])


def _exact_mul(constant, v):
    """(high, low) 32-bit halves of constant * v in limbs of 16 bits."""
    m = 0xFFFF
    a0, a1, b0, b1 = constant & m, constant >> 16, v & m, v >> 16
    t = a0 * b0
    mid = a1 * b0 + (t >> 16)
    other = a0 * b1 + (mid & m)
    return a1 * b1 + (mid >> 16) + (other >> 16), ((other & m) << 16) | (t & m)


def _exact_dropout(case, s):
    x = s["src"].double().view(-1)
    blocks = torch.arange((x.numel() + 3) // 4, device="cuda", dtype=torch.int64) + s["offset"]
    c = [blocks % 2**32, blocks // 2**32, torch.zeros_like(blocks), torch.zeros_like(blocks)]
    for r in range(10):
        key = ((s["seed"] % 2**32 + r * 0x9E3779B9) % 2**32, (s["seed"] // 2**32 + r * 0xBB67AE85) % 2**32)
        h0, l0 = _exact_mul(0xD2511F53, c[0])
        h1, l1 = _exact_mul(0xCD9E8D57, c[2])
        c = [h1 ^ c[1] ^ key[0], l1, h0 ^ c[3] ^ key[1], l0]
    words = torch.empty((blocks.numel(), 4), dtype=torch.int64, device="cuda")
    for j in range(4):
        words[:, j] = c[j]
    kept = words.view(-1)[:x.numel()].double() / 2.0**32 >= round(case["p"] * 2.0**32) / 2.0**32
    y = torch.zeros_like(x)
    y[kept] = x[kept] / (1.0 - case["p"])
    if case["residual"]:
        y += s["residual"].double().view(-1)
    return [y.view(s["src"].shape)]


def exact(case, seed):
    s = prepare(case, seed)["torch"]
    if case["op"] == "recurrence":
        return _exact_recurrence(case, s)
    if case["op"] == "group_norm":
        return _exact_group_norm(case, s)
    return _exact_dropout(case, s)

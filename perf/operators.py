"""Measured cases of the 8-bit operators: a linear layer on 8-bit integers with a scale for each token and channel,
the root-mean-square norm that feeds it, activation checkpoints in 8 bits, and the weight gradient taken from them.

Matrices of tokens are held a token after the other (``[tokens, features]``, row pitch ``ld`` elements), weights a
channel after the other; an 8-bit row ``q`` with its scale ``s`` stands for the values ``s * q``.

  linear      y[t, n]  = sx[t] * sw[n] * sum_k qx[t, k] * qw[n, k]  (+ bias[n])
  norm        h = x + r (FP32, also written back rounded to x's type),  p = h * g (FP32),  P = max_k |p|,
              q = round(127 p / P),  s = P * rsqrt(mean_k h^2 + eps) / 127
  checkpoint  P = max_k |x|;  s = P / 127, or the least power of two with 127 s >= P;  q = round(x / s); then the values
              s * q again, rounded to x's type, as a backward pass reads them
  wgrad       dw[n, k] = c[n, k] + sum_t dy[t, n] * s[t] * q[t, k]

Roundings to 8 bits go to the nearest, halves to the even; a row of zeros has s = 0 and q = 0.
"""
import importlib
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


# ------------------------------------------------------------------------------------------------------------ cases
def _linear(name, tokens, channels, features, dtype, bias, ld_extra=0):
    return {"name": name, "op": "linear", "tokens": tokens, "channels": channels, "features": features, "dtype": dtype,
            "bias": bias, "ld_extra": ld_extra}


def _norm(name, tokens, features, dtype, residual):
    return {"name": name, "op": "norm", "tokens": tokens, "features": features, "dtype": dtype, "residual": residual}


def _checkpoint(name, tokens, features, dtype, pow2):
    return {"name": name, "op": "checkpoint", "tokens": tokens, "features": features, "dtype": dtype, "pow2": pow2}


def _wgrad(name, tokens, channels, features, dtype, out, accumulate):
    return {"name": name, "op": "wgrad", "tokens": tokens, "channels": channels, "features": features, "dtype": dtype,
            "out": out, "accumulate": accumulate}


def listed():
    return [
        # one token through a square projection: reads the weights and little else, latency counts
        _linear("linear_1_token", 1, 4096, 4096, "bf16", False),
        # a batch of sequences that decode together, an output width and a feature count that fill no tile
        _linear("linear_23_tokens", 23, 8200, 8190, "fp16", True, ld_extra=32),
        # a short prompt: too few tiles for the whole device without a finer cut
        _linear("linear_short_prompt", 509, 4096, 4096, "bf16", True),
        # a long prompt or a large batch: bound by the matrix product
        _linear("linear_long_prompt", 8192, 8192, 8192, "bf16", False),
        # the norm in front of a projection while a few sequences decode
        _norm("norm_5_tokens", 5, 4100, "fp16", True),
        # the same over a long prompt: bound by memory
        _norm("norm_long_prompt", 8192, 8192, "bf16", True),
        # a checkpoint of a small ragged activation with the finest scale
        _checkpoint("checkpoint_small", 37, 1001, "fp32", False),
        # a checkpoint of a layer's activations, restored for the backward pass
        _checkpoint("checkpoint_layer", 16384, 4096, "bf16", True),
        # few tokens: the gradient itself is most of the traffic
        _wgrad("wgrad_77_tokens", 77, 2048, 2048, "fp16", "fp16", False),
        # a small layer over many tokens: the sum over tokens has to be cut
        _wgrad("wgrad_small_layer", 16384, 1000, 1024, "bf16", "bf16", False),
        # a layer's gradient, added to the FP32 gradient kept over micro-batches
        _wgrad("wgrad_layer", 8192, 4096, 4096, "bf16", "fp32", True),
        # a wide layer, ragged in every direction
        _wgrad("wgrad_wide", 4099, 11001, 4104, "bf16", "bf16", False),
    ]


def _size(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]; every other one as it falls, the others multiples of 64."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and hi >= 64:
        n = max(64, n // 64 * 64)
    return max(lo, min(hi, n))


def draw(rng):
    op = rng.choice(["linear", "norm", "checkpoint", "wgrad"])
    if op == "linear":
        return {"op": op, "tokens": _size(rng, 1, 8192), "channels": _size(rng, 256, 8192), "features": _size(rng, 256, 8192),
                "dtype": rng.choice(["bf16", "fp16", "fp32"]), "bias": rng.random() < 0.5, "ld_extra": rng.choice([0, 0, 16, 128])}
    if op == "norm":
        return {"op": op, "tokens": _size(rng, 1, 8192), "features": _size(rng, 256, 8192),
                "dtype": rng.choice(["bf16", "fp16", "fp32"]), "residual": rng.random() < 0.7}
    if op == "checkpoint":
        return {"op": op, "tokens": _size(rng, 16, 16384), "features": _size(rng, 256, 8192),
                "dtype": rng.choice(["bf16", "fp16", "fp32"]), "pow2": rng.random() < 0.6}
    return {"op": op, "tokens": _size(rng, 16, 16384), "channels": _size(rng, 256, 4096), "features": _size(rng, 256, 4096),
            "dtype": rng.choice(["bf16", "fp16"]), "out": rng.choice(["bf16", "fp16", "fp32"]), "accumulate": rng.random() < 0.5}


# ----------------------------------------------------------------------------------------------------------- inputs
def _pitch(features, extra=0):
    """Row pitch of 8-bit matrices: whole 16-byte units, as a program that lays out its weights and buffers once takes it."""
    return (features + 15) // 16 * 16 + extra


def _activations(gen, tokens, features, dtype):
    """Normal values with a few channels far above the others and tokens of different size, as inside a network."""
    x = torch.randn(tokens, features, generator=gen, device="cuda")
    wide = torch.rand(features, generator=gen, device="cuda") < 0.004
    x = x * torch.where(wide, 12.0, 1.0) * torch.exp(0.5 * torch.randn(tokens, 1, generator=gen, device="cuda"))
    return x.to(dtype)


def _rows8(x, pitch, pow2=False):
    """8-bit rows of x with their scales, by the definition."""
    peak = x.double().abs().amax(1, keepdim=True)
    if pow2:
        s = torch.exp2(torch.ceil(torch.log2(peak / 127.0)))
        s = torch.where(127.0 * s / 2 >= peak, s / 2, torch.where(127.0 * s < peak, 2 * s, s))   # log2 next to a border
        q = torch.round(x.double() / s)
    else:
        s = peak / 127.0
        q = torch.round(127.0 * x.double() / peak)
    out = torch.zeros(x.shape[0], pitch, dtype=torch.int8, device=x.device)
    out[:, :x.shape[1]] = torch.nan_to_num(q).to(torch.int8)
    return out, s.reshape(-1).float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, t, k = case["op"], case["tokens"], case["features"]
    dtype = TYPES[case["dtype"]]
    state = {"op": op, "t": t, "k": k, "dtype": dtype}
    new = lambda *shape, of=dtype: torch.empty(*shape, dtype=of, device="cuda")   # noqa: E731
    if op == "linear":
        n, ld = case["channels"], _pitch(k, case["ld_extra"])
        qx, sx = _rows8(_activations(gen, t, k, torch.float32), ld)
        qw, sw = _rows8(0.02 * torch.randn(n, k, generator=gen, device="cuda"), ld)
        bias = torch.randn(n, generator=gen, device="cuda") if case["bias"] else None
        state.update(n=n, ld=ld, qx=qx, sx=sx, qw=qw, sw=sw, bias=bias, y=new(t, n))
    elif op == "norm":
        x = _activations(gen, t, k, dtype)
        r = (3.0 * _activations(gen, t, k, torch.float32)).to(dtype) if case["residual"] else None
        g = (1.0 + 0.2 * torch.randn(k, generator=gen, device="cuda")).to(dtype)
        state.update(x=x, r=r, g=g, h=new(t, k) if r is not None else None, ld=_pitch(k), values=new(t, k))
        state.update(q=new(t, state["ld"], of=torch.int8), s=new(t, of=torch.float32))
    elif op == "checkpoint":
        x = _activations(gen, t, k, dtype)
        state.update(x=x, pow2=case["pow2"], ld=_pitch(k), values=new(t, k))
        state.update(q=new(t, state["ld"], of=torch.int8), s=new(t, of=torch.float32))
    else:
        n, ld = case["channels"], _pitch(k)
        q, s = _rows8(_activations(gen, t, k, torch.bfloat16), ld, pow2=True)
        pitch = (n + 7) // 8 * 8
        dy = torch.zeros(t, pitch, dtype=dtype, device="cuda")
        dy[:, :n] = (0.01 * torch.randn(t, n, generator=gen, device="cuda")
                     * torch.exp(0.5 * torch.randn(t, 1, generator=gen, device="cuda"))).to(dtype)
        out = TYPES[case["out"]]
        c = (0.1 * torch.randn(n, k, generator=gen, device="cuda")).to(out) if case["accumulate"] else None
        state.update(n=n, ld=ld, pitch=pitch, q=q, s=s, dy=dy, c=c, dw=new(n, k, of=out), out=out)
    return state


# ------------------------------------------------------------------------------------------------------- plain forms
def _plain(state):
    k = state["k"]
    if state["op"] == "linear":
        y = (state["qx"][:, :k].float() @ state["qw"][:, :k].float().T) * state["sx"][:, None] * state["sw"]
        return (y if state["bias"] is None else y + state["bias"]).to(state["dtype"])
    if state["op"] == "norm":
        h = state["x"].float()
        if state["r"] is not None:
            h = h + state["r"].float()
        p = h * state["g"].float()
        peak = p.abs().amax(1, keepdim=True)
        q = torch.nan_to_num(torch.round(127.0 * p.double() / peak.double())).float()   # 64 bits: values next to a border
        s = peak * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) / 127.0
        values = (q * s).to(state["dtype"])
        return (values, s[:, 0]) if state["r"] is None else (values, s[:, 0], h.to(state["dtype"]))
    if state["op"] == "checkpoint":
        x = state["x"].float()
        peak = x.abs().amax(1, keepdim=True)
        if state["pow2"]:
            s = torch.exp2(torch.ceil(torch.log2(peak.double() / 127.0)))
            s = torch.where(127.0 * s / 2 >= peak, s / 2, torch.where(127.0 * s < peak, 2 * s, s)).float()
            q = torch.nan_to_num(torch.round(x / s))
        else:
            s = peak / 127.0
            q = torch.nan_to_num(torch.round(127.0 * x.double() / peak.double())).float()   # 64 bits: values next to a border
        return (q * s).to(state["dtype"]), s[:, 0]
    x = state["q"][:, :k].float() * state["s"][:, None]
    dw = state["dy"][:, :state["n"]].float().T @ x
    return (dw if state["c"] is None else dw + state["c"].float()).to(state["out"])


# ------------------------------------------------------------------------------------------------------- own kernels
_runners = {}


def _runner():
    """The handle of the 8-bit operators on the current device, opened once."""
    device = torch.cuda.current_device()
    if device not in _runners:
        importlib.import_module("amdgpu-arch-gemm_b200")
        import kernels
        from runner.api import SgemmRunner
        _runners[device] = SgemmRunner(*kernels.ensure(kernels.DEFAULT_I8), device)
    return _runners[device]


def _kernels(state):
    r, stream = _runner(), torch.cuda.current_stream().cuda_stream
    op, t, k, ld = state["op"], state["t"], state["k"], state["ld"]
    if op == "linear":
        r.i8_linear(state["qw"], state["sw"], state["qx"], state["sx"], state["y"], state["n"], t, k, bias=state["bias"],
                    ldw=ld, ldx=ld, stream=stream)
        return state["y"]
    if op == "norm":
        r.i8_rmsnorm(state["x"], state["g"], state["q"], state["s"], k, t, residual=state["r"], sum_out=state["h"], eps=EPS,
                     ldq=ld, stream=stream)
        r.i8_restore(state["q"], state["s"], state["values"], k, t, ldq=ld, stream=stream)
        return (state["values"], state["s"]) if state["r"] is None else (state["values"], state["s"], state["h"])
    if op == "checkpoint":
        r.i8_quantize(state["x"], state["q"], state["s"], k, t, pow2=state["pow2"], ldq=ld, stream=stream)
        r.i8_restore(state["q"], state["s"], state["values"], k, t, ldq=ld, stream=stream)
        return state["values"], state["s"]
    r.i8_wgrad(state["q"], state["s"], state["dy"], state["dw"], k, state["n"], t, c=state["c"],
               beta=0.0 if state["c"] is None else 1.0, ldq=ld, lddy=state["pitch"], stream=stream)
    return state["dw"]


def run(state):
    return _kernels(state) if own else _plain(state)


# -------------------------------------------------------------------------------------------------------------- work
def work(case):
    op, t, k, e = case["op"], case["tokens"], case["features"], 4 if case["dtype"] == "fp32" else 2
    if op == "linear":
        n = case["channels"]
        return {"bytes": t * k + n * k + 4 * (t + n) + t * n * e + (4 * n if case["bias"] else 0), "flops": 2 * t * n * k}
    if op == "norm":   # x (and r) read, q and its scales written, h written, the values q stands for written
        return {"bytes": t * k * (e + 1 + e + (2 * e if case["residual"] else 0)) + 4 * t + k * e, "flops": 8 * t * k}
    if op == "checkpoint":   # x read, q written for the time in between, read again, the values written
        return {"bytes": t * k * (e + 1 + 1 + e) + 8 * t, "flops": 4 * t * k}
    n, o = case["channels"], 4 if case["out"] == "fp32" else 2
    return {"bytes": t * k + 4 * t + t * n * e + n * k * o * (2 if case["accumulate"] else 1), "flops": 2 * t * n * k}


# ------------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """The definitions in 64 bits.  (The sum h and the product p of the norm are FP32 numbers by definition: what q is
    rounded from does not depend on the order of a sum.)"""
    st = prepare(case, seed)
    t, k = st["t"], st["k"]
    wide = torch.float64
    if st["op"] == "linear":
        y = torch.matmul(st["qx"].to(wide)[:, :k], st["qw"].to(wide)[:, :k].t())
        y = torch.einsum("tn,t,n->tn", y, st["sx"].to(wide), st["sw"].to(wide))
        return y if st["bias"] is None else y + st["bias"].to(wide)
    if st["op"] == "wgrad":
        dw = torch.matmul(st["dy"].to(wide)[:, :st["n"]].t(), st["q"].to(wide)[:, :k] * st["s"].to(wide).reshape(t, 1))
        return dw if st["c"] is None else dw + st["c"].to(wide)
    x = st["x"].to(wide)
    factor = torch.ones(t, 1, dtype=wide, device="cuda")
    if st["op"] == "norm":
        if st["r"] is not None:
            x = (x + st["r"].to(wide)).float().to(wide)
        factor = 1.0 / torch.sqrt((x * x).sum(1, keepdim=True) / k + EPS)
        total, x = x, (x * st["g"].to(wide)).float().to(wide)
    peak = x.abs().max(1, keepdim=True).values
    if st.get("pow2"):
        mantissa, exponent = torch.frexp(peak)              # peak = mantissa * 2^exponent, mantissa in [0.5, 1)
        step = torch.ldexp(torch.ones_like(peak), exponent - 7 + (mantissa > 127.0 / 128.0))
    else:
        step = peak / 127.0
    q = torch.where(peak > 0, x / torch.where(peak > 0, step, 1.0), 0.0)
    if not st.get("pow2"):
        q = torch.where(peak > 0, x * 127.0 / torch.where(peak > 0, peak, 1.0), 0.0)
    q = torch.round(q)
    s = step * factor
    if st["op"] == "norm" and st["r"] is not None:
        return q * s, s.reshape(-1), total
    return q * s, s.reshape(-1)

"""Workloads of the gated feed-forward and microscaled 4-bit operators, each with its plain form.

Operators:
  gated_linear            h = act(x Wg^T) * (x Wu^T)                 x [T, D], Wg and Wu [F, D], 16 bits
  gated_linear_backward   dx, dWg, dWu from dh                        nothing kept from the forward pass
  quantize_mxfp4 / dequantize_mxfp4   blocks of 32 values: E2M1 elements, one E8M0 scale (a power of two)
  linear_mxfp4            y = q(x) q(W)^T                             weights quantised once, x in the call
  gated_linear_mxfp4      h = act(q(x) q(Wg)^T) * (q(x) q(Wu)^T)      the same block served in 4 bits

`run` computes the plain form (elementary torch operations in 32 bits, one rounding at the end), or,
with `own` set, calls tenzor_b200.ops.  `exact` restates each definition in 64 bits.
"""
import math

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BLOCK = 32  # values that share one scale


# ---- the cases ---------------------------------------------------------------------------------------

def listed():
    return [
        # one token of a serving loop: the two weight matrices are read once, latency counts
        {"name": "gated one token", "op": "gated", "dtype": "bf16", "act": "silu", "T": 1, "D": 2048, "F": 6144},
        # the packed tokens of the framework's default encoder batch at its own widths (384 -> 1536)
        {"name": "gated encoder batch", "op": "gated", "dtype": "f16", "act": "gelu", "T": 18106, "D": 384, "F": 1536},
        # a long prompt or a training batch of a wide model: bound by the matrix products
        {"name": "gated long", "op": "gated", "dtype": "bf16", "act": "silu", "T": 8192, "D": 4096, "F": 8192},
        # a small fine-tuning step with ragged sizes
        {"name": "backward ragged", "op": "gated_bwd", "dtype": "f16", "act": "gelu_erf", "T": 77, "D": 384, "F": 1000},
        # training on the encoder batch: few weight tiles, a long sum over tokens
        {"name": "backward encoder batch", "op": "gated_bwd", "dtype": "bf16", "act": "gelu", "T": 18106, "D": 384, "F": 1536},
        # training a wide model
        {"name": "backward long", "op": "gated_bwd", "dtype": "bf16", "act": "silu", "T": 8192, "D": 4096, "F": 8192},
        # activations of a few tokens, there and back
        {"name": "quantise tokens", "op": "quant", "dtype": "bf16", "T": 8, "K": 4096},
        # a large weight matrix at load, there and back
        {"name": "quantise weights", "op": "quant", "dtype": "bf16", "T": 8192, "K": 8192},
        # one token through a 4-bit projection
        {"name": "fp4 linear one token", "op": "linear4", "dtype": "bf16", "T": 1, "K": 4096, "N": 4096},
        # a prompt through a large 4-bit projection
        {"name": "fp4 linear long", "op": "linear4", "dtype": "f16", "T": 8192, "K": 8192, "N": 8192},
        # a batch of decoding sequences through the 4-bit block
        {"name": "fp4 gated tokens", "op": "gated4", "dtype": "bf16", "act": "silu", "T": 16, "D": 4096, "F": 8192},
        # the encoder batch served in 4 bits
        {"name": "fp4 gated encoder batch", "op": "gated4", "dtype": "bf16", "act": "gelu", "T": 18106, "D": 384, "F": 1536},
    ]


_LARGEST = 8192 * 4096 * 8192  # multiply-adds of one product of the largest case


def _spread(rng, lo, hi, step):
    """A multiple of `step` in [lo, hi], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["gated", "gated", "gated_bwd", "gated_bwd", "quant", "linear4", "linear4", "gated4"])
    dt = rng.choice(["bf16", "f16"])
    T = _spread(rng, 1, 18200, 1)
    if op == "quant":
        return {"op": op, "dtype": rng.choice(["bf16", "f16", "f32"]), "T": _spread(rng, 1, 8192, 1), "K": _spread(rng, 32, 8192, 32)}
    if op == "linear4":
        c = {"op": op, "dtype": dt, "T": T, "K": _spread(rng, 32, 8192, 32), "N": _spread(rng, 8, 8192, 8)}
        while 3 * c["T"] * c["K"] * c["N"] > _LARGEST:
            c["T"] //= 2
        return c
    step = 32 if op == "gated4" else 8
    c = {"op": op, "dtype": dt, "act": rng.choice(["silu", "gelu", "gelu_erf", "relu", "sigmoid"]), "T": T,
         "D": _spread(rng, 128, 4096, step), "F": _spread(rng, 256, 8192, step)}
    while c["T"] * c["D"] * c["F"] > _LARGEST:
        c["T"] //= 2
    return c


def work(case):
    T, op = case["T"], case["op"]
    e = 4 if case["dtype"] == "f32" else 2
    if op == "quant":
        return {"bytes": 2 * e * T * case["K"], "flops": 0}
    if op == "linear4":
        K, N = case["K"], case["N"]
        return {"bytes": e * T * K + N * (K // 2 + K // BLOCK) + e * T * N, "flops": 2 * T * K * N}
    D, F = case["D"], case["F"]
    if op == "gated":
        return {"bytes": e * (T * D + 2 * F * D + T * F), "flops": 4 * T * D * F}
    if op == "gated4":
        return {"bytes": e * T * D + 2 * F * (D // 2 + D // BLOCK) + e * T * F, "flops": 4 * T * D * F}
    # both projections again, dx, and the two weights' gradients
    return {"bytes": e * (2 * T * D + 4 * F * D + T * F), "flops": 12 * T * D * F}


# ---- what a program has in hand ----------------------------------------------------------------------

_ctx = None


def _ops():
    """The framework's entry points and this process's context."""
    global _ctx
    from tenzor_b200 import ops
    if _ctx is None:
        from tenzor_b200.runtime import Context
        _ctx = Context(torch.cuda.current_device())
    return ops, _ctx


def _inputs(case, seed):
    """The tensors of a case, in its type, the same for every form."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, op, T = _DT[case["dtype"]], case["op"], case["T"]

    def normal(shape, std):
        return torch.randn(shape, generator=gen, device="cuda").mul_(std).to(dt)

    K = case["K"] if "K" in case else case["D"]
    x = torch.randn((T, K), generator=gen, device="cuda")
    if op in ("quant", "linear4", "gated4"):  # a few channels of activations are much larger than the others
        loud = torch.rand(K, generator=gen, device="cuda") < 0.01
        x = torch.where(loud, x * 12.0, x)
    got = {"x": x.to(dt)}
    if op == "linear4":
        got["w"] = normal((case["N"], K), K ** -0.5)
    elif op != "quant":
        got["wg"] = normal((case["F"], K), K ** -0.5)
        got["wu"] = normal((case["F"], K), K ** -0.5)
    if op == "gated_bwd":
        got["dh"] = normal((T, case["F"]), 0.05)
    return got


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    if case["op"] == "linear4":  # a serving program keeps its weights in 4 bits only
        w = s.pop("w")
        if own:
            ops, ctx = _ops()
            s["w4"] = ops.quantize_mxfp4(ctx, w)
        else:
            s["w4"] = _encode(w)
    elif case["op"] == "gated4":
        wg, wu = s.pop("wg"), s.pop("wu")
        if own:
            ops, ctx = _ops()
            s["w4"] = ops.pack_gated_mxfp4(ctx, wg, wu)
        else:
            s["w4"] = (_encode(wg), _encode(wu))
    return s


# ---- the plain forms ---------------------------------------------------------------------------------

def _act(name, g):
    if name == "silu":
        return g * torch.sigmoid(g)
    if name == "gelu":
        return 0.5 * g * (1.0 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g * g * g)))
    if name == "gelu_erf":
        return 0.5 * g * (1.0 + torch.erf(g * 0.7071067811865476))
    if name == "relu":
        return torch.clamp(g, min=0.0)
    return torch.sigmoid(g)


def _act_grad(name, g):
    if name == "silu":
        s = torch.sigmoid(g)
        return s * (1.0 + g * (1.0 - s))
    if name == "gelu":
        t = torch.tanh(0.7978845608028654 * (g + 0.044715 * g * g * g))
        return 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * 0.7978845608028654 * (1.0 + 0.134145 * g * g)
    if name == "gelu_erf":
        return 0.5 * (1.0 + torch.erf(g * 0.7071067811865476)) + g * torch.exp(-0.5 * g * g) * 0.3989422804014327
    if name == "relu":
        return (g > 0).to(g.dtype)
    s = torch.sigmoid(g)
    return s * (1.0 - s)


def _encode(x):
    """(element codes [T, K] 0..15, scale codes [T, K / 32]) of x: the scale is 2^(floor(log2 max|x|) - 2) over
    32 values, the elements round to the nearest of 0 .5 1 1.5 2 3 4 6, ties to the even code, and saturate."""
    b = x.float().reshape(x.shape[0], -1, BLOCK)
    a = b.abs()
    scale = torch.clamp((a.amax(dim=-1).view(torch.int32) >> 23) - 2, min=0)
    y = a * ((254 - scale) << 23).view(torch.float32).unsqueeze(-1)
    code = ((y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0))
    code = code.to(torch.uint8) + 8 * (b < 0).to(torch.uint8)
    return code.reshape(x.shape), scale.to(torch.uint8)


def _decode(codes):
    """The 32-bit values that the codes stand for."""
    code, scale = codes
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0],
                        device=code.device)
    v = grid[code.to(torch.int32)].reshape(code.shape[0], -1, BLOCK)
    s = torch.exp2(scale.to(torch.float32) - 127.0).unsqueeze(-1)
    return (v * s).reshape(code.shape)


def _plain(s):
    case = s["case"]
    op, dt, x = case["op"], s["x"].dtype, s["x"]
    if op == "quant":
        return _decode(_encode(x)).to(dt)
    if op == "linear4":
        return (_decode(_encode(x)) @ _decode(s["w4"]).t()).to(dt)
    if op == "gated4":
        xf = _decode(_encode(x))
        wg, wu = _decode(s["w4"][0]), _decode(s["w4"][1])
        return (_act(case["act"], xf @ wg.t()) * (xf @ wu.t())).to(dt)
    xf, wg, wu = x.float(), s["wg"].float(), s["wu"].float()
    g, u = xf @ wg.t(), xf @ wu.t()
    if op == "gated":
        return (_act(case["act"], g) * u).to(dt)
    dh = s["dh"].float()
    dg, du = dh * u * _act_grad(case["act"], g), dh * _act(case["act"], g)
    return {"dx": (dg @ wg + du @ wu).to(dt), "dw_gate": (dg.t() @ xf).to(dt), "dw_up": (du.t() @ xf).to(dt)}


def run(state):
    if not own:
        return _plain(state)
    ops, ctx = _ops()
    case = state["case"]
    op, x = case["op"], state["x"]
    if op == "quant":
        return ops.dequantize_mxfp4(ctx, ops.quantize_mxfp4(ctx, x), x.dtype)
    if op == "linear4":
        return ops.linear_mxfp4(ctx, x, state["w4"])
    if op == "gated4":
        return ops.gated_linear_mxfp4(ctx, x, state["w4"], case["act"])
    if op == "gated":
        return ops.gated_linear(ctx, x, state["wg"], state["wu"], case["act"])
    dx, dwg, dwu = ops.gated_linear_backward(ctx, x, state["wg"], state["wu"], state["dh"], case["act"])
    return {"dx": dx, "dw_gate": dwg, "dw_up": dwu}


# ---- the definitions in 64 bits ----------------------------------------------------------------------

def _nearest4(x):
    """q(x) in 64 bits, from the definition: the grid's spacing at |x| / scale is a power of two."""
    v = x.double().reshape(x.shape[0], x.shape[1] // BLOCK, BLOCK)
    top = v.abs().amax(dim=2, keepdim=True)
    _, e = torch.frexp(top)  # top = m 2^e with m in [0.5, 1)
    e = torch.where(top > 0, e - 1 - 2, torch.full_like(e, -127)).clamp(min=-127)
    s = torch.ldexp(torch.ones_like(top), e)
    y = v / s
    _, f = torch.frexp(y.abs())
    step = torch.ldexp(torch.full_like(y, 0.5), (f - 1).clamp(min=0, max=2))
    q = torch.round(y / step) * step  # ties to even
    return (q.clamp(min=-6.0, max=6.0) * s).reshape(x.shape)


def exact(case, seed):
    v = _inputs(case, seed)
    op = case["op"]
    if op == "quant":
        return _nearest4(v["x"])
    if op == "linear4":
        return torch.einsum("tk,nk->tn", _nearest4(v["x"]), _nearest4(v["w"]))
    q = _nearest4 if op == "gated4" else torch.Tensor.double
    x, wg, wu = q(v["x"]), q(v["wg"]), q(v["wu"])
    g = torch.einsum("td,fd->tf", x, wg).requires_grad_(op == "gated_bwd")
    u = torch.einsum("td,fd->tf", x, wu).requires_grad_(op == "gated_bwd")
    fn = torch.nn.functional
    a = {"silu": fn.silu, "gelu": lambda z: fn.gelu(z, approximate="tanh"), "gelu_erf": fn.gelu, "relu": fn.relu,
         "sigmoid": torch.sigmoid}[case["act"]](g)
    if op != "gated_bwd":
        return a * u
    dg, du = torch.autograd.grad(a * u, (g, u), v["dh"].double())
    return {"dx": torch.einsum("tf,fd->td", dg, wg) + torch.einsum("tf,fd->td", du, wu),
            "dw_gate": torch.einsum("tf,td->fd", dg, x), "dw_up": torch.einsum("tf,td->fd", du, x)}

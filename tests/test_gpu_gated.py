"""Gated feed-forward block (forward and backward) against plain 64-bit formulas.

Tolerances, elementwise and derived from the arithmetic:
  U       unit roundoff of the 16-bit type (2^-8 bf16, 2^-11 f16), TINY half its smallest subnormal
  S(n)    a sum of n products in f32 on the tensor core: one rounding or truncation (2^-23) per 16 products
          and one per partial sum, relative to the sum of the absolute products: (n / 16 + 20) 2^-23
  ACT     the fast exponential and reciprocal: 2^-19 of the value's scale
"""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}
U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134}
ACTS = ["silu", "gelu", "gelu_erf", "relu", "sigmoid"]
ACT = 2.0 ** -19


def act64(name, g):
    fn = torch.nn.functional
    return {"silu": fn.silu, "gelu": lambda z: fn.gelu(z, approximate="tanh"), "gelu_erf": fn.gelu, "relu": fn.relu,
            "sigmoid": torch.sigmoid}[name](g)


def S(n):
    return (n / 16 + 20) * 2.0 ** -23


def make(T, D, F, dt, seed=0, wscale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s, std=1.0):
        return (torch.randn(*s, generator=gen, device="cuda") * std).to(DT[dt])

    return r(T, D), r(F, D, std=wscale * D ** -0.5), r(F, D, std=wscale * D ** -0.5), r(T, F, std=0.1)


def reference(x, wg, wu, dh, act):
    """h and the gradients in 64 bits, and the bounds of h, dx, dwg, dwu."""
    dt = {v: k for k, v in DT.items()}[x.dtype]
    u16, tiny = U[dt], TINY[dt]
    x, wg, wu, dh = x.double(), wg.double(), wu.double(), dh.double()
    g = (x @ wg.t()).requires_grad_(True)
    u = (x @ wu.t()).requires_grad_(True)
    a = act64(act, g)
    h = a * u
    dg, du = torch.autograd.grad(h, (g, u), dh)
    (da,) = torch.autograd.grad(act64(act, g).sum(), g)
    g, u, a, h = g.detach(), u.detach(), a.detach(), h.detach()
    D, F, T = x.shape[1], wg.shape[0], x.shape[0]
    eg, eu = S(D) * (x.abs() @ wg.abs().t()), S(D) * (x.abs() @ wu.abs().t())
    scale = 1.0 + g.abs()
    ea = 1.13 * eg + ACT * scale  # |act'| <= 1.13
    th = u16 * h.abs() + (1 + u16) * (u.abs() * ea + a.abs() * eu + ea * eu) + tiny
    # |act''| <= 1 except at relu's corner, where the sign of g is not certain
    ed = (da.abs() + (g.abs() <= eg).double() + 1) * eg + ACT * scale
    if act == "relu":
        ed = torch.where(g.abs() <= eg, torch.ones_like(g), torch.zeros_like(g))
    edg = dh.abs() * (u.abs() * ed + da.abs() * eu + ed * eu)
    edg = edg + u16 * (dg.abs() + edg) + tiny
    edu = dh.abs() * ea
    edu = edu + u16 * (du.abs() + edu) + tiny
    dx, dwg, dwu = dg @ wg + du @ wu, dg.t() @ x, du.t() @ x
    sx = (dg.abs() + edg) @ wg.abs() + (du.abs() + edu) @ wu.abs()
    tx = edg @ wg.abs() + edu @ wu.abs() + S(2 * F) * sx
    tg = edg.t() @ x.abs() + S(T) * ((dg.abs() + edg).t() @ x.abs())
    tu = edu.t() @ x.abs() + S(T) * ((du.abs() + edu).t() @ x.abs())
    tx, tg, tu = (t + u16 * (v.abs() + t) + tiny for t, v in ((tx, dx), (tg, dwg), (tu, dwu)))
    return (h, dx, dwg, dwu), (th, tx, tg, tu)


def near(got, want, tol, what):
    assert got.shape == want.shape, (got.shape, want.shape)
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((got.double() - want).abs().max()), float(tol.max()))


def run(ctx, x, wg, wu, dh, act):
    from tenzor_b200 import ops
    h = ops.gated_linear(ctx, x, wg, wu, act)
    dx, dwg, dwu = ops.gated_linear_backward(ctx, x, wg, wu, dh, act)
    torch.cuda.synchronize()
    ctx.check_status()
    return h, dx, dwg, dwu


def check(ctx, x, wg, wu, dh, act):
    want, tol = reference(x, wg, wu, dh, act)
    for g, w, t, n in zip(run(ctx, x, wg, wu, dh, act), want, tol, ("h", "dx", "dw_gate", "dw_up")):
        near(g, w, t, n)


SIZES = [(1, 8, 8), (1, 384, 1536), (2, 64, 72), (3, 2048, 264), (7, 72, 2000), (8, 384, 1536), (9, 40, 8), (16, 1024, 520),
         (17, 136, 136), (31, 200, 96), (64, 384, 1000), (77, 384, 1000), (127, 128, 128), (128, 8, 264), (129, 64, 384),
         (256, 256, 512), (300, 1000, 328), (513, 520, 776), (1000, 384, 1536), (4099, 128, 264),
         (5003, 384, 1544), (9000, 448, 520), (20000, 256, 264), (700, 768, 2048), (2100, 1160, 336), (100, 64, 9736)]


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("T,D,F", SIZES)
def test_sizes(ctx, T, D, F, dt):
    check(ctx, *make(T, D, F, dt, seed=T + D + F), "silu")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("T", [3, 150])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_activations(ctx, act, T, dt):
    check(ctx, *make(T, 128, 200, dt, seed=T), act)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("T", [4, 140])
def test_large_gates_saturate(ctx, act, T):
    """Gates of a few hundred: every activation and derivative reaches its limits without an infinity or NaN."""
    x, wg, wu, dh = make(T, 64, 96, "bf16", seed=5, wscale=1.0)
    for o in run(ctx, x, (wg.float() * 300).to(wg.dtype), wu, dh, act):
        assert torch.isfinite(o).all()
    if act in ("relu", "sigmoid"):
        return
    h = run(ctx, x, (wg.float() * 300).to(wg.dtype), wu, dh, act)[0]
    g = x.double() @ (wg.float() * 300).to(wg.dtype).double().t()
    u = x.double() @ wu.double().t()
    sure = g.abs() > 60
    want = torch.where(g > 0, g * u, torch.zeros_like(g))
    assert ((h.double() - want).abs()[sure] <= 2.0 ** -7 * want.abs()[sure] + 1e-3).all()


@pytest.mark.parametrize("T", [5, 200])
def test_strided_rows(ctx, T):
    x, wg, wu, dh = make(T, 128, 136, "bf16", seed=3)
    xb = torch.full((T, 128 + 64), float("nan"), device="cuda", dtype=x.dtype)
    db = torch.full((T, 136 + 8), float("nan"), device="cuda", dtype=x.dtype)
    xb[:, 64:], db[:, :136] = x, dh
    check(ctx, xb[:, 64:], wg, wu, db[:, :136], "gelu")


@pytest.mark.parametrize("T", [6, 135])
def test_weights_as_halves_of_one_matrix(ctx, T):
    x, wg, wu, dh = make(T, 64, 80, "f16", seed=9)
    w = torch.cat([wg, wu])
    check(ctx, x, w[:80], w[80:], dh, "silu")


@pytest.mark.parametrize("T", [7, 140])
def test_bad_values_stay_in_their_rows(ctx, T):
    """A NaN or infinite token spoils its own row of h and dx; the weights' gradients sum over tokens and show it."""
    x, wg, wu, dh = make(T, 64, 72, "bf16", seed=4)
    clean = run(ctx, x, wg, wu, dh, "silu")
    x[2, 5] = float("nan")
    x[4, 9] = float("inf")
    h, dx, dwg, dwu = run(ctx, x, wg, wu, dh, "silu")
    keep = [r for r in range(T) if r not in (2, 4)]
    assert torch.equal(h[keep], clean[0][keep]) and torch.equal(dx[keep], clean[1][keep])
    assert torch.isnan(h[2]).all() and torch.isnan(dx[2]).all() and not torch.isfinite(h[4]).any()
    assert torch.isnan(dwg[:, 5]).all() and torch.isnan(dwu[:, 5]).all()


@pytest.mark.parametrize("act", ACTS)
def test_gradient_against_differences(ctx, act):
    """<dx, v> and <dW, V> against central differences of the 64-bit forward formula."""
    from tenzor_b200 import ops
    x, wg, wu, dh = make(70, 72, 88, "f16", seed=21)
    grads = ops.gated_linear_backward(ctx, x, wg, wu, dh, act)
    _, (_, *tol) = reference(x, wg, wu, dh, act)
    base = [t.double() for t in (x, wg, wu)]
    gen = torch.Generator(device="cuda").manual_seed(2)
    eps = 1e-5

    def loss(v):
        return float((act64(act, v[0] @ v[1].t()) * (v[0] @ v[2].t()) * dh.double()).sum())

    for i in range(3):
        v = torch.randn(base[i].shape, generator=gen, device="cuda", dtype=torch.float64)
        up, dn = list(base), list(base)
        up[i], dn[i] = base[i] + eps * v, base[i] - eps * v
        diff = (loss(up) - loss(dn)) / (2 * eps)
        bound = float((tol[i] * v.abs()).sum()) + 1e-4  # the differences' own error: eps^2 and 2^-52 / eps
        if act == "relu":
            bound += 0.02  # corners crossed within eps
        assert abs(float((grads[i].double() * v).sum()) - diff) <= bound


def test_repeats_are_bit_equal(ctx):
    a = make(700, 136, 200, "bf16", seed=8)
    one, two = run(ctx, *a, "gelu"), run(ctx, *a, "gelu")
    assert all(torch.equal(p, q) for p, q in zip(one, two))


def test_no_tokens(ctx):
    from tenzor_b200 import ops
    x, wg, wu, dh = make(4, 64, 72, "bf16")
    assert ops.gated_linear(ctx, x[:0], wg, wu).shape == (0, 72)
    dx, dwg, dwu = ops.gated_linear_backward(ctx, x[:0], wg, wu, dh[:0])
    assert dx.shape == (0, 64) and not dwg.any() and not dwu.any()


def test_other_stream_and_graph(ctx):
    from tenzor_b200 import ops
    x, wg, wu, dh = make(300, 128, 136, "f16", seed=6)
    want = run(ctx, x, wg, wu, dh, "silu")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = (ops.gated_linear(ctx, x, wg, wu), *ops.gated_linear_backward(ctx, x, wg, wu, dh))
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = (ops.gated_linear(ctx, x, wg, wu), *ops.gated_linear_backward(ctx, x, wg, wu, dh))
    for t in got:
        t.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_refusals(ctx):
    from tenzor_b200 import TenzorError, _lib, ops
    x, wg, wu, dh = make(4, 64, 72, "bf16")
    with pytest.raises(TypeError):
        ops.gated_linear(ctx, x.float(), wg, wu)
    with pytest.raises(ValueError):
        ops.gated_linear(ctx, x, wg.half(), wu)
    with pytest.raises(ValueError):
        ops.gated_linear(ctx, x, wg, wu[:64])
    with pytest.raises(ValueError):
        ops.gated_linear(ctx, x, wg, wu, act="tanh")
    with pytest.raises(ValueError):
        ops.gated_linear(ctx, x, wg, wu, out=torch.empty(4, 64, device="cuda", dtype=x.dtype))
    with pytest.raises(ValueError):
        ops.gated_linear(ctx, x.t().contiguous().t(), wg, wu)
    with pytest.raises(ValueError):
        ops.gated_linear(ctx, x.cpu(), wg, wu)
    with pytest.raises(ValueError):
        ops.gated_linear_backward(ctx, x, wg, wu, dh[:2])
    with pytest.raises(TenzorError) as e:  # a width that is no multiple of 8
        ops.gated_linear(ctx, x[:, :60].contiguous(), wg[:, :60].contiguous(), wu[:, :60].contiguous())
    assert e.value.code == _lib.TZ_EINVAL
    wide = torch.zeros(4, 68, device="cuda", dtype=x.dtype)
    with pytest.raises(TenzorError):  # a row stride that is no multiple of 8
        ops.gated_linear(ctx, wide[:, :64], wg, wu)
    odd = torch.zeros(4 * 64 + 1, device="cuda", dtype=x.dtype)[1:].view(4, 64)
    with pytest.raises(TenzorError):  # an address that is no multiple of 16 bytes
        ops.gated_linear(ctx, odd, wg, wu)
    Lb, p = _lib.lib(), (lambda t: C.c_void_p(t.data_ptr()))
    assert Lb.tz_gated_linear_backward(ctx.handle, p(x), 64, p(wg), p(wu), p(dh), 72, p(x), p(wg), p(wu), p(x), 1, 4, 64, 72,
                                       _lib.OP["silu"], 1, None) == _lib.TZ_EINVAL
    assert "workspace" in Lb.tz_get_last_error().decode()
    assert Lb.tz_gated_linear(ctx.handle, p(x), 64, p(wg), p(wu), p(dh), 4, 64, 72, _lib.OP["exp"], 1, None) == _lib.TZ_EINVAL
    assert Lb.tz_gated_linear(ctx.handle, p(x), 64, p(wg), p(wu), p(dh), 4, 64, 72, _lib.OP["silu"], 7, None) == _lib.TZ_EINVAL
    assert Lb.tz_gated_linear(None, p(x), 64, p(wg), p(wu), p(dh), 4, 64, 72, _lib.OP["silu"], 1, None) == _lib.TZ_EINVAL


@pytest.mark.parametrize("reserve", [100, 140, 146])
def test_few_sms(reserve):
    """Leaving SMs to other kernels cuts the grids: more tiles per CTA, other splits, the same results."""
    from tenzor_b200.runtime import Context
    c = Context(0)
    c.set_sm_reserve(reserve)
    for T, D, F in ((5, 384, 1536), (700, 384, 1544), (300, 520, 328)):
        check(c, *make(T, D, F, "bf16", seed=T), "gelu")
    c.close()


@pytest.mark.parametrize("T", [1, 6, 40, 300])
def test_outputs_that_overlap_are_refused(ctx, T):
    """Other CTAs still read what an overlapping output would overwrite."""
    from tenzor_b200 import TenzorError, _lib, ops
    x, wg, wu, dh = make(T, 64, 64, "bf16")
    buf = torch.zeros(T * 64 + 64 * 64 + T * 64, device="cuda", dtype=x.dtype)
    at = lambda n, rows: buf[n:n + rows * 64].view(rows, 64)  # noqa: E731
    for a, gate, up, out in ((x, wg, wu, x), (at(8, T), wg, wu, at(0, T)), (at(0, T), wg, wu, at(T * 64 - 8, T)),
                             (x, at(T * 64, 64), wu, at(8 + 64, T)), (x, wg, at(0, 64), at(64 * 64 - 8, T))):
        with pytest.raises(TenzorError) as e:
            ops.gated_linear(ctx, a, gate, up, out=out)
        assert e.value.code == _lib.TZ_EINVAL and "overlaps" in str(e.value)
    # touching, or in the gap between two rows, is no overlap
    assert torch.equal(ops.gated_linear(ctx, at(0, T), wg, wu, out=at(T * 64, T)), torch.zeros_like(x))
    wide = torch.zeros(2, 64 + 128 + 8, device="cuda", dtype=x.dtype)
    wide[:, :64] = x[0]
    gap = wide.view(-1)[64:192].view(2, 64)
    assert torch.equal(ops.gated_linear(ctx, wide[:, :64], wg, wu, out=gap), ops.gated_linear(ctx, x[:1].repeat(2, 1), wg, wu))
    with pytest.raises(TenzorError):
        ops.gated_linear(ctx, wide[:, :64], wg, wu, out=wide.view(-1)[80:208].view(2, 64))

    Lb, p = _lib.lib(), (lambda t: C.c_void_p(t.data_ptr()))
    need = C.c_size_t()
    assert Lb.tz_gated_linear_backward_workspace(ctx.sm_count, T, 64, 64, C.byref(need)) == 0
    ws = torch.zeros(need.value, device="cuda", dtype=torch.uint8)
    good = {"dx": torch.empty_like(x), "dw_gate": torch.empty_like(wg), "dw_up": torch.empty_like(wu), "ws": ws}

    def call(**other):
        o = {**good, **other}
        return Lb.tz_gated_linear_backward(ctx.handle, p(x), 64, p(wg), p(wu), p(dh), 64, p(o["dx"]), p(o["dw_gate"]), p(o["dw_up"]), p(o["ws"]),
                                           need.value, T, 64, 64, _lib.OP["silu"], 1, None)

    for bad in ({"dx": x}, {"dx": dh}, {"dx": wg}, {"dw_gate": wg}, {"dw_up": wg}, {"dw_up": good["dw_gate"]}, {"dw_gate": good["dx"]}, {"ws": x},
                {"ws": good["dw_up"]}, {"dx": ws}):
        assert call(**bad) == _lib.TZ_EINVAL and "overlaps" in Lb.tz_get_last_error().decode(), bad
    assert call() == 0
    torch.cuda.synchronize()


class _KernelNode(C.Structure):  # CUDA_KERNEL_NODE_PARAMS of the driver API
    _fields_ = [("func", C.c_void_p), *((n, C.c_uint) for n in ("gx", "gy", "gz", "bx", "by", "bz", "smem")), ("params", C.c_void_p),
                ("extra", C.c_void_p), ("kern", C.c_void_p), ("ctx", C.c_void_p)]


def captured_grids(fn):
    """(blocks, dynamic shared memory) of every kernel that fn launches."""
    cu = C.CDLL("libcuda.so.1")
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g):
        keep = fn()
    graph, n = C.c_void_p(g.raw_cuda_graph()), C.c_size_t()
    assert cu.cuGraphGetNodes(graph, None, C.byref(n)) == 0
    nodes = (C.c_void_p * n.value)()
    assert cu.cuGraphGetNodes(graph, nodes, C.byref(n)) == 0
    got = []
    for node in nodes:
        kind, k = C.c_int(), _KernelNode()
        assert cu.cuGraphNodeGetType(C.c_void_p(node), C.byref(kind)) == 0
        if kind.value == 0:  # a kernel
            assert cu.cuGraphKernelNodeGetParams_v2(C.c_void_p(node), C.byref(k)) == 0
            got.append((k.gx * k.gy * k.gz, k.smem))
    del keep
    return got


@pytest.mark.parametrize("reserve", [0, 16, 100, 146])
@pytest.mark.parametrize("T", [1, 16, 20, 32, 100, 300])
def test_reserved_sms_stay_free(reserve, T):
    """No product kernel (all of them use shared memory for their operands) launches more CTAs than there are SMs left;
    more feature tiles than that are taken one lot after the other, with the same result."""
    from tenzor_b200 import ops
    from tenzor_b200.runtime import Context
    c = Context(0)
    x, wg, wu, dh = make(T, 64, 151 * 128 - 40, "bf16", seed=T)
    want = (ops.gated_linear(c, x, wg, wu), *ops.gated_linear_backward(c, x, wg, wu, dh))
    c.set_sm_reserve(reserve)

    def call():
        return ops.gated_linear(c, x, wg, wu), *ops.gated_linear_backward(c, x, wg, wu, dh)

    grids = [blocks for blocks, smem in captured_grids(call) if smem > 0]
    assert len(grids) >= 3 and (reserve == 0 or max(grids) <= c.sm_count - reserve), grids
    got = call()
    torch.cuda.synchronize()
    c.check_status()
    assert torch.equal(got[0], want[0])  # h: one sum over all of D, whatever the grid
    _, tol = reference(x, wg, wu, dh, "silu")
    for g, w, t in zip(got[1:], want[1:], tol[1:]):  # the gradients' sums are split by the SMs in use
        near(g, w.double(), 2 * t, (T, reserve))
    c.close()


def test_reserve_set_through_the_c_abi():
    """The backward call sizes its workspace for the SMs that the library uses, however the reserve was set."""
    from tenzor_b200 import _lib
    from tenzor_b200.runtime import Context
    c = Context(0)
    a = make(3000, 384, 264, "bf16", seed=1)
    c.set_sm_reserve(140)
    check(c, *a, "silu")
    for reserve in (0, 116):  # more SMs, more splits: more partial sums than for the reserve above
        assert _lib.lib().tz_cuda_set_sm_reserve(c.handle, reserve) == 0
        check(c, *a, "silu")
        assert c.sm_reserve == reserve
    c.close()


def test_no_sm_left_is_refused():
    from tenzor_b200 import TenzorError, ops
    from tenzor_b200.runtime import Context
    c = Context(0)
    c.set_sm_reserve(147)
    x, wg, wu, dh = make(300, 64, 72, "bf16")
    with pytest.raises(TenzorError):
        ops.gated_linear(c, x, wg, wu)
    c.close()


def test_more_than_2_to_31_elements(ctx):
    """h, dg and du of 2.2e9 elements: the last rows against the 64-bit formulas, and the weights' gradients as the
    sum of those of two halves of the tokens."""
    from tenzor_b200 import ops
    T, D, F = 530_001, 64, 4104
    x, wg, wu, _ = make(T, D, F, "bf16", seed=1)
    dh = torch.empty((T, F), device="cuda", dtype=torch.bfloat16).normal_(0, 0.1, generator=torch.Generator(device="cuda").manual_seed(2))
    h = ops.gated_linear(ctx, x, wg, wu, "silu")
    dx, dwg, dwu = ops.gated_linear_backward(ctx, x, wg, wu, dh, "silu")
    for at in (slice(0, 200), slice(T - 200, T)):
        (wh, wdx, _, _), (th, tdx, _, _) = reference(x[at], wg, wu, dh[at], "silu")
        near(h[at], wh, th, "h")
        near(dx[at], wdx, tdx, "dx")
    del h, dx
    half = 265_024
    a = ops.gated_linear_backward(ctx, x[:half], wg, wu, dh[:half], "silu")
    b = ops.gated_linear_backward(ctx, x[half:], wg, wu, dh[half:], "silu")
    for whole, p, q in ((dwg, a[1], b[1]), (dwu, a[2], b[2])):
        want = p.double() + q.double()
        rms = want.square().mean().sqrt()  # rounding of the three results, and of sums of 530 k products in f32
        assert ((whole.double() - want).abs() <= 3 * U["bf16"] * (want.abs() + rms)).all()

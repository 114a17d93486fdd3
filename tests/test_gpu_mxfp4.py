"""MXFP4 quantiser and products against the format's definition in 64 bits.

The quantiser is compared exactly.  Products of E2M1 values are exact, so a product differs from the 64-bit
one by its f32 sum (one rounding or truncation, 2^-23, per 64 products and 8 more for joined partial sums,
relative to the sum of the absolute products) and by the rounding to the output's type (U, TINY)."""
import ctypes as C

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}
GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def quant64(x):
    """(values, element codes, scale codes) of a float array [rows, cols], from the definition."""
    x = x.astype(np.float64)
    b = x.reshape(x.shape[0], -1, 32)
    top = np.abs(b).max(axis=2)
    _, e = np.frexp(np.where(np.isfinite(top) & (top > 0), top, 1.0))
    code = np.where(top > 0, np.maximum(e - 3, -127), -127) + 127
    s = np.ldexp(1.0, code - 127)[..., None]
    y = np.abs(np.where(np.isfinite(b), b, 0.0)) / s
    d = np.abs(np.minimum(y, 6.0)[..., None] - GRID)  # distance to every grid point
    low = d.min(axis=-1, keepdims=True)
    even = np.where(d == low, np.arange(8) % 2, 2).argmin(axis=-1)  # of two equally near codes the even one
    q = np.where(np.signbit(b), -GRID[even], GRID[even]) * s
    bad = ~np.isfinite(top)
    q[bad] = np.nan
    code = np.where(bad, 255, code)
    return q.reshape(x.shape), (even + 8 * np.signbit(b)).reshape(x.shape), code


def scale_codes(q):
    """The scale codes [rows, cols / 32] of an Mxfp4, from its documented layout."""
    kc = -(-q.cols // 128)
    raw = q.scales.cpu().numpy()
    r, b = np.meshgrid(np.arange(q.rows), np.arange(q.cols // 32), indexing="ij")
    return raw[((r // 128) * kc + b // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4]


def element_codes(q):
    raw = q.codes.cpu().numpy()
    return np.stack([raw & 15, raw >> 4], axis=-1).reshape(q.rows, q.cols)


def rand(rows, cols, dt, seed, spread=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, cols), generator=gen, device="cuda")
    if spread:  # scales over several binades
        x = x * torch.exp2(torch.randint(-6, 5, (rows, cols // 32, 1), generator=gen, device="cuda").float()).expand(-1, -1, 32).reshape(rows, cols)
    return x.to(DT[dt])


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 32), (2, 64), (3, 96), (5, 160), (31, 224), (33, 256), (127, 288), (128, 384), (129, 512), (300, 4096)])
def test_quantiser_exact(ctx, rows, cols, dt):
    from tenzor_b200 import ops
    x = rand(rows, cols, dt, rows + cols)
    q = ops.quantize_mxfp4(ctx, x)
    want, codes, scales = quant64(x.float().cpu().numpy())
    assert np.array_equal(scale_codes(q), scales)
    assert np.array_equal(element_codes(q), codes)
    for out in ("f32", "bf16"):
        assert np.array_equal(ops.dequantize_mxfp4(ctx, q, DT[out]).double().cpu().numpy(), want)
    f16 = torch.from_numpy(want).to(torch.float16)  # one rounding where f16 is too narrow
    assert torch.equal(ops.dequantize_mxfp4(ctx, q, torch.float16).cpu(), f16)


def test_ties_saturation_and_edges(ctx):
    from tenzor_b200 import ops
    x = torch.zeros(12, 32)
    x[0, :10] = torch.tensor([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.9, -0.25])
    x[1, :3] = torch.tensor([7.99, 5.01, -7.5])  # above the largest code: saturates
    x[2] = -0.0
    x[3, 0] = 2.0 ** -149  # subnormal maximum: the smallest scale
    x[4, 1] = 2.0 ** -126
    x[5, 2] = 3.0e38
    x[6, 7] = float("inf")
    x[7, 8] = float("nan")
    x[8, 9] = -float("inf")
    x[9] = torch.arange(32) * 2.0 ** -130
    x[10, 0], x[10, 1] = 1.0, 2.0 ** -140
    x = x.cuda()
    q = ops.quantize_mxfp4(ctx, x)
    want, codes, scales = quant64(x.cpu().numpy())
    assert np.array_equal(scale_codes(q), scales)
    ok = scales[:, 0] != 255
    assert np.array_equal(element_codes(q)[ok], codes[ok])
    got = ops.dequantize_mxfp4(ctx, q).double().cpu().numpy()
    assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_quantiser_strided_rows(ctx, dt):
    from tenzor_b200 import ops
    x = rand(37, 96, dt, 1)
    wide = torch.full((37, 160), float("nan"), device="cuda", dtype=x.dtype)
    wide[:, 32:128] = x
    a, b = ops.quantize_mxfp4(ctx, wide[:, 32:128]), ops.quantize_mxfp4(ctx, x)
    assert torch.equal(a.codes, b.codes) and np.array_equal(scale_codes(a), scale_codes(b))


def product64(x, w, bias=None):
    a = torch.from_numpy(quant64(x.float().cpu().numpy())[0]).cuda()
    b = torch.from_numpy(quant64(w.float().cpu().numpy())[0]).cuda()
    y = a @ b.t()
    err = (x.shape[1] / 64 + 8) * 2.0 ** -23 * (a.abs() @ b.abs().t())
    if bias is not None:
        y = y + bias.double()
        err = err + 2.0 ** -24 * (y.abs() + err)
    return y, err


def near(got, want, tol, what=""):
    assert got.shape == want.shape
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((got.double() - want).abs().max()), float(tol.max()))


SIZES = [(1, 32, 8), (1, 4096, 1024), (2, 64, 16), (3, 96, 200), (5, 160, 136), (8, 2048, 512), (9, 224, 24), (16, 1024, 1000),
         (17, 288, 192), (31, 512, 384), (33, 320, 392), (64, 4096, 264), (65, 448, 200), (127, 128, 128), (128, 256, 576),
         (129, 384, 1536), (257, 1536, 384), (300, 1056, 328), (1000, 384, 1536), (3000, 96, 72), (70, 256, 15000)]


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_linear_sizes(ctx, M, K, N, dt):
    from tenzor_b200 import ops
    x, w = rand(M, K, dt, M + K), (rand(N, K, dt, N).float() * K ** -0.5).to(DT[dt])
    bias = torch.randn(N, device="cuda") if M % 2 else None
    y = ops.linear_mxfp4(ctx, x, ops.quantize_mxfp4(ctx, w), bias)
    torch.cuda.synchronize()
    ctx.check_status()
    want, err = product64(x, w, bias)
    near(y, want, err + U[dt] * (want.abs() + err) + TINY[dt])


@pytest.mark.parametrize("M", [4, 200])
def test_linear_of_quantised_input_and_output_types(ctx, M):
    from tenzor_b200 import ops
    x, w = rand(M, 192, "bf16", 3), rand(104, 192, "f16", 4)
    xq, wq = ops.quantize_mxfp4(ctx, x), ops.quantize_mxfp4(ctx, w)
    want, err = product64(x, w)
    for dt in ("f32", "f16", "bf16"):
        tol = err + U[dt] * (want.abs() + err) + TINY[dt]
        a = ops.linear_mxfp4(ctx, x, wq, out_dtype=DT[dt])
        near(a, want, tol)
        near(ops.linear_mxfp4(ctx, xq, wq, out_dtype=DT[dt]), want, tol)
    assert ops.linear_mxfp4(ctx, xq, wq).dtype == torch.float32
    out = torch.empty_like(a)
    assert ops.linear_mxfp4(ctx, x, wq, out=out) is out and torch.equal(out, a)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_erf", "relu", "sigmoid"])
@pytest.mark.parametrize("T,D,F", [(1, 32, 16), (1, 2048, 512), (6, 160, 112), (16, 1024, 208), (33, 512, 48), (140, 96, 336), (520, 384, 1536), (100, 160, 7520)])
def test_gated(ctx, act, T, D, F):
    from test_gpu_gated import act64
    from tenzor_b200 import ops
    dt = "bf16" if T % 2 else "f16"
    x, wg, wu = rand(T, D, dt, T), rand(F, D, dt, 1), rand(F, D, dt, 2)
    wg, wu = (wg.float() * 0.5 * D ** -0.5).to(DT[dt]), (wu.float() * 0.5 * D ** -0.5).to(DT[dt])
    h = ops.gated_linear_mxfp4(ctx, x, ops.pack_gated_mxfp4(ctx, wg, wu), act)
    torch.cuda.synchronize()
    ctx.check_status()
    (g, eg), (u, eu) = product64(x, wg), product64(x, wu)
    a = act64(act, g)
    ea = 1.13 * eg + 2.0 ** -19 * (1 + g.abs())  # |act'| <= 1.13; the fast exponential
    err = u.abs() * ea + a.abs() * eu + ea * eu
    near(h, a * u, err + U[dt] * ((a * u).abs() + err) + TINY[dt])


@pytest.mark.parametrize("M", [3, 150])
def test_bad_values_stay_in_their_rows(ctx, M):
    from tenzor_b200 import ops
    x, w = rand(M, 256, "bf16", 8), ops.quantize_mxfp4(ctx, rand(72, 256, "bf16", 9))
    clean = ops.linear_mxfp4(ctx, x, w)
    x[1, 40], x[2, 200] = float("nan"), float("inf")
    y = ops.linear_mxfp4(ctx, x, w)
    keep = [r for r in range(M) if r not in (1, 2)]
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[1:3]).all()


@pytest.mark.parametrize("M", [5, 150])
def test_extreme_scales(ctx, M):
    """Scales at both ends of f32: products of a tiny and a huge block."""
    from tenzor_b200 import ops
    x = rand(M, 64, "f32", 1, spread=False) * 2.0 ** -100
    w = rand(40, 64, "f32", 2, spread=False) * 2.0 ** 110
    y = ops.linear_mxfp4(ctx, x, ops.quantize_mxfp4(ctx, w))
    want, err = product64(x, w)
    near(y, want, err + U["f32"] * want.abs())


@pytest.mark.parametrize("M", [1, 7, 200])
def test_repeats_streams_and_graphs(ctx, M):
    from tenzor_b200 import ops
    x, w = rand(M, 1024, "bf16", 5), ops.quantize_mxfp4(ctx, rand(520, 1024, "bf16", 6))
    want = ops.linear_mxfp4(ctx, x, w)
    assert torch.equal(want, ops.linear_mxfp4(ctx, x, w))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.linear_mxfp4(ctx, x, w)
    s.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ops.linear_mxfp4(ctx, x, w)
    got.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_no_rows(ctx):
    from tenzor_b200 import ops
    w = ops.quantize_mxfp4(ctx, rand(16, 64, "bf16", 1))
    x = torch.empty((0, 64), device="cuda", dtype=torch.bfloat16)
    q = ops.quantize_mxfp4(ctx, x)
    assert ops.dequantize_mxfp4(ctx, q).shape == (0, 64)
    assert ops.linear_mxfp4(ctx, x, w).shape == (0, 16) and ops.linear_mxfp4(ctx, q, w).shape == (0, 16)
    wp = ops.pack_gated_mxfp4(ctx, rand(16, 64, "bf16", 1), rand(16, 64, "bf16", 2))
    assert ops.gated_linear_mxfp4(ctx, x, wp).shape == (0, 16)


def test_refusals(ctx):
    from tenzor_b200 import TenzorError, _lib, ops
    x = rand(4, 64, "bf16", 1)
    w = ops.quantize_mxfp4(ctx, rand(16, 64, "bf16", 2))
    wp = ops.pack_gated_mxfp4(ctx, rand(16, 64, "bf16", 1), rand(16, 64, "bf16", 2))
    with pytest.raises(TypeError):
        ops.quantize_mxfp4(ctx, x.double())
    with pytest.raises(ValueError):
        ops.quantize_mxfp4(ctx, x[:, :48].contiguous())
    with pytest.raises(ValueError):
        ops.quantize_mxfp4(ctx, x.cpu())
    with pytest.raises(ValueError):
        ops.linear_mxfp4(ctx, x[:, :32].contiguous(), w)
    with pytest.raises(ValueError):
        ops.linear_mxfp4(ctx, x, wp)
    with pytest.raises(ValueError):
        ops.gated_linear_mxfp4(ctx, x, w)
    with pytest.raises(TypeError):
        ops.gated_linear_mxfp4(ctx, x.float(), wp)
    with pytest.raises(ValueError):
        ops.gated_linear_mxfp4(ctx, x, wp, act="exp")
    with pytest.raises(ValueError):
        ops.dequantize_mxfp4(ctx, wp)
    with pytest.raises(ValueError):
        ops.linear_mxfp4(ctx, x, w, bias=torch.zeros(16, device="cuda", dtype=torch.float16))
    with pytest.raises(ValueError):
        ops.pack_gated_mxfp4(ctx, x, x)
    with pytest.raises(TenzorError):
        ops.linear_mxfp4(ctx, x, ops.quantize_mxfp4(ctx, rand(12, 64, "bf16", 2)))
    with pytest.raises(TenzorError):
        ops.quantize_mxfp4(ctx, torch.zeros(4 * 64 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(4, 64))
    Lb, p = _lib.lib(), (lambda t: C.c_void_p(t.data_ptr()))
    x = rand(40, 64, "bf16", 1)
    y = torch.empty(40, 16, device="cuda", dtype=torch.bfloat16)
    assert Lb.tz_linear_mxfp4(ctx.handle, p(x), 64, 2, p(w.codes), p(w.scales), None, p(y), 2, p(y), 16, 40, 64, 16, None) == _lib.TZ_EINVAL
    assert "workspace" in Lb.tz_get_last_error().decode()
    assert Lb.tz_linear_mxfp4(ctx.handle, p(x), 64, 3, p(w.codes), p(w.scales), None, p(y), 2, p(y), 16, 4, 64, 16, None) == _lib.TZ_EINVAL
    assert Lb.tz_quantize_mxfp4(None, p(x), 64, 2, p(w.codes), p(w.scales), 4, 64, None) == _lib.TZ_EINVAL
    assert Lb.tz_mxfp4_scale_bytes(-1, 64) == 0 and Lb.tz_mxfp4_scale_bytes(129, 160) == 2 * 2 * 512


def test_example_trains_and_serves(ctx):
    """The example's whole path: training with the 16-bit kernels, serving with the 4-bit ones."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "gated_block.py")
    spec = importlib.util.spec_from_file_location("gated_block", path)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    losses, cos, same = ex.main(["--dim", "128", "--ffn", "256", "--tokens", "1024", "--steps", "40"])
    assert losses[-1] < 0.5 * losses[0]
    # Each 4-bit operand is off by up to a quarter of its value (E2M1 keeps one fraction bit), 0.1 rms; four of them
    # (x, the two weights, h and Wd in turn) leave an angle of about 0.2 to 0.25.
    assert float(cos.mean()) > 0.95
    assert same <= 2.0 ** -6  # the kernels of one token and of a batch round h to 16 bits, then to 4, from other sums


@pytest.mark.parametrize("reserve", [100, 146])
def test_few_sms(reserve):
    from tenzor_b200 import ops
    from tenzor_b200.runtime import Context
    c = Context(0)
    c.set_sm_reserve(reserve)
    for M, K, N in ((3, 512, 1000), (700, 288, 1544)):
        x, w = rand(M, K, "bf16", M), rand(N, K, "bf16", N)
        y = ops.linear_mxfp4(c, x, ops.quantize_mxfp4(c, w))
        want, err = product64(x, w)
        near(y, want, err + U["bf16"] * (want.abs() + err))
    c.close()


@pytest.mark.parametrize("M", [1, 20, 40, 300])
def test_outputs_that_overlap_are_refused(ctx, M):
    from tenzor_b200 import TenzorError, _lib, ops
    x, w = rand(M, 64, "bf16", 1), ops.quantize_mxfp4(ctx, rand(64, 64, "bf16", 2))
    wp = ops.pack_gated_mxfp4(ctx, rand(64, 64, "bf16", 1), rand(64, 64, "bf16", 2))
    bias = torch.zeros(64 + 64 * M, device="cuda")
    calls = [lambda: ops.linear_mxfp4(ctx, x, w, out=x), lambda: ops.gated_linear_mxfp4(ctx, x, wp, out=x),
             lambda: ops.linear_mxfp4(ctx, x, w, bias=bias[:64], out_dtype=torch.float32, out=bias[60:60 + 64 * M].view(M, 64))]
    if M <= 20:  # outputs inside the weights' codes and scales
        for q, f in ((w, ops.linear_mxfp4), (wp, ops.gated_linear_mxfp4)):
            for end in (M * 128, q.buf.numel()):
                calls.append(lambda q=q, f=f, end=end: f(ctx, x, q, out=q.buf[end - M * 128:end].view(torch.bfloat16).view(M, 64)))
    for call in calls:
        with pytest.raises(TenzorError) as e:
            call()
        assert e.value.code == _lib.TZ_EINVAL and "overlaps" in str(e.value)
    Lb = _lib.lib()
    v = torch.zeros(8 * M * 64, device="cuda")
    a = v.data_ptr()
    n = M * 64 * 4
    for codes, scales in ((a, a + n), (a + 16, a + n), (a + n, a + n), (a + n, a), (a + n - 16, a + 2 * n)):
        assert Lb.tz_quantize_mxfp4(ctx.handle, a, 64, 0, codes, scales, M, 64, None) == _lib.TZ_EINVAL
        assert "overlaps" in Lb.tz_get_last_error().decode()
    for out in (w.codes_ptr, w.scales_ptr):
        assert Lb.tz_dequantize_mxfp4(ctx.handle, w.codes_ptr, w.scales_ptr, out, 2, 64, 64, None) == _lib.TZ_EINVAL
    assert Lb.tz_gemm_mxfp4(ctx.handle, w.codes_ptr, w.scales_ptr, w.codes_ptr, w.scales_ptr, None, w.codes_ptr, 2, 64, 64, 64, None) == _lib.TZ_EINVAL
    g = torch.zeros(64, 64, device="cuda", dtype=torch.bfloat16)
    assert Lb.tz_pack_gated_mxfp4(ctx.handle, g.data_ptr(), g.data_ptr(), 2, g.data_ptr(), wp.scales_ptr, 64, 64, None) == _lib.TZ_EINVAL
    need = C.c_size_t()
    assert Lb.tz_linear_mxfp4_workspace(M, 64, 64, C.byref(need)) == 0
    if need.value:
        big = torch.zeros(need.value + M * 128, device="cuda", dtype=torch.uint8)
        y = torch.empty_like(x)
        for ws in (big.data_ptr(), w.codes_ptr, x.data_ptr()):
            out = big.data_ptr() if ws == big.data_ptr() else y.data_ptr()
            assert Lb.tz_linear_mxfp4(ctx.handle, x.data_ptr(), 64, 2, w.codes_ptr, w.scales_ptr, None, out, 2, ws, need.value, M, 64, 64,
                                      None) == _lib.TZ_EINVAL
            assert "overlaps" in Lb.tz_get_last_error().decode()


def gated64(x, wg, wu, act):
    """The gated block on quantised operands in 64 bits, and the bound of a 16-bit result."""
    from test_gpu_gated import act64
    dt = {v: k for k, v in DT.items()}[x.dtype]
    (g, eg), (u, eu) = product64(x, wg), product64(x, wu)
    a = act64(act, g)
    ea = 1.13 * eg + 2.0 ** -19 * (1 + g.abs())  # |act'| <= 1.13; the fast exponential
    err = u.abs() * ea + a.abs() * eu + ea * eu
    return a * u, err + U[dt] * ((a * u).abs() + err) + TINY[dt]


@pytest.mark.parametrize("reserve", [0, 16, 100, 146])
@pytest.mark.parametrize("M", [1, 16, 20, 32, 100, 300])
def test_reserved_sms_stay_free(reserve, M):
    """No product kernel (all of them use shared memory for their operands) launches more CTAs than there are SMs left."""
    from test_gpu_gated import captured_grids
    from tenzor_b200 import ops
    from tenzor_b200.runtime import Context
    c = Context(0)
    x, w = rand(M, 160, "bf16", M), rand(151 * 128 - 40, 160, "bf16", 1)
    wg, wu = (0.08 * rand(151 * 64 - 32, 160, "bf16", k) for k in (2, 3))
    wq, wp = ops.quantize_mxfp4(c, w), ops.pack_gated_mxfp4(c, wg, wu)
    c.set_sm_reserve(reserve)

    def call():
        return ops.linear_mxfp4(c, x, wq), ops.gated_linear_mxfp4(c, x, wp, "gelu")

    grids = [blocks for blocks, smem in captured_grids(call) if smem > 0]
    assert len(grids) >= 2 and (reserve == 0 or max(grids) <= c.sm_count - reserve), grids
    y, h = call()
    torch.cuda.synchronize()
    c.check_status()
    want, err = product64(x, w)
    near(y, want, err + U["bf16"] * (want.abs() + err))
    near(h, *gated64(x, wg, wu, "gelu"))
    c.close()


@pytest.mark.parametrize("act", ["silu", "gelu_erf", "relu"])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("T,D,F", [(17, 160, 112), (17, 32, 16), (20, 4096, 1024), (24, 288, 80), (31, 512, 208), (32, 2080, 208), (32, 256, 4016)])
def test_gated_17_to_32_tokens(ctx, T, D, F, dt, act):
    """The few-row kernel's form for 32 rows: both of its column passes, both MMA issuers, splits, partial tiles."""
    from tenzor_b200 import ops
    x, wg, wu = rand(T, D, dt, T), rand(F, D, dt, 1), rand(F, D, dt, 2)
    wg, wu = (wg.float() * 0.5 * D ** -0.5).to(DT[dt]), (wu.float() * 0.5 * D ** -0.5).to(DT[dt])
    h = ops.gated_linear_mxfp4(ctx, x, ops.pack_gated_mxfp4(ctx, wg, wu), act)
    torch.cuda.synchronize()
    ctx.check_status()
    near(h, *gated64(x, wg, wu, act))


@pytest.mark.parametrize("waves", [2, 3])
@pytest.mark.parametrize("M", [16, 17, 32])
def test_few_rows_of_many_weights(ctx, M, waves):
    """From the third wave of 128-row weight tiles on, 17 to 32 rows take the persistent kernel; up to 16 stay."""
    from test_gpu_gated import captured_grids
    from tenzor_b200 import ops
    tiles = 2 * ctx.sm_count + (waves - 2) * 3
    x, w = rand(M, 96, "bf16", M), rand(tiles * 128 - 32, 96, "bf16", 1)
    wg, wu = (rand(tiles * 64 - 16, 96, "bf16", k) * 0.1 for k in (2, 3))
    wq, wp = ops.quantize_mxfp4(ctx, w), ops.pack_gated_mxfp4(ctx, wg, wu)
    grids = [blocks for blocks, smem in captured_grids(lambda: (ops.linear_mxfp4(ctx, x, wq), ops.gated_linear_mxfp4(ctx, x, wp))) if smem > 0]
    assert len(grids) == 2
    if M <= 16 or waves == 2:
        assert grids == [tiles, tiles]
    else:
        assert max(grids) <= ctx.sm_count
    want, err = product64(x, w)
    near(ops.linear_mxfp4(ctx, x, wq), want, err + U["bf16"] * (want.abs() + err))
    near(ops.gated_linear_mxfp4(ctx, x, wp), *gated64(x, wg, wu, "silu"))
    ctx.check_status()


@pytest.mark.parametrize("reserve", [100, 140, 146])
@pytest.mark.parametrize("T,D,F", [(3, 512, 496), (16, 2048, 1040), (20, 288, 400), (32, 1056, 1040), (100, 96, 208), (700, 288, 768)])
def test_gated_few_sms(reserve, T, D, F):
    from tenzor_b200 import ops
    from tenzor_b200.runtime import Context
    c = Context(0)
    c.set_sm_reserve(reserve)
    x, wg, wu = rand(T, D, "f16", T), rand(F, D, "f16", 1), rand(F, D, "f16", 2)
    wg, wu = (wg.float() * 0.5 * D ** -0.5).half(), (wu.float() * 0.5 * D ** -0.5).half()
    h = ops.gated_linear_mxfp4(c, x, ops.pack_gated_mxfp4(c, wg, wu), "gelu")
    torch.cuda.synchronize()
    c.check_status()
    near(h, *gated64(x, wg, wu, "gelu"))
    c.close()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("F,D", [(16, 32), (48, 160), (144, 96), (80, 1056)])
def test_packed_pair_layout(ctx, F, D, dt):
    """16 rows of the gate's codes and scales, then 16 of the up projection's, and so on."""
    from tenzor_b200 import ops
    wg, wu = rand(F, D, dt, 1), rand(F, D, dt, 2)
    q = ops.pack_gated_mxfp4(ctx, wg, wu)
    assert q.gated and q.shape == (2 * F, D)
    (_, cg, sg), (_, cu, su) = (quant64(w.float().cpu().numpy()) for w in (wg, wu))
    mixed = lambda a, b: np.stack([a.reshape(F // 16, 16, -1), b.reshape(F // 16, 16, -1)], axis=1).reshape(2 * F, -1)  # noqa: E731
    assert np.array_equal(element_codes(q), mixed(cg, cu)) and np.array_equal(scale_codes(q), mixed(sg, su))


def quantise_into_ones(ctx, x, other=None):
    """quantize_mxfp4(x), or pack_gated_mxfp4(x, other), into memory that is all ones: scale code 255, a NaN, wherever
    nothing is written."""
    from tenzor_b200 import _lib, ops
    q = ops.Mxfp4(x.shape[0] * (1 if other is None else 2), x.shape[1], x, gated=other is not None)
    q.buf.fill_(255)
    dt, stream = ops._DTF[x.dtype], ops.CUDA_STREAM_LEGACY
    if other is None:
        rc = _lib.lib().tz_quantize_mxfp4(ctx.ptr, x.data_ptr(), q.cols, dt, q.codes_ptr, q.scales_ptr, q.rows, q.cols, stream)
    else:
        rc = _lib.lib().tz_pack_gated_mxfp4(ctx.ptr, x.data_ptr(), other.data_ptr(), dt, q.codes_ptr, q.scales_ptr, x.shape[0], q.cols, stream)
    assert rc == 0
    return q


@pytest.mark.parametrize("K", [32, 64, 96, 160, 224, 288, 1056, 1312])
@pytest.mark.parametrize("M", [3, 20, 40, 300])
def test_scales_past_the_rows_end_and_of_absent_rows(ctx, M, K):
    """Scale bytes of blocks past a row's end are written as 0 (an MMA of 64 values reads one of them where K is an odd
    multiple of 32), and what the scales of absent rows hold reaches no result."""
    from tenzor_b200 import ops
    x, w = rand(M, K, "bf16", M), rand(72, K, "bf16", K)
    wg, wu = (rand(80, K, "bf16", k) * 0.04 for k in (1, 2))
    xq, wq, wp = quantise_into_ones(ctx, x), quantise_into_ones(ctx, w), quantise_into_ones(ctx, wg, wu)
    for q in (xq, wq, wp):
        raw = q.scales.cpu().numpy().reshape(-(-q.rows // 128), -1, 32, 4, 4)  # row block, chunk, row % 32, row / 32, block
        rows = raw.transpose(0, 3, 2, 1, 4).reshape(raw.shape[0] * 128, -1)
        assert (rows[:q.rows, K // 32:] == 0).all() and (rows[q.rows:] == 255).all()
    want, err = product64(x, w)
    for dt in ("f32", "bf16"):
        for a in (x, xq):
            near(ops.linear_mxfp4(ctx, a, wq, out_dtype=DT[dt]), want, err + U[dt] * (want.abs() + err) + TINY[dt])
    near(ops.gated_linear_mxfp4(ctx, x, wp, "silu"), *gated64(x, wg, wu, "silu"))


def test_more_than_2_to_31_elements(ctx):
    from tenzor_b200 import ops
    rows, cols = 1_050_007, 2080
    x = torch.empty((rows, cols), device="cuda", dtype=torch.bfloat16).normal_(generator=torch.Generator(device="cuda").manual_seed(3))
    q = ops.quantize_mxfp4(ctx, x)
    y = ops.dequantize_mxfp4(ctx, q, torch.bfloat16)
    for at in (slice(0, 64), slice(rows - 64, rows)):
        assert np.array_equal(y[at].double().cpu().numpy(), quant64(x[at].float().cpu().numpy())[0])
    del y, q
    M, K, N = 530_001, 96, 4104
    x, w = x.view(-1)[:M * K].view(M, K), rand(N, K, "bf16", 1)
    y = ops.linear_mxfp4(ctx, x, ops.quantize_mxfp4(ctx, w))
    for at in (slice(0, 64), slice(M - 64, M)):
        want, err = product64(x[at], w)
        near(y[at], want, err + U["bf16"] * (want.abs() + err))


@pytest.mark.parametrize("M,K", [(16, 8192), (16, 8448), (17, 8192), (32, 12320), (3, 16384)])
def test_long_rows(ctx, M, K):
    """Row lengths at which x no longer fits the few-rows kernel's shared memory, or only in more splits."""
    from tenzor_b200 import ops
    x, w = rand(M, K, "f16", M, spread=False), (rand(40, K, "f16", 40, spread=False).float() * K ** -0.5).half()
    want, err = product64(x, w)
    tol = err + U["f16"] * (want.abs() + err) + TINY["f16"]
    for times in (1, 500):  # the same 40 weight rows again and again
        y = ops.linear_mxfp4(ctx, x, ops.quantize_mxfp4(ctx, w.repeat(times, 1)))
        near(y, want.repeat(1, times), tol.repeat(1, times), (M, K, times))


@pytest.mark.parametrize("reserve,M,K,N", [(146, 32, 16384, 128), (146, 17, 15872, 800), (130, 20, 16384, 1000), (130, 32, 16640, 1000),
                                           (146, 16, 16384, 128), (146, 2, 32768, 120)])
def test_long_rows_and_few_sms(reserve, M, K, N):
    """So few SMs that a cluster of two would give each CTA more of x than its shared memory holds, or just as much."""
    from tenzor_b200 import ops
    from tenzor_b200.runtime import Context
    c = Context(0)
    c.set_sm_reserve(reserve)
    x, w = rand(M, K, "f16", M, spread=False), (rand(N, K, "f16", N, spread=False).float() * K ** -0.5).half()
    y = ops.linear_mxfp4(c, x, ops.quantize_mxfp4(c, w))
    want, err = product64(x, w)
    near(y, want, err + U["f16"] * (want.abs() + err) + TINY["f16"])
    c.check_status()
    c.close()

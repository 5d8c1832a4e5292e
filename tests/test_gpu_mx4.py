"""MXFP4 rows (wrs_mx4_quantize, wrs_mx4_dequantize) bit for bit against the format's
definition, and the projections with them (wrs_linear_mx4) against float64 products
of the values that the codes stand for."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from gpu_util import host, note

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
E2M1 = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])


@pytest.fixture(scope="module")
def ctx(wrs):
    c = wrs.Context(0)
    c.use_torch_stream()
    return c


def pack_f64(x):
    """Codes and scales of float64 rows, element by element from the definition."""
    rows, cols = x.shape
    b = x.reshape(-1, 32)
    top = np.abs(b).max(axis=1)
    bad = ~np.isfinite(top)
    exp = np.frexp(np.where(bad | (top == 0), 1.0, top))[1] - 1  # floor(log2)
    e = np.where(top == 0, -127, np.maximum(exp - 2, -127))
    y = np.abs(np.where(np.isfinite(b), b, 0.0)) / np.exp2(e.astype(float))[:, None]
    dist = np.abs(y[:, :, None] - E2M1)
    # nearest; of two at one distance the even code
    code = np.argmin(dist + 1e-9 * (np.arange(8) % 2) * (dist > 0), axis=2)
    code += 8 * np.signbit(b)
    code = np.where(bad[:, None], 0, code).reshape(rows, cols).astype(np.uint8)
    scale = np.where(bad, 255, e + 127).astype(np.uint8).reshape(rows, -1)
    return code[:, 0::2] | (code[:, 1::2] << 4), scale


def unpack_f64(codes, scales):
    code = np.stack([codes & 15, codes >> 4], axis=2).reshape(codes.shape[0], -1)
    v = np.where(code & 8, -1.0, 1.0) * E2M1[code & 7]
    s = np.exp2(scales.astype(float) - 127)
    s[scales == 255] = np.nan
    return v * np.repeat(s, 32, axis=1)


def values(rng, rows, cols, kind):
    x = rng.standard_normal((rows, cols))
    if kind == "wide":  # blocks of very different size
        x *= np.exp2(rng.integers(-12, 12, (rows, cols // 32))).repeat(32, axis=1)
    if kind == "edges":  # halfway cases, powers of two, zeros of both signs
        mid = np.array([.25, .75, 1.25, 1.75, 2.5, 3.5, 5, 7, 4, 6, 7.999, 0, -0.0, -.25, -5, 3])
        x = rng.choice(mid, (rows, cols))
        x[0] = 0.0
        x[-1] = -0.0
    return x


@pytest.mark.parametrize("kind", ["normal", "wide", "edges"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (17, 64), (130, 1280), (5, 5120)])
def test_quantize_is_the_definition(wrs, ctx, rows, cols, dtype, kind):
    note(f"mx4_quantize {rows}x{cols} {dtype} {kind}")
    x = torch.from_numpy(values(np.random.default_rng(rows + cols), rows, cols, kind)).to(
        DT[dtype]).cuda()
    got = wrs.mx4_quantize(x, ctx=ctx)
    codes, scales = pack_f64(x.double().cpu().numpy())
    assert np.array_equal(got.scales.cpu().numpy(), scales)
    assert np.array_equal(got.codes.cpu().numpy(), codes)
    back = torch.empty_like(x)
    wrs.mx4_dequantize(got, back, ctx=ctx)
    want = torch.from_numpy(unpack_f64(codes, scales)).to(DT[dtype])
    assert torch.equal(back.cpu(), want)
    assert torch.equal(torch.signbit(back.cpu()), torch.signbit(want))


def test_quantize_at_the_ends_of_f32(wrs, ctx):
    # subnormal blocks (scale 2^-127), the largest finite values, infinities and NaN
    note("mx4_quantize of extreme blocks")
    rng = np.random.default_rng(5)
    x = rng.standard_normal((9, 64)).astype(np.float32)
    x[0] *= np.float32(1e-39)
    x[1] *= np.float32(2.0 ** -126)
    x[2] *= np.float32(2.0 ** -124)
    x[3] = np.sign(x[3]) * np.float32(3.4028235e38)
    x[4, 3] = np.inf
    x[5, 40] = np.nan
    x[6, 63] = -np.inf
    x[7, :32] = np.float32(1e-45)
    x[8, 5] = np.float32(1e38)
    t = torch.from_numpy(x).cuda()
    got = wrs.mx4_quantize(t, ctx=ctx)
    codes, scales = pack_f64(x.astype(np.float64))
    assert np.array_equal(got.scales.cpu().numpy(), scales)
    assert np.array_equal(got.codes.cpu().numpy(), codes)
    back = torch.empty_like(t)
    wrs.mx4_dequantize(got, back, ctx=ctx)
    with np.errstate(over="ignore"):
        want = unpack_f64(codes, scales).astype(np.float32)
    assert np.array_equal(back.cpu().numpy(), want, equal_nan=True)


def test_every_code_and_scale_comes_back(wrs, ctx):
    note("mx4_dequantize of all codes and scales")
    codes = np.tile(np.arange(256, dtype=np.uint8), (256, 1))  # 512 values a row
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 16, axis=1)
    m = wrs.Mx4(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda())
    ref = unpack_f64(codes, scales)
    for dtype in ("f32", "f16", "bf16"):
        out = torch.empty((256, 512), dtype=DT[dtype], device="cuda")
        wrs.mx4_dequantize(m, out, ctx=ctx)
        want = torch.from_numpy(ref).to(DT[dtype])
        got = out.cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want)), dtype
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want)), dtype


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_strided_rows(wrs, ctx, dtype):
    note(f"mx4 strided rows {dtype}")
    wide = torch.randn((37, 264), device="cuda").to(DT[dtype])
    x = wide[:, 8:8 + 192]
    got = wrs.mx4_quantize(x, ctx=ctx)
    same = wrs.mx4_quantize(x.contiguous(), ctx=ctx)
    assert torch.equal(got.codes, same.codes) and torch.equal(got.scales, same.scales)
    out = torch.full((37, 264), 7.0, dtype=DT[dtype], device="cuda")
    wrs.mx4_dequantize(got, out[:, 8:200], ctx=ctx)
    flat = torch.empty((37, 192), dtype=DT[dtype], device="cuda")
    wrs.mx4_dequantize(got, flat, ctx=ctx)
    assert torch.equal(out[:, 8:200], flat)
    assert bool((out[:, :8] == 7).all()) and bool((out[:, 200:] == 7).all())


def gelu(y):
    return 0.5 * y * (1.0 + np.tanh(0.7978846 * y * (1.0 + 0.044715 * y * y)))


def reference(x, w, b, act, out_dtype):
    """Result and how far it may be off: f32 sums of n_in products with operands in up to
    two parts, (n_in + 16) u of the absolute sum; GELU's own arithmetic 16 u of its
    argument (and it stretches an error by at most 1.13); one rounding to the output type,
    half a step, and its smallest step."""
    y = x @ w.T + (b if b is not None else 0.0)
    err = (x.shape[1] + 16) * U32 * (np.abs(x) @ np.abs(w).T + (np.abs(b) if b is not None else 0))
    if act:
        err = 1.13 * err + 16 * U32 * np.abs(y)
        y = gelu(y)
    tiny = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}[out_dtype]
    return y, err + (np.abs(y) + err) * HALF_STEP[out_dtype] + tiny


def make(wrs, ctx, rng, n_out, n_in, spread=0):
    w = rng.standard_normal((n_out, n_in)) * n_in ** -0.5
    if spread:
        w *= np.exp2(rng.integers(-spread, spread + 1, (n_out, n_in // 32))).repeat(32, axis=1)
    m = wrs.mx4_quantize(torch.from_numpy(w.astype(np.float32)).cuda(), ctx=ctx)
    return m, unpack_f64(m.codes.cpu().numpy(), m.scales.cpu().numpy())


def run(wrs, ctx, x_dtype, rows, n_in, n_out, groups=1, out="f32", act=None, bias=True, seed=0,
        spread=0):
    rng = np.random.default_rng(seed + rows + n_in + n_out)
    ws = [make(wrs, ctx, rng, n_out, n_in, spread) for _ in range(groups)]
    x = torch.from_numpy(rng.standard_normal((rows, n_in)).astype(np.float32)).cuda()
    if x_dtype == "mx4":
        x = wrs.mx4_quantize(x, ctx=ctx)
        ref = unpack_f64(x.codes.cpu().numpy(), x.scales.cpu().numpy())
    else:
        x = x.to(DT[x_dtype])
        ref = x.double().cpu().numpy()
    bs = [rng.standard_normal(n_out).astype(np.float32) if bias and g != 1 else None
          for g in range(groups)]
    outs = [torch.full((rows, n_out), float("nan"), dtype=DT[out], device="cuda")
            for _ in range(groups)]
    wrs.linear_mx4(x, [w for w, _ in ws],
                   [None if b is None else torch.from_numpy(b).cuda() for b in bs] if bias else None,
                   outs, act=act, ctx=ctx)
    for (_, w), b, o in zip(ws, bs, outs):
        y, tol = reference(ref, w, None if b is None else b.astype(np.float64), act, out)
        err = np.abs(host(o).astype(np.float64) - y)
        assert np.all(err <= tol), (float(err.max()), float((err / tol).max()))


@pytest.mark.parametrize("x_dtype", ["f32", "f16", "bf16", "mx4"])
@pytest.mark.parametrize("rows", [1, 2, 5, 6, 8, 9, 11, 16, 17, 33, 64, 129, 300])
def test_rows(wrs, ctx, rows, x_dtype):
    note(f"linear_mx4 rows={rows} {x_dtype}")
    run(wrs, ctx, x_dtype, rows, 256, 192)


@pytest.mark.parametrize("x_dtype", ["f32", "f16", "bf16", "mx4"])
@pytest.mark.parametrize("rows", [3, 40])
@pytest.mark.parametrize("n_in,n_out", [(64, 1), (64, 7), (128, 65), (192, 16), (320, 50),
                                        (1280, 129), (5120, 33), (448, 515)])
def test_shapes(wrs, ctx, n_in, n_out, rows, x_dtype):
    note(f"linear_mx4 {rows} x {n_in} -> {n_out} {x_dtype}")
    run(wrs, ctx, x_dtype, rows, n_in, n_out, seed=1)


@pytest.mark.parametrize("x_dtype", ["f32", "f16", "bf16", "mx4"])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [4, 70])
def test_outputs_groups_and_gelu(wrs, ctx, rows, out, x_dtype):
    note(f"linear_mx4 groups and gelu, {rows} rows {x_dtype} -> {out}")
    run(wrs, ctx, x_dtype, rows, 192, 100, groups=3, out=out, act="gelu", seed=2)
    run(wrs, ctx, x_dtype, rows, 192, 128, groups=8, out=out, bias=False, seed=3)


@pytest.mark.parametrize("x_dtype", ["f32", "f16", "bf16", "mx4"])
@pytest.mark.parametrize("rows", [1, 6, 10, 12, 16])
@pytest.mark.parametrize("n_in,n_out,groups", [(1280, 1280, 3), (5120, 1280, 1), (8192, 16, 1),
                                               (512, 40000, 1), (2624, 20000, 1)])
def test_few_rows_of_every_grid(wrs, ctx, n_in, n_out, groups, rows, x_dtype):
    # small and large grids, x whole in LDS or in pieces
    note(f"linear_mx4 {rows} x {n_in} -> {n_out} x {groups} {x_dtype}")
    run(wrs, ctx, x_dtype, rows, n_in, n_out, groups=groups, seed=6)


@pytest.mark.parametrize("x_dtype", ["f32", "f16", "bf16", "mx4"])
@pytest.mark.parametrize("rows", [5, 150])
def test_large_product(wrs, ctx, rows, x_dtype):
    note(f"linear_mx4 {rows} x 1280 -> 5120 {x_dtype}")
    run(wrs, ctx, x_dtype, rows, 1280, 5120, seed=4)


@pytest.mark.parametrize("x_dtype", ["f32", "f16", "bf16", "mx4"])
@pytest.mark.parametrize("rows", [3, 50])
@pytest.mark.parametrize("spread", [8, 40])
def test_scales_of_very_different_blocks(wrs, ctx, spread, rows, x_dtype):
    note(f"linear_mx4 scales spread by 2^{2 * spread}, {rows} rows {x_dtype}")
    run(wrs, ctx, x_dtype, rows, 256, 70, spread=spread, seed=5)


@pytest.mark.parametrize("x_dtype", ["f32", "f16", "bf16", "mx4"])
@pytest.mark.parametrize("rows", [3, 50])
def test_small_weights_that_decide(wrs, ctx, rows, x_dtype):
    # Each row of weights has one block 2^60 above the others, which meets x of zero: the
    # result is the small blocks' alone.
    note(f"linear_mx4 small weights, {rows} rows {x_dtype}")
    rng = np.random.default_rng(6)
    n_in, n_out = 256, 70
    w = rng.standard_normal((n_out, n_in))
    w[:, 64:96] *= 2.0 ** 60
    x = rng.standard_normal((rows, n_in))
    x[:, 64:96] = 0.0
    m = wrs.mx4_quantize(torch.from_numpy(w.astype(np.float32)).cuda(), ctx=ctx)
    xt = torch.from_numpy(x.astype(np.float32)).cuda()
    if x_dtype == "mx4":
        xt = wrs.mx4_quantize(xt, ctx=ctx)
        xr = unpack_f64(xt.codes.cpu().numpy(), xt.scales.cpu().numpy())
    else:
        xt = xt.to(DT[x_dtype])
        xr = xt.double().cpu().numpy()
    out = torch.empty((rows, n_out), device="cuda")
    wrs.linear_mx4(xt, [m], None, [out], ctx=ctx)
    y, tol = reference(xr, unpack_f64(m.codes.cpu().numpy(), m.scales.cpu().numpy()), None, None,
                       "f32")
    assert np.all(np.abs(host(out) - y) <= tol)


@pytest.mark.parametrize("x_dtype", ["f32", "bf16", "mx4"])
@pytest.mark.parametrize("rows", [2, 40])
def test_very_large_and_small_scales(wrs, ctx, rows, x_dtype):
    # rows of weights at 2^-100 .. 2^100 (x at 1): results of the same size
    note(f"linear_mx4 rows of weights from 2^-100 to 2^100, {rows} rows {x_dtype}")
    rng = np.random.default_rng(8)
    n_in, n_out = 128, 41
    size = np.exp2(np.linspace(-100, 100, n_out).round())
    w = rng.standard_normal((n_out, n_in)) * size[:, None]
    m = wrs.mx4_quantize(torch.from_numpy(w.astype(np.float32)).cuda(), ctx=ctx)
    xt = torch.from_numpy(rng.standard_normal((rows, n_in)).astype(np.float32)).cuda()
    if x_dtype == "mx4":
        xt = wrs.mx4_quantize(xt, ctx=ctx)
        xr = unpack_f64(xt.codes.cpu().numpy(), xt.scales.cpu().numpy())
    else:
        xt = xt.to(DT[x_dtype])
        xr = xt.double().cpu().numpy()
    out = torch.empty((rows, n_out), device="cuda")
    wrs.linear_mx4(xt, [m], None, [out], ctx=ctx)
    y, tol = reference(xr, unpack_f64(m.codes.cpu().numpy(), m.scales.cpu().numpy()), None, None,
                       "f32")
    assert np.all(np.abs(host(out) - y) <= tol)


@pytest.mark.parametrize("x_dtype", ["f32", "f16", "bf16", "mx4"])
@pytest.mark.parametrize("rows", [3, 40])
def test_nan_and_infinity_stay_in_their_rows(wrs, ctx, rows, x_dtype):
    # a NaN scale reaches its output feature alone, a non-finite row of x its own row
    note(f"linear_mx4 with NaN, {rows} rows {x_dtype}")
    rng = np.random.default_rng(9)
    n_in, n_out = 192, 70
    w = rng.standard_normal((n_out, n_in)).astype(np.float32)
    w[11, 100] = np.nan
    x = rng.standard_normal((rows, n_in)).astype(np.float32)
    x[1, 7] = np.inf
    m = wrs.mx4_quantize(torch.from_numpy(w).cuda(), ctx=ctx)
    xt = torch.from_numpy(x).cuda()
    xt = wrs.mx4_quantize(xt, ctx=ctx) if x_dtype == "mx4" else xt.to(DT[x_dtype])
    out = torch.empty((rows, n_out), device="cuda")
    wrs.linear_mx4(xt, [m], None, [out], ctx=ctx)
    got = host(out)
    assert np.all(np.isnan(got[:, 11]))
    assert not np.any(np.isfinite(got[1]))
    keep_r = [i for i in range(rows) if i != 1]
    keep_c = [i for i in range(n_out) if i != 11]
    assert np.all(np.isfinite(got[np.ix_(keep_r, keep_c)]))


@pytest.mark.parametrize("x_dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [5, 90])
def test_strided_input_and_head_major_output(wrs, ctx, rows, x_dtype):
    note(f"linear_mx4 strides, {rows} rows {x_dtype}")
    rng = np.random.default_rng(10)
    n_in, n_out = 128, 200  # 4 heads of 64, the last of 8
    m, w = make(wrs, ctx, rng, n_out, n_in)
    wide = torch.from_numpy(rng.standard_normal((rows, 3 * n_in)).astype(np.float32)).to(
        DT[x_dtype]).cuda()
    x = wide[:, n_in:2 * n_in]
    hs = rows * 64 + 32
    out = torch.full((4 * hs + 5,), 7.0, device="cuda")
    wrs.linear_mx4(x, [m], None, [out], out_row_stride=64, out_head_stride=hs, ctx=ctx)
    y, tol = reference(x.double().cpu().numpy(), w, None, None, "f32")
    got = host(out)
    seen = np.zeros(got.size, bool)
    for h in range(4):
        n = min(64, n_out - 64 * h)
        at = h * hs + 64 * np.arange(rows)[:, None] + np.arange(n)
        seen[at] = True
        assert np.all(np.abs(got[at] - y[:, 64 * h:64 * h + n]) <= tol[:, 64 * h:64 * h + n])
    assert np.all(got[~seen] == 7.0)


@pytest.mark.parametrize("x_dtype", ["f32", "f16", "mx4"])
@pytest.mark.parametrize("rows", [4, 64])
def test_odd_places_of_out_and_bias(wrs, ctx, rows, x_dtype):
    # out and bias at any element, rows of odd length
    note(f"linear_mx4 unaligned out and bias, {rows} rows {x_dtype}")
    rng = np.random.default_rng(12)
    n_in, n_out = 128, 67
    m, w = make(wrs, ctx, rng, n_out, n_in)
    x = torch.from_numpy(rng.standard_normal((rows, n_in)).astype(np.float32)).cuda()
    xr = x.double().cpu().numpy()
    if x_dtype == "mx4":
        x = wrs.mx4_quantize(x, ctx=ctx)
        xr = unpack_f64(x.codes.cpu().numpy(), x.scales.cpu().numpy())
    elif x_dtype == "f16":
        x = x.half()
        xr = x.double().cpu().numpy()
    b = rng.standard_normal(n_out + 1).astype(np.float32)
    bias = torch.from_numpy(b).cuda()[1:]
    for out in ("f32", "f16"):
        buf = torch.full((rows * (n_out + 2) + 3,), 7.0, dtype=DT[out], device="cuda")
        wrs.linear_mx4(x, [m], [bias], [buf[1:]], out_row_stride=n_out + 2, ctx=ctx)
        got = host(buf)
        y, tol = reference(xr, w, b[1:].astype(np.float64), None, out)
        at = 1 + (n_out + 2) * np.arange(rows)[:, None] + np.arange(n_out)
        assert np.all(np.abs(got[at] - y) <= tol)
        rest = np.ones(got.size, bool)
        rest[at] = False
        assert np.all(got[rest] == 7.0)


def test_captured_and_replayed(wrs):
    note("linear_mx4 and mx4_quantize captured")
    c = wrs.Context(0)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        c.use_torch_stream()
        rng = np.random.default_rng(14)
        for rows, x_dtype in ((5, "f32"), (100, "f32"), (100, "f16"), (100, "mx4")):
            m, w = make(wrs, c, rng, 320, 256)
            x = torch.empty((rows, 256), dtype=torch.float16 if x_dtype == "f16" else torch.float32,
                            device="cuda")
            packed = wrs.Mx4.empty(rows, 256)
            out = torch.empty((rows, 320), device="cuda")

            def call(o):
                src = wrs.mx4_quantize(x, packed, ctx=c) if x_dtype == "mx4" else x
                wrs.linear_mx4(src, [m], None, [o], ctx=c)

            side.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                call(out)
            for _ in range(4):
                x.copy_(torch.randn(rows, 256))
                out.fill_(float("nan"))
                g.replay()
                side.synchronize()
                eager = torch.empty_like(out)
                call(eager)
                side.synchronize()
                assert torch.equal(out, eager)
    c.close()


def test_empty_calls(wrs, ctx):
    note("linear_mx4 of nothing")
    m = wrs.mx4_quantize(torch.randn((4, 64), device="cuda"), ctx=ctx)
    wrs.linear_mx4(torch.empty((0, 64), device="cuda"), [m], None,
                   [torch.empty((0, 4), device="cuda")], ctx=ctx)
    e = wrs.mx4_quantize(torch.empty((0, 64), device="cuda"), ctx=ctx)
    assert e.shape == (0, 64)
    wrs.mx4_dequantize(e, torch.empty((0, 64), device="cuda"), ctx=ctx)


def test_refusals(wrs, ctx):
    note("mx4 refusals (no launch)")
    x = torch.randn((4, 96), device="cuda")
    with pytest.raises(AssertionError):  # not a multiple of 32
        wrs.mx4_quantize(torch.randn((4, 40), device="cuda"), ctx=ctx)
    with pytest.raises(TypeError):
        wrs.mx4_quantize(x.double(), ctx=ctx)
    with pytest.raises(TypeError):
        wrs.mx4_quantize(x.T, ctx=ctx)
    with pytest.raises(TypeError):
        wrs.mx4_quantize(x.cpu(), wrs.Mx4.empty(4, 96), ctx=ctx)
    with pytest.raises(RuntimeError):  # rows off 16 bytes
        wrs.mx4_quantize(torch.randn((4, 97), device="cuda")[:, :96], ctx=ctx)
    with pytest.raises(AssertionError):
        wrs.mx4_quantize(x, wrs.Mx4.empty(3, 96), ctx=ctx)
    m = wrs.mx4_quantize(x, ctx=ctx)
    out = torch.empty((4, 4), device="cuda")
    with pytest.raises(RuntimeError):  # n_in % 64
        wrs.linear_mx4(x, [m], None, [out], ctx=ctx)
    w = wrs.mx4_quantize(torch.randn((4, 128), device="cuda"), ctx=ctx)
    x = torch.randn((4, 128), device="cuda")
    with pytest.raises(AssertionError):  # out too short
        wrs.linear_mx4(x, [w], None, [torch.empty((3, 4), device="cuda")], ctx=ctx)
    with pytest.raises(AssertionError):  # widths
        wrs.linear_mx4(x[:, :64], [w], None, [out], ctx=ctx)
    with pytest.raises(AssertionError):  # groups
        wrs.linear_mx4(x, [w] * 9, None, [out] * 9, ctx=ctx)
    with pytest.raises(AssertionError):  # bias
        wrs.linear_mx4(x, [w], [torch.zeros(5, device="cuda")], [out], ctx=ctx)
    with pytest.raises(TypeError):
        wrs.linear_mx4(x, [w], None, [out.cpu()], ctx=ctx)
    with pytest.raises(KeyError):
        wrs.linear_mx4(x, [w], None, [out], act="tanh", ctx=ctx)
    with pytest.raises(RuntimeError):  # x rows off 16 bytes
        wrs.linear_mx4(torch.randn((4, 129), device="cuda")[:, :128], [w], None, [out], ctx=ctx)
    with pytest.raises(AssertionError):  # negative stride
        wrs.linear_mx4(x, [w], None, [out], out_row_stride=-4, ctx=ctx)


def test_addresses_and_strides_that_are_refused(wrs, ctx):
    """Scales at odd bytes, rows whose last one lies at 2^64 and beyond (no launch)."""
    w = wrs.mx4_quantize(torch.randn((4, 128), device="cuda"), ctx=ctx)
    x = torch.randn((4, 128), device="cuda")
    out = torch.empty((4, 4), device="cuda")
    odd = torch.empty(64, device="cuda", dtype=torch.uint8)[1:17].view(4, 4)
    shifted = wrs.Mx4(w.codes, odd)
    for rows, weights in ((x, shifted), (shifted, w)):
        with pytest.raises(RuntimeError):
            wrs.linear_mx4(rows, [weights], None, [out], ctx=ctx)
    lib = wrs._lib.lib()
    p, q, s = (ctypes.c_void_p(t.data_ptr()) for t in (x, w.codes, w.scales))
    wraps = 6148914691236517208  # three times it is 2^64 + 8
    for stride in (2**62, wraps):
        assert lib.wrs_mx4_quantize(ctx.handle, 0, p, 512, stride, 4, 128, q, 256, s, 16) < 0
        assert lib.wrs_mx4_dequantize(ctx.handle, q, 256, s, 16, 4, 128, 0, p, 512, stride) < 0
        ws, ss = (ctypes.c_void_p * 1)(q.value), (ctypes.c_void_p * 1)(s.value)
        o, n = (ctypes.c_void_p * 1)(out.data_ptr()), (ctypes.c_size_t * 1)(16)
        assert lib.wrs_linear_mx4(ctx.handle, 0, p, None, 512, stride, 1, ws, ss, None, 4, 128, 4,
                                  0, 0, o, n, 4, 64) < 0
        assert lib.wrs_linear_mx4(ctx.handle, 0, p, None, 512, 128, 1, ws, ss, None, 4, 128, 4,
                                  0, 0, o, n, stride, 64) < 0
        assert lib.wrs_linear_mx4(ctx.handle, 0, p, None, 512, 128, 1, ws, ss, None, 4, 128, 4,
                                  0, 0, o, n, 4, 64) == 0
    torch.cuda.synchronize()


@pytest.mark.parametrize("rows,n_in,n_out,groups,x_dtype", [
    (5, 5120, 1280, 1, "f32"), (16, 5120, 1280, 1, "f32"), (7, 4096, 1031, 1, "f16"),
    (16, 1600, 48, 3, "f32"), (13, 5056, 17, 5, "f32"), (16, 5120, 2048, 1, "bf16"),
    (16, 65536, 16, 1, "f32"),
])
def test_long_rows_whose_columns_split(wrs, ctx, rows, n_in, n_out, groups, x_dtype):
    """Few rows over few features and many columns; the splits are the same ones each time."""
    note(f"linear_mx4 {rows} x {n_in} -> {n_out} x {groups} {x_dtype}, split")
    run(wrs, ctx, x_dtype, rows, n_in, n_out, groups=groups, act="gelu", seed=8)
    x = torch.randn((rows, n_in), device="cuda").to(DT[x_dtype])
    ws = [wrs.mx4_quantize(torch.randn((n_out, n_in), device="cuda"), ctx=ctx)
          for _ in range(groups)]
    outs = [[torch.empty((rows, n_out), device="cuda") for _ in ws] for _ in range(4)]
    for o in outs:
        wrs.linear_mx4(x, ws, None, o, ctx=ctx)
    torch.cuda.synchronize()
    for o in outs[1:]:
        for a, b in zip(outs[0], o):
            assert torch.equal(a, b)


def test_long_rows_captured_before_and_after_the_scratch(wrs):
    """A context's first call, captured, finds no scratch and sums in one piece; the graphs
    captured later split, and share scratch and counters with each other and eager calls."""
    note("linear_mx4 5 x 5120 -> 128, captured before any eager call")
    c = wrs.Context(0)
    side = torch.cuda.Stream()
    rng = np.random.default_rng(15)
    with torch.cuda.stream(side):
        c.use_torch_stream()
        m, w = make(wrs, c, rng, 128, 5120)
        x = torch.empty((5, 5120), device="cuda")
        outs = [torch.empty((5, 128), device="cuda") for _ in range(3)]
        eager = torch.empty((5, 128), device="cuda")
        side.synchronize()
        graphs = []
        for i, o in enumerate(outs):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                wrs.linear_mx4(x, [m], None, [o], ctx=c)
            graphs.append(g)
            if i == 0:
                wrs.linear_mx4(x, [m], None, [eager], ctx=c)
                side.synchronize()
        for _ in range(4):
            x.copy_(torch.from_numpy(rng.standard_normal((5, 5120)).astype(np.float32)))
            for o in outs:
                o.fill_(float("nan"))
            for g in graphs + graphs[1:]:
                g.replay()
            wrs.linear_mx4(x, [m], None, [eager], ctx=c)
            side.synchronize()
            y, tol = reference(x.double().cpu().numpy(), w, None, None, "f32")
            assert np.all(np.abs(host(outs[0]).astype(np.float64) - y) <= tol)
            assert torch.equal(outs[1], eager) and torch.equal(outs[2], eager)
            assert np.all(np.abs(host(eager).astype(np.float64) - y) <= tol)
    c.close()


def test_new_rows_for_a_context_on_another_stream(wrs):
    """A new Mx4's memory may still be written by torch's stream when it is allocated."""
    note("mx4_quantize into new rows, the context on its own stream")
    c = wrs.Context(0)
    x = torch.randn((4096, 4096), device="cuda")
    want = wrs.Mx4.empty(4096, 4096)
    torch.cuda.synchronize()
    wrs.mx4_quantize(x, want, ctx=c)
    torch.cuda.synchronize()
    before = torch.empty((4096, 2048), dtype=torch.uint8, device="cuda")
    for i in range(300):
        before.fill_(i % 7)
    del before
    got = wrs.mx4_quantize(x, ctx=c)
    torch.cuda.synchronize()
    assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
    c.close()


@pytest.mark.parametrize("x_dtype", ["f32", "f16", "bf16", "mx4"])
@pytest.mark.parametrize("n_in", [64, 192, 320, 576])
@pytest.mark.parametrize("rows,n_out", [(130, 3850), (1500, 1530), (2100, 2500)])
def test_tiles_of_every_size_at_their_edges(wrs, ctx, rows, n_out, n_in, x_dtype):
    """Tiles of 64 x 64, 128 x 128 and 256 x 128, whole ones and the last, over few columns."""
    note(f"linear_mx4 {rows} x {n_in} -> {n_out} {x_dtype}")
    run(wrs, ctx, x_dtype, rows, n_in, n_out, out="f16" if n_in == 192 else "f32",
        act="gelu" if n_in == 320 else None, seed=16)


@pytest.mark.parametrize("x_dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows,n_out", [(130, 3850), (1500, 1530), (2100, 2500)])
def test_large_tiles_formed_again(wrs, ctx, rows, n_out, x_dtype):
    """A row of x and a feature's scales that 16-bit operands of a tile cannot hold."""
    note(f"linear_mx4 {rows} x 256 -> {n_out} {x_dtype}, values out of f16's range")
    rng = np.random.default_rng(17)
    w = rng.standard_normal((n_out, 256)) / 16
    w[77] *= 2.0 ** 40
    w[-1] *= 2.0 ** -50
    m = wrs.mx4_quantize(torch.from_numpy(w.astype(np.float32)).cuda(), ctx=ctx)
    wf = unpack_f64(m.codes.cpu().numpy(), m.scales.cpu().numpy())
    x = rng.standard_normal((rows, 256)).astype(np.float32)
    if x_dtype == "f32":
        x[5] *= 2.0 ** 60
        x[-1] *= 2.0 ** -70
    xt = torch.from_numpy(x).cuda().to(DT[x_dtype])
    out = torch.full((rows, n_out), float("nan"), device="cuda")
    wrs.linear_mx4(xt, [m], None, [out], ctx=ctx)
    y, tol = reference(xt.double().cpu().numpy(), wf, None, None, "f32")
    err = np.abs(host(out).astype(np.float64) - y)
    assert np.all(err <= tol), (float(err.max()), float((err / tol).max()))


def test_rows_between_the_outputs_stay(wrs, ctx):
    """Whole tiles stored into wider rows write nothing beside them."""
    note("linear_mx4 2100 x 128 -> 2560 into rows of 2600")
    m = wrs.mx4_quantize(torch.randn((2560, 128), device="cuda"), ctx=ctx)
    x = torch.randn((2100, 128), device="cuda").half()
    wide = torch.full((2101, 2600), 7.0, device="cuda", dtype=torch.float16)
    flat = torch.empty((2100, 2560), device="cuda", dtype=torch.float16)
    wrs.linear_mx4(x, [m], None, [wide], out_row_stride=2600, ctx=ctx)
    wrs.linear_mx4(x, [m], None, [flat], ctx=ctx)
    assert torch.equal(wide[:2100, :2560], flat)
    assert bool((wide[:, 2560:] == 7).all()) and bool((wide[2100] == 7).all())


@pytest.mark.parametrize("rows,n_in,n_out,groups,x_dtype", [
    (17, 5120, 1280, 1, "f32"), (64, 5120, 1280, 1, "f16"), (130, 5120, 1280, 1, "f32"),
    (33, 2112, 500, 3, "f32"), (90, 4160, 77, 2, "bf16"), (20, 65536, 16, 1, "f32"),
    (40, 5056, 1, 8, "f16"),
])
def test_small_tiles_whose_columns_split(wrs, ctx, rows, n_in, n_out, groups, x_dtype):
    """Tiles over few features and many columns; the splits are the same ones each time."""
    note(f"linear_mx4 {rows} x {n_in} -> {n_out} x {groups} {x_dtype}, tiles split")
    run(wrs, ctx, x_dtype, rows, n_in, n_out, groups=groups, act="gelu", seed=18)
    x = torch.randn((rows, n_in), device="cuda")
    if x_dtype == "f32":
        x[3] *= 2.0 ** 40  # one split's range is another's too: a tile formed again in all
    x = x.to(DT[x_dtype])
    ws = [wrs.mx4_quantize(torch.randn((n_out, n_in), device="cuda"), ctx=ctx)
          for _ in range(groups)]
    outs = [[torch.empty((rows, n_out), device="cuda") for _ in ws] for _ in range(4)]
    for o in outs:
        wrs.linear_mx4(x, ws, None, o, ctx=ctx)
    torch.cuda.synchronize()
    for o in outs[1:]:
        for a, b in zip(outs[0], o):
            assert torch.equal(a, b)
    for w, o in zip(ws, outs[0]):
        y, tol = reference(x.double().cpu().numpy(),
                           unpack_f64(w.codes.cpu().numpy(), w.scales.cpu().numpy()), None, None,
                           "f32")
        assert np.all(np.abs(host(o).astype(np.float64) - y) <= tol)


def test_split_tiles_captured(wrs):
    note("linear_mx4 40 x 5120 -> 192, captured before and after an eager call")
    c = wrs.Context(0)
    side = torch.cuda.Stream()
    rng = np.random.default_rng(19)
    with torch.cuda.stream(side):
        c.use_torch_stream()
        m, w = make(wrs, c, rng, 192, 5120)
        x = torch.empty((40, 5120), device="cuda")
        outs = [torch.empty((40, 192), device="cuda") for _ in range(3)]
        eager = torch.empty((40, 192), device="cuda")
        side.synchronize()
        graphs = []
        for i, o in enumerate(outs):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                wrs.linear_mx4(x, [m], None, [o], ctx=c)
            graphs.append(g)
            if i == 0:
                wrs.linear_mx4(x, [m], None, [eager], ctx=c)
                side.synchronize()
        for _ in range(4):
            x.copy_(torch.from_numpy(rng.standard_normal((40, 5120)).astype(np.float32)))
            for o in outs:
                o.fill_(float("nan"))
            for g in graphs + graphs[1:]:
                g.replay()
            wrs.linear_mx4(x, [m], None, [eager], ctx=c)
            side.synchronize()
            y, tol = reference(x.double().cpu().numpy(), w, None, None, "f32")
            assert np.all(np.abs(host(outs[0]).astype(np.float64) - y) <= tol)
            assert torch.equal(outs[1], eager) and torch.equal(outs[2], eager)
            assert np.all(np.abs(host(eager).astype(np.float64) - y) <= tol)
    c.close()


@pytest.mark.parametrize("x_dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("octaves", [20, 25])
@pytest.mark.parametrize("rows,n_out", [(3, 70), (17, 70), (50, 70), (130, 3850), (1500, 1530),
                                        (2100, 2500)])
def test_small_x_that_decides(wrs, ctx, rows, n_out, octaves, x_dtype):
    """The large values of every row of x meet weights of 0 (in blocks with others): the result
    is the small values' alone, 2^-octaves of them. Two parts of f32 x leave 2^-22 of a value,
    which reference() counts, or 2^-43."""
    note(f"linear_mx4 {rows} x 256 -> {n_out} {x_dtype}, x at 2^-{octaves} beside large values")
    rng = np.random.default_rng(20)
    w = rng.standard_normal((n_out, 256)) / 16
    w[:, 64:72] = w[:, 250:] = 0.0
    m = wrs.mx4_quantize(torch.from_numpy(w.astype(np.float32)).cuda(), ctx=ctx)
    x = rng.standard_normal((rows, 256)).astype(np.float32)
    small = np.ones(256, bool)
    small[64:72] = small[250:] = False
    x[:, small] *= np.float32(2.0 ** -octaves)
    x[:, ~small] *= 30
    xt = torch.from_numpy(x).cuda().to(DT[x_dtype])
    out = torch.full((rows, n_out), float("nan"), device="cuda")
    wrs.linear_mx4(xt, [m], None, [out], ctx=ctx)
    wf = unpack_f64(m.codes.cpu().numpy(), m.scales.cpu().numpy())
    y, tol = reference(xt.double().cpu().numpy(), wf, None, None, "f32")
    if x_dtype == "f32":
        tol = tol + 2.0 ** -43 * np.abs(wf).sum(axis=1)
    err = np.abs(host(out).astype(np.float64) - y)
    assert np.all(err <= tol), (float(err.max()), float((err / tol).max()))


@pytest.mark.parametrize("x_dtype", ["f32", "f16", "bf16", "mx4"])
@pytest.mark.parametrize("rows,n_out", [(3, 70), (50, 70), (130, 3850), (1500, 1530), (2100, 2500)])
def test_blocks_of_zeros_leave_the_others_alone(wrs, ctx, rows, n_out, x_dtype):
    """Padded columns and pruned rows: blocks of zeros, which quantise to the scale 2^-127. The
    results are bit for bit those of the same zeros under a scale of 1."""
    note(f"linear_mx4 {rows} x 256 -> {n_out} {x_dtype}, blocks of zeros")
    rng = np.random.default_rng(21)
    w = rng.standard_normal((n_out, 256)) / 16
    w[:, 224:] = 0.0
    w[5] = w[n_out - 1] = 0.0
    w[:, 32:64] *= rng.random((n_out, 1)) < 0.5
    w[9, 64:96] = -0.0
    m = wrs.mx4_quantize(torch.from_numpy(w.astype(np.float32)).cuda(), ctx=ctx)
    other = wrs.Mx4(m.codes, torch.where(m.scales == 0, 127, m.scales).to(torch.uint8))
    assert int((m.scales == 0).sum()) > n_out
    x = torch.from_numpy(rng.standard_normal((rows, 256)).astype(np.float32)).cuda()
    if x_dtype == "mx4":
        x = wrs.mx4_quantize(x, ctx=ctx)
        xr = unpack_f64(x.codes.cpu().numpy(), x.scales.cpu().numpy())
    else:
        x = x.to(DT[x_dtype])
        xr = x.double().cpu().numpy()
    outs = [torch.full((rows, n_out), float("nan"), device="cuda") for _ in range(2)]
    for weights, out in zip((m, other), outs):
        wrs.linear_mx4(x, [weights], None, [out], ctx=ctx)
    y, tol = reference(xr, unpack_f64(m.codes.cpu().numpy(), m.scales.cpu().numpy()), None, None,
                       "f32")
    for out in outs:
        assert np.all(np.abs(host(out).astype(np.float64) - y) <= tol)
    assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("x_dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("byte", [1, 114, 115, 133, 200, 247, 254, 255])
@pytest.mark.parametrize("rows", [3, 50])
def test_zeros_under_any_scale(wrs, ctx, rows, byte, x_dtype):
    """A block of zeros is 0 under every scale but the NaN, which stays one."""
    note(f"linear_mx4 {rows} rows {x_dtype}, zeros under the scale byte {byte}")
    rng = np.random.default_rng(22)
    w = rng.standard_normal((70, 128)) / 8
    w[11, 32:64] = 0.0
    m = wrs.mx4_quantize(torch.from_numpy(w.astype(np.float32)).cuda(), ctx=ctx)
    m.scales[11, 1] = byte
    x = torch.from_numpy(rng.standard_normal((rows, 128)).astype(np.float32)).cuda().to(DT[x_dtype])
    out = torch.full((rows, 70), float("nan"), device="cuda")
    wrs.linear_mx4(x, [m], None, [out], ctx=ctx)
    y, tol = reference(x.double().cpu().numpy(),
                       unpack_f64(m.codes.cpu().numpy(), m.scales.cpu().numpy()), None, None, "f32")
    got = host(out).astype(np.float64)
    if byte == 255:
        assert np.all(np.isnan(got[:, 11]))
        got[:, 11] = y[:, 11] = tol[:, 11] = 0.0
    assert np.all(np.abs(got - y) <= tol)


@pytest.mark.parametrize("x_dtype", ["f32", "f16", "bf16", "mx4"])
@pytest.mark.parametrize("rows,n_in,n_out,groups", [
    (5, 64, 512, 1), (16, 256, 512, 1), (5, 1280, 5120, 1), (8, 1280, 51866, 1),  # the stream
    (16, 1600, 48, 3), (5, 5120, 1280, 1), (16, 5120, 1280, 1), (16, 65536, 16, 1),  # split
    (40, 64, 512, 1), (33, 256, 70, 1), (130, 1280, 1280, 3), (1500, 1280, 1530, 1),  # tiles
    (2100, 256, 2500, 1), (300, 5120, 5120, 1),
    (33, 2112, 500, 3), (17, 5120, 1280, 1), (130, 5120, 1280, 1), (20, 65536, 16, 1),  # split
])
def test_norm_of_the_error(wrs, ctx, rows, n_in, n_out, groups, x_dtype):
    """The whole result's error against its norm, which unlike a bound of the absolute sums sees
    a part of x that is lost. Roundings of random terms add in squares: each of the n f32 sums is
    off by u / sqrt(3) of what it holds then, sqrt(k / n) of the result after k products, and the
    operands of each product by 2^-22 / sqrt(3): sqrt(n / 6 + 16 / 3) u, here twice that (one
    f16 part alone leaves about 2e-4, two bf16 parts 4e-6)."""
    note(f"linear_mx4 {rows} x {n_in} -> {n_out} x {groups} {x_dtype}, norm of the error")
    rng = np.random.default_rng(23)
    x = torch.from_numpy(rng.standard_normal((rows, n_in)).astype(np.float32)).cuda()
    if x_dtype == "mx4":
        x = wrs.mx4_quantize(x, ctx=ctx)
        xr = unpack_f64(x.codes.cpu().numpy(), x.scales.cpu().numpy())
    else:
        x = x.to(DT[x_dtype])
        xr = x.double().cpu().numpy()
    ws = [make(wrs, ctx, rng, n_out, n_in) for _ in range(groups)]
    outs = [torch.full((rows, n_out), float("nan"), device="cuda") for _ in ws]
    wrs.linear_mx4(x, [w for w, _ in ws], None, outs, ctx=ctx)
    for (_, w), out in zip(ws, outs):
        y = xr @ w.T
        off = np.linalg.norm(host(out).astype(np.float64) - y) / np.linalg.norm(y)
        assert off <= 2 * U32 * np.sqrt(n_in / 6 + 16 / 3), off


@pytest.mark.parametrize("x_dtype", ["f32", "f16", "bf16", "mx4"])
@pytest.mark.parametrize("rows", [1, 5, 16, 17, 130, 2100])
def test_gelu_is_one_function_for_any_rows(wrs, ctx, rows, x_dtype):
    """GELU of numbers that the products give exactly, small results among them, relative to
    themselves: x / (1 + exp(-2 u)) is off by its exponential's argument, whose constants and
    four operations round, 6 u of 2 u(x), and by a few roundings of the rest."""
    note(f"linear_mx4 {rows} rows {x_dtype}, gelu")
    w = torch.zeros((640, 64), device="cuda")
    w[:, 3] = torch.arange(640, device="cuda") % 3 - 1.0
    m = wrs.mx4_quantize(w, ctx=ctx)
    x = torch.zeros((rows, 64), device="cuda")
    x[:, 3] = torch.linspace(-6, 6, rows, device="cuda") if rows > 1 else -4.0
    x = x.bfloat16().float()
    if x_dtype == "mx4":
        x = wrs.mx4_quantize(x, ctx=ctx)
        xr = unpack_f64(x.codes.cpu().numpy(), x.scales.cpu().numpy())
    else:
        x = x.to(DT[x_dtype])
        xr = x.double().cpu().numpy()
    out = torch.full((rows, 640), float("nan"), device="cuda")
    wrs.linear_mx4(x, [m], None, [out], act="gelu", ctx=ctx)
    y = xr @ unpack_f64(m.codes.cpu().numpy(), m.scales.cpu().numpy()).T
    two_u = 2 * 0.7978846 * np.abs(y) * (1 + 0.044715 * y * y)
    ref = gelu(y)
    assert np.all(np.abs(host(out) - ref) <= (6 * two_u + 16) * U32 * np.abs(ref))


@pytest.mark.parametrize("x_dtype", ["f32", "f16", "bf16", "mx4"])
@pytest.mark.parametrize("rows", [1, 6, 40, 300])
@pytest.mark.parametrize("pad", [0, 1, 8])
def test_groups_side_by_side_in_wider_rows(wrs, ctx, rows, pad, x_dtype):
    """q, k and v as column slices of one tensor, its rows on 16 bytes or not; what lies between
    them stays."""
    note(f"linear_mx4 {rows} rows {x_dtype} into slices of rows padded by {pad}")
    rng = np.random.default_rng(24)
    d = 192
    ws = [make(wrs, ctx, rng, d, 128) for _ in range(3)]
    x = torch.from_numpy(rng.standard_normal((rows, 128)).astype(np.float32)).cuda()
    if x_dtype == "mx4":
        x = wrs.mx4_quantize(x, ctx=ctx)
        xr = unpack_f64(x.codes.cpu().numpy(), x.scales.cpu().numpy())
    else:
        x = x.to(DT[x_dtype])
        xr = x.double().cpu().numpy()
    for out in ("f32", "f16", "bf16"):
        wide = torch.full((rows + 1, 3 * d + 3 * pad), 7.0, dtype=DT[out], device="cuda")
        at = [g * (d + pad) + pad for g in range(3)]
        wrs.linear_mx4(x, [w for w, _ in ws], None, [wide[:, a:a + d] for a in at],
                       out_row_stride=wide.shape[1], ctx=ctx)
        got, rest = host(wide).astype(np.float64), np.ones(wide.shape, bool)
        for a, (_, w) in zip(at, ws):
            y, tol = reference(xr, w, None, None, out)
            assert np.all(np.abs(got[:rows, a:a + d] - y) <= tol)
            rest[:rows, a:a + d] = False
        assert np.all(got[rest] == 7.0)


@pytest.mark.parametrize("rows", [3, 16, 40, 300])
@pytest.mark.parametrize("octaves", [100, 115, 130])
def test_f32_x_next_to_the_smallest(wrs, ctx, rows, octaves):
    """f32 x goes in bf16 parts where two f16 ones do not hold it; their last bit is 2^-133."""
    note(f"linear_mx4 {rows} rows f32 at 2^-{octaves}")
    rng = np.random.default_rng(25)
    w = rng.standard_normal((70, 128)) * 2.0 ** 60
    m = wrs.mx4_quantize(torch.from_numpy(w.astype(np.float32)).cuda(), ctx=ctx)
    wf = unpack_f64(m.codes.cpu().numpy(), m.scales.cpu().numpy())
    x = torch.from_numpy((rng.standard_normal((rows, 128)) * 2.0 ** -octaves).astype(np.float32))
    out = torch.full((rows, 70), float("nan"), device="cuda")
    wrs.linear_mx4(x.cuda(), [m], None, [out], ctx=ctx)
    y, tol = reference(x.double().numpy(), wf, None, None, "f32")
    assert np.all(np.abs(host(out) - y) <= tol + 2.0 ** -133 * np.abs(wf).sum(axis=1))

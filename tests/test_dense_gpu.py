"""Norm, 8-bit product and gated feed-forward against plain implementations in 64 bits."""
import pytest
import torch

import dense_ref as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def capi():
    from graphiler_b200 import capi as c
    return c


def randn(*shape, seed=0, scale=1.0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


# ---- norm -----------------------------------------------------------------------------------------------------------

NORM_SHAPES = [(1, 1), (1, 8), (3, 7), (5, 64), (2, 128), (257, 129), (33, 256), (1, 1000), (600, 1001), (64, 1024), (1, 4096), (9, 5000), (3, 8192),
               (2, 12345), (2, 16400), (2, 40000), (77, 16), (33, 40), (1000, 56), (9, 120)]


@pytest.mark.parametrize("m,n", NORM_SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("with_res", [False, True])
def test_rms_norm(m, n, dtype, with_res):
    x, w = randn(m, n, seed=1, dtype=dtype), randn(n, seed=2, dtype=dtype if n % 2 else F32)
    res = randn(m, n, seed=3, scale=3.0, dtype=dtype) if with_res else None
    got = capi().rms_norm(x, w, 1e-5, residual=res, return_rstd=True)
    r, rstd, y = ref.rms_norm(x, res, w, 1e-5)
    ref.close(got[0], y, ref.FP32 * y.abs(), what="y")
    if with_res:
        assert torch.equal(got[1], r)
    ref.close(got[-1], rstd[:, 0], ref.FP32 * rstd[:, 0], what="rstd")


@pytest.mark.parametrize("m,n", NORM_SHAPES + [(700, 24), (2000, 512)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("with_dr", [False, True])
def test_rms_norm_grad(m, n, dtype, with_dr):
    r, w = randn(m, n, seed=1, dtype=dtype), randn(n, seed=2, dtype=F32 if n % 2 else dtype)
    dy, dr = randn(m, n, seed=3, dtype=dtype), randn(m, n, seed=4, dtype=dtype) if with_dr else None
    _, rstd = capi().rms_norm(r, w, 1e-6, return_rstd=True)
    dx, dw = capi().rms_norm_grad(r, w, rstd, dy, dr)
    _, rstd64, _ = ref.rms_norm(r, None, w, 1e-6)
    want_dx, want_dw, size, size_dw = ref.rms_norm_grad(r, rstd64, w, dy, dr)
    ref.close(dx, want_dx, ref.FP32 * size, what="dx")
    # a lane adds the rows that it meets one after the other in fp32: fewer than m additions, half a step of the running sum each
    ref.close(dw, want_dw, (ref.FP32 + m * 2.0 ** -24) * size_dw, what="dw")


@pytest.mark.parametrize("offset", [1, 3])
def test_rms_norm_unaligned_base(offset):
    base, w = randn(offset + 5 * 256, seed=1, dtype=BF16), randn(256, seed=2, dtype=BF16)
    x = base[offset:].view(5, 256)
    _, _, y = ref.rms_norm(x, None, w, 1e-6)
    ref.close(capi().rms_norm(x, w), y, ref.FP32 * y.abs())


def test_rms_norm_zero_rows_and_special_values():
    x = randn(4, 256, seed=1)
    x[1] = 0
    x[2, 7] = float("inf")
    x[3, 9] = float("nan")
    w = randn(256, seed=2)
    y = capi().rms_norm(x, w, 0.0)
    assert torch.isfinite(y[0]).all() and torch.isnan(y[1]).all() and torch.isnan(y[3]).all()      # 0 / 0 with eps = 0
    assert torch.isnan(y[2, 7]) and (y[2, :7] == 0).all()
    assert (capi().rms_norm(x, w, 1e-6)[1] == 0).all()


def near_border(v, full):
    """Whether v / full lies within 2^-20 of a border between two codes: there the sum of squares' own rounding decides."""
    a = (v / full).abs()
    return ref.fp8_round(a * (1 + 2.0 ** -20)) != ref.fp8_round(a * (1 - 2.0 ** -20))


@pytest.mark.parametrize("m,n", NORM_SHAPES + [(300, 2048)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("with_res", [False, True])
def test_rms_norm_fp8(m, n, dtype, with_res):
    x, w = randn(m, n, seed=1, dtype=dtype), randn(n, seed=2, dtype=dtype)
    res = randn(m, n, seed=3, dtype=dtype) if with_res else None
    got = capi().rms_norm_fp8(x, w, 1e-6, residual=res)
    q, r = got if with_res else (got, None)
    want_r, _, y = ref.rms_norm(x, res, w, 1e-6)
    want, s = ref.quantize_rows(y)
    if with_res:
        assert torch.equal(r, want_r)
    assert torch.equal(q.scales.double(), s)
    full = s.repeat_interleave(128, dim=1)[:, :n]
    same = ref.rows_value(q) == want
    assert (same | near_border(y, full)).all()
    pad = q.values.as_strided((m, -(-n // 16) * 16), (q.values.stride(0) if m > 1 else -(-n // 16) * 16, 1))
    assert (pad.view(torch.uint8)[:, n:] == 0).all()


# ---- quantisers -----------------------------------------------------------------------------------------------------

def special_rows(m, n, dtype):
    x = randn(m, n, seed=5, dtype=dtype) * torch.exp2(torch.arange(m).cuda() % 24 - 12.0)[:, None].to(dtype)
    if n > 3:
        x[0, :4] = torch.tensor([0.0, -0.0, float("inf"), float("nan")], dtype=dtype)
    if m > 1:
        x[1] = 0
    return x


@pytest.mark.parametrize("m,n", [(1, 1), (2, 16), (77, 24), (31, 64), (18, 104), (3, 127), (4, 128), (5, 129), (7, 1000), (130, 2050), (64, 4096)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_quantize_and_dequantize(m, n, dtype):
    x = special_rows(m, n, dtype)
    q = capi().quantize_fp8(x)
    want, s = ref.quantize_rows(x.double())
    assert torch.equal(q.scales.double(), s)
    assert torch.equal(torch.nan_to_num(ref.rows_value(q), nan=-7.0), torch.nan_to_num(want, nan=-7.0))
    for out in (F32, BF16, F16):
        y = capi().dequantize_fp8(q, out)
        assert torch.equal(torch.nan_to_num(y, nan=-7.0), torch.nan_to_num(want.float().to(out), nan=-7.0))


def test_quantize_extremes():
    x = torch.zeros(6, 128, device="cuda")
    x[0, 3], x[1, 3], x[2, 3], x[3, 3], x[4, 3], x[5, 3] = 3.4028234e38, 1e-45, 448.0, 448.00003, 2.0 ** -117, -1.75
    q = capi().quantize_fp8(x)
    want, s = ref.quantize_rows(x.double())
    assert torch.equal(q.scales.double(), s) and torch.equal(ref.rows_value(q), want)


@pytest.mark.parametrize("t,k,n", [(1, 1, 1), (1, 128, 128), (2, 130, 100), (3, 1000, 257), (1, 64, 4096)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_quantize_weight(t, k, n, dtype):
    w = randn(t, k, n, seed=6, dtype=dtype)
    w[0, 0, 0] = float("nan")
    q = capi().quantize_fp8_weight(w)
    want, s = ref.quantize_weight(w)
    assert torch.equal(q.scales.double(), s)
    assert torch.equal(torch.nan_to_num(ref.weight_value(q), nan=-7.0), torch.nan_to_num(want, nan=-7.0))


# ---- 8-bit product --------------------------------------------------------------------------------------------------

def codes(m, k, seed):
    """Rows in 8 bits with scales that are no powers of two."""
    c = capi()
    q = c.quantize_fp8(randn(m, k, seed=seed))
    return c.Fp8Rows(q.values, q.scales * (1 + 0.3 * randn(*q.scales.shape, seed=seed + 1).abs()))


def weights(t, k, n, seed):
    c = capi()
    q = c.quantize_fp8_weight(randn(t, k, n, seed=seed))
    return c.Fp8Weight(q.values, q.scales * (1 + 0.3 * randn(*q.scales.shape, seed=seed + 1).abs()))


def check_mm(x, w, ptr, dtype, out=None):
    y = capi().segment_mm_fp8(x, w, None if ptr is None else torch.tensor(ptr, dtype=torch.int32, device="cuda"), out_dtype=dtype, out=out)
    xv, wv = ref.rows_value(x), ref.weight_value(w)
    for i, (a, b) in enumerate(zip((ptr or [0, xv.shape[0]]), (ptr or [0, xv.shape[0]])[1:])):
        want = xv[a:b] @ wv[i].t()
        ref.close(y[a:b], want, ref.sum_loss(xv.shape[1], fp8=True) * (xv[a:b].abs() @ wv[i].abs().t()), what=f"type {i}")
    return y


@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 128, 128), (1, 16, 24), (2, 200, 65), (128, 128, 256), (129, 384, 300), (100, 1000, 777), (1, 4096, 4096),
                                   (7, 2048, 1000), (1000, 640, 1500), (300, 5000, 64), (4096, 256, 512), (640, 129, 20000),
                                   (5000, 500, 2100), (260, 2000, 3000)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_mm_fp8(m, k, n, dtype):
    check_mm(codes(m, k, 10), weights(1, k, n, 20), None, dtype)


@pytest.mark.parametrize("ptr", [[0, 0, 5, 5, 300], [0, 1, 2, 3, 4], [0, 128, 256, 300, 300], [0, 0, 0, 0, 0], [3, 130, 140, 150, 280]])
@pytest.mark.parametrize("k,n", [(128, 128), (1000, 300), (4096, 40)])
def test_mm_fp8_typed(ptr, k, n):
    m = 300
    out = torch.full((m, n), 7.0, device="cuda", dtype=BF16)
    y = check_mm(codes(m, k, 10), weights(4, k, n, 20), ptr, BF16, out=out)
    assert y is out and (out[:ptr[0]] == 7).all() and (out[ptr[-1]:] == 7).all()      # rows of no type stay


def test_mm_fp8_long_types():
    check_mm(codes(4100, 300, 10), weights(3, 300, 2100, 20), [0, 1500, 1500, 4100], BF16)


def test_mm_fp8_many_types():
    ptr = [0]
    for i in range(100):
        ptr.append(ptr[-1] + (i * 7) % 23)
    check_mm(codes(ptr[-1], 256, 10), weights(100, 256, 48, 20), ptr, F16)


def nan_padding(c, q):
    """The same codes in rows whose padding holds the NaN code."""
    k = q.values.shape[-1]
    wide = torch.full((*q.values.shape[:-1], (k + 15) // 16 * 16 + 16), 0x7f, dtype=torch.uint8, device="cuda")
    wide[..., :k] = q.values.view(torch.uint8)
    return type(q)(wide.view(torch.float8_e4m3fn)[..., :k], q.scales)


@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 15, 16, 17])
@pytest.mark.parametrize("k,n", [(1, 17), (15, 8), (130, 129), (1000, 300), (1024, 16), (3200, 1001)])
def test_fp8_few_rows(m, k, n):
    """Single tokens and small batches, whatever the rows' padding holds; the gated form too."""
    c = capi()
    x, w, wu = nan_padding(c, codes(m, k, 10)), nan_padding(c, weights(1, k, n, 20)), nan_padding(c, weights(1, k, n, 30))
    y = check_mm(x, w, None, F16)
    check_mm(x, w, None, F32)
    assert torch.equal(y, c.segment_mm_fp8(c.Fp8Rows(x.values, x.scales.contiguous()), w, out_dtype=F16))
    h = c.gated_linear_fp8(x, w, wu, "relu", out_dtype=F32)
    xv, gv, uv = ref.rows_value(x), ref.weight_value(w)[0].t(), ref.weight_value(wu)[0].t()
    g, u, loss = xv @ gv, xv @ uv, ref.sum_loss(k, fp8=True)
    dg, du = loss * (xv.abs() @ gv.abs()), loss * (xv.abs() @ uv.abs())
    ref.close(h, g.clamp(min=0) * u, dg * u.abs() + du * g.abs() + dg * du + 2.0 ** -22 * (g * u).abs())
    z, want = c.gated_linear_fp8(x, w, wu, "relu"), c.quantize_fp8(h)
    assert torch.equal(z.scales, want.scales) and torch.equal(z.values.view(torch.uint8), want.values.view(torch.uint8))


def test_fp8_few_rows_nan_stays_in_its_row():
    c = capi()
    a = randn(12, 300, seed=1)
    clean = c.segment_mm_fp8(c.quantize_fp8(a), weights(1, 300, 130, 3), out_dtype=F32)
    a[5, 299] = float("nan")
    y = c.segment_mm_fp8(c.quantize_fp8(a), weights(1, 300, 130, 3), out_dtype=F32)
    keep = torch.arange(12, device="cuda") != 5
    assert torch.isnan(y[5]).all() and torch.equal(y[keep], clean[keep])


def test_mm_fp8_scale_layouts_and_views():
    c = capi()
    x, w = codes(40, 600, 1), weights(1, 600, 96, 2)
    y = check_mm(x, w, None, F32)
    assert torch.equal(y, c.segment_mm_fp8(c.Fp8Rows(x.values, x.scales.contiguous()), w, out_dtype=F32))
    wide = torch.zeros(40, 1024, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    wide.view(torch.uint8)[:, 16:616] = x.values.view(torch.uint8)
    assert torch.equal(y, c.segment_mm_fp8(c.Fp8Rows(wide[:, 16:616], x.scales), w, out_dtype=F32))


def test_mm_fp8_nan_stays_in_its_row():
    c = capi()
    a = randn(200, 256, seed=1)
    clean = c.segment_mm_fp8(c.quantize_fp8(a), weights(1, 256, 130, 3), out_dtype=F32)
    a[17, 100] = float("nan")
    y = c.segment_mm_fp8(c.quantize_fp8(a), weights(1, 256, 130, 3), out_dtype=F32)
    assert torch.isnan(y[17]).all()
    keep = torch.arange(200, device="cuda") != 17
    assert torch.equal(y[keep], clean[keep])


# ---- gated feed-forward ---------------------------------------------------------------------------------------------

GATED_SHAPES = [(1, 1, 1), (1, 64, 64), (3, 7, 9), (2, 8, 130), (128, 64, 128), (129, 200, 136), (100, 1001, 77), (1, 2048, 1024), (5, 520, 1400),
                (700, 96, 264), (2000, 256, 320), (3000, 264, 1000), (1300, 2056, 400)]


def gated_inputs(m, k, f, dtype, transposed):
    x, dh = randn(m, k, seed=1, dtype=dtype), randn(m, f, seed=4, dtype=dtype)
    if transposed:
        wg, wu = (randn(f, k, seed=s, scale=k ** -0.5, dtype=dtype).t() for s in (2, 3))
    else:
        wg, wu = (randn(k, f, seed=s, scale=k ** -0.5, dtype=dtype) for s in (2, 3))
    return x, wg, wu, dh


@pytest.mark.parametrize("m,k,f", GATED_SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_gated(m, k, f, dtype, transposed, act):
    x, wg, wu, _ = gated_inputs(m, k, f, dtype, transposed)
    want, err, (g64, u64, _, _, eg, eu) = ref.gated(x, wg, wu, act)
    ref.close(capi().gated_linear(x, wg, wu, act), want, err, what="h")
    h, g, u = capi().gated_linear(x, wg, wu, act, return_projections=True)
    ref.close(h, want, err, what="h")
    ref.close(g[:, :f], g64, eg, what="g")
    ref.close(u[:, :f], u64, eu, what="u")


@pytest.mark.parametrize("m,k,f", GATED_SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_gated_grad(m, k, f, dtype, transposed, act):
    c = capi()
    x, wg, wu, dh = gated_inputs(m, k, f, dtype, transposed)
    if act == "relu":
        # an element whose g the sums' rounding could carry over 0 has a gradient of its own accord: it gets none from above
        _, _, (g64, _, _, _, eg, _) = ref.gated(x, wg, wu, act)
        dh = torch.where(g64.abs() > eg, dh, torch.zeros_like(dh))
    _, g, u = c.gated_linear(x, wg, wu, act, return_projections=True)
    got = c.gated_linear_grad(dh, g, u, x, wg, wu, act)
    for name, a, (want, err) in zip(("dx", "dwg", "dwu"), got, ref.gated_grad(dh, x, wg, wu, act, dtype)):
        ref.close(a, want, err, what=name)
    for name, a, (want, err) in zip(("dx", "dwg", "dwu"), c.gated_linear_grad(dh, None, None, x, wg, wu, act), ref.gated_grad(dh, x, wg, wu, act, dtype)):
        ref.close(a, want, err, what=name + " with the projections made again")
    only = c.gated_linear_grad(dh, g, u, x, wg, wu, act, want_dw=False)
    assert torch.equal(only[0], got[0]) and only[1] is None
    only = c.gated_linear_grad(dh, g, u, x, wg, wu, act, want_dx=False)
    assert only[0] is None and torch.equal(only[1], got[1]) and torch.equal(only[2], got[2])


@pytest.mark.parametrize("m,k,f", [(1, 128, 128), (1, 4096, 1000), (3, 200, 65), (129, 384, 300), (300, 1000, 777), (2000, 256, 640), (2500, 300, 1200)])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16, torch.float8_e4m3fn])
def test_gated_fp8(m, k, f, act, dtype):
    c = capi()
    x, wg, wu = codes(m, k, 1), weights(1, k, f, 3), weights(1, k, f, 5)
    wg, wu = (c.Fp8Weight(w.values, w.scales * k ** -0.5) for w in (wg, wu))
    xv, gv, uv = ref.rows_value(x), ref.weight_value(wg)[0].t(), ref.weight_value(wu)[0].t()
    want, err, (g, u, a, _, eg, eu) = ref.gated(xv, gv, uv, act)
    more = ref.sum_loss(k, fp8=True) / ref.sum_loss(k)
    err = err * max(more, 1.0)
    got = c.gated_linear_fp8(x, wg, wu, act, out_dtype=dtype)
    if dtype != torch.float8_e4m3fn:
        ref.close(got, want, err, what="h")
        return
    # a code is off by at most half a step: 2^-4 of the value, 2^-10 of the scale near 0
    v, full = ref.rows_value(got), got.scales.double().repeat_interleave(128, dim=1)[:, :f]
    assert ((v - want).abs() <= err + torch.maximum((want.abs() + err) * 2.0 ** -4, full * 2.0 ** -10)).all()
    big = ref.blocks(want.abs(), [1]).amax(dim=2)
    e = ref.blocks(err, [1]).amax(dim=2)
    lo, hi = ref.fp8_scale((big - e).clamp(min=0)), ref.fp8_scale(big + e)
    assert ((got.scales.double() >= lo) & (got.scales.double() <= hi)).all()


def test_long_sums_of_one_sign():
    """131,072 positive terms: no chain of tensor-core additions (16 terms each) is longer than 2048, each loses at most 2^-23 of the sum."""
    m, k = 2432, 131072
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w = (torch.rand(*s, generator=g, device="cuda").bfloat16() for s in ((m, k), (k, m)))
    _, got, _ = capi().gated_linear(x, w, w, "relu", return_projections=True)
    rows = torch.arange(0, m, 97, device="cuda")
    want = sum(x[rows, a:a + 16384].double() @ w[a:a + 16384].double() for a in range(0, k, 16384))
    assert float(((got[rows, :m].double() - want) / want).abs().max()) <= 2048 * 2.0 ** -23 + ref.FP32


# ---- autograd -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("shape", [(5, 64), (2, 3, 40), (257,)])
def test_autograd_norm(shape):
    from graphiler_b200 import dense
    x, res, dy, dr = (randn(*shape, seed=s).requires_grad_(s < 3) for s in (1, 2, 3, 4))
    w = randn(shape[-1], seed=5).requires_grad_(True)
    y, r = dense.rms_norm(x, w, 1e-6, residual=res)
    dx, dres, dw = torch.autograd.grad((y, r), (x, res, w), (dy, dr))
    assert torch.equal(dx, dres) and dx.shape == x.shape
    n = shape[-1]
    r64, rstd, _ = ref.rms_norm(x.detach().view(-1, n), res.detach().view(-1, n), w.detach(), 1e-6)
    want, want_dw, size, size_dw = ref.rms_norm_grad(r64, rstd, w.detach(), dy.view(-1, n), dr.view(-1, n))
    ref.close(dx.view(-1, n), want, ref.FP32 * size)
    ref.close(dw, want_dw, 2 * ref.FP32 * size_dw)
    # only one of the two outputs goes on
    y, r = dense.rms_norm(x, w, 1e-6, residual=res)
    assert torch.equal(torch.autograd.grad(r, (x, res), dr)[0], dr)
    y, r = dense.rms_norm(x, w, 1e-6, residual=res)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    want, want_dw, size, size_dw = ref.rms_norm_grad(r64, rstd, w.detach(), dy.view(-1, n), None)
    ref.close(dx.view(-1, n), want, ref.FP32 * size)
    y = dense.rms_norm(x, w, 1e-6)
    assert torch.autograd.grad(y.sum(), (x, w))[0].shape == x.shape


def test_norm_gradient_against_differences():
    c = capi()
    from graphiler_b200 import dense
    x, w, dy = randn(3, 96, seed=1).requires_grad_(True), randn(96, seed=2), randn(3, 96, seed=3)
    dx, = torch.autograd.grad(dense.rms_norm(x, w, 1e-3), x, dy)
    d, h = randn(3, 96, seed=4), 2.0 ** -6
    f = lambda t: (c.rms_norm((x.detach() + t * d).contiguous(), w, 1e-3).double() * dy.double()).sum()
    # central differences: O(h^2) of the third derivative (of order 1 here, 288 terms) and the two values' rounding over 2 h
    size = float((c.rms_norm(x.detach(), w, 1e-3).abs() * dy.abs()).sum())
    assert abs(float((f(h) - f(-h)) / (2 * h) - (dx.double() * d.double()).sum())) <= 288 * h * h + 2 * size * 2.0 ** -22 / (2 * h)


@pytest.mark.parametrize("needs", [(True, True, True), (True, False, False), (False, True, False), (False, False, True)])
def test_autograd_gated(needs):
    from graphiler_b200 import dense
    x, wg, wu, dh = gated_inputs(6, 40, 56, BF16, False)
    x = x.view(2, 3, 40)
    for t, n in zip((x, wg, wu), needs):
        t.requires_grad_(n)
    h = dense.gated_linear(x, wg, wu, "silu")
    assert h.shape == (2, 3, 56)
    want = ref.gated_grad(dh, x.detach().view(6, 40), wg.detach(), wu.detach(), "silu", BF16)
    got = torch.autograd.grad(h, [t for t, n in zip((x, wg, wu), needs) if n], dh.view(2, 3, 56))
    for a, (v, err) in zip(got, [w for w, n in zip(want, needs) if n]):
        ref.close(a.reshape(v.shape), v, err)
    with torch.no_grad():
        assert not dense.gated_linear(x, wg, wu).requires_grad


def test_gated_gradient_against_differences():
    """Along a direction d: the differences of h itself, in 64 bits, against the kernel's gradients."""
    c = capi()
    x, wg, wu, dh = gated_inputs(4, 32, 48, F16, False)
    _, g, u = c.gated_linear(x, wg, wu, "gelu", return_projections=True)
    got = c.gated_linear_grad(dh, g, u, x, wg, wu, "gelu")
    bounds = ref.gated_grad(dh, x, wg, wu, "gelu", F16)
    args, h = [x.double(), wg.double(), wu.double()], 1e-5
    for i, (a, (_, err)) in enumerate(zip(got, bounds)):
        d = randn(*args[i].shape, seed=9).double()
        f = lambda t: (ref.gated(*[v + t * d if j == i else v for j, v in enumerate(args)], "gelu")[0] * dh.double()).sum()
        num = (f(h) - f(-h)) / (2 * h)
        bound = float(((err + ref.half_step(F16) * a.double().abs() + 2.0 ** -25) * d.abs()).sum()) + 1e-5 * float((a.double().abs() * d.abs()).sum())
        assert abs(float(num - (a.double() * d).sum())) <= bound


# ---- the operators together -------------------------------------------------------------------------------------------

def ff_inputs(n, d, f, dtype):
    p = {"norm_weight": 1 + 0.2 * randn(d, seed=7), "gate_weight": randn(d, f, seed=8, scale=d ** -0.5), "up_weight": randn(d, f, seed=9, scale=d ** -0.5),
         "down_weight": randn(f, d, seed=10, scale=f ** -0.5)}
    return randn(n, d, seed=11, dtype=dtype), randn(n, d, seed=12, dtype=dtype), {k: v.to(dtype) for k, v in p.items()}


def ff_ref(h, res, p, rows=lambda v: v, weight=lambda w: w.double()):
    """The block in 64 bits; `rows` and `weight`: what is rounded on the way."""
    r = h if res is None else (h.float() + res.float()).to(h.dtype)
    y = rows(ref.rms_norm(r, None, p["norm_weight"], 1e-6)[2])
    g, u = y @ weight(p["gate_weight"]), y @ weight(p["up_weight"])
    return r.double() + rows(ref.act(g, "silu")[0] * u) @ weight(p["down_weight"])


@pytest.mark.parametrize("n,d,f", [(1, 64, 128), (50, 96, 200), (300, 256, 640)])
@pytest.mark.parametrize("with_res", [False, True])
def test_feed_forward_layer(n, d, f, with_res):
    from graphiler_b200 import layers
    h, res, p = ff_inputs(n, d, f, BF16)
    res = res if with_res else None
    leaves = [t.requires_grad_(True) for t in (h, *p.values())] + ([res.requires_grad_(True)] if with_res else [])
    out = layers.feed_forward_layer(h, p, residual=res)
    want = ff_ref(h.detach(), None if res is None else res.detach(), {k: v.detach() for k, v in p.items()})
    # every element of n, of the gated rows, of the product and of the sum is rounded once, half a step of bf16 each: relative to
    # the values' own size, and the three products average what is random in it; four half steps of the largest value cover the sum
    assert float((out.detach().double() - want).abs().max()) <= 4 * ref.half_step(BF16) * float(want.abs().max()) * 2
    grads = torch.autograd.grad(out, leaves, torch.ones_like(out))
    # the same through 64-bit autograd
    leaves64 = [t.detach().double().requires_grad_(True) for t in leaves]
    h64, w64 = leaves64[0], dict(zip(p, leaves64[1:1 + len(p)]))
    r = h64 + (leaves64[-1] if with_res else 0)
    y = r * torch.rsqrt(r.square().mean(dim=1, keepdim=True) + 1e-6) * w64["norm_weight"]
    o = r + (torch.nn.functional.silu(y @ w64["gate_weight"]) * (y @ w64["up_weight"])) @ w64["down_weight"]
    for a, b in zip(grads, torch.autograd.grad(o, leaves64, torch.ones_like(o))):
        # eight roundings of half a step on the longest way (sum, n, gated rows, their gradients, dx, the norm's gradient)
        assert float((a.double() - b).norm()) <= 8 * ref.half_step(BF16) * float(b.norm())


@pytest.mark.parametrize("n,d,f", [(1, 128, 256), (50, 200, 333), (700, 512, 1024)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_feed_forward_layer_fp8(n, d, f, dtype):
    from graphiler_b200 import layers
    h, res, p = ff_inputs(n, d, f, dtype)
    q = layers.prepare_feed_forward_fp8(p)
    got = layers.feed_forward_layer_fp8(h, q, residual=res)
    want = ff_ref(h, res, p, rows=lambda v: ref.quantize_rows(v)[0], weight=lambda w: ref.quantize_weight(w[None])[0][0].t())
    # codes next to a border may fall on its other side: a share of about 2^-20 / 2^-4 of them moves by 2^-3 in n, which moves g and u by
    # 2^-3 sqrt(2^-16) = 2^-11 relative, so that a share of 2^-7 of the second codes moves by 2^-3: 2^-6.5 of the product; plus the output's rounding
    r = (h.float() + res.float()).double()
    assert float((got.double() - want).norm()) <= 2.0 ** -6.5 * float((want - r).norm()) + 2 * ref.half_step(dtype) * float(want.norm())


# ---- two calls at once, captured calls, streams ---------------------------------------------------------------------------

def test_two_streams_at_once():
    c = capi()
    x, w = codes(500, 2048, 1), weights(1, 2048, 640, 2)
    a, b = randn(300, 512, seed=3, dtype=BF16), randn(512, 384, seed=4, dtype=BF16)
    want = c.segment_mm_fp8(x, w), c.gated_linear(a, b, b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(5):
        with torch.cuda.stream(s1):
            got.append(c.segment_mm_fp8(x, w))
        with torch.cuda.stream(s2):
            got.append(c.gated_linear(a, b, b))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g, want[i % 2])


def test_first_call_of_a_thread():
    """A thread that has made no CUDA call yet, its memory in the allocator's cache: as autograd's threads at the first backward pass."""
    import threading
    c = capi()
    x, w = randn(300, 256, seed=1, dtype=BF16), randn(256, 512, seed=2, dtype=BF16)
    q, qw = codes(300, 256, 3), weights(1, 256, 512, 4)
    dh = randn(300, 512, seed=5, dtype=BF16)
    calls = [lambda: c.gated_linear(x, w, w), lambda: c.segment_mm_fp8(q, qw), lambda: c.gated_linear_grad(dh, None, None, x, w, w)[1]]
    want = [f() for f in calls]
    spare = [f() for f in calls]
    torch.cuda.synchronize()
    del spare                                        # the threads' outputs take these blocks
    got = []
    for f in calls:
        t = threading.Thread(target=lambda: got.append(f()))
        t.start()
        t.join()
    torch.cuda.synchronize()
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_calls_keep_their_scratch_apart():
    """Two graphs whose calls need scratch (k is split), replayed in turn and with new inputs."""
    c = capi()
    w = weights(1, 4096, 512, 2)
    ws = [randn(2048, 256, seed=s, dtype=BF16) for s in (5, 6)]
    xs = [codes(3, 4096, 1), codes(5, 4096, 7)]
    rows = [randn(4, 2048, seed=8, dtype=BF16), randn(9, 2048, seed=9, dtype=BF16)]
    def call(i):
        y, r = c.rms_norm(rows[i], ws[0][:, 0].contiguous(), residual=rows[i])
        return c.segment_mm_fp8(xs[i], w), c.gated_linear(y, *ws)
    want = [call(0), call(1)]
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(i))
        graphs.append(g)
    for _ in range(3):
        for i in (0, 1, 1, 0):
            graphs[i].replay()
        torch.cuda.synchronize()
        for o, v in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, v))
    rows[0].copy_(randn(4, 2048, seed=20, dtype=BF16))
    graphs[0].replay()
    assert torch.equal(outs[0][1], call(0)[1])
    del graphs, outs


def test_captured_training_step():
    from graphiler_b200 import dense
    x, wg, wu, dh = gated_inputs(40, 96, 128, BF16, False)
    nw, leaves = torch.ones(96, device="cuda", dtype=BF16).requires_grad_(True), [t.requires_grad_(True) for t in (x, wg, wu)]
    def step():
        h = dense.gated_linear(dense.rms_norm(x, nw), wg, wu, "gelu")
        return torch.autograd.grad(h, leaves + [nw], dh)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del g


def test_capture_beside_a_living_graph_is_refused():
    """An eager graph of the same leaves, recorded on the default stream, lives: a captured backward pass would reach that stream."""
    from graphiler_b200 import capi as c, dense
    x, wg, wu, dh = gated_inputs(40, 96, 128, BF16, False)
    nw = torch.ones(96, device="cuda", dtype=BF16).requires_grad_(True)
    wg.requires_grad_(True)
    kept = dense.gated_linear(dense.rms_norm(x, nw), wg, wu)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = x + 1
        with pytest.raises(c.GphlError, match="default stream"):
            dense.rms_norm(x, nw)
        with pytest.raises(c.GphlError, match="default stream"):
            dense.gated_linear(x, wg, wu)
        with torch.no_grad():
            h = dense.gated_linear(x, wg, wu)
    g.replay()
    torch.cuda.synchronize()
    with torch.no_grad():
        assert torch.equal(h, dense.gated_linear(x, wg, wu)) and torch.equal(y, x + 1)
    del kept, g
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dw, dn = torch.autograd.grad(dense.gated_linear(dense.rms_norm(x, nw), wg, wu), (wg, nw), dh)
    g.replay()
    want = torch.autograd.grad(dense.gated_linear(dense.rms_norm(x, nw), wg, wu), (wg, nw), dh)
    assert torch.equal(dw, want[0]) and torch.equal(dn, want[1])
    del g


@pytest.mark.filterwarnings("ignore:The AccumulateGrad node's stream")
def test_capture_after_a_warm_up_whose_outputs_are_kept():
    """The usual recipe: warm-up on a side stream, its last outputs still there, then the capture."""
    from graphiler_b200 import dense
    x, wg, wu, dh = gated_inputs(40, 96, 128, BF16, False)
    nw = torch.ones(96, device="cuda", dtype=BF16).requires_grad_(True)
    leaves = [nw, wg.requires_grad_(True), wu.requires_grad_(True)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            for t in leaves:
                t.grad = None
            y = dense.gated_linear(dense.rms_norm(x, nw), wg, wu)
            y.backward(dh)
        want = [t.grad for t in leaves]
    torch.cuda.current_stream().wait_stream(s)
    for t in leaves:
        t.grad = None
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dense.gated_linear(dense.rms_norm(x, nw), wg, wu).backward(dh)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(t.grad, v) for t, v in zip(leaves, want))
    del g, y


def test_results_repeat_bit_for_bit():
    c = capi()
    x, wg, wu, dh = gated_inputs(1500, 96, 264, BF16, False)
    first = c.gated_linear_grad(dh, None, None, x, wg, wu)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, c.gated_linear_grad(dh, None, None, x, wg, wu)))
    r, w, rstd = x, wg[:, 0].contiguous(), c.rms_norm(x, wg[:, 0].contiguous(), return_rstd=True)[1]
    first = c.rms_norm_grad(r, w, rstd, x)
    assert all(torch.equal(a, b) for a, b in zip(first, c.rms_norm_grad(r, w, rstd, x)))


def test_codes_repeat_over_many_tiles():
    """Long k and more tiles than blocks: the warps that share a row's scale run ahead of one another into the next tile."""
    c = capi()
    x, wg, wu = codes(1000, 2600, 1), weights(1, 2600, 6000, 2), weights(1, 2600, 6000, 3)
    first = c.gated_linear_fp8(x, wg, wu)
    h = c.gated_linear_fp8(x, wg, wu, out_dtype=F32)
    want = c.quantize_fp8(h)                       # the same fp32 values, quantised by themselves
    for _ in range(20):
        got = c.gated_linear_fp8(x, wg, wu)
        assert torch.equal(got.values.view(torch.uint8), first.values.view(torch.uint8)) and torch.equal(got.scales, first.scales)
    assert torch.equal(first.scales, want.scales) and torch.equal(first.values.view(torch.uint8), want.values.view(torch.uint8))


def test_no_wait_ran_out():
    assert capi().tc_wait_timeouts() == 0


# ---- empty inputs ------------------------------------------------------------------------------------------------------

def test_empty_inputs():
    c = capi()
    e = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype, device="cuda")
    assert c.rms_norm(e(0, 64), e(64)).shape == (0, 64) and c.rms_norm(e(3, 0), e(0)).shape == (3, 0)
    dx, dw = c.rms_norm_grad(e(0, 64), e(64) + 1, e(0, dtype=F32), e(0, 64))
    assert dx.shape == (0, 64) and (dw == 0).all()
    q = c.quantize_fp8(e(0, 64))
    assert q.values.shape == (0, 64) and c.dequantize_fp8(q).shape == (0, 64)
    w = c.quantize_fp8_weight(e(64, 32))
    assert c.segment_mm_fp8(q, w).shape == (0, 32)
    assert c.segment_mm_fp8(c.quantize_fp8(e(5, 64)), c.quantize_fp8_weight(e(64, 0))).shape == (5, 0)
    assert (c.segment_mm_fp8(c.quantize_fp8(e(5, 0)), c.quantize_fp8_weight(e(0, 32))) == 0).all()
    assert (c.gated_linear(e(5, 0), e(0, 8), e(0, 8)) == 0).all() and c.gated_linear(e(0, 4), e(4, 8), e(4, 8)).shape == (0, 8)
    dx, dg, du = c.gated_linear_grad(e(0, 8), None, None, e(0, 4), e(4, 8) + 1, e(4, 8))
    assert dx.shape == (0, 4) and (dg == 0).all() and (du == 0).all()
    h = c.gated_linear_fp8(c.quantize_fp8(e(0, 64)), w, w)
    assert h.values.shape == (0, 32)
    z = c.gated_linear_fp8(c.quantize_fp8(e(4, 64)), w, w)
    assert (c.dequantize_fp8(z) == 0).all()

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

"""Dense operators at the edges of what is documented: results over their inputs, infinities, tails, long sums, empty products."""
import ctypes

import pytest
import torch

import dense_ref as ref

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
F8 = torch.float8_e4m3fn
CODE = {F32: 0, BF16: 1, F16: 2}


@pytest.fixture(scope="module", autouse=True)
def built():
    from graphiler_b200 import build
    build.build_all()


def capi():
    from graphiler_b200 import capi as c
    return c


def randn(*shape, seed=0, scale=1.0, dtype=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def c_call(name, *args):
    """An entry of the C ABI on the current stream; tensors go as addresses."""
    c = capi()
    args = [None if a is None else ctypes.c_void_p(a.data_ptr()) if isinstance(a, torch.Tensor) else a for a in args]
    c._check(getattr(c.lib(), name)(*args, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)), name)


# ---- results over inputs, as the C ABI allows ---------------------------------------------------------------------------

WIDTHS = [64, 256, 1001, 4096, 9001, 16384, 16400, 20001]


@pytest.mark.gpu
@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("over", ["y is x", "r is x", "r is residual", "y is x, r is residual"])
def test_norm_over_its_inputs(n, dtype, over):
    m = 200
    x, res, w = randn(m, n, seed=1, dtype=dtype), randn(m, n, seed=2, dtype=dtype), randn(n, seed=3, dtype=dtype)
    y, r, rstd = capi().rms_norm(x, w, 1e-6, residual=res, return_rstd=True)
    a, b, got_rstd = x.clone(), res.clone(), torch.empty(m, device="cuda")
    got_y = a if "y is x" in over else torch.empty_like(x)
    got_r = a if "r is x" in over else b if "r is residual" in over else torch.empty_like(x)
    c_call("gphl_rms_norm", CODE[dtype], m, n, a, b, w, CODE[dtype], 1e-6, got_y, got_r, got_rstd)
    assert torch.equal(got_y, y) and torch.equal(got_r, r) and torch.equal(got_rstd, rstd)


@pytest.mark.gpu
@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("over", ["x", "residual"])
def test_norm_to_codes_over_its_inputs(n, over):
    m, pad, blocks = 70, -(-n // 16) * 16, -(-n // 128)
    x, res, w = randn(m, n, seed=1, dtype=BF16), randn(m, n, seed=2, dtype=BF16), randn(n, seed=3, dtype=BF16)
    q, r = capi().rms_norm_fp8(x, w, 1e-6, residual=res)
    a, b = x.clone(), res.clone()
    codes, scales = torch.empty(m, pad, dtype=torch.uint8, device="cuda"), torch.empty(blocks, m, device="cuda")
    got_r = a if over == "x" else b
    c_call("gphl_rms_norm_fp8", 1, m, n, a, b, w, 1, 1e-6, codes, pad, scales, m, got_r)
    assert torch.equal(got_r, r) and torch.equal(scales.t(), q.scales) and torch.equal(codes[:, :n], q.values.view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("over", ["dy", "dr"])
def test_norm_gradient_over_its_inputs(n, dtype, over):
    """More rows than the 64 groups in which dw of wide rows is summed."""
    m, c = 200, capi()
    r, w, dy, dr = (randn(*s, seed=i, dtype=dtype) for i, s in enumerate([(m, n), (n,), (m, n), (m, n)]))
    _, rstd = c.rms_norm(r, w, 1e-6, return_rstd=True)
    dx, dw = c.rms_norm_grad(r, w, rstd, dy, dr)
    _, rstd64, _ = ref.rms_norm(r, None, w, 1e-6)
    want_dx, want_dw, size, size_dw = ref.rms_norm_grad(r, rstd64, w, dy, dr)
    ref.close(dx, want_dx, ref.FP32 * size, what="dx")
    ref.close(dw, want_dw, (ref.FP32 + m * 2.0 ** -24) * size_dw, what="dw")
    a, b, got = dy.clone(), dr.clone(), torch.empty_like(w)
    work = torch.empty(c.lib().gphl_rms_norm_grad_workspace_bytes(CODE[dtype], m, n), dtype=torch.uint8, device="cuda")
    out = a if over == "dy" else b
    c_call("gphl_rms_norm_grad", CODE[dtype], m, n, r, w, CODE[dtype], rstd, a, b, out, got, work)
    assert torch.equal(out, dx) and torch.equal(got, dw)


# ---- infinities and tails of the activations ----------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,k", [(1, 8), (300, 8), (2, 4096)])
def test_relu_of_infinities(m, k, dtype):
    """g of -inf gives 0, of +inf +inf, of NaN NaN; with gradients from above, that of u is 0 where act is (k = 4096: k is split)."""
    c = capi()
    x, wg, wu = torch.ones(m, k, dtype=dtype, device="cuda"), torch.ones(k, 40, dtype=dtype, device="cuda"), torch.ones(k, 40, dtype=dtype, device="cuda")
    wg[0, 3], wg[0, 5], wg[0, 7], wg[0, 9] = float("-inf"), float("inf"), float("nan"), -2.0 * k
    h, g, u = c.gated_linear(x, wg, wu, "relu", return_projections=True)
    want = torch.full((40,), float(k) * k, device="cuda")
    want[3], want[5], want[7], want[9] = 0, float("inf"), float("nan"), 0
    assert torch.equal(torch.nan_to_num(h, nan=-7.0), torch.nan_to_num(want.to(dtype).expand(m, 40), nan=-7.0))
    dh = torch.ones(m, 40, dtype=dtype, device="cuda")
    for kept in ((g, u), (None, None)):
        _, dwg, dwu = c.gated_linear_grad(dh, *kept, x, wg, wu, "relu", want_dx=False)
        for col in (3, 9):
            assert (dwg[:, col] == 0).all() and (dwu[:, col] == 0).all()
        assert torch.isinf(dwu[:, 5]).all() and torch.isnan(dwu[:, 7]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 8, 40, 300])
def test_relu_of_infinities_in_8_bits(m):
    """Scales whose product is beyond fp32: g = -inf, h = 0, as a value and as codes."""
    c = capi()
    row = lambda v, s: c.Fp8Rows(torch.full((m, 128), v, device="cuda").to(F8), torch.full((m, 1), s, device="cuda"))
    weight = lambda v, s: c.Fp8Weight(torch.full((1, 32, 128), v, device="cuda").to(F8), torch.full((1, 1, 1), s, device="cuda"))
    x, wg, wu = row(1.0, 2.0 ** 100), weight(-1.0, 2.0 ** 100), weight(1.0, 2.0 ** -100)
    assert (c.gated_linear_fp8(x, wg, wu, "relu", out_dtype=F32) == 0).all()
    assert (c.dequantize_fp8(c.gated_linear_fp8(x, wg, wu, "relu")) == 0).all()


def gelu_bound(g):
    """Relative error of Phi(g): fp32 arithmetic of a fit that is right to 2^-22 and two approximate instructions (2^-19 in all), and the exponent
    g^2 / 2, two products and a rounded constant: 1.5 * 2^-24 of it each way and 2^-23 of room."""
    return 2.0 ** -19 + g.square() * 2.0 ** -23


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 40])
def test_gelu_keeps_its_leading_digits_8_bits(m):
    """g over the e4m3 values of [-12, 12] with u = 1, results in 32 bits: relative to the value itself, also where it is small."""
    c = capi()
    codes = torch.arange(256, dtype=torch.int32, device="cuda").to(torch.uint8).view(F8).float()
    g = codes[codes.abs() <= 12].sort().values
    n = g.numel()
    wg, wu = torch.zeros(1, n, 16, device="cuda"), torch.zeros(1, n, 16, device="cuda")
    wg[0, :, 0], wu[0, :, 1] = g, 1.0
    x = torch.zeros(m, 16, device="cuda")
    x[:, :2] = 1.0
    one = torch.ones(m, 1, device="cuda"), torch.ones(1, -(-n // 128), 1, device="cuda")
    h = c.gated_linear_fp8(c.Fp8Rows(x.to(F8), one[0]), c.Fp8Weight(wg.to(F8), one[1]), c.Fp8Weight(wu.to(F8), one[1]), "gelu", out_dtype=F32)
    want = g.double() * torch.exp(torch.special.log_ndtr(g.double()))
    ref.close(h, want.expand(m, n), (gelu_bound(g.double()) * want.abs()).expand(m, n), what="gelu")


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("m", [1, 300])
def test_activations_of_large_values(act, m):
    """+inf stays, NaN stays, and far below 0 nothing is left."""
    x, wg, wu = (torch.ones(*s, dtype=BF16, device="cuda") for s in ((m, 8), (8, 40), (8, 40)))
    wg[0, 3], wg[0, 5], wg[0, 7], wg[0, 9] = float("inf"), float("nan"), 1e30, -1e30
    h = capi().gated_linear(x, wg, wu, act).float()
    assert (h[:, 3] == float("inf")).all() and torch.isnan(h[:, 5]).all() and (h[:, 9] == 0).all()
    ref.close(h[:, 7].bfloat16(), (8 * wg[0, 7].double()).expand(m), (ref.FP32 * 8e30 * torch.ones(m, dtype=torch.float64, device="cuda")))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_gelu_keeps_its_leading_digits_with_gradients(dtype):
    """One row: the weights' gradients are dg and du themselves.  u = 2^10, so that fp16 holds the tail."""
    c = capi()
    g = torch.arange(-96, 49, device="cuda") / 16.0                   # -6 .. 3, exact in both types
    n, size = g.numel(), 1024.0
    wg, wu = torch.zeros(8, n, device="cuda"), torch.zeros(8, n, device="cuda")
    wg[0], wu[1] = g, size
    x, wg, wu, dh = torch.ones(1, 8, device="cuda").to(dtype), wg.to(dtype), wu.to(dtype), torch.full((1, n), 4.0, dtype=dtype, device="cuda")
    h, gg, uu = c.gated_linear(x, wg, wu, "gelu", return_projections=True)
    assert torch.equal(gg[0, :n], g) and (uu[0, :n] == size).all()
    g = g.double()
    phi, dens = torch.special.ndtr(g), torch.exp(-g * g / 2) / (2 * torch.pi) ** 0.5
    act, err = g * phi, gelu_bound(g) * (g * phi).abs()
    ref.close(h, (size * act)[None], (size * err)[None], what="h")
    # act' = Phi + g phi: the second term's exponential is off by as much, and the sum cancels near g = -0.75
    dact, derr = phi + g * dens, gelu_bound(g) * (phi + g.abs() * dens)
    for kept in ((gg, uu), (None, None)):
        _, dwg, dwu = c.gated_linear_grad(dh, *kept, x, wg, wu, "gelu", want_dx=False)
        ref.close(dwu[0], 4 * act, 4 * err, what="du")
        ref.close(dwg[0], 4 * size * dact, 4 * size * derr, what="dg")


# ---- the layers -----------------------------------------------------------------------------------------------------------

def ff_params(d, f, dtype=BF16):
    return {"norm_weight": 1 + 0.2 * randn(d, seed=7).to(dtype), "gate_weight": randn(d, f, seed=8, scale=d ** -0.5, dtype=dtype),
            "up_weight": randn(d, f, seed=9, scale=d ** -0.5, dtype=dtype), "down_weight": randn(f, d, seed=10, scale=f ** -0.5, dtype=dtype)}


@pytest.mark.gpu
@pytest.mark.parametrize("with_res", [False, True])
def test_the_serving_layer_records_no_gradients(with_res):
    """Not a part of them either: the sum with the input would pass its own on and nothing of the rest."""
    from graphiler_b200 import layers
    q = layers.prepare_feed_forward_fp8(ff_params(96, 200))
    h, res = randn(50, 96, seed=1, dtype=BF16), randn(50, 96, seed=2, dtype=BF16) if with_res else None
    want = layers.feed_forward_layer_fp8(h, q, residual=res)
    kept = h.clone()
    h.requires_grad_(True)
    got = layers.feed_forward_layer_fp8(h, q, residual=None if res is None else res.requires_grad_(True))
    assert not got.requires_grad and torch.equal(got, want) and torch.equal(h, kept)


# ---- the typed product's arguments ------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_mm_fp8_of_an_empty_inner_dimension(dtype):
    """Sums of nothing: zeros in the rows of any type, with a pointer as without; rows of no type stay."""
    c = capi()
    x = c.Fp8Rows(torch.empty(300, 0, dtype=torch.uint8, device="cuda").view(F8), torch.empty(300, 0, device="cuda"))
    w = lambda t: c.Fp8Weight(torch.empty(t, 40, 0, dtype=torch.uint8, device="cuda").view(F8), torch.empty(t, 1, 0, device="cuda"))
    assert (c.segment_mm_fp8(x, w(1), out_dtype=dtype) == 0).all()
    out = torch.full((300, 40), 7.0, dtype=dtype, device="cuda")
    y = c.segment_mm_fp8(x, w(3), torch.tensor([5, 40, 40, 290], dtype=torch.int32, device="cuda"), out=out)
    assert y is out and (out[:5] == 7).all() and (out[5:290] == 0).all() and (out[290:] == 7).all()
    y = c.segment_mm_fp8(x, w(3), torch.tensor([0, 40, 40, 300], dtype=torch.int32, device="cuda"), out_dtype=dtype)
    assert y.dtype == dtype and (y == 0).all()


def test_mm_fp8_says_that_it_writes_out():
    """The registration's schema, by which graph passes keep the write in its place."""
    capi()._op("segment_mm_fp8")
    args = {a.name: a for a in torch.ops.my_ops.segment_mm_fp8.default._schema.arguments}
    assert "out" in args and args["out"].alias_info is not None and args["out"].alias_info.is_write
    assert not any(a.alias_info for n, a in args.items() if n != "out")


@pytest.mark.gpu
def test_mm_fp8_counts_its_write():
    """What autograd kept of `out` is known to have changed."""
    c = capi()
    x, w = c.quantize_fp8(randn(4, 64, seed=1)), c.quantize_fp8_weight(randn(64, 32, seed=2))
    out = torch.ones(4, 32, device="cuda")
    a = torch.ones(4, 32, device="cuda", requires_grad=True)
    loss = (a * out).sum()
    assert c.segment_mm_fp8(x, w, out=out) is out and out._version == 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with pytest.raises(c.GphlError, match="gradients"):
        c.segment_mm_fp8(x, w, out=torch.ones(4, 32, device="cuda", requires_grad=True))
    with torch.no_grad():
        c.segment_mm_fp8(x, w, out=torch.ones(4, 32, device="cuda", requires_grad=True))
    with torch.inference_mode():
        assert torch.equal(c.segment_mm_fp8(x, w, out=torch.ones(4, 32, device="cuda")), out)


# ---- derivatives that there are not ------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_is_refused(requires_grad):
    """A tangent is not dropped without a word."""
    from graphiler_b200 import dense
    from torch.autograd import forward_ad as fw
    args = [randn(4, 64, seed=1, dtype=BF16), randn(64, seed=2, dtype=BF16), randn(4, 64, seed=3, dtype=BF16), randn(64, 32, seed=4, dtype=BF16),
            randn(64, 32, seed=5, dtype=BF16)]
    with fw.dual_level():
        for i in range(5):
            x, w, res, wg, wu = (fw.make_dual(a.clone().requires_grad_(requires_grad), torch.ones_like(a)) if i == j else a for j, a in enumerate(args))
            if i < 3:
                with pytest.raises(capi().GphlError, match="forward"):
                    dense.rms_norm(x, w, residual=res)
            if i in (0, 3, 4):
                with pytest.raises(capi().GphlError, match="forward"):
                    dense.gated_linear(x, wg, wu)


# ---- long sums ----------------------------------------------------------------------------------------------------------------

CHAIN = 32768            # values of k that one tensor-core sum may gather


@pytest.mark.parametrize("m", [8192, 300_000, 8_388_608, 8_500_000, 100_000_000, 2_000_000_000])
def test_gated_weight_gradients_have_room_for_all_parts(m):
    """dW sums over the rows in parts of at most CHAIN, whose fp32 sums lie in the workspace behind dg and du."""
    k, f = 64, 72
    room = capi().lib().gphl_gated_grad_workspace_bytes(m, k, f) - 2 * -(-m * f * 2 // 256) * 256
    parts = -(-m // CHAIN)
    assert parts == 1 or room >= parts * 2 * k * f * 4


@pytest.mark.gpu
def test_gated_weight_gradients_of_very_many_rows():
    """Sums over 100 million rows, of one sign.  u and du are 1 (x's first column times the first rows of the weights, dh = 1), so that nothing is
    rounded before the sum.  A chain of CHAIN values loses at most 2^-23 with each of its CHAIN / 16 additions, the join half a step of
    the running sum with each of at most 64 + parts / 64."""
    c, m, n = capi(), 100_000_000, 8
    g = torch.Generator(device="cuda").manual_seed(1)
    x = (torch.rand(m, n, generator=g, device="cuda", dtype=F16) + 1) * 2.0 ** -13
    x[:, 0] = 1
    w = torch.zeros(n, n, dtype=F16, device="cuda")
    w[0] = 1
    _, _, dwu = c.gated_linear_grad(torch.ones(m, n, dtype=F16, device="cuda"), None, None, x, w, w, "relu", want_dx=False)
    want = sum(x[a:a + 10_000_000].double().sum(dim=0) for a in range(0, m, 10_000_000))[1:, None].expand(n - 1, n)
    parts = -(-m // CHAIN)
    ref.close(dwu[1:], want, (CHAIN / 16 * 2.0 ** -23 + (64 + parts / 64) * 2.0 ** -24) * want, what="dWu")


@pytest.mark.gpu
@pytest.mark.parametrize("n", [16400, 1 << 20, 1 << 24])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_of_very_wide_rows(n, dtype):
    """Equal values: every addition of a running sum rounds the same way."""
    c = capi()
    x, dy, w = (torch.full(s, v, device="cuda").to(dtype) for s, v in (((2, n), 1.1), ((2, n), 1.3), ((n,), 0.9)))
    y, rstd = c.rms_norm(x, w, 0.0, return_rstd=True)
    _, rstd64, want = ref.rms_norm(x, None, w, 0.0)
    ref.close(rstd, rstd64[:, 0], ref.FP32 * rstd64[:, 0], what="rstd")
    ref.close(y, want, ref.FP32 * want, what="y")
    dx, dw = c.rms_norm_grad(x, w, rstd, dy)
    want, want_dw, size, size_dw = ref.rms_norm_grad(x, rstd64, w, dy, None)
    ref.close(dx, want, ref.FP32 * size, what="dx")
    ref.close(dw, want_dw, ref.FP32 * size_dw, what="dw")
    q = c.rms_norm_fp8(x, w, 0.0)
    want, _ = ref.quantize_rows(ref.rms_norm(x, None, w, 0.0)[2])
    assert torch.equal(ref.rows_value(q), want)


# ---- refusals, by their reasons ---------------------------------------------------------------------------------------------------

REASONS = {
    "norm: width": r"rows \(m, n\) and a weight", "norm: residual's shape": "residual must have", "norm: residual's type": "residual must have",
    "norm: weight's type": "weight must have", "norm: integers": "rows must be float32", "norm: negative eps": "eps must not", "norm: strided rows": "contiguous",
    "norm8: width": r"rows \(m, n\) and a weight", "norm grad: rstd": "rstd must hold", "norm grad: dy": "gradients must have",
    "quantize: dimensions": "quantize_fp8 needs rows", "quantize: doubles": "rows must be float32", "quantize weight: dimensions": r"needs \(k, n\) or",
    "dequantize: output type": "output must be float32", "dequantize: scales' shape": "scales of shape",
    "mm8: inner dimension": "inner dimensions differ", "mm8: rows not 16 bytes apart": "16-byte boundaries", "mm8: values' type": "must be float8_e4m3fn",
    "mm8: several types, no pointer": "need a type pointer", "mm8: pointer's length": "type pointer must hold", "mm8: pointer's type": "type pointer must hold",
    "mm8: output type": "output must be float32", "mm8: out's shape": r"out must be \(m, n\)",
    "gated: activation": "unknown activation", "gated: float32": "bfloat16 or float16", "gated: mixed types": "must have one type",
    "gated: weights' shapes": r"two weights \(k, f\)", "gated: inner dimension": r"two weights \(k, f\)", "gated: one weight transposed": "or their transposes",
    "gated: strided rows": "contiguous", "gated grad: dh": "dh must have", "gated grad: g alone": "projections that gated_linear returned",
    "gated8: several types": r"two weights \(1, f, k\)", "gated8: weights' shapes": r"two weights \(1, f, k\)", "gated8: activation": "unknown activation",
    "gated8: output type": "output must be float32", "dense norm: width": r"\(\.\.\., n\) and a weight", "dense gated: inner dimension": r"\(\.\.\., k\) and two weights",
}


def refused_calls(device):
    from test_dense_refusals import calls
    return calls(device)


def test_every_refusal_has_a_reason():
    assert set(REASONS) == set(refused_calls("cpu"))


@pytest.mark.gpu
@pytest.mark.parametrize("what", sorted(REASONS))
def test_refused_for_its_reason(what):
    with pytest.raises(capi().GphlError, match=REASONS[what]):
        refused_calls("cuda")[what]()


OPERATORS = ["norm", "norm grad", "norm8", "quantize", "quantize weight", "dequantize", "mm8", "gated", "gated grad", "gated8", "dense norm", "dense gated"]


def good_calls(device):
    """A call of each operator that nothing is wrong with but, on the CPU, the device."""
    from graphiler_b200 import dense
    c = capi()
    e = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype, device=device)
    x, v, w, q = e(4, 64), e(64), e(64, 32), c.Fp8Rows(e(4, 64, dtype=torch.uint8).view(F8), e(4, 1, dtype=F32))
    qw = c.Fp8Weight(e(1, 32, 64, dtype=torch.uint8).view(F8), e(1, 1, 1, dtype=F32))
    return dict(zip(OPERATORS, [
        lambda: c.rms_norm(x, v), lambda: c.rms_norm_grad(x, v, e(4, dtype=F32), x), lambda: c.rms_norm_fp8(x, v), lambda: c.quantize_fp8(x),
        lambda: c.quantize_fp8_weight(w), lambda: c.dequantize_fp8(q), lambda: c.segment_mm_fp8(q, qw), lambda: c.gated_linear(x, w, w),
        lambda: c.gated_linear_grad(e(4, 32), None, None, x, w, w), lambda: c.gated_linear_fp8(q, qw, qw), lambda: dense.rms_norm(x, v),
        lambda: dense.gated_linear(x, w, w)]))


@pytest.mark.parametrize("what", OPERATORS)
def test_no_cpu_path(what):
    with pytest.raises(capi().GphlError, match="need CUDA tensors"):
        good_calls("cpu")[what]()


@pytest.mark.gpu
@pytest.mark.parametrize("what", OPERATORS)
def test_the_same_call_on_the_gpu(what):
    good_calls("cuda")[what]()


# ---- after an attention layer -------------------------------------------------------------------------------------------------------

def block(r, p, rows=lambda v: v, weight=lambda w: w.double()):
    """r + (silu(n Wg) * (n Wu)) Wd in 64 bits; `rows` and `weight`: what is rounded on the way."""
    n = rows(ref.rms_norm(r, None, p["norm_weight"], 1e-6)[2])
    g, u = n @ weight(p["gate_weight"]), n @ weight(p["up_weight"])
    return r.double() + rows(ref.act(g, "silu")[0] * u) @ weight(p["down_weight"])


@pytest.mark.gpu
def test_feed_forward_after_attention():
    """The attention layer puts out 32 bits: the 8-bit form takes them, the 16-bit form takes them cast and refuses them as they are."""
    from graphiler_b200 import layers, synthetic
    w = synthetic.make_c4(scale=0.01).to("cuda")
    a = layers.hgt_layer(layers.PreparedGraph(w.graph), w.feats, w.params, int(w.hyper["heads"]), w.hyper["sqrt_dk"])
    d = a.shape[1]
    p = ff_params(d, 3 * d + 8)
    with pytest.raises(capi().GphlError, match="type|bfloat16"):
        layers.feed_forward_layer(a, {k: v.float() for k, v in p.items()})
    h = a.bfloat16()
    got, want = layers.feed_forward_layer(h, p), block(h, p)
    # n, the gated rows, the product and the sum are rounded once each: four half steps of the largest value, and as much for what the products add up
    assert float((got.double() - want).abs().max()) <= 8 * ref.half_step(BF16) * float(want.abs().max())
    p32 = {k: v.float() for k, v in p.items()}
    got = layers.feed_forward_layer_fp8(a, layers.prepare_feed_forward_fp8(p32))
    want = block(a, p32, rows=lambda v: ref.quantize_rows(v)[0], weight=lambda w: ref.quantize_weight(w[None])[0][0].t())
    assert got.dtype == F32
    # codes beside a border fall on its other side for a share of 2^-16 of n, which moves g and u by 2^-11 and a share of 2^-7 of the second codes by 2^-3
    assert float((got.double() - want).norm()) <= 2.0 ** -6.5 * float((want - a.double()).norm()) + 2 * ref.half_step(F32) * float(want.norm())


# ---- offsets beyond 32 bits -----------------------------------------------------------------------------------------------------------

BLOCK_ROWS, REPS, FAR = 656, 400, 8200            # 262,400 rows of 8200: 2.15e9 values


def repeated(*shape, seed, dtype=BF16):
    """A block of rows, again and again: every block has to come out as the first one does."""
    return randn(BLOCK_ROWS, *shape, seed=seed, dtype=dtype).repeat(REPS, 1)


def blocks_alike(y):
    first = y[:BLOCK_ROWS]
    return all(torch.equal(y[a:a + BLOCK_ROWS], first) for a in range(0, y.shape[0], BLOCK_ROWS))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [FAR, FAR + 1])
def test_norms_of_far_rows(n):
    c = capi()
    x, res, w = repeated(n, seed=1), repeated(n, seed=2), randn(n, seed=3, dtype=BF16)
    y, r, rstd = c.rms_norm(x, w, residual=res, return_rstd=True)
    assert blocks_alike(y) and blocks_alike(r) and blocks_alike(rstd)
    _, _, want = ref.rms_norm(x[:8], res[:8], w, 1e-6)
    ref.close(y[:8], want, ref.FP32 * want.abs())
    dx, dw = c.rms_norm_grad(r, w, rstd, y, res)
    assert blocks_alike(dx) and torch.isfinite(dw).all()
    del dx, y, r
    q, r = c.rms_norm_fp8(x, w, residual=res)
    assert blocks_alike(q.values.view(torch.uint8)) and blocks_alike(q.scales) and blocks_alike(r)
    del q, r, res
    q = c.quantize_fp8(x)
    assert blocks_alike(q.values.view(torch.uint8)) and blocks_alike(q.scales)
    assert blocks_alike(c.dequantize_fp8(q, BF16))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [FAR, FAR + 1])
def test_products_of_far_rows(n):
    c = capi()
    x, w = repeated(128, seed=1), randn(128, n, seed=2, dtype=BF16)
    x8, w8 = c.quantize_fp8(x), c.quantize_fp8_weight(w)
    y = c.segment_mm_fp8(x8, w8)
    assert blocks_alike(y)
    want = ref.rows_value(x8)[:8] @ ref.weight_value(w8)[0].t()
    ref.close(y[:8], want, ref.sum_loss(128, fp8=True) * (ref.rows_value(x8)[:8].abs() @ ref.weight_value(w8)[0].t().abs()))
    del y
    q = c.gated_linear_fp8(x8, w8, w8)
    assert blocks_alike(q.values.view(torch.uint8)) and blocks_alike(q.scales)
    del q
    h, g, u = c.gated_linear(x, w, w, return_projections=True)
    assert blocks_alike(h) and blocks_alike(g[:, :n]) and blocks_alike(u[:, :n])
    dx, _, _ = c.gated_linear_grad(h, g, u, x, w, w)
    assert blocks_alike(dx)
    del g, u
    again, _, _ = c.gated_linear_grad(h, None, None, x, w, w)
    assert torch.equal(again, dx)

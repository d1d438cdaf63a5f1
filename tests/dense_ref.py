"""The dense operators restated in 64 bits for the tests, with bounds of the kernels' rounding.

A rounding to type t is off by at most half a step, eps(t) / 2 relative.  A tensor-core sum is taken to lose at most 2^-22 of
the sum of magnitudes with each of its additions (one per 16 or 32 values of k and per block), fp32 elementwise chains 2^-20 relative."""
import torch

BLK = 128
FP32 = 2.0 ** -20


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def fp8_scale(amax):
    """The smallest power of two s >= 2^-126 with amax <= 448 s."""
    f, e = torch.frexp(amax.double())
    e = torch.where(amax > 0, e - 9 + (f > 0.875), torch.full_like(e, -126)).clamp(min=-126)
    return torch.ldexp(torch.ones_like(amax, dtype=torch.float64), e)


def fp8_round(v):
    """e4m3 value nearest to v (float64, |v| <= 448), ties to even; NaN stays."""
    a = v.abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    return torch.sign(v) * torch.round(a / step) * step


def blocks(v, dims):
    """v padded with zeros to whole blocks of 128 along `dims`, each such dimension split in two."""
    for d in sorted(dims, reverse=True):
        n = v.shape[d]
        pad = [0, 0] * v.dim()
        pad[2 * (v.dim() - 1 - d) + 1] = -n % BLK
        v = torch.nn.functional.pad(v, pad)
        v = v.reshape(v.shape[:d] + (v.shape[d] // BLK, BLK) + v.shape[d + 1:])
    return v


def finite(v):
    return torch.where(torch.isfinite(v), v, torch.zeros_like(v))


def quantize_rows(y):
    """(values that the codes stand for, scales) of float64 rows."""
    m, k = y.shape
    s = fp8_scale(blocks(finite(y).abs(), [1]).amax(dim=2)) if k else y.new_zeros(m, 0)
    full = s.repeat_interleave(BLK, dim=1)[:, :k]
    return torch.where(torch.isfinite(y), fp8_round(finite(y) / full), torch.full_like(y, float("nan"))) * full, s


def quantize_weight(w):
    """(T, K, N) -> values (T, N, K), scales (T, nb, kb)."""
    t, k, n = w.shape
    v = w.double().transpose(1, 2)
    s = fp8_scale(blocks(finite(v).abs(), [1, 2]).amax(dim=(2, 4)))
    full = s.repeat_interleave(BLK, dim=1)[:, :n].repeat_interleave(BLK, dim=2)[:, :, :k]
    return torch.where(torch.isfinite(v), fp8_round(finite(v) / full), torch.full_like(v, float("nan"))) * full, s


def rows_value(q):
    """float64 values of Fp8Rows."""
    m, k = q.values.shape
    return q.values.float().double() * q.scales.double().repeat_interleave(BLK, dim=1)[:, :k]


def weight_value(w):
    t, n, k = w.values.shape
    return w.values.float().double() * w.scales.double().repeat_interleave(BLK, dim=1)[:, :n].repeat_interleave(BLK, dim=2)[:, :, :k]


def rms_norm(x, res, w, eps):
    r = x if res is None else (x.float() + res.float()).to(x.dtype)
    rd = r.double()
    rstd = 1 / torch.sqrt(rd.square().mean(dim=1, keepdim=True) + eps)
    return r, rstd, rd * rstd * w.double()


def rms_norm_grad(r, rstd, w, dy, dr):
    xhat = r.double() * rstd
    g = dy.double() * w.double()
    mean = (g * xhat).mean(dim=1, keepdim=True)
    dx = rstd * (g - xhat * mean) + (0 if dr is None else dr.double())
    size = rstd * (g.abs() + xhat.abs() * (g * xhat).abs().mean(dim=1, keepdim=True)) + (0 if dr is None else dr.double().abs())
    return dx, (dy.double() * xhat).sum(dim=0), size, (dy.double() * xhat).abs().sum(dim=0)


def act(g, name):
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if name == "gelu":
        c = torch.special.ndtr(g)
        return g * c, c + g * torch.exp(-g * g / 2) * (0.5 / torch.pi) ** 0.5
    return g.clamp(min=0), (g > 0).to(g.dtype)


def sum_loss(k, fp8=False):
    """Relative loss of a tensor-core sum over k, of the sum of magnitudes."""
    return (k / (32 if fp8 else 16) + 8 + (k / 128 if fp8 else 0)) * 2.0 ** -22


def gated(x, wg, wu, name):
    """h in 64 bits and the bound of its error before the last rounding; also g, u and their bounds."""
    x, wg, wu = x.double(), wg.double(), wu.double()
    g, u = x @ wg, x @ wu
    a, da = act(g, name)
    eg, eu = (x.abs() @ wg.abs()) * sum_loss(x.shape[1]), (x.abs() @ wu.abs()) * sum_loss(x.shape[1])
    err = 1.13 * u.abs() * eg + (a.abs() + 1.13 * eg) * eu + FP32 * (g.abs() * u.abs())     # |act'| <= 1.13; act in fast fp32, |act(g)| <= |g|
    return a * u, err, (g, u, a, da, eg, eu)


def gated_grad(dh, x, wg, wu, name, dtype):
    """dx, dWg, dWu in 64 bits and bounds of their errors before the last rounding."""
    h, _, (g, u, a, da, eg, eu) = gated(x, wg, wu, name)
    dh, x, wg, wu = dh.double(), x.double(), wg.double(), wu.double()
    dg, du = dh * u * da, dh * a
    # |act''| <= 1 for the smooth ones; for relu the sign of g must be certain (checked by the caller)
    edg = dh.abs() * (1.13 * eu + (u.abs() + eu) * (eg if name != "relu" else 0) + FP32 * (u.abs() + u.abs() * g.abs()))
    edu = dh.abs() * (1.13 * eg + FP32 * g.abs())
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0          # half a step of fp16's subnormals
    edg, edu = edg + (half_step(dtype) * (dg.abs() + edg)).clamp(min=tiny), edu + (half_step(dtype) * (du.abs() + edu)).clamp(min=tiny)
    f, m = wg.shape[1], x.shape[0]
    dx = dg @ wg.t() + du @ wu.t()
    edx = edg @ wg.abs().t() + edu @ wu.abs().t() + sum_loss(2 * f) * (dg.abs() @ wg.abs().t() + du.abs() @ wu.abs().t())
    out = [(dx, edx)]
    for d, e in ((dg, edg), (du, edu)):
        out.append((x.t() @ d, x.abs().t() @ e + sum_loss(m) * (x.abs().t() @ d.abs())))
    return out


def close(got, want, err, dtype=None, what=""):
    """got (rounded to dtype) within half a step of a value no further than err from want."""
    dtype = dtype or got.dtype
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134 if dtype == torch.bfloat16 else 2.0 ** -150
    bound = err + (half_step(dtype) * (want.abs() + err)).clamp(min=tiny)
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / bound).max()):.3g} x the bound"

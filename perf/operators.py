"""The dense operators of a transformer block on node rows: what is measured of them.

Operators: root-mean-square norm with the residual's addition (16 / 32 bits with its backward pass, or e4m3 with a scale per row and
128 columns; scales are powers of two, so that scaling rounds nothing), the typed product of e4m3 rows with e4m3 weights (a scale per 128 values / per 128 x 128 values), and the gated feed-forward
h = act(x Wg) * (x Wu) (16 bits with its backward pass; e4m3 for serving), alone and as the chain norm -> gated -> product.
"""
import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6
BLK = 128
ACTS = ("silu", "gelu", "relu")


def listed():
    return [
        # one token's hidden state on its way into an 8-bit projection: launch latency alone
        {"name": "norm8 1 token", "op": "norm8", "m": 1, "d": 4096, "dt": "bf16"},
        # a long prompt's rows
        {"name": "norm8 32k rows", "op": "norm8", "m": 32768, "d": 8192, "dt": "bf16"},
        # odd width, single precision, as the layers of this library keep their node rows
        {"name": "norm step odd f32", "op": "norm", "m": 10007, "d": 1001, "dt": "f32"},
        # training over the node rows of a large graph: many short rows
        {"name": "norm step nodes", "op": "norm", "m": 600000, "d": 256, "dt": "bf16"},
        # single-token decoding: bound by the weights' bytes
        {"name": "mm8 1 token", "op": "mm8", "m": 1, "k": 4096, "n": 8192, "t": 1, "dt": "bf16"},
        # node rows grouped by type, ragged groups (one of them empty), widths that end inside a block
        {"name": "mm8 typed odd", "op": "mm8", "m": 5003, "k": 1000, "n": 777, "t": 7, "dt": "f16"},
        # a prompt's projection
        {"name": "mm8 16k rows", "op": "mm8", "m": 16384, "k": 8192, "n": 8192, "t": 1, "dt": "bf16"},
        # decoding a small batch in 16 bits, no gradients
        {"name": "gated 5 tokens", "op": "gated", "m": 5, "k": 4096, "f": 11264, "act": "silu", "dt": "bf16"},
        # odd sizes, fp16, the smooth activation
        {"name": "gated step odd f16", "op": "gated_step", "m": 1537, "k": 520, "f": 1400, "act": "gelu", "dt": "f16"},
        # training step on long sequences
        {"name": "gated step 8k rows", "op": "gated_step", "m": 8192, "k": 4096, "f": 11264, "act": "silu", "dt": "bf16"},
        # training step over a graph's node rows: many rows, narrow weights
        {"name": "gated step nodes", "op": "gated_step", "m": 300000, "k": 256, "f": 1024, "act": "silu", "dt": "bf16"},
        # the chain as it is served: norm -> gated -> product, all in 8 bits
        {"name": "block8 2k rows", "op": "block8", "m": 2048, "k": 4096, "f": 11264, "act": "silu", "dt": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["norm8", "norm", "mm8", "gated", "gated_step", "block8"])
    dt = rng.choice(["bf16", "bf16", "f16"])
    if op in ("norm8", "norm"):
        d = _log(rng, 64, 8192)
        if rng.random() < 0.5:
            d = max(16, d // 16 * 16)
        return {"op": op, "m": _log(rng, 1, min(600000, 32768 * 8192 // 4 // d)), "d": d, "dt": rng.choice(["bf16", "f16", "f32"])}
    act = rng.choice(ACTS)
    k, f = _log(rng, 128, 4096), _log(rng, 128, 11264)
    if rng.random() < 0.6:                       # widths of networks are mostly round; the others are odd ones
        k, f = max(64, k // 64 * 64), max(64, f // 64 * 64)
    most = 8192 * 4096 * 11264 // 4
    m = _log(rng, 1, max(2, min(100000, most // (k * f))))
    if op == "mm8":
        t = rng.choice([1, 1, 2, 5, 16])
        return {"op": op, "m": m, "k": k, "n": f, "t": t, "dt": dt}
    return {"op": op, "m": m, "k": k, "f": f, "act": act, "dt": dt}


# ---- inputs -----------------------------------------------------------------------------------------------------

def _randn(g, *shape, dt=torch.float32, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda").mul_(scale).to(dt)


def _pointer(m, t, seed):
    """Ragged groups: cut points at random places, the first group of several empty."""
    g = torch.Generator().manual_seed(seed + 1)
    cuts = torch.sort(torch.randint(0, m + 1, (max(t - 1, 0),), generator=g)).values.tolist()
    if cuts:
        cuts[0] = 0
    return torch.tensor([0] + cuts + [m], dtype=torch.int32, device="cuda")


def _scale(amax):
    """The smallest power of two s >= 2^-126 with amax <= 448 s."""
    f, e = torch.frexp(amax)                    # amax = f 2^e, 1/2 <= f < 1; 448 = 0.875 * 2^9
    e = torch.where(amax > 0, e - 9 + (f > 0.875), -126).clamp_min(-126)
    return torch.ldexp(torch.ones_like(amax), e)


def _quant_rows(v):
    """e4m3 values and scales of the rows of v: (M, K), (M, ceil(K / 128))."""
    m, k = v.shape
    nb = -(-k // BLK)
    b = torch.nn.functional.pad(v, (0, nb * BLK - k)).view(m, nb, BLK)
    s = _scale(b.abs().amax(dim=2))
    return (b / s.unsqueeze(2)).view(m, nb * BLK)[:, :k].to(torch.float8_e4m3fn), s


def _quant_weight(w):
    """w (T, K, N) -> e4m3 (T, N, K) and scales (T, ceil(N / 128), ceil(K / 128)), one per 128 x 128 values."""
    t, k, n = w.shape
    nb, kb = -(-n // BLK), -(-k // BLK)
    p = torch.nn.functional.pad(w.float().transpose(1, 2), (0, kb * BLK - k, 0, nb * BLK - n)).view(t, nb, BLK, kb, BLK)
    s = _scale(p.abs().amax(dim=(2, 4)))
    q = p / s[:, :, None, :, None]
    return q.view(t, nb * BLK, kb * BLK)[:, :n, :k].to(torch.float8_e4m3fn), s


def _padded(q):
    """The same values with rows that start on 16-byte boundaries, as the library's quantisers lay them out."""
    k = q.shape[-1]
    kp = -(-k // 16) * 16
    out = torch.zeros(*q.shape[:-1], kp, dtype=torch.uint8, device=q.device)
    out[..., :k] = q.view(torch.uint8)
    return out.view(torch.float8_e4m3fn)[..., :k]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, m, dt = case["op"], case["m"], DT[case["dt"]]
    s = {"case": case}
    if op in ("norm8", "norm"):
        d = case["d"]
        # rows of a residual stream: some rows much larger than others, a few large columns
        size = torch.exp(_randn(g, m, 1, scale=0.7))
        cols = torch.exp(_randn(g, 1, d, scale=0.7))
        s["x"] = (_randn(g, m, d) * size * cols).to(dt)
        s["res"] = (_randn(g, m, d) * size * cols).to(dt)
        s["w"] = (1.0 + 0.2 * _randn(g, d)).to(dt)
        if op == "norm":
            s["dy"], s["dr"] = _randn(g, m, d, dt=dt), _randn(g, m, d, dt=dt)
            for n in ("x", "res", "w"):
                s[n].requires_grad_(True)
        return s
    if op == "mm8":
        k, n, t = case["k"], case["n"], case["t"]
        q, s["xs"] = _quant_rows(_randn(g, m, k) * torch.exp(_randn(g, m, 1, scale=0.7)))
        w, s["ws"] = _quant_weight(_randn(g, t, k, n, scale=k ** -0.5))
        s["x8"], s["w8"] = _padded(q), _padded(w)
        s["ptr"] = _pointer(m, t, seed) if t > 1 else None
        s["xs"] = s["xs"].t().contiguous().t()      # one block's scales of consecutive rows lie together, as the quantisers lay them out
        return s
    k, f = case["k"], case["f"]
    s["x"] = _randn(g, m, k, dt=dt)
    wg, wu = _randn(g, k, f, dt=dt, scale=k ** -0.5), _randn(g, k, f, dt=dt, scale=k ** -0.5)
    if op == "block8":
        s["res"], s["w"] = _randn(g, m, k, dt=dt), (1.0 + 0.2 * _randn(g, k)).to(dt)
        wd = _randn(g, 1, f, k, scale=f ** -0.5)
        for name, w in (("g", wg.unsqueeze(0)), ("u", wu.unsqueeze(0)), ("d", wd)):
            q, sc = _quant_weight(w)
            s[name + "8"], s[name + "s"] = _padded(q), sc
        return s
    s["wg"], s["wu"] = wg, wu
    if op == "gated_step":
        s["dh"] = _randn(g, m, f, dt=dt)
        for n in ("x", "wg", "wu"):
            s[n].requires_grad_(True)
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------

def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    from graphiler_b200 import capi, dense

    case = s["case"]
    op = case["op"]
    if op == "norm8":
        q, r = capi.rms_norm_fp8(s["x"], s["w"], EPS, residual=s["res"])
        return {"y": capi.dequantize_fp8(q, torch.bfloat16), "r": r}       # 4 significant bits times a power of two: exact
    if op == "norm":
        y, r = dense.rms_norm(s["x"], s["w"], EPS, residual=s["res"])
        dx, dres, dw = torch.autograd.grad((y, r), (s["x"], s["res"], s["w"]), (s["dy"], s["dr"]))
        return {"y": y, "r": r, "dx": dx, "dres": dres, "dw": dw}
    if op == "mm8":
        return {"y": capi.segment_mm_fp8(capi.Fp8Rows(s["x8"], s["xs"]), capi.Fp8Weight(s["w8"], s["ws"]), s["ptr"], out_dtype=DT[case["dt"]])}
    if op == "gated":
        return {"h": capi.gated_linear(s["x"], s["wg"], s["wu"], case["act"])}
    if op == "gated_step":
        h = dense.gated_linear(s["x"], s["wg"], s["wu"], case["act"])
        dx, dwg, dwu = torch.autograd.grad(h, (s["x"], s["wg"], s["wu"]), s["dh"])
        return {"h": h, "dx": dx, "dwg": dwg, "dwu": dwu}
    n8, r = capi.rms_norm_fp8(s["x"], s["w"], EPS, residual=s["res"])
    h8 = capi.gated_linear_fp8(n8, capi.Fp8Weight(s["g8"], s["gs"]), capi.Fp8Weight(s["u8"], s["us"]), case["act"])
    y = capi.segment_mm_fp8(h8, capi.Fp8Weight(s["d8"], s["ds"]), out_dtype=DT[case["dt"]])
    return {"y": y, "r": r}


def _act(g, act):
    """act(g) and its derivative."""
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if act == "gelu":
        c = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
        return g * c, c + g * torch.exp(-0.5 * g * g) * (0.5 / torch.pi) ** 0.5
    p = (g > 0).to(g.dtype)
    return g * p, p


def _norm(x, res, w):
    """The stored sum r, 1 / rms and the normalised rows, float32."""
    r = (x.float() + res.float()).to(x.dtype)
    rf = r.float()
    rstd = torch.rsqrt(rf.square().mean(dim=1, keepdim=True) + EPS)
    return r, rstd, rf * rstd * w.float()


def _rows(q, sc):
    return q.float() * sc.repeat_interleave(BLK, dim=1)[:, :q.shape[1]]


def _weight(q, sc):
    t, n, k = q.shape
    return q.float() * sc.repeat_interleave(BLK, dim=1)[:, :n].repeat_interleave(BLK, dim=2)[:, :, :k]


def _plain(s):
    with torch.no_grad():
        case = s["case"]
        op, dt = case["op"], DT[case["dt"]]
        if op == "norm8":
            r, _, y = _norm(s["x"], s["res"], s["w"])
            return {"y": _rows(*_quant_rows(y)).bfloat16(), "r": r}
        if op == "norm":
            r, rstd, y = _norm(s["x"], s["res"], s["w"])
            xhat = r.float() * rstd
            dy = s["dy"].float()
            g = dy * s["w"].float()
            dx = (s["dr"].float() + rstd * (g - xhat * (g * xhat).mean(dim=1, keepdim=True))).to(dt)
            return {"y": y.to(dt), "r": r, "dx": dx, "dres": dx, "dw": (dy * xhat).sum(dim=0).to(dt)}
        if op == "mm8":
            x, w = _rows(s["x8"], s["xs"]), _weight(s["w8"], s["ws"])
            if s["ptr"] is None:
                return {"y": (x @ w[0].t()).to(dt)}
            ptr = s["ptr"].tolist()
            return {"y": torch.cat([x[a:b] @ w[i].t() for i, (a, b) in enumerate(zip(ptr, ptr[1:]))]).to(dt)}
        if op == "block8":
            r, _, y = _norm(s["x"], s["res"], s["w"])
            n = _rows(*_quant_rows(y))
            h = _act(n @ _weight(s["g8"], s["gs"])[0].t(), case["act"])[0] * (n @ _weight(s["u8"], s["us"])[0].t())
            return {"y": (_rows(*_quant_rows(h)) @ _weight(s["d8"], s["ds"])[0].t()).to(dt), "r": r}
        x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
        g, u = x @ wg, x @ wu
        a, da = _act(g, case["act"])
        if op == "gated":
            return {"h": (a * u).to(dt)}
        dh = s["dh"].float()
        dg, du = dh * u * da, dh * a
        return {"h": (a * u).to(dt), "dx": (dg @ wg.t() + du @ wu.t()).to(dt), "dwg": (x.t() @ dg).to(dt), "dwu": (x.t() @ du).to(dt)}


# ---- the work of a pass -----------------------------------------------------------------------------------------

def work(case):
    op, m, b = case["op"], case["m"], SIZE[case["dt"]]
    if op == "norm8":
        d = case["d"]
        return {"bytes": m * d * (3 * b + 2) + d * b, "flops": 6 * m * d}
    if op == "norm":
        d = case["d"]
        return {"bytes": m * d * 8 * b + 2 * d * b, "flops": 16 * m * d}
    if op == "mm8":
        k, n, t = case["k"], case["n"], case["t"]
        kb = -(-k // BLK)
        return {"bytes": m * k + t * k * n + m * n * b + 4 * (m * kb + t * kb * -(-n // BLK)), "flops": 2 * m * k * n}
    k, f = case["k"], case["f"]
    if op == "gated":
        return {"bytes": b * (m * k + 2 * k * f + m * f), "flops": 4 * m * k * f}
    if op == "gated_step":
        return {"bytes": b * (2 * m * k + 4 * k * f + 2 * m * f), "flops": 12 * m * k * f}
    return {"bytes": 4 * m * k * b + 3 * k * f, "flops": 6 * m * k * f}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------

SECONDS_FLOPS = 1.2e13          # double-precision products a second, well below the card's rate


def exact(case, seed):
    if work(case)["flops"] > 18 * SECONDS_FLOPS and case["op"] not in ("norm", "norm8"):
        return None
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm8": _exact_norm8, "norm": _exact_norm, "mm8": _exact_mm8, "block8": _exact_block}.get(case["op"], _exact_gated)(s)


def _chunks(m, width):
    step = max(1, (1 << 26) // max(1, width))
    return [(a, min(m, a + step)) for a in range(0, m, step)]


def _exact_q(y):
    """The e4m3 code's value of each element and the scale of each block, from 64-bit rows."""
    q, sc = torch.empty_like(y), []
    for c in range(0, y.shape[1], BLK):
        part = y[:, c:c + BLK]
        scale = torch.exp2(torch.ceil(torch.log2(part.abs().max(dim=1, keepdim=True).values / 448)).clamp(min=-126))
        v = part.abs() / scale
        step = torch.exp2(torch.floor(torch.log2(v.clamp(min=2.0 ** -6))) - 3)              # 3 bits behind the leading one, 2^-9 at the least
        q[:, c:c + BLK] = torch.round(v / step) * step * torch.sign(part)                    # ties to even
        sc.append(scale)
    return q, torch.cat(sc, dim=1)


def _exact_y(s, a, b):
    # the sum is kept in the rows' own type: what the next layer adds to is what is normalised
    r = (s["x"][a:b].double() + s["res"][a:b].double()).to(s["x"].dtype)
    rd = r.double()
    rms = torch.sqrt((rd * rd).sum(dim=1, keepdim=True) / rd.shape[1] + EPS)
    return r, rd / rms, rms


def _exact_norm8(s):
    m, d = s["x"].shape
    parts = []
    for a, b in _chunks(m, d):
        _, xh, _ = _exact_y(s, a, b)
        q, sc = _exact_q(xh * s["w"].double())
        r = s["x"][a:b].double() + s["res"][a:b].double()
        parts.append((q * sc.repeat_interleave(BLK, dim=1)[:, :d], r))
    return {"y": torch.cat([p[0] for p in parts]), "r": torch.cat([p[1] for p in parts])}


def _exact_norm(s):
    m, d = s["x"].shape
    w, dw, parts = s["w"].double(), 0, []
    for a, b in _chunks(m, d):
        _, xh, rms = _exact_y(s, a, b)
        dy = s["dy"][a:b].double()
        dw = dw + torch.einsum("md,md->d", dy, xh)
        inner = torch.einsum("md,md->m", dy * w, xh).unsqueeze(1) / d
        dx = s["dr"][a:b].double() + (dy * w - xh * inner) / rms
        parts.append((xh * w, s["x"][a:b].double() + s["res"][a:b].double(), dx))
    y, r, dx = (torch.cat([p[i] for p in parts]) for i in range(3))
    return {"y": y, "r": r, "dx": dx, "dres": dx, "dw": dw}


def _exact_product(q, sc, w, ws):
    """sum over the blocks of 128 of the two scales times the block's product."""
    y = torch.zeros(q.shape[0], w.shape[0], dtype=torch.float64, device=q.device)
    of_n = torch.arange(w.shape[0], device=q.device) // BLK
    for i, c in enumerate(range(0, q.shape[1], BLK)):
        part = q[:, c:c + BLK].double() @ w[:, c:c + BLK].double().t()
        y += part * sc[:, i:i + 1].double() * ws[of_n, i].double()
    return y


def _exact_mm8(s):
    ptr = [0, s["x8"].shape[0]] if s["ptr"] is None else s["ptr"].tolist()
    return {"y": torch.cat([_exact_product(s["x8"][a:b].float(), s["xs"][a:b], s["w8"][i].float(), s["ws"][i]) for i, (a, b) in enumerate(zip(ptr, ptr[1:]))])}


def _exact_act(g, act):
    if act == "silu":
        p = 1 / (1 + torch.exp(-g))
        return g * p, p + g * p * (1 - p)
    if act == "gelu":
        p = torch.special.ndtr(g)
        return g * p, p + g * torch.exp(-g * g / 2) / (2 * torch.pi) ** 0.5
    return torch.clamp(g, min=0), torch.heaviside(g, torch.zeros((), dtype=g.dtype, device=g.device))


def _exact_block(s):
    case = s["case"]
    r, xh, _ = _exact_y(s, 0, case["m"])
    q, sc = _exact_q(xh * s["w"].double())
    g = _exact_product(q, sc, s["g8"][0].float(), s["gs"][0])
    u = _exact_product(q, sc, s["u8"][0].float(), s["us"][0])
    q, sc = _exact_q(_exact_act(g, case["act"])[0] * u)
    return {"y": _exact_product(q, sc, s["d8"][0].float(), s["ds"][0]), "r": s["x"].double() + s["res"].double()}


def _exact_gated(s):
    case = s["case"]
    x, wg, wu = s["x"].double(), s["wg"].double(), s["wu"].double()
    g, u = torch.mm(x, wg), torch.mm(x, wu)
    a, da = _exact_act(g, case["act"])
    if case["op"] == "gated":
        return {"h": a * u}
    dh = s["dh"].double()
    dg, du = dh * da * u, dh * a
    return {"h": a * u, "dx": torch.mm(dg, wg.t()) + torch.mm(du, wu.t()), "dwg": torch.mm(x.t(), dg), "dwu": torch.mm(x.t(), du)}

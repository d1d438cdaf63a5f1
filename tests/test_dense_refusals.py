"""What the dense operators refuse, checked before anything is launched."""
import pytest
import torch

from graphiler_b200 import capi, dense

F8 = torch.float8_e4m3fn


def rows(m=4, k=64, dtype=torch.bfloat16, device="cpu"):
    return torch.zeros(m, k, dtype=dtype, device=device)


def calls(device):
    """(what is wrong, a call that is refused)."""
    x, w, v = rows(device=device), rows(64, 32, device=device), torch.zeros(64, dtype=torch.bfloat16, device=device)
    q = capi.Fp8Rows(torch.zeros(4, 64, dtype=torch.uint8, device=device).view(F8), torch.zeros(4, 1, device=device))
    qw = capi.Fp8Weight(torch.zeros(1, 32, 64, dtype=torch.uint8, device=device).view(F8), torch.zeros(1, 1, 1, device=device))
    qw2 = capi.Fp8Weight(torch.zeros(2, 32, 64, dtype=torch.uint8, device=device).view(F8), torch.zeros(2, 1, 1, device=device))
    odd = capi.Fp8Rows(torch.zeros(4, 72, dtype=torch.uint8, device=device).view(F8)[:, :63], torch.zeros(4, 1, device=device))
    f = lambda t: t.float()
    return {
        "norm: width": lambda: capi.rms_norm(x, v[:32]),
        "norm: residual's shape": lambda: capi.rms_norm(x, v, residual=x[:2]),
        "norm: residual's type": lambda: capi.rms_norm(x, v, residual=f(x)),
        "norm: weight's type": lambda: capi.rms_norm(x, v.half()),
        "norm: integers": lambda: capi.rms_norm(x.int(), v.int()),
        "norm: negative eps": lambda: capi.rms_norm(x, v, eps=-1.0),
        "norm: strided rows": lambda: capi.rms_norm(rows(4, 128, device=device)[:, :64], v),
        "norm8: width": lambda: capi.rms_norm_fp8(x, v[:32]),
        "norm grad: rstd": lambda: capi.rms_norm_grad(x, v, f(v), x),
        "norm grad: dy": lambda: capi.rms_norm_grad(x, v, torch.zeros(4, device=device), f(x)),
        "quantize: dimensions": lambda: capi.quantize_fp8(v),
        "quantize: doubles": lambda: capi.quantize_fp8(x.double()),
        "quantize weight: dimensions": lambda: capi.quantize_fp8_weight(v),
        "dequantize: output type": lambda: capi.dequantize_fp8(q, torch.float64),
        "dequantize: scales' shape": lambda: capi.dequantize_fp8(capi.Fp8Rows(q.values, q.scales[:, :0])),
        "mm8: inner dimension": lambda: capi.segment_mm_fp8(capi.Fp8Rows(q.values[:, :32], q.scales), qw),
        "mm8: rows not 16 bytes apart": lambda: capi.segment_mm_fp8(odd, capi.Fp8Weight(qw.values[..., :63], qw.scales)),
        "mm8: values' type": lambda: capi.segment_mm_fp8(capi.Fp8Rows(x, q.scales), qw),
        "mm8: several types, no pointer": lambda: capi.segment_mm_fp8(q, qw2),
        "mm8: pointer's length": lambda: capi.segment_mm_fp8(q, qw2, torch.zeros(2, dtype=torch.int32, device=device)),
        "mm8: pointer's type": lambda: capi.segment_mm_fp8(q, qw2, torch.zeros(3, dtype=torch.int64, device=device)),
        "mm8: output type": lambda: capi.segment_mm_fp8(q, qw, out_dtype=torch.float64),
        "mm8: out's shape": lambda: capi.segment_mm_fp8(q, qw, out=rows(4, 16, device=device)),
        "gated: activation": lambda: capi.gated_linear(x, w, w, "tanh"),
        "gated: float32": lambda: capi.gated_linear(f(x), f(w), f(w)),
        "gated: mixed types": lambda: capi.gated_linear(x, w, w.half()),
        "gated: weights' shapes": lambda: capi.gated_linear(x, w, w[:, :16]),
        "gated: inner dimension": lambda: capi.gated_linear(x, w[:32], w[:32]),
        "gated: one weight transposed": lambda: capi.gated_linear(x, w, rows(32, 64, device=device).t()),
        "gated: strided rows": lambda: capi.gated_linear(rows(4, 128, device=device)[:, :64], w, w),
        "gated grad: dh": lambda: capi.gated_linear_grad(x, None, None, x, w, w),
        "gated grad: g alone": lambda: capi.gated_linear_grad(rows(4, 32, device=device), torch.zeros(4, 32, device=device), None, x, w, w),
        "gated8: several types": lambda: capi.gated_linear_fp8(q, qw2, qw2),
        "gated8: weights' shapes": lambda: capi.gated_linear_fp8(q, qw, qw2),
        "gated8: activation": lambda: capi.gated_linear_fp8(q, qw, qw, "swish"),
        "gated8: output type": lambda: capi.gated_linear_fp8(q, qw, qw, out_dtype=torch.float64),
        "dense norm: width": lambda: dense.rms_norm(x, v[:32]),
        "dense gated: inner dimension": lambda: dense.gated_linear(x, w[:32], w[:32]),
    }


@pytest.fixture(scope="module", autouse=True)
def built():
    from graphiler_b200 import build
    build.build_all()


@pytest.mark.parametrize("what", sorted(calls("cpu")))
def test_refused_on_the_cpu(what):
    """There is no CPU path; shapes, types and devices are checked on the host."""
    with pytest.raises(capi.GphlError):
        calls("cpu")[what]()


@pytest.mark.gpu
@pytest.mark.parametrize("what", sorted(calls("cpu")))
def test_refused_on_the_gpu(what):
    before = capi.launch_count()
    with pytest.raises(capi.GphlError):
        calls("cuda")[what]()
    assert capi.launch_count() == before


def test_good_arguments_on_the_cpu_are_refused_for_their_device():
    with pytest.raises(capi.GphlError, match="CUDA"):
        capi.rms_norm(rows(), torch.zeros(64, dtype=torch.bfloat16))
    with pytest.raises(capi.GphlError, match="CUDA"):
        capi.gated_linear(rows(), rows(64, 32), rows(64, 32))


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    x, w = rows(device="cuda").requires_grad_(True), torch.ones(64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="first derivatives"):
        torch.autograd.grad(dense.rms_norm(x, w).sum(), x, create_graph=True)
    g = rows(64, 32, device="cuda")
    with pytest.raises(RuntimeError, match="first derivatives"):
        torch.autograd.grad(dense.gated_linear(x, g, g).sum(), x, create_graph=True)


@pytest.mark.gpu
def test_changed_inputs_are_noticed():
    x = torch.randn(4, 64, device="cuda").bfloat16().requires_grad_(True)
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda").requires_grad_(True)
    r = torch.randn(4, 64, device="cuda").bfloat16()
    y, s = dense.rms_norm(x, w, residual=r)
    s.add_(1)                                    # r is kept for the backward pass
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    x = torch.randn(2, 3, 64, device="cuda").bfloat16()
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda").requires_grad_(True)
    g = torch.randn(64, 32, device="cuda").bfloat16().requires_grad_(True)
    for y in (dense.rms_norm(x, w), dense.gated_linear(x, g, g)):
        x.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


@pytest.mark.gpu
def test_codes_without_padding_behind_the_last_row_are_refused():
    s = torch.ones(3, 1, device="cuda")
    whole = torch.zeros(3 * 48, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).as_strided((3, 36), (48, 1))
    assert capi.segment_mm_fp8(capi.Fp8Rows(whole, s), capi.quantize_fp8_weight(torch.ones(36, 16, device="cuda"))).shape == (3, 16)
    short = torch.zeros(3 * 48 - 12, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).as_strided((3, 36), (48, 1))
    with pytest.raises(capi.GphlError, match="padded"):
        capi.segment_mm_fp8(capi.Fp8Rows(short, s), capi.quantize_fp8_weight(torch.ones(36, 16, device="cuda")))

"""Operands whose offsets leave 32 bits: what lies at their end has the bits of the same values at their beginning."""
import math

import pytest
import torch

from flexflow_train_b200.ops import kernels as K

pytestmark = pytest.mark.gpu


def test_rms_norm_of_more_than_2_31_elements():
    rows, cols, few = 2 ** 20 + 2 ** 16, 2048, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for t in (x, dy):
        t[:few] = torch.randn(few, cols, generator=g, device="cuda").bfloat16()
        t[-few:] = t[:few]
    assert x.numel() > 2 ** 31
    gamma = torch.randn(cols, generator=g, device="cuda").bfloat16()
    rstd = torch.empty(rows, device="cuda")
    y = K.rmsnorm_fwd(x, gamma, 1e-5, rstd=rstd)
    assert y[:few].abs().sum() > 0 and torch.equal(y[:few], y[-few:]) and torch.equal(rstd[:few], rstd[-few:]) and not y[few:-few].any()
    dgamma = torch.empty_like(gamma)
    K.rmsnorm_bwd(dy, x, gamma, rstd, y, dgamma, torch.empty(K.rmsnorm_bwd_scratch(rows, cols), device="cuda"))
    assert y[:few].abs().sum() > 0 and torch.equal(y[:few], y[-few:]) and not y[few:-few].any()
    want = 2 * (dy[:few].double() * x[:few].double() * rstd[:few, None].double()).sum(0)
    size = 2 * (dy[:few].double() * x[:few].double() * rstd[:few, None].double()).abs().sum(0)
    # rounded to bf16 once; each term's two products and the sums of 128 terms in 32 bits
    assert ((dgamma.double() - want).abs() <= 2.0 ** -8 * want.abs() + 200 * 2.0 ** -24 * size).all()


def test_gradient_norm_of_more_than_2_32_elements():
    n = 2 ** 32 + 12345
    grad = torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda")
    grads = K.GradientList([grad])
    norm = K.clip_gradients(grads, math.sqrt(n) / 4).item()        # half of the norm
    assert abs(norm - math.sqrt(n) / 2) <= 2.0 ** -23 * norm
    assert grad.min().item() == grad.max().item() == 0.25


@pytest.mark.parametrize("D,KH", [(128, 4), (64, 2)])
def test_attention_over_matrices_of_more_than_2_31_elements(D, KH):
    B, S, H = 2200 * 128 // D, 160, 8
    ld = 6144                                                      # the heads lie in wide rows
    g = torch.Generator(device="cuda").manual_seed(2)

    def rows():
        t = torch.zeros(B * S, ld, dtype=torch.bfloat16, device="cuda")
        t[:S] = torch.randn(S, ld, generator=g, device="cuda").bfloat16()
        t[-S:] = t[:S]
        return t

    def heads(t):
        return t[:, :H * D], t[:, H * D:(H + KH) * D], t[:, (H + KH) * D:(H + 2 * KH) * D]

    qkv, dqkv = rows(), rows()
    assert qkv.numel() > 2 ** 31
    (q, k, v), (dq, dk, dv) = heads(qkv), heads(dqkv)
    out = torch.empty(B * S, H * D, dtype=torch.bfloat16, device="cuda")
    dout = torch.zeros_like(out)
    dout[:S] = torch.randn(S, H * D, generator=g, device="cuda").bfloat16()
    dout[-S:] = dout[:S]
    lse = torch.empty(B, H, S, device="cuda")
    spans = K.attention_spans(torch.zeros(B, S, dtype=torch.int32, device="cuda"))
    sizes = dict(B=B, S=S, H=H, KH=KH, D=D, scale=D ** -0.5)
    K.span_attention_fwd(q, k, v, out, lse, spans, **sizes)
    scratch = torch.empty(K.span_attention_bwd_scratch_floats(B, H, S), device="cuda")
    K.span_attention_bwd(q, k, v, out, lse, dout, dq, dk, dv, scratch, spans, **sizes)
    assert K.span_attention_last_error() == 0
    for t in (out, dq, dk, dv):
        assert t[:S].abs().sum() > 0 and torch.equal(t[:S], t[-S:])
    assert torch.equal(lse[0], lse[-1])
    one = dict(sizes, B=1)
    first = torch.empty(S, H * D, dtype=torch.bfloat16, device="cuda")
    K.span_attention_fwd(q[:S], k[:S], v[:S], first, torch.empty(1, H, S, device="cuda"), spans[:1], **one)
    assert torch.equal(first, out[:S])

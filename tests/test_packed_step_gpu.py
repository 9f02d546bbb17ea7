"""The operators of a packed-document step together, as a training loop uses them: spans, two layers' norms and attention between projections, their
gradients, clipping, Adam; against the same model in 64 bits under autograd."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from flexflow_train_b200.ops import kernels as K  # noqa: E402

from span_reference import spans_of, visible  # noqa: E402

B, S, H, KH, D, E, LAYERS, CAP, EPS = 2, 200, 4, 2, 32, 96, 2, 20.0, 1e-6
QKV = (H + 2 * KH) * D


def parameters(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *s: (torch.randn(*s, generator=g, device="cuda") / math.sqrt(s[-1])).bfloat16()  # noqa: E731
    return [{"gamma": 1 + 0.1 * new(1, E)[0], "qkv": new(QKV, E), "out": new(E, H * D)} for _ in range(LAYERS)]


def step(params, x, target, doc, prompt):
    """h = x + sum over layers of out(attention(qkv(norm(h)))), loss = sum h target; gradients of all parameters."""
    spans = K.attention_spans(doc, prompt)
    sizes = dict(B=B, S=S, H=H, KH=KH, D=D, scale=1.0 / math.sqrt(D), cap=CAP)
    rows, saved, residual, branch = B * S, [], x, None
    for p in params:
        y, rstd = torch.empty_like(x), torch.empty(rows, device="cuda")
        h = residual if branch is None else torch.empty_like(x)
        if branch is None:
            K.rmsnorm_fwd(residual, p["gamma"], EPS, out=y, rstd=rstd)
        else:
            K.rmsnorm_fwd(branch, p["gamma"], EPS, residual=residual, xsum=h, out=y, rstd=rstd)
        qkv = K.matmul_nt(y, p["qkv"])
        q, k, v = qkv[:, :H * D], qkv[:, H * D:(H + KH) * D], qkv[:, (H + KH) * D:]
        o, lse = torch.empty(rows, H * D, device="cuda", dtype=torch.bfloat16), torch.empty(B, H, S, device="cuda")
        K.span_attention_fwd(q, k, v, o, lse, spans, **sizes)
        branch = K.matmul_nt(o, p["out"])
        saved.append((h, y, rstd, q, k, v, o, lse))
        residual = h
    grads, dh = [], target                       # the gradient of the last sum reaches its branch and its residual alike
    for p, (h, y, rstd, q, k, v, o, lse) in zip(reversed(params), reversed(saved)):
        do = K.matmul_nn(dh, p["out"])
        dqkv = torch.empty(rows, QKV, device="cuda", dtype=torch.bfloat16)
        scratch = torch.empty(K.span_attention_bwd_scratch_floats(B, H, S), device="cuda")
        K.span_attention_bwd(q, k, v, o, lse, do, dqkv[:, :H * D], dqkv[:, H * D:(H + KH) * D], dqkv[:, (H + KH) * D:], scratch, spans, **sizes)
        dx, dgamma = torch.empty_like(h), torch.empty_like(p["gamma"])
        room = torch.empty(K.rmsnorm_bwd_scratch(rows, E), device="cuda")
        K.rmsnorm_bwd(K.matmul_nn(dqkv, p["qkv"]), h, p["gamma"], rstd, dx, dgamma, room, dsum=dh)
        grads.append({"gamma": dgamma, "qkv": K.matmul_tn(dqkv, y), "out": K.matmul_tn(dh, o)})
        dh = dx
    return grads[::-1], dh


def in_64_bits(params, x, target, seen):
    leaves = [{n: t.double().requires_grad_() for n, t in p.items()} for p in params]
    first = x.double().requires_grad_()
    h = first
    for p in leaves:
        y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS) * p["gamma"]
        qkv = y @ p["qkv"].T
        heads = lambda t, n: t.reshape(B, S, n, D).permute(0, 2, 1, 3)  # noqa: E731
        q, k, v = heads(qkv[:, :H * D], H), heads(qkv[:, H * D:(H + KH) * D], KH), heads(qkv[:, (H + KH) * D:], KH)
        k, v = k.repeat_interleave(H // KH, 1), v.repeat_interleave(H // KH, 1)
        s = CAP * torch.tanh(q @ k.transpose(-1, -2) / math.sqrt(D) / CAP)
        p_ = torch.softmax(s.masked_fill(~seen[:, None], -1e30), -1) * seen.any(-1)[:, None, :, None]
        h = h + (p_ @ v).permute(0, 2, 1, 3).reshape(B * S, H * D) @ p["out"].T
    (h * target.double()).sum().backward()
    return [{n: t.grad for n, t in p.items()} for p in leaves], first.grad


def test_gradients_clipping_and_update_of_a_packed_step():
    g = torch.Generator(device="cuda").manual_seed(7)
    params = parameters(3)
    x, target = (torch.randn(B * S, E, generator=g, device="cuda").bfloat16() for _ in range(2))
    doc = torch.full((B, S), -1, dtype=torch.int32)
    doc[0, :70], doc[0, 70:160], doc[1, 20:200] = 0, 1, 5
    prompt = torch.zeros(B, S, dtype=torch.bool)
    prompt[0, 70:100] = True
    seen = visible(spans_of(doc, prompt), S).cuda()
    grads, dx = step(params, x, target, doc.cuda(), prompt.cuda())
    want, want_x = in_64_bits(params, x, target, seen)
    assert K.span_attention_last_error() == 0
    # Along a layer a value is rounded to bf16 in the norm, the projection, P, the context, the output projection and the sum, and its gradient
    # as often on the way back: 12 roundings a layer of at most 2^-8 of what they round, 2 layers, in the 2-norm of a whole gradient
    bound = 12 * LAYERS * 2.0 ** -8
    for p, w in zip(grads, want):
        for n in p:
            assert ((p[n].double() - w[n]).norm() / w[n].norm()).item() < bound, n
    assert ((dx.double() - want_x).norm() / want_x.norm()).item() < bound
    flat = [p[n] for p in grads for n in p]
    norm = math.sqrt(sum((t.double() ** 2).sum().item() for t in flat))
    arena = torch.cat([t.reshape(-1) for t in flat])
    master = torch.cat([p[n].reshape(-1).float() for p in params for n in p])
    start, m, v, shadow = master.clone(), torch.zeros_like(master), torch.zeros_like(master), torch.empty_like(arena)
    lst = K.GradientList(flat)
    got = K.gradient_norm(lst)
    assert abs(got.item() - norm) <= 3e-7 * norm
    K.adam_update(master, m, v, arena, shadow, 0.1, 0.9, 0.999, 1e-8, grad_norm=got, max_grad_norm=norm / 4)
    K.clip_gradients(lst, norm / 4)
    scaled = arena.double() / 4
    # the optimizer's factor and the clipped tensors are the same scale (32 bits against the gradients' own type)
    assert ((m.double() - 0.1 * scaled).abs() <= 1e-6 * scaled.abs() + 1e-30).all()
    clipped = torch.cat([t.reshape(-1) for t in flat]).double()
    assert ((clipped - scaled).abs() <= (2.0 ** -8 + 1e-6) * scaled.abs() + 2.0 ** -126).all()
    assert torch.equal(shadow, master.bfloat16()) and not torch.equal(master, start)

"""What the operators of a packed-document training step refuse, on tensors in host memory: refusals come before anything is launched."""
import pytest
import torch

from flexflow_train_b200.ops import kernels as K

pytestmark = pytest.mark.skipif(not K.available(), reason="kernel library not built")

B, S, H, KH, D = 2, 16, 4, 2, 64


def refused(what, call):
    with pytest.raises(K.KernelError, match=what):
        call()


# ---------------------------------------------------------------------------------------------- attention
def attention(name="fwd", **change):
    sizes = dict(B=B, S=S, H=H, KH=KH, D=D, scale=0.125, cap=0.0, slopes=None)
    sizes.update({k: change.pop(k) for k in list(change) if k in sizes})
    b, s, h, kh, d = (sizes[n] for n in ("B", "S", "H", "KH", "D"))
    bf = lambda n: torch.zeros(b * s, n * d, dtype=torch.bfloat16)  # noqa: E731
    t = dict(q=bf(h), k=bf(kh), v=bf(kh), out=bf(h), lse=torch.zeros(b, h, s), spans=torch.zeros(b, s, 2, dtype=torch.int32))
    if name == "bwd":
        t.update(dout=bf(h), dq=bf(h), dk=bf(kh), dv=bf(kh), scratch=torch.zeros(K.span_attention_bwd_scratch_floats(b, h, s)))
    t.update(change)
    if name == "fwd":
        return K.span_attention_fwd(t["q"], t["k"], t["v"], t["out"], t["lse"], t["spans"], **sizes)
    return K.span_attention_bwd(t["q"], t["k"], t["v"], t["out"], t["lse"], t["dout"], t["dq"], t["dk"], t["dv"], t["scratch"], t["spans"], **sizes)


@pytest.mark.parametrize("name", ["fwd", "bwd"])
def test_attention_refuses(name):
    bf = lambda rows, cols: torch.zeros(rows, cols, dtype=torch.bfloat16)  # noqa: E731
    refused("CPU tensor", lambda: attention(name))
    refused("key head", lambda: attention(name, KH=3))
    refused("key head", lambda: attention(name, KH=8))
    for d in (4, 60, 136, 256):
        refused("head dim", lambda: attention(name, D=d))
    refused("scale", lambda: attention(name, scale=0.0))
    refused("scale", lambda: attention(name, scale=-1.0))
    refused("scale", lambda: attention(name, scale=float("nan")))
    refused("cap", lambda: attention(name, cap=-1.0))
    refused("cap", lambda: attention(name, cap=float("inf")))
    refused("cap", lambda: attention(name, cap=0.126 * 2.0**30))
    refused("slopes", lambda: attention(name, slopes=torch.zeros(H + 1)))
    refused("slopes", lambda: attention(name, slopes=torch.zeros(H, dtype=torch.float64)))
    refused("spans", lambda: attention(name, spans=torch.zeros(B, S, 2, dtype=torch.int64)))
    refused("spans", lambda: attention(name, spans=torch.zeros(B, 2, S, dtype=torch.int32).transpose(1, 2)))
    refused("q must be", lambda: attention(name, q=torch.zeros(B * S, H * D, dtype=torch.float16)))
    refused("q must be", lambda: attention(name, q=bf(B * S + 1, H * D)))
    refused("k must be", lambda: attention(name, k=bf(B * S, KH * D - 8)))
    refused("v must be", lambda: attention(name, v=bf(KH * D, B * S).t()))
    refused("16-byte boundary", lambda: attention(name, q=bf(B * S, H * D + 8)[:, 1:H * D + 1]))
    refused("multiple of 8", lambda: attention(name, k=bf(B * S, KH * D + 4)[:, :KH * D]))
    refused("16-byte boundary", lambda: attention(name, v=bf(1, KH * D).expand(B * S, KH * D)))
    refused("lse", lambda: attention(name, lse=torch.zeros(B, S, H)))
    refused("lse", lambda: attention(name, lse=torch.zeros(B, H, S, dtype=torch.bfloat16)))
    packed = bf(B * S, (H + 2 * KH) * D)
    q, k, v = packed[:, :H * D], packed[:, H * D:(H + KH) * D], packed[:, (H + KH) * D:]
    refused("CPU tensor", lambda: attention(name, q=q, k=k, v=v))              # views side by side are fine
    if name == "fwd":
        refused("out and q share", lambda: attention(name, q=q, k=k, v=v, out=packed[:, KH * D:(H + KH) * D]))
        refused("out and q share", lambda: attention(name, q=q, k=k, v=v, out=q))
        refused("out and v share", lambda: attention(name, v=packed[:, :KH * D], out=packed[:, D:(H + 1) * D]))
    else:
        refused("scratch", lambda: attention(name, scratch=torch.zeros(3)))
        refused("scratch", lambda: attention(name, scratch=None))
        refused("dq and dk share", lambda: attention(name, dq=q, dk=packed[:, :KH * D]))
        both = bf(B * S, KH * D)
        refused("dk and dv share", lambda: attention(name, dk=both, dv=both))


def test_spans_refuse():
    doc = torch.zeros(2, 8, dtype=torch.int32)
    refused("CPU tensor", lambda: K.attention_spans(doc))
    refused("int32", lambda: K.attention_spans(doc.long()))
    refused("int32", lambda: K.attention_spans(doc[0]))
    refused("prompt", lambda: K.attention_spans(doc, torch.zeros(2, 7, dtype=torch.bool)))
    refused("prompt", lambda: K.attention_spans(doc, torch.zeros(2, 8)))
    refused("CPU tensor", lambda: K.attention_spans(doc, torch.zeros(2, 8, dtype=torch.bool), causal=False))
    refused("out is", lambda: K.attention_spans(doc, out=torch.zeros(2, 8, dtype=torch.int32)))
    both = torch.zeros(2, 8, 2, dtype=torch.int32)
    refused("share memory", lambda: K.attention_spans(both.view(-1)[:16].view(2, 8), out=both))


# ---------------------------------------------------------------------------------------------- RMS norm
def test_rmsnorm_refuses():
    x, g, r = torch.zeros(4, 32), torch.zeros(32), torch.zeros(4)
    refused("CPU tensor", lambda: K.rmsnorm_fwd(x, g, 1e-6))
    refused("2-D", lambda: K.rmsnorm_fwd(x[0], g, 1e-6))
    refused("bf16 or fp32", lambda: K.rmsnorm_fwd(x.half(), g.half(), 1e-6))
    refused("gamma", lambda: K.rmsnorm_fwd(x, g.bfloat16(), 1e-6))
    refused("gamma", lambda: K.rmsnorm_fwd(x, g[:16], 1e-6))
    refused("shape and dtype", lambda: K.rmsnorm_fwd(x, g, 1e-6, residual=x.bfloat16()))
    refused("shape and dtype", lambda: K.rmsnorm_fwd(x, g, 1e-6, out=torch.zeros(4, 31)))
    refused("with a residual", lambda: K.rmsnorm_fwd(x, g, 1e-6, xsum=x.clone()))
    refused("rstd", lambda: K.rmsnorm_fwd(x, g, 1e-6, rstd=r[:3]))
    refused("elements", lambda: K.rmsnorm_fwd(torch.zeros(4, 0), torch.zeros(0), 1e-6))
    for shape in ((2**31 - 4096, 1), (1, 2**30 + 1)):              # loops' steps past the end would leave 32 bits
        refused("elements", lambda: K.rmsnorm_fwd(torch.zeros(1, 1).expand(shape), g, 1e-6))  # noqa: B023
    flat = torch.zeros(300)
    refused("share memory", lambda: K.rmsnorm_fwd(flat[:128].view(4, 32), g, 1e-6, out=flat[32:160].view(4, 32)))
    same = torch.zeros(4, 32)
    refused("share memory", lambda: K.rmsnorm_fwd(x, g, 1e-6, residual=x.clone(), xsum=same, out=same))
    big = torch.zeros(K.rmsnorm_bwd_scratch(4, 32))
    refused("CPU tensor", lambda: K.rmsnorm_bwd(x, x.clone(), g, r, x.clone(), g.clone(), big))
    refused("scratch", lambda: K.rmsnorm_bwd(x, x.clone(), g, r, x.clone(), g.clone(), big[:-1]))
    refused("scratch", lambda: K.rmsnorm_bwd(x, x.clone(), g, r, x.clone(), g.clone(), None))
    refused("dgamma", lambda: K.rmsnorm_bwd(x, x.clone(), g, r, x.clone(), g.bfloat16(), big))
    refused("needed", lambda: K.rmsnorm_bwd(x, x.clone(), g, None, x.clone(), g.clone(), big))
    refused("share memory", lambda: K.rmsnorm_bwd(x, x.clone(), g, r, flat[:128].view(4, 32), flat[100:132], big))
    refused("dgamma and gamma share", lambda: K.rmsnorm_bwd(x, x.clone(), g, r, x.clone(), g, big))
    one = torch.zeros(1, 32)
    refused("out and gamma share", lambda: K.rmsnorm_fwd(one, g, 1e-6, out=g.view(1, 32)))
    exact = torch.zeros(K.rmsnorm_bwd_scratch(4, 32) // 32, 32)
    refused("scratch and x share|shape", lambda: K.rmsnorm_bwd(x, exact[:4], g, r, x.clone(), g.clone(), exact.view(-1)))
    refused("rstd and a share", lambda: K.rmsnorm_fwd(flat[:4].view(4, 1), torch.zeros(1), 1e-6, rstd=flat[:4]))


# ---------------------------------------------------------------------------------------------- clipping
def test_gradient_list_refuses():
    a, b = torch.zeros(10), torch.zeros(4, 4, dtype=torch.bfloat16)
    refused("CPU tensor", lambda: K.GradientList([a, b]))
    refused("no gradients", lambda: K.GradientList([]))
    refused("dtype", lambda: K.GradientList([a, torch.zeros(3, dtype=torch.float64)]))
    refused("one output", lambda: K.GradientList([a, b], out=[a.clone()]))
    refused("shape and dtype", lambda: K.GradientList([a], out=[a.bfloat16()]))
    refused("shape and dtype", lambda: K.GradientList([a], out=[torch.zeros(11)]))
    refused("share memory", lambda: K.GradientList([a, a]))
    refused("share memory", lambda: K.GradientList([a[:6], a[5:]]))
    refused("share memory", lambda: K.GradientList([a, torch.zeros(10)], out=[torch.zeros(10), a]))
    refused("non-contiguous|CPU", lambda: K.GradientList([torch.zeros(4, 4).t()]))


# ---------------------------------------------------------------------------------------------- devices
class _On:
    """Stands in for a tensor on a device of a machine with several."""

    def __init__(self, device):
        self.device_index = device

    def get_device(self):
        return self.device_index


def test_operands_on_another_device_than_the_current_one(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    monkeypatch.setattr(K, "_raw_stream", lambda device: 1000 + device)
    assert K._launch_stream(_On(1), None, _On(1)) == 1001
    refused("current device", lambda: K._launch_stream(_On(0), _On(0)))
    refused("cuda:1 and on cuda:0", lambda: K._launch_stream(_On(1), None, _On(0)))
    refused("CPU tensor", lambda: K._launch_stream(_On(1), _On(-1)))
    refused("CPU tensor", lambda: K._launch_stream(_On(-1), _On(1)))

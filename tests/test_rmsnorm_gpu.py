"""RMS norm with the residual's addition, forward and backward, against the formula in 64 bits.

Bounds: what is stored in bf16 is off by at most U = 2^-8 of its value (half a step), in fp32 by 2^-24; sums of up to 20000 products in 32 bits,
added over threads and warps, and the reciprocal square root by less than E = 1e-5 of the sum of the terms' sizes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from flexflow_train_b200.ops import kernels as K  # noqa: E402

E = 1.0e-5
EPS = 1e-6
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def tensor(g, shape, dtype, scale=1.0, shift=0):
    """A contiguous tensor; `shift` elements past an allocation's start."""
    flat = torch.empty(shape[0] * shape[1] + shift, dtype=dtype, device="cuda")
    t = flat[shift:].view(shape)
    t.copy_(torch.randn(shape, generator=g, device="cuda") * scale)
    return t


def within(got, value, bound, name):
    off = (got.double() - value).abs()
    assert (off <= bound).all(), f"{name}: {(off / bound.clamp_min(1e-300)).max().item():.2f} of the bound"


def both(rows, cols, dtype, shift=0, residual=True, dsum=True, accumulate=False, inplace=False, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(rows * 31 + cols)
    u = UNIT[dtype]
    x, r = tensor(g, (rows, cols), dtype, spread, shift), tensor(g, (rows, cols), dtype, 2.0 * spread, shift)
    gamma = (1.0 + 0.2 * torch.randn(cols, generator=g, device="cuda")).to(dtype)
    dy, ds = tensor(g, (rows, cols), dtype, 1.0, shift), tensor(g, (rows, cols), dtype, 1.0, shift)
    h = (x.float() + r.float()).to(dtype) if residual else x.clone()
    hd, gd, dyd, dsd = h.double(), gamma.double(), dy.double(), ds.double()
    rstd = torch.full((rows,), 7.0, device="cuda")
    y = x if inplace else torch.full_like(x, 7.0)
    xsum = (r if inplace else torch.full_like(x, 7.0)) if residual else None
    K.rmsnorm_fwd(x, gamma, EPS, residual=r if residual else None, xsum=xsum, out=y, rstd=rstd)
    root = 1.0 / torch.sqrt((hd * hd).mean(1) + EPS)
    if residual:
        assert torch.equal(xsum, h)
    within(rstd, root, E * root, "rstd")
    value = hd * root[:, None] * gd
    within(y, value, (u + E) * value.abs(), "y")
    dx = dy if inplace else torch.full_like(x, 7.0)
    dgamma = torch.full_like(gamma, 0.5)
    scratch = torch.full((K.rmsnorm_bwd_scratch(rows, cols),), float("nan"), device="cuda")
    K.rmsnorm_bwd(dy, h, gamma, rstd, dx, dgamma, scratch, dsum=ds if dsum else None, accumulate_params=accumulate)
    part = dyd * gd
    mean = (part * hd).mean(1, keepdim=True)
    extra = dsd if dsum else torch.zeros_like(dsd)
    k = root[:, None] ** 2 * mean
    value = root[:, None] * (part - hd * k) + extra
    terms = root[:, None] * (part.abs() + hd.abs() * root[:, None] ** 2 * (part * hd).abs().mean(1, keepdim=True)) + extra.abs()
    within(dx, value, u * value.abs() + E * terms, "dx")
    each = dyd * hd * root[:, None]
    value = each.sum(0) + (0.5 if accumulate else 0.0)
    within(dgamma, value, u * value.abs() + E * (each.abs().sum(0) + 0.5), "dgamma")
    return y, dx, dgamma


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 8), (2, 31), (9, 33), (130, 256), (1300, 256), (64, 300), (1200, 512), (50, 1000), (77, 1001),
                                       (600, 1024), (301, 2048), (40, 2056), (33, 4096), (5, 8192), (7, 16384), (3, 16392), (4, 20000), (2, 2049)])
def test_norm_and_gradients_against_the_formula(rows, cols, dtype):
    both(rows, cols, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(200, 512), (9, 2048), (3, 12000)])
def test_addresses_that_are_no_multiple_of_16_bytes(rows, cols, dtype):
    both(rows, cols, dtype, shift=1)


@pytest.mark.parametrize("residual,dsum,accumulate,inplace", [(False, False, False, False), (True, False, True, False), (False, True, False, True), (True, True, True, True)])
@pytest.mark.parametrize("rows,cols", [(100, 512), (31, 2048), (2, 18000), (13, 77)])
def test_forms(rows, cols, residual, dsum, accumulate, inplace):
    both(rows, cols, torch.bfloat16, residual=residual, dsum=dsum, accumulate=accumulate, inplace=inplace)


@pytest.mark.parametrize("spread", [1e-12, 1e12])
def test_rows_of_tiny_and_of_large_values(spread):
    """Mean squares of 1e-24, which eps dwarfs, and of 1e24."""
    both(65, 640, torch.float32, spread=spread)


def test_rows_of_zeros_give_zeros():
    x = torch.zeros(4, 512, device="cuda", dtype=torch.bfloat16)
    y = K.rmsnorm_fwd(x, torch.ones(512, device="cuda", dtype=torch.bfloat16), EPS)
    assert (y == 0).all()


def test_no_rows():
    x = torch.empty(0, 64, device="cuda")
    gamma, dgamma = torch.ones(64, device="cuda"), torch.full((64,), 3.0, device="cuda")
    rstd = torch.empty(0, device="cuda")
    assert K.rmsnorm_fwd(x, gamma, EPS).shape == (0, 64)
    K.rmsnorm_bwd(x, x.clone(), gamma, rstd, x.clone(), dgamma, None)
    assert (dgamma == 0).all()
    dgamma.fill_(3.0)
    K.rmsnorm_bwd(x, x.clone(), gamma, rstd, x.clone(), dgamma, None, accumulate_params=True)
    assert (dgamma == 3).all()


def test_gradients_against_differences():
    """d(sum y dy + sum h ds)/dx along a direction by central differences in 64 bits."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x, dy, ds, way = (torch.randn(40, 320, generator=g, device="cuda") for _ in range(4))
    gamma, wayg = torch.randn(320, generator=g, device="cuda"), torch.randn(320, generator=g, device="cuda")
    rstd, dx, dgamma = torch.empty(40, device="cuda"), torch.empty_like(x), torch.empty_like(gamma)
    K.rmsnorm_fwd(x, gamma, EPS, rstd=rstd)
    K.rmsnorm_bwd(dy, x, gamma, rstd, dx, dgamma, torch.empty(K.rmsnorm_bwd_scratch(40, 320), device="cuda"), dsum=ds)

    def loss(a, b):
        return (a / torch.sqrt((a * a).mean(1, keepdim=True) + EPS) * b * dy.double() + a * ds.double()).sum()

    h = 1e-5
    slope = (loss(x.double() + h * way, gamma.double() + h * wayg) - loss(x.double() - h * way, gamma.double() - h * wayg)) / (2 * h)
    mine = (dx.double() * way).sum() + (dgamma.double() * wayg).sum()
    # 12800 terms of size 1, each off by some 1e-7, and h^2 / 6 of the third derivative
    assert abs(mine - slope).item() < 12800 * 4e-7


def test_same_bits_on_another_stream_and_replayed():
    first = both(999, 1024, torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = both(999, 1024, torch.bfloat16)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    g = torch.Generator(device="cuda").manual_seed(1)
    x, r = tensor(g, (64, 2048), torch.bfloat16), tensor(g, (64, 2048), torch.bfloat16)
    gamma, s, y = torch.ones(2048, device="cuda", dtype=torch.bfloat16), torch.empty_like(x), torch.empty_like(x)
    K.rmsnorm_fwd(x, gamma, EPS, residual=r, xsum=s, out=y)
    want = y.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.rmsnorm_fwd(x, gamma, EPS, residual=r, xsum=s, out=y)
    y.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)

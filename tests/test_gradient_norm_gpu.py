"""The norm of a list of gradients and clipping by it, against 64 bits.  The sum is held in 64 bits, groups of up to 8 squares in 32: the norm
is off by less than 8 * 2^-24 / 2 + 2^-24 (its own rounding) = 3e-7.  A clipped value is off by half a step of its type and the scale's 2^-24."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from flexflow_train_b200.ops import kernels as K  # noqa: E402

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
SHAPES = [(1,), (7, 3), (0, 5), (128, 128), (16384,), (16385,), (3, 16383), (40000,), (1, 1, 9)]


def gradients(dtypes, seed=0, scale=1e-2, shapes=SHAPES):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(s, generator=g, device="cuda") * scale).to(dtypes[i % len(dtypes)]) for i, s in enumerate(shapes)]


def norm_of(tensors):
    return math.sqrt(sum((t.double() ** 2).sum().item() for t in tensors))


def clipped_as(before, after, scale):
    for b, a in zip(before, after):
        want = b.double() * scale
        u = UNIT[b.dtype]
        least = 2.0 ** -25 if b.dtype == torch.float16 else 2.0 ** -126      # half a step of the smallest numbers
        assert ((a.double() - want).abs() <= (u + 2.0 ** -22) * want.abs() + least).all()


@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16], [torch.float16], [torch.bfloat16, torch.float32, torch.float16]])
@pytest.mark.parametrize("factor", [0.25, 0.999, 1.5])
def test_norm_and_clipping(dtypes, factor):
    grads = gradients(dtypes)
    before = [t.clone() for t in grads]
    n = norm_of(grads)
    lst = K.GradientList(grads)
    assert abs(K.gradient_norm(lst).item() - n) <= 3e-7 * n
    assert abs(K.clip_gradients(lst, n * factor).item() - n) <= 3e-7 * n
    if factor > 1:
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
    else:
        clipped_as(before, grads, factor)


def test_clipping_into_other_tensors_leaves_the_gradients_alone():
    grads = gradients([torch.bfloat16, torch.float32], seed=2)
    before = [t.clone() for t in grads]
    out = [torch.full_like(t, 9.0) for t in grads]
    out[3] = grads[3]                                     # one of them in place
    n = norm_of(grads)
    lst = K.GradientList(grads, out=out)
    K.clip_gradients(lst, 2 * n)
    assert all(torch.equal(a, b) for a, b in zip(out, before))
    K.clip_gradients(lst, 0.3 * n)
    clipped_as(before, out, 0.3)
    assert all(torch.equal(a, b) for i, (a, b) in enumerate(zip(grads, before)) if i != 3)


def test_neighbours_in_one_buffer_and_odd_addresses():
    flat = torch.full((100003,), 5.0, device="cuda", dtype=torch.bfloat16)
    grads = [flat[1:1000], flat[1000:1000], flat[1000:50001], flat[50003:100000]]
    before = [t.clone() for t in grads]
    n = norm_of(grads)
    norm = K.clip_gradients(K.GradientList(grads), 0.5 * n).item()
    assert abs(norm - n) <= 3e-7 * n
    clipped_as(before, grads, 0.5)
    assert (flat[[0, 50001, 50002, 100000, 100002]] == 5).all()


@pytest.mark.parametrize("value", [1e30, 1e-30, 1e-22, 3e18])
def test_values_whose_squares_leave_32_bits(value):
    t = torch.full((5000,), value, device="cuda")
    t[::7] = 0
    n = norm_of([t])
    lst = K.GradientList([t])
    assert abs(K.gradient_norm(lst).item() - n) <= 3e-7 * n
    K.clip_gradients(lst, n / 2)
    assert abs(norm_of([t]) - n / 2) <= 1e-6 * n


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_norm_that_is_not_finite_leaves_the_gradients(bad):
    for dtype in UNIT:
        t = torch.ones(3000, device="cuda", dtype=dtype)
        t[1234] = bad
        before = t.clone()
        n = K.clip_gradients(K.GradientList([t]), 1.0).item()
        assert math.isnan(n) if math.isnan(bad) else n == math.inf
        assert torch.equal(torch.nan_to_num(t, nan=7.0), torch.nan_to_num(before, nan=7.0))


def test_zero_gradients_and_zero_norm():
    t = torch.zeros(500, device="cuda")
    lst = K.GradientList([t])
    assert K.clip_gradients(lst, 1.0).item() == 0 and (t == 0).all()
    t.fill_(2.0)
    K.clip_gradients(lst, 0.0)
    assert (t == 0).all()
    nothing = K.GradientList([torch.empty(0, device="cuda")])
    assert K.clip_gradients(nothing, 1.0).item() == 0


def test_same_bits_again_on_another_stream_and_replayed():
    grads = gradients([torch.bfloat16, torch.float32], seed=4, shapes=[(300, 1000), (5000,), (70000,)] * 9)
    out = [torch.empty_like(t) for t in grads]
    lst = K.GradientList(grads, out=out)
    n = K.clip_gradients(lst, 0.1).clone()
    first = [t.clone() for t in out]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = K.clip_gradients(lst, 0.1).clone()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(n, again) and all(torch.equal(a, b) for a, b in zip(first, out))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        K.clip_gradients(lst, 0.1)
    for t in out:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(n, lst.norm) and all(torch.equal(a, b) for a, b in zip(first, out))


def test_two_lists_at_once():
    a, b = gradients([torch.float32], seed=5, shapes=[(200000,)]), gradients([torch.float32], seed=6, shapes=[(150000,)])
    la, lb = K.GradientList(a), K.GradientList(b)
    na, nb = norm_of(a), norm_of(b)
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        with torch.cuda.stream(s[0]):
            ra = K.gradient_norm(la)
        with torch.cuda.stream(s[1]):
            rb = K.gradient_norm(lb)
    torch.cuda.synchronize()
    assert abs(ra.item() - na) <= 3e-7 * na and abs(rb.item() - nb) <= 3e-7 * nb

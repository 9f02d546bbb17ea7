"""Attention over spans of keys, and the spans of packed documents, against their definitions (64 bits; bounds in span_reference.py)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from flexflow_train_b200.ops import kernels as K  # noqa: E402

from span_reference import reference, spans_of, visible  # noqa: E402


def documents_of(lengths, S):
    """One row of document numbers: (length) a document, (-length) padding; the rest padding."""
    row, n = [], 0
    for i, length in enumerate(lengths):
        row += [(i if length > 0 else -1)] * abs(length)
        n += abs(length)
    return (row + [-1] * S)[:S]


def random_documents(B, S, mean, seed, padding=True):
    g = torch.Generator().manual_seed(seed)
    rows = []
    for b in range(B):
        lengths = []
        while sum(map(abs, lengths)) < S:
            n = 1 + int(torch.randint(0, max(2 * mean, 1), (1,), generator=g))
            lengths.append(-n if padding and torch.rand(1, generator=g) < 0.2 else n)
        rows.append(documents_of(lengths, S))
    return torch.tensor(rows, dtype=torch.int32)


@pytest.mark.parametrize("B,S,mean", [(1, 1, 1), (3, 7, 2), (2, 129, 20), (2, 1024, 90), (1, 1025, 3000), (3, 2500, 700), (2, 5000, 1)])
@pytest.mark.parametrize("form", ["causal", "prompt", "both"])
def test_spans_follow_the_definition(B, S, mean, form):
    doc = random_documents(B, S, mean, seed=S + mean)
    prompt = None
    if form == "prompt":
        g = torch.Generator().manual_seed(S)
        prompt = torch.rand(B, S, generator=g) < (0.9 if S % 2 else 0.999)
    got = K.attention_spans(doc.cuda(), None if prompt is None else prompt.cuda(), causal=form != "both")
    assert torch.equal(got.cpu(), spans_of(doc, prompt, causal=form != "both"))


@pytest.mark.parametrize("S,mean", [(17 * 1024, 900), (17 * 1024 + 1, 30000), (40000, 6000), (20000, 1)])
@pytest.mark.parametrize("form", ["causal", "prompt", "both"])
def test_spans_of_long_rows(S, mean, form):
    """Rows whose pieces are told of one another by a launch of their own."""
    doc = random_documents(2, S, mean, seed=S)
    prompt = None
    if form == "prompt":                     # a document's flags end in its own piece, at a piece's border, pieces later, or with it
        prompt = torch.ones(2, S, dtype=torch.bool)
        prompt[0, torch.randint(0, S, (max(1, S // 5000),), generator=torch.Generator().manual_seed(S))] = False
        prompt[0, 5 * 1024] = prompt[0, 9 * 1024 - 1] = False
    got = K.attention_spans(doc.cuda(), None if prompt is None else prompt.cuda(), causal=form != "both")
    assert torch.equal(got.cpu(), spans_of(doc, prompt, causal=form != "both"))


@pytest.mark.parametrize("S,mean", [(7, 2), (1024, 90), (2500, 700)])
def test_prompts_of_documents_that_are_seen_from_both_sides(S, mean):
    doc = random_documents(3, S, mean, seed=S)
    prompt = torch.rand(3, S, generator=torch.Generator().manual_seed(S)) < 0.9
    got = K.attention_spans(doc.cuda(), prompt.cuda(), causal=False).cpu()
    assert torch.equal(got, spans_of(doc, prompt, causal=False)) and torch.equal(got, spans_of(doc, None, causal=False))


def test_spans_of_runs_that_cross_many_blocks_and_of_flags_that_end_there():
    S = 6000
    doc = torch.zeros(4, S, dtype=torch.int32)
    doc[1, 1024:] = 1
    doc[2, 1023:3000] = 5
    doc[3, 5999:] = -7
    prompt = torch.zeros(4, S, dtype=torch.uint8)
    prompt[0, :4096] = 1
    prompt[1, :1024] = 2                 # any value that is not zero
    prompt[1, 2047:] = 1                 # not from the document's first token on: no prompt
    prompt[2, 1023:3000] = 1
    prompt[3] = 1
    got = K.attention_spans(doc.cuda(), prompt.cuda(), causal=True)
    assert torch.equal(got.cpu(), spans_of(doc, prompt))
    # a number that comes back later is another document
    again = torch.tensor([[3, 3, 4, 3, 3, -1, -1, 4]], dtype=torch.int32)
    assert torch.equal(K.attention_spans(again.cuda()).cpu(), spans_of(again))


def make(B, S, H, KH, D, seed, dtype=torch.bfloat16, wide=0):
    """q, k, v as views into one packed matrix (with `wide` columns to the right that belong to nobody), dout."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = torch.randn(B * S, (H + 2 * KH) * D + wide, generator=g, device="cuda").to(dtype)
    dout = torch.randn(B * S, H * D, generator=g, device="cuda").to(dtype)
    return qkv, qkv[:, :H * D], qkv[:, H * D:(H + KH) * D], qkv[:, (H + KH) * D:(H + 2 * KH) * D], dout


def run(q, k, v, dout, spans, backward=True, grads=None, **sizes):
    B, S, H, KH, D = (sizes[n] for n in ("B", "S", "H", "KH", "D"))
    out = torch.full((B * S, H * D), 7.0, device="cuda", dtype=torch.bfloat16)
    lse = torch.full((B, H, S), 7.0, device="cuda")
    K.span_attention_fwd(q, k, v, out, lse, spans, **sizes)
    got = {"out": out, "lse": lse}
    if backward:
        dq, dk, dv = grads if grads is not None else (torch.full((B * S, n * D), 7.0, device="cuda", dtype=torch.bfloat16) for n in (H, KH, KH))
        scratch = torch.full((K.span_attention_bwd_scratch_floats(B, H, S),), float("nan"), device="cuda")
        K.span_attention_bwd(q, k, v, out, lse, dout, dq, dk, dv, scratch, spans, **sizes)
        got.update(dq=dq, dk=dk, dv=dv)
    assert K.span_attention_last_error() == 0
    return got


def check(got, want):
    for name, (value, bound) in want.items():
        if name not in got:
            continue
        off = (got[name].double() - value).abs()
        assert torch.isfinite(got[name]).all(), name
        worst = (off / bound.clamp_min(1e-300)).max().item()
        assert (off <= bound).all(), f"{name}: {worst:.2f} of the bound, off by up to {off.max().item():.3g}"


def mask(kind, B, S, seed):
    if kind == "full":
        return K.attention_spans(torch.zeros(B, S, dtype=torch.int32, device="cuda"), causal=False)
    if kind == "causal":
        return K.attention_spans(torch.zeros(B, S, dtype=torch.int32, device="cuda"))
    doc = random_documents(B, S, max(S // 4, 1), seed).cuda()
    if kind == "documents":
        return K.attention_spans(doc)
    if kind == "both":
        return K.attention_spans(doc, causal=False)
    if kind == "prefix":
        g = torch.Generator(device="cuda").manual_seed(seed)
        return K.attention_spans(doc, torch.rand(B, S, generator=g, device="cuda") < 0.97)
    # any spans at all: beyond either end, empty, the whole sequence
    g = torch.Generator(device="cuda").manual_seed(seed)
    a = torch.randint(-S // 2 - 2, S + 3, (B, S), generator=g, device="cuda", dtype=torch.int32)
    n = torch.randint(-3, 2 * S, (B, S), generator=g, device="cuda", dtype=torch.int32)
    return torch.stack([a, a + n], -1).contiguous()


CASES = [
    # B, S, H, KH, D, mask, cap, bias
    (1, 1, 1, 1, 64, "causal", 0.0, False), (2, 1, 4, 2, 128, "full", 20.0, True), (3, 3, 2, 1, 8, "causal", 0.0, True),
    (1, 127, 2, 2, 64, "documents", 0.0, False), (2, 128, 3, 1, 128, "causal", 30.0, False), (1, 129, 4, 4, 72, "prefix", 0.0, True),
    (2, 256, 2, 2, 64, "any", 5.0, True), (1, 257, 6, 2, 128, "any", 0.0, False), (2, 300, 8, 1, 32, "documents", 50.0, True),
    (1, 384, 4, 2, 96, "both", 0.0, False), (2, 513, 4, 4, 128, "documents", 50.0, False), (1, 640, 3, 3, 112, "prefix", 2.0, False),
    (2, 1000, 4, 2, 64, "causal", 0.0, True), (1, 1024, 8, 8, 128, "causal", 0.0, False), (1, 1300, 5, 1, 40, "full", 0.0, True),
    (2, 1537, 2, 1, 128, "documents", 0.0, True), (40, 260, 4, 2, 64, "causal", 0.0, False), (1, 2048, 16, 4, 128, "prefix", 30.0, True),
]


@pytest.mark.parametrize("B,S,H,KH,D,kind,cap,bias", CASES)
def test_attention_and_gradients_against_the_formula(B, S, H, KH, D, kind, cap, bias):
    spans = mask(kind, B, S, seed=S * 7 + H)
    slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device="cuda") if bias else None
    _, q, k, v, dout = make(B, S, H, KH, D, seed=S + D)
    sizes = dict(B=B, S=S, H=H, KH=KH, D=D, scale=1.0 / math.sqrt(D), cap=cap, slopes=slopes)
    check(run(q, k, v, dout, spans, **sizes), reference(q, k, v, spans, dout=dout, **sizes))


FEW = 8


@pytest.mark.parametrize("S,mean", [(1, 1), (2, 2), (3, 3), (5, 2), (8, 8), (131, 3), (400, 2)])
@pytest.mark.parametrize("H,KH,D,kind,cap,bias", [(1, 1, 64, "full", 0.0, False), (1, 1, 32, "causal", 0.0, True), (4, 2, 128, "both", 20.0, False),
                                                  (3, 1, 72, "documents", 0.5, True), (2, 2, 8, "documents", 0.0, False)])
def test_queries_that_see_few_keys(S, mean, H, KH, D, kind, cap, bias):
    """Their gradients are differences of a few products: the bound has no rounding of O in it."""
    B = 3
    if kind in ("both", "documents"):
        spans = K.attention_spans(random_documents(B, S, mean, seed=S).cuda(), causal=kind == "documents")
    elif S > FEW:                            # windows
        at = torch.arange(S, dtype=torch.int32, device="cuda").expand(B, S)
        spans = torch.stack([at - (3 if kind == "full" else 7), at + (4 if kind == "full" else 0)], -1).contiguous()
    else:
        spans = mask(kind, B, S, seed=S)
    slopes = torch.linspace(0.1, 1.0, H, device="cuda") if bias else None
    _, q, k, v, dout = make(B, S, H, KH, D, seed=S + D)
    sizes = dict(B=B, S=S, H=H, KH=KH, D=D, scale=1.0 / math.sqrt(D), cap=cap, slopes=slopes)
    check(run(q, k, v, dout, spans, **sizes), reference(q, k, v, spans, dout=dout, few=FEW, **sizes))


@pytest.mark.parametrize("cap,scale", [(0.0, 2.0), (3.0, 1.0), (30.0, 4.0)])
def test_scores_far_apart(cap, scale):
    """Maxima that move by much more than 2^8 from tile to tile, and scores at the cap's flat end."""
    B, S, H, KH, D = 1, 700, 2, 2, 64
    _, q, k, v, dout = make(B, S, H, KH, D, seed=5)
    k.mul_(torch.linspace(0.1, 4.0, S, device="cuda").to(torch.bfloat16)[:, None])
    spans = mask("causal", B, S, 0)
    sizes = dict(B=B, S=S, H=H, KH=KH, D=D, scale=scale / math.sqrt(D), cap=cap)
    want = reference(q, k, v, spans, dout=dout, **sizes)
    # scores of some hundreds: 32 bits hold them to 2^-24 of their terms' size, which the probabilities take up as it is
    size = scale / math.sqrt(D) * (q.double().abs().reshape(S, H, D).norm(dim=-1).max() * k.double().reshape(S, H, D).norm(dim=-1).max()).item()
    more = 1.0 + size * D * 2.0 ** -24 / 4.0e-4
    check(run(q, k, v, dout, spans, **sizes), {n: (x, e * more) for n, (x, e) in want.items() if n != "lse"})


@pytest.mark.parametrize("D,KH", [(64, 4), (128, 1), (72, 2)])
def test_tokens_that_nobody_sees_may_hold_anything(D, KH):
    B, S, H = 2, 700, 4
    doc = torch.tensor([documents_of([100, -30, 200, -1, 150, -100, 60], S), documents_of([-140, 300, -5, 1, -7, 130], S)], dtype=torch.int32).cuda()
    spans = K.attention_spans(doc)
    qkv, q, k, v, dout = make(B, S, H, KH, D, seed=D)
    sizes = dict(B=B, S=S, H=H, KH=KH, D=D, scale=1.0 / math.sqrt(D), cap=10.0)
    clean = run(q, k, v, dout, spans, **sizes)
    pad = (doc < 0).reshape(-1)
    for fill in (float("nan"), float("inf"), -3.0e38):
        for t in (qkv, dout):
            t[pad] = fill
        got = run(q, k, v, dout, spans, **sizes)
        for name in clean:
            assert torch.equal(got[name], clean[name]), (name, fill)
    for name in ("out", "dq", "dk", "dv"):
        assert (clean[name][pad] == 0).all()
    assert (clean["lse"].permute(0, 2, 1)[doc < 0] == 0).all()


def test_all_rows_empty():
    B, S, H, KH, D = 2, 200, 2, 1, 64
    _, q, k, v, dout = make(B, S, H, KH, D, seed=1)
    spans = torch.tensor([1, 0], dtype=torch.int32, device="cuda").expand(B, S, 2).contiguous()
    got = run(q, k, v, dout, spans, B=B, S=S, H=H, KH=KH, D=D, scale=0.125)
    assert all((t == 0).all() for t in got.values())


def test_outputs_in_wider_matrices_leave_the_rest_alone():
    B, S, H, KH, D = 1, 333, 3, 1, 72
    _, q, k, v, dout = make(B, S, H, KH, D, seed=2, wide=24)
    spans = mask("prefix", B, S, 3)
    sizes = dict(B=B, S=S, H=H, KH=KH, D=D, scale=0.1)
    packed = torch.full((B * S + 2, (H + 2 * KH) * D + 16), 5.0, device="cuda", dtype=torch.bfloat16)
    inner = packed[1:-1]
    grads = (inner[:, :H * D], inner[:, H * D:(H + KH) * D], inner[:, (H + KH) * D:(H + 2 * KH) * D])
    check(run(q, k, v, dout, spans, grads=grads, **sizes), reference(q, k, v, spans, dout=dout, **sizes))
    assert (packed[0] == 5).all() and (packed[-1] == 5).all() and (inner[:, (H + 2 * KH) * D:] == 5).all()


def test_same_inputs_same_bits_on_another_stream_and_replayed():
    B, S, H, KH, D = 2, 900, 6, 2, 128
    _, q, k, v, dout = make(B, S, H, KH, D, seed=9)
    spans = mask("documents", B, S, 4)
    sizes = dict(B=B, S=S, H=H, KH=KH, D=D, scale=1.0 / math.sqrt(D), cap=30.0)
    first = run(q, k, v, dout, spans, **sizes)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run(q, k, v, dout, spans, **sizes)
    torch.cuda.current_stream().wait_stream(side)
    out, lse = torch.empty_like(first["out"]), torch.empty_like(first["lse"])
    dq, dk, dv = (torch.empty_like(first[n]) for n in ("dq", "dk", "dv"))
    scratch = torch.empty(K.span_attention_bwd_scratch_floats(B, H, S), device="cuda")
    doc = random_documents(B, S, S // 4, 4).cuda()
    own = torch.empty(B, S, 2, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        K.attention_spans(doc, out=own)
        K.span_attention_fwd(q, k, v, out, lse, own, **sizes)
        K.span_attention_bwd(q, k, v, out, lse, dout, dq, dk, dv, scratch, own, **sizes)
    for _ in range(3):
        for t in (out, lse, dq, dk, dv, scratch):
            t.fill_(float("nan"))
        graph.replay()
    torch.cuda.synchronize()
    for name, t in (("out", out), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        assert torch.equal(first[name], second[name]) and torch.equal(first[name], t), name


def test_gradients_against_differences():
    """The derivative of sum(out * dout) along a direction, by central differences of the formula in 64 bits, against the kernels' gradients."""
    B, S, H, KH, D = 1, 150, 4, 2, 64
    _, q, k, v, dout = make(B, S, H, KH, D, seed=11)
    spans = mask("prefix", B, S, 5)
    slopes = torch.tensor([0.3, 0.1, 0.05, 0.01], device="cuda")
    sizes = dict(B=B, S=S, H=H, KH=KH, D=D, scale=1.0 / math.sqrt(D), cap=4.0, slopes=slopes)
    got = run(q, k, v, dout, spans, **sizes)
    want = reference(q, k, v, spans, dout=dout, **sizes)
    g = torch.Generator(device="cuda").manual_seed(1)
    for name, base in (("dq", q), ("dk", k), ("dv", v)):
        way = torch.randn(base.shape, generator=g, device="cuda", dtype=torch.float64)
        h = 1e-4

        def loss(x):
            at = {"dq": q, "dk": k, "dv": v}
            at[name] = x
            return (reference(at["dq"], at["dk"], at["dv"], spans, **sizes)["out"][0] * dout.double()).sum()

        slope = ((loss(base.double() + h * way) - loss(base.double() - h * way)) / (2 * h)).item()
        mine = (got[name].double() * way).sum().item()
        # each element off by at most its bound; differences are off by h^2 / 6 of the third derivative, some 1e-8 times the sizes here
        assert abs(mine - slope) <= (want[name][1] * way.abs()).sum().item() + 1e-5 * abs(slope), (name, mine, slope)


def test_long_sequence_rows_against_the_formula():
    """A long causal sequence at shared heads: the last rows, and the gradients of the first keys, which every query reaches."""
    B, S, H, KH, D = 1, 8192, 2, 1, 64
    _, q, k, v, dout = make(B, S, H, KH, D, seed=21)
    spans = mask("causal", B, S, 0)
    sizes = dict(B=B, S=S, H=H, KH=KH, D=D, scale=1.0 / math.sqrt(D))
    check(run(q, k, v, dout, spans, **sizes), reference(q, k, v, spans, dout=dout, **sizes))


def test_visible_is_what_the_plain_masks_say():
    """The spans of the plain masks are those masks."""
    S = 40
    at = torch.arange(S)
    zero = torch.zeros(1, S, dtype=torch.int32, device="cuda")
    assert torch.equal(visible(K.attention_spans(zero), S)[0].cpu(), at[None] <= at[:, None])
    assert visible(K.attention_spans(zero, causal=False), S).all()
    flags = torch.zeros(1, S, dtype=torch.bool, device="cuda")
    flags[0, :9] = True
    assert torch.equal(visible(K.attention_spans(zero, flags), S)[0].cpu(), (at[None] <= at[:, None]) | (at[None] < 9))


@pytest.mark.parametrize("D,KH", [(128, 16), (64, 4)])
def test_many_passes_give_the_same_bits(D, KH):
    """Warps of a block run apart by as much as the barriers let them: many blocks, many passes."""
    B, S, H = 4, 1536, 16
    _, q, k, v, dout = make(B, S, H, KH, D, seed=31)
    spans = mask("documents", B, S, 6)
    sizes = dict(B=B, S=S, H=H, KH=KH, D=D, scale=1.0 / math.sqrt(D), cap=50.0)
    first = run(q, k, v, dout, spans, **sizes)
    for _ in range(30):
        again = run(q, k, v, dout, spans, **sizes)
        assert all(torch.equal(first[n], again[n]) for n in first)


@pytest.mark.parametrize("cap", [1e-3, 0.05, 300.0, 3000.0, 1e5, 1e8])
def test_caps_far_from_the_scores(cap):
    """Caps that every score is far beyond, and caps that no score comes near: the same operator."""
    B, S, H, KH, D = 1, 200, 2, 2, 64
    _, q, k, v, dout = make(B, S, H, KH, D, seed=41)
    spans = mask("causal", B, S, 0)
    sizes = dict(B=B, S=S, H=H, KH=KH, D=D, scale=1.0 / math.sqrt(D), cap=cap)
    check(run(q, k, v, dout, spans, **sizes), reference(q, k, v, spans, dout=dout, **sizes))


@pytest.mark.parametrize("slope", [0.0, -0.05, 4.0])
def test_slopes_of_any_sign(slope):
    B, S, H, KH, D = 1, 300, 2, 1, 64
    _, q, k, v, dout = make(B, S, H, KH, D, seed=43)
    spans = mask("full", B, S, 0)
    sizes = dict(B=B, S=S, H=H, KH=KH, D=D, scale=1.0 / math.sqrt(D), slopes=torch.tensor([slope, 0.01], device="cuda"))
    check(run(q, k, v, dout, spans, **sizes), reference(q, k, v, spans, dout=dout, **sizes))


@pytest.mark.parametrize("B,S", [(0, 5), (3, 0)])
def test_nothing_to_do(B, S):
    H, KH, D = 2, 1, 64
    _, q, k, v, dout = make(B, S, H, KH, D, seed=1)
    assert K.attention_spans(torch.zeros(B, S, dtype=torch.int32, device="cuda")).shape == (B, S, 2)
    spans = torch.zeros(B, S, 2, dtype=torch.int32, device="cuda")
    assert run(q, k, v, dout, spans, B=B, S=S, H=H, KH=KH, D=D, scale=0.1)["dq"].shape == (0, H * D)


FIRST_CALL = """
import torch
from flexflow_train_b200.ops import kernels as K
B, S, H, KH, D = 1, 300, 2, 1, 64
g = torch.Generator(device="cuda").manual_seed(0)
new = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()
q, k, v, dout = new(S, H * D), new(S, D), new(S, D), new(S, H * D)
out, dq, dk, dv = (torch.empty_like(t) for t in (q, q, k, v))
x, gamma, y, dx, dgamma = new(S, 128), new(128), new(S, 128), new(S, 128), new(128)
lse, rstd = torch.empty(B, H, S, device="cuda"), torch.empty(S, device="cuda")
doc = torch.zeros(B, S, dtype=torch.int32, device="cuda")
spans = torch.empty(B, S, 2, dtype=torch.int32, device="cuda")
scratch, room = torch.empty(K.span_attention_bwd_scratch_floats(B, H, S), device="cuda"), torch.empty(K.rmsnorm_bwd_scratch(S, 128), device="cuda")
grads = K.GradientList([dq, dk, dv, dgamma])
sizes = dict(B=B, S=S, H=H, KH=KH, D=D, scale=0.125, cap=20.0)

def step():
    K.attention_spans(doc, out=spans)
    K.span_attention_fwd(q, k, v, out, lse, spans, **sizes)
    K.span_attention_bwd(q, k, v, out, lse, dout, dq, dk, dv, scratch, spans, **sizes)
    K.rmsnorm_fwd(x, gamma, 1e-6, out=y, rstd=rstd)
    K.rmsnorm_bwd(y, x, gamma, rstd, dx, dgamma, room)
    K.clip_gradients(grads, 1.0)

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    step()
graph.replay()
torch.cuda.synchronize()
kept = [t.clone() for t in (out, lse, dq, dk, dv, y, dx, dgamma, grads.norm)]
step()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(kept, (out, lse, dq, dk, dv, y, dx, dgamma, grads.norm)))
print("same")
"""


def test_the_first_calls_of_a_process_may_be_captured():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("same"), r.stdout + r.stderr


def test_calls_on_two_streams_at_once():
    """Passes of different head dims and masks side by side give the bits that they give alone."""
    jobs = []
    for D, KH, S, cap in ((64, 2, 700, 0.0), (128, 4, 900, 30.0)):
        B, H = 2, 4
        _, q, k, v, dout = make(B, S, H, KH, D, seed=D)
        spans = K.attention_spans(random_documents(B, S, 150, seed=D).cuda())
        sizes = dict(B=B, S=S, H=H, KH=KH, D=D, scale=1.0 / math.sqrt(D), cap=cap, slopes=None)
        jobs.append((q, k, v, dout, spans, sizes, run(q, k, v, dout, spans, **sizes), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for q, k, v, dout, spans, sizes, _, stream in jobs:
            B, S, H, KH, D = (sizes[n] for n in ("B", "S", "H", "KH", "D"))
            with torch.cuda.stream(stream):
                out, lse = torch.empty(B * S, H * D, dtype=torch.bfloat16, device="cuda"), torch.empty(B, H, S, device="cuda")
                dq, dk, dv = (torch.empty(B * S, n * D, dtype=torch.bfloat16, device="cuda") for n in (H, KH, KH))
                scratch = torch.empty(K.span_attention_bwd_scratch_floats(B, H, S), device="cuda")
                K.span_attention_fwd(q, k, v, out, lse, spans, **sizes)
                K.span_attention_bwd(q, k, v, out, lse, dout, dq, dk, dv, scratch, spans, **sizes)
            got.append({"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv, "scratch": scratch})
        torch.cuda.synchronize()
        for (*_, want, _stream), g in zip(jobs, got):
            assert all(torch.equal(g[n], want[n]) for n in want)
    assert K.span_attention_last_error() == 0


def test_spans_of_long_rows_replayed():
    """Their pieces' summaries lie in memory of the graph's own."""
    S = 20000
    doc = random_documents(2, S, 4000, seed=1).cuda()
    want, other = K.attention_spans(doc), K.attention_spans(torch.zeros_like(doc))
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        K.attention_spans(doc, out=out)
    graph.replay()
    assert torch.equal(out, want)
    doc.zero_()
    between = K.attention_spans(torch.ones_like(doc))            # an eager call has a scratch of its own
    graph.replay()
    assert torch.equal(out, other) and torch.equal(between, other)

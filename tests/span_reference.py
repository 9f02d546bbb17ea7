"""Attention over spans of keys in 64 bits, and how far the kernels' 16-bit results may be from it.

The bounds count roundings, each off by at most half a step of bf16 relative to the value (U = 2^-8), on the formula's own terms:
  O   = sum P v: P is rounded before the product, O when it is stored                     |dO|  <= U (|O| + P|V|)
  dV  = sum P^T do: the same                                                              |ddV| <= U (|dV| + P^T|dO|)
  dS  = P c (dP - delta) is rounded; delta = do . O takes O as it was stored             |ddS| <= U |dS| + P c |do| . |dO|
  dQ  = scale dS K, rounded when stored                                                   |ddQ| <= U |dQ| + scale ddS |K|, dK alike
  c   = 1 - t^2 with t = tanh in 32 bits, to 4e-7 of itself (the polynomials' error, twice the exponential form's, with their roundings): c is off
        by up to 2 * 4e-7 + 2^-23 < TANH = 1e-6 of 1, which is all there is to it where t is next to 1: a term of p |do| . |v| without c
SLACK (of the same sums) covers what is held in 32 bits: scores of up to 128 products and exponents (a few 1e-6 each), the exponential and
tanh (3e-6), accumulation over up to some thousand terms (1e-4 in the worst case), and second-order terms (U^2 = 1.5e-5)."""
import math

import torch

U = 2.0 ** -8
SLACK = 4.0e-4
TANH = 1.0e-6


def visible(spans, S):
    at = torch.arange(S, device=spans.device)
    return (at[None, None] >= spans[..., :1]) & (at[None, None] <= spans[..., 1:])          # [B, S, S]


def reference(q, k, v, spans, *, B, S, H, KH, D, scale, cap=0.0, slopes=None, dout=None, few=0):
    """Values and bounds of out (and lse), and with `dout` of dq, dk, dv: {name: (value, bound)}, matrices of [B*S, heads*D] in 64 bits.
    Rows that nothing may touch (tokens that nobody sees, queries with empty spans) may hold NaN.  few: queries that see so many keys at most have
    a delta in 32 bits, no rounded O in it."""
    seen = visible(spans, S)
    some = seen.any(-1)                                       # queries that see a key
    heads = lambda t, n: t.double().reshape(B, S, n, D).permute(0, 2, 1, 3)  # noqa: E731
    clean = lambda t, rows: torch.where(rows[:, None, :, None], t, torch.zeros_like(t))  # noqa: E731
    q = clean(heads(q, H), some)
    k, v = (clean(heads(t, KH), seen.any(1)).repeat_interleave(H // KH, 1) for t in (k, v))
    u = scale * q @ k.transpose(-1, -2)
    t = torch.tanh(u / cap) if cap > 0 else None
    x = u if t is None else cap * t
    if slopes is not None:
        at = torch.arange(S, device=q.device, dtype=torch.float64)
        x = x - slopes.double()[None, :, None, None] * (at[:, None] - at[None]).abs()
    x = x.masked_fill(~seen[:, None], -math.inf)
    lse = torch.where(some[:, None], torch.logsumexp(x, -1), torch.zeros((), dtype=torch.float64, device=q.device))
    p = torch.exp(x - lse[..., None])
    out = p @ v
    e_out = U * (out.abs() + p @ v.abs()) + SLACK * (p @ v.abs())
    flat = lambda z, n: z.permute(0, 2, 1, 3).reshape(B * S, n * D)  # noqa: E731
    res = {"out": (flat(out, H), flat(e_out, H)), "lse": (lse / math.log(2.0), 1e-5 + 3e-6 * lse.abs())}
    if dout is None:
        return res
    do = clean(heads(dout, H), some)
    c = torch.ones_like(p) if t is None else 1.0 - t * t
    share = lambda z: z.reshape(B, KH, H // KH, S, D).sum(2)  # noqa: E731
    dp = do @ v.transpose(-1, -2)
    delta = (do * out).sum(-1, keepdim=True)
    ds = p * c * (dp - delta)
    whole = p * (do.abs() @ v.abs().transpose(-1, -2) + (do.abs() * out.abs()).sum(-1, keepdim=True))
    many = (seen.sum(-1) > few)[:, None, :, None]
    e_ds = U * ds.abs() + p * c * many * (do.abs() * e_out).sum(-1, keepdim=True) + (SLACK * c + (TANH if cap > 0 else 0.0)) * whole
    dq, dk, dv = scale * ds @ k, share(scale * ds.transpose(-1, -2) @ q), share(p.transpose(-1, -2) @ do)
    m_dv = share(p.transpose(-1, -2) @ do.abs())
    tiny = 1e-30
    res["dq"] = (flat(dq, H), flat(U * dq.abs() + scale * e_ds @ k.abs() + tiny, H))
    res["dk"] = (flat(dk, KH), flat(U * dk.abs() + share(scale * e_ds.transpose(-1, -2) @ q.abs()) + tiny, KH))
    res["dv"] = (flat(dv, KH), flat(U * (dv.abs() + m_dv) + SLACK * m_dv + tiny, KH))
    return res


def spans_of(documents, prompt=None, causal=True):
    """Spans by the definition, token by token."""
    rows = []
    for b, row in enumerate(documents.tolist()):
        flags = None if prompt is None else prompt[b].tolist()
        line, t = [], 0
        while t < len(row):
            end = t
            while end + 1 < len(row) and row[end + 1] == row[t]:
                end += 1
            lead = t
            while flags is not None and lead <= end and flags[lead]:
                lead += 1
            line += [[0, -1] if row[t] < 0 else [t, max(i, lead - 1) if causal else end] for i in range(t, end + 1)]
            t = end + 1
        rows.append(line)
    return torch.tensor(rows, dtype=torch.int32).reshape(documents.shape[0], documents.shape[1], 2)

"""The operators of a language model's training step on packed documents, and the calls their speed is measured on.

Four operators that are used together: the key spans of a batch of packed documents (`attention_spans`), attention over such spans
with capped or distance-biased scores and shared key / value heads (`span_attention_fwd` / `_bwd`), the RMS norm with the residual's
addition (`rmsnorm_fwd` / `_bwd`), and clipping by the global norm of a list of gradients (`clip_gradients`).  Where ``own`` is false
`run` computes them from elementary torch operations in 32 bits.
"""
import math

import torch

own = False

BF16, F32 = "bf16", "fp32"
_TYPES = {BF16: torch.bfloat16, F32: torch.float32}
_LOG2E = 1.4426950408889634


def listed():
    return [
        # The mask of a small language model's batch (8 x 256 tokens): a launch or two, once per step.
        {"name": "spans_small", "op": "spans", "batch": 8, "seq": 256, "document": 90, "prompt": False, "causal": True},
        # The mask of a batch of long packed sequences with prompts that are seen from both sides.
        {"name": "spans_long", "op": "spans", "batch": 16, "seq": 16384, "document": 1500, "prompt": True, "causal": True},
        # One short sequence through the smallest heads, forward and backward: latency of the launches.
        {"name": "attention_short_train", "op": "attention", "train": True, "batch": 1, "seq": 128, "heads": 8, "kv_heads": 8, "head_dim": 64,
         "mask": "documents", "document": 60, "cap": 0.0, "bias": False},
        # Scoring a batch of documents whose length is no multiple of anything, linear distance bias, four heads to a key head.
        {"name": "attention_odd_forward", "op": "attention", "train": False, "batch": 4, "seq": 1001, "heads": 16, "kv_heads": 4, "head_dim": 128,
         "mask": "causal", "document": 0, "cap": 0.0, "bias": True},
        # Scoring one long sequence, causal, capped scores, shared key heads.
        {"name": "attention_long_forward", "op": "attention", "train": False, "batch": 1, "seq": 8192, "heads": 16, "kv_heads": 4, "head_dim": 128,
         "mask": "causal", "document": 0, "cap": 30.0, "bias": False},
        # The headline model's heads (16 of 128) on packed documents, training.
        {"name": "attention_packed_train", "op": "attention", "train": True, "batch": 8, "seq": 2048, "heads": 16, "kv_heads": 16, "head_dim": 128,
         "mask": "documents", "document": 700, "cap": 50.0, "bias": False},
        # Prompts seen from both sides, answers causal, heads of 64 with a distance bias and shared key heads, training.
        {"name": "attention_prefix_train", "op": "attention", "train": True, "batch": 8, "seq": 1024, "heads": 12, "kv_heads": 4, "head_dim": 64,
         "mask": "prefix", "document": 400, "cap": 0.0, "bias": True},
        # The residual stream of one short prompt: latency.
        {"name": "rmsnorm_short_forward", "op": "rmsnorm", "train": False, "rows": 128, "cols": 512, "dtype": BF16},
        # The headline model's residual stream (32 x 1024 tokens of 2048), forward and backward.
        {"name": "rmsnorm_train", "op": "rmsnorm", "train": True, "rows": 32768, "cols": 2048, "dtype": BF16},
        # 32-bit rows of a width that is no multiple of a vector.
        {"name": "rmsnorm_odd_train", "op": "rmsnorm", "train": True, "rows": 4004, "cols": 1001, "dtype": F32},
        # The gradients of a small classifier: a handful of tensors, 32 bits.
        {"name": "clip_small", "op": "clip", "layers": 2, "width": 512, "dtype": F32, "clipped": True},
        # The gradients of eight layers of the headline model: weights in 16 bits, norms in 32, biases of odd lengths among them.
        {"name": "clip_layers", "op": "clip", "layers": 8, "width": 2048, "dtype": BF16, "clipped": True},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["spans", "attention", "attention", "rmsnorm", "clip"])
    if op == "spans":
        seq = _spread(rng, 1, 16384)
        return {"op": op, "batch": _spread(rng, 1, max(1, min(64, 262144 // seq))), "seq": seq, "document": _spread(rng, 1, seq),
                "prompt": rng.random() < 0.5, "causal": rng.random() < 0.7}
    if op == "attention":
        seq = _spread(rng, 1, 8192)
        kv = rng.choice([1, 2, 3, 4, 8])
        heads = kv * rng.choice([1, 1, 2, 3, 4])
        # no more score pairs than the largest listed case has
        batch = _spread(rng, 1, max(1, min(16, int(5.0e8 / (float(seq) * seq * heads)))))
        train = rng.random() < 0.6 and float(seq) * seq * heads * batch < 3.0e8
        return {"op": op, "train": train, "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv,
                "head_dim": rng.choice([32, 64, 64, 72, 96, 128, 128]), "mask": rng.choice(["causal", "documents", "prefix", "full"]),
                "document": _spread(rng, 1, seq), "cap": rng.choice([0.0, 0.0, 20.0, 50.0]), "bias": rng.random() < 0.4}
    if op == "rmsnorm":
        cols = _spread(rng, 1, 16384)
        return {"op": op, "train": rng.random() < 0.6, "rows": _spread(rng, 1, max(1, min(32768, 33554432 // cols))), "cols": cols,
                "dtype": rng.choice([BF16, BF16, F32])}
    return {"op": op, "layers": rng.randint(1, 8), "width": _spread(rng, 8, 1536), "dtype": rng.choice([BF16, F32]), "clipped": rng.random() < 0.7}


# ---------------------------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 9973 + 17)


def _normal(gen, shape, scale, dtype):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _documents(gen, batch, seq, mean):
    """Document numbers of `batch` packed sequences: lengths around `mean`, the last eighth of every other sequence padding (-1)."""
    ends = torch.rand(batch, seq, generator=gen, device="cuda") < 1.0 / max(mean, 1)
    numbers = torch.cumsum(ends.to(torch.int32), 1, dtype=torch.int32)
    padded = torch.arange(seq, device="cuda")[None, :] >= torch.tensor([seq - seq // 8 if b % 2 else seq for b in range(batch)], device="cuda")[:, None]
    return torch.where(padded, torch.full_like(numbers, -1), numbers).contiguous()


def _prompt(gen, documents):
    """Flags of the first tokens of each document: as many as a draw per document says, and a few stray ones, which are no prompt."""
    batch, seq = documents.shape
    place = torch.arange(seq, device="cuda").expand(batch, seq)
    starts = torch.ones_like(documents, dtype=torch.bool)
    starts[:, 1:] = documents[:, 1:] != documents[:, :-1]
    first = torch.where(starts, place, torch.zeros_like(place)).cummax(1).values
    length = torch.randint(0, max(2, seq // 4), (batch, seq), generator=gen, device="cuda")
    stray = torch.rand(batch, seq, generator=gen, device="cuda") < 0.05
    return ((place - first < length.gather(1, first)) | stray) & (documents >= 0)


def _spans_plain(documents, prompt, causal):
    """[B, S, 2]: first and last token that each token sees."""
    batch, seq = documents.shape
    place = torch.arange(seq, device=documents.device, dtype=torch.int32).expand(batch, seq)
    starts = torch.ones_like(documents, dtype=torch.bool)
    starts[:, 1:] = documents[:, 1:] != documents[:, :-1]
    ends = torch.ones_like(starts)
    ends[:, :-1] = starts[:, 1:]
    low = torch.where(starts, place, torch.zeros_like(place)).cummax(1).values
    last = torch.where(ends, place, torch.full_like(place, seq)).flip(1).cummin(1).values.flip(1)
    if causal:
        high = place
        if prompt is not None:
            # the first token from each place on that is not flagged, or that opens the next document
            stop = torch.where(prompt, torch.where(ends, place + 1, torch.full_like(place, seq)), place).flip(1).cummin(1).values.flip(1)
            high = torch.maximum(place, stop.gather(1, low.long()) - 1)
    else:
        high = last
    padded = documents < 0
    return torch.stack([torch.where(padded, torch.zeros_like(low), low), torch.where(padded, torch.full_like(high, -1), high)], -1).to(torch.int32)


def _slopes(heads):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], dtype=torch.float32, device="cuda")


def _gradient_shapes(case):
    """Shapes of a model's gradients, and which of them are in the case's type (the rest are in 32 bits)."""
    w, shapes = case["width"], []
    for _ in range(case["layers"]):
        shapes += [((3 * w, w), True), ((w, w), True), ((4 * w, w), True), ((w, 4 * w), True), ((4 * w + 1,), True), ((w,), False), ((w,), False)]
    return shapes


def prepare(case, seed):
    gen = _generator(seed)
    state = dict(case)
    if case["op"] == "spans":
        state["documents"] = _documents(gen, case["batch"], case["seq"], case["document"])
        state["flags"] = _prompt(gen, state["documents"]) if case["prompt"] else None
        state["spans"] = torch.empty(case["batch"], case["seq"], 2, dtype=torch.int32, device="cuda")
    elif case["op"] == "attention":
        b, s, h, kh, d = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "head_dim"))
        # one projection's output holds queries, keys and values side by side
        qkv = _normal(gen, (b * s, (h + 2 * kh) * d), 1.0, torch.bfloat16)
        state["q"], state["k"], state["v"] = qkv[:, :h * d], qkv[:, h * d:(h + kh) * d], qkv[:, (h + kh) * d:]
        state["scale"] = 1.0 / math.sqrt(d)
        state["slopes"] = _slopes(h) if case["bias"] else None
        if case["mask"] in ("documents", "prefix"):
            numbers = _documents(gen, b, s, case["document"])
            flags = _prompt(gen, numbers) if case["mask"] == "prefix" else None
        else:
            numbers, flags = torch.zeros(b, s, dtype=torch.int32, device="cuda"), None
        state["spans"] = _spans_plain(numbers, flags, case["mask"] != "full").contiguous()
        state["out"] = torch.empty(b * s, h * d, dtype=torch.bfloat16, device="cuda")
        state["lse"] = torch.empty(b, h, s, dtype=torch.float32, device="cuda")
        if case["train"]:
            state["dout"] = _normal(gen, (b * s, h * d), 1.0, torch.bfloat16)
            dqkv = torch.empty_like(qkv)
            state["dq"], state["dk"], state["dv"] = dqkv[:, :h * d], dqkv[:, h * d:(h + kh) * d], dqkv[:, (h + kh) * d:]
    elif case["op"] == "rmsnorm":
        t = _TYPES[case["dtype"]]
        shape = (case["rows"], case["cols"])
        state["x"], state["residual"] = _normal(gen, shape, 0.5, t), _normal(gen, shape, 2.0, t)
        state["gamma"] = (1.0 + 0.1 * torch.randn(case["cols"], generator=gen, device="cuda")).to(t)
        state["sum"], state["y"] = torch.empty(shape, dtype=t, device="cuda"), torch.empty(shape, dtype=t, device="cuda")
        state["rstd"] = torch.empty(case["rows"], dtype=torch.float32, device="cuda")
        if case["train"]:
            state["dy"], state["dsum"] = _normal(gen, shape, 1.0, t), _normal(gen, shape, 1.0, t)
            state["dx"], state["dgamma"] = torch.empty(shape, dtype=t, device="cuda"), torch.empty(case["cols"], dtype=t, device="cuda")
    else:
        t = _TYPES[case["dtype"]]
        shapes = _gradient_shapes(case)
        state["grads"] = [_normal(gen, shape, 2.0e-3, t if typed else torch.float32) for shape, typed in shapes]
        # the clipped gradients of each type end up side by side in one buffer, as a flat optimizer takes them
        sizes = [(math.prod(shape) + 63) // 64 * 64 for shape, _ in shapes]
        wide = [not typed or t == torch.float32 for _, typed in shapes]
        flat = {k: torch.zeros(max(1, sum(n for n, w in zip(sizes, wide) if w == k)), dtype=torch.float32 if k else t, device="cuda")
                for k in (False, True)}
        at, state["clipped_grads"] = {False: 0, True: 0}, []
        for (shape, _), n, w in zip(shapes, sizes, wide):
            state["clipped_grads"].append(flat[w][at[w]:at[w] + math.prod(shape)].view(shape))
            at[w] += n
        state["flat"] = [flat[k] for k in (False, True) if at[k]]
        total = sum(math.prod(shape) for shape, _ in shapes)
        # the norm is near 2e-3 sqrt(total); three tenths of that are clipped to, four times that leaves the gradients as they are
        state["max_norm"] = 2.0e-3 * math.sqrt(total) * (0.3 if case["clipped"] else 4.0)
        if own:
            from flexflow_train_b200.ops import kernels as K
            state["list"] = K.GradientList(state["grads"], out=state["clipped_grads"])
    return state


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _run_own(state)
    return {"spans": _run_spans, "attention": _run_attention, "rmsnorm": _run_rmsnorm, "clip": _run_clip}[state["op"]](state)


def _run_own(state):
    from flexflow_train_b200.ops import kernels as K
    op = state["op"]
    if op == "spans":
        return K.attention_spans(state["documents"], state["flags"], causal=state["causal"], out=state["spans"])
    if op == "attention":
        sizes = dict(B=state["batch"], S=state["seq"], H=state["heads"], KH=state["kv_heads"], D=state["head_dim"], scale=state["scale"],
                     cap=state["cap"], slopes=state["slopes"])
        K.span_attention_fwd(state["q"], state["k"], state["v"], state["out"], state["lse"], state["spans"], **sizes)
        if not state["train"]:
            return state["out"], state["lse"]
        scratch = torch.empty(K.span_attention_bwd_scratch_floats(state["batch"], state["heads"], state["seq"]), dtype=torch.float32, device="cuda")
        K.span_attention_bwd(state["q"], state["k"], state["v"], state["out"], state["lse"], state["dout"], state["dq"], state["dk"], state["dv"],
                             scratch, state["spans"], **sizes)
        return state["out"], state["dq"], state["dk"], state["dv"]
    if op == "rmsnorm":
        K.rmsnorm_fwd(state["x"], state["gamma"], 1e-6, residual=state["residual"], xsum=state["sum"], out=state["y"], rstd=state["rstd"])
        if not state["train"]:
            return state["y"], state["sum"]
        scratch = torch.empty(K.rmsnorm_bwd_scratch(state["rows"], state["cols"]), dtype=torch.float32, device="cuda")
        K.rmsnorm_bwd(state["dy"], state["sum"], state["gamma"], state["rstd"], state["dx"], state["dgamma"], scratch, dsum=state["dsum"])
        return state["y"], state["sum"], state["dx"], state["dgamma"]
    norm = K.clip_gradients(state["list"], state["max_norm"])
    return [norm] + state["flat"]


def _run_spans(state):
    state["spans"].copy_(_spans_plain(state["documents"], state["flags"], state["causal"]))
    return state["spans"]


def _heads(matrix, batch, seq, heads, dim):
    return matrix.float().reshape(batch, seq, heads, dim).permute(0, 2, 1, 3)


def _run_attention(state):
    b, s, h, kh, d = (state[n] for n in ("batch", "seq", "heads", "kv_heads", "head_dim"))
    q, k, v = _heads(state["q"], b, s, h, d), _heads(state["k"], b, s, kh, d), _heads(state["v"], b, s, kh, d)
    k, v = k.repeat_interleave(h // kh, 1), v.repeat_interleave(h // kh, 1)
    scores = torch.matmul(q, k.transpose(-1, -2)) * state["scale"]
    slope = None
    if state["cap"] > 0:
        scores = torch.tanh(scores / state["cap"])
        slope = 1.0 - scores * scores if state["train"] else None
        scores = scores * state["cap"]
    place = torch.arange(s, device="cuda")
    if state["slopes"] is not None:
        scores = scores - state["slopes"][None, :, None, None] * (place[:, None] - place[None, :]).abs().float()
    low, high = state["spans"][..., 0], state["spans"][..., 1]
    visible = ((place[None, None, :] >= low[:, :, None]) & (place[None, None, :] <= high[:, :, None]))[:, None]
    scores = scores.masked_fill(~visible, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    scores = torch.exp(scores - top)
    total = scores.sum(-1, keepdim=True)
    probs = scores / torch.where(total > 0, total, torch.ones_like(total))
    del scores
    out = torch.matmul(probs, v)
    back = lambda x, n: x.permute(0, 2, 1, 3).reshape(b * s, n * d).to(torch.bfloat16)  # noqa: E731
    state["out"].copy_(back(out, h))
    if not state["train"]:
        lse = torch.where(total > 0, (top + torch.log(total)) * _LOG2E, torch.zeros_like(total))
        state["lse"].copy_(lse[..., 0])
        return state["out"], state["lse"]
    dout = _heads(state["dout"], b, s, h, d)
    dv = torch.matmul(probs.transpose(-1, -2), dout)
    delta = (dout * out).sum(-1, keepdim=True)
    ds = torch.matmul(dout, v.transpose(-1, -2)).sub_(delta).mul_(probs)
    del probs
    if slope is not None:
        ds.mul_(slope)
    dq = torch.matmul(ds, k) * state["scale"]
    dk = torch.matmul(ds.transpose(-1, -2), q) * state["scale"]
    share = lambda x: x.reshape(b, kh, h // kh, s, d).sum(2)  # noqa: E731
    state["dq"].copy_(back(dq, h))
    state["dk"].copy_(back(share(dk), kh))
    state["dv"].copy_(back(share(dv), kh))
    return state["out"], state["dq"], state["dk"], state["dv"]


def _run_rmsnorm(state):
    state["sum"].copy_(state["x"].float() + state["residual"].float())
    h = state["sum"].float()
    rstd = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6)
    gamma = state["gamma"].float()
    state["y"].copy_(h * rstd * gamma)
    if not state["train"]:
        return state["y"], state["sum"]
    dy = state["dy"].float()
    g = dy * gamma
    state["dx"].copy_(rstd * (g - h * (rstd * rstd * (g * h).mean(-1, keepdim=True))) + state["dsum"].float())
    state["dgamma"].copy_((dy * (h * rstd)).sum(0, dtype=torch.float64))
    return state["y"], state["sum"], state["dx"], state["dgamma"]


def _run_clip(state):
    squares = torch.stack([g.float().square().sum(dtype=torch.float64) for g in state["grads"]]).sum()
    norm = torch.sqrt(squares)
    scale = torch.clamp(state["max_norm"] / norm, max=1.0).float()
    [c.copy_(g.float() * scale) for g, c in zip(state["grads"], state["clipped_grads"])]
    return [norm.float().reshape(1)] + state["flat"]


# ---------------------------------------------------------------------------------------------------------------- work
def _visible_pairs(case):
    """Query-key pairs of the case's masks: exact where lengths decide, of one draw where documents do."""
    b, s = case["batch"], case["seq"]
    if case["mask"] == "full":
        return b * s * s
    if case["mask"] == "causal":
        return b * (s * (s + 1) // 2)
    import random
    rng, pairs = random.Random(1), 0
    for row in range(b):
        left = s - s // 8 if row % 2 else s
        while left > 0:
            n = min(left, 1 + int(rng.expovariate(1.0 / max(case["document"], 1))))
            pairs += n * (n + 1) // 2
            if case["mask"] == "prefix":
                p = min(n, rng.randrange(max(2, s // 4)))
                pairs += p * (p - 1) // 2
            left -= n
    return pairs


def work(case):
    if case["op"] == "spans":
        n = case["batch"] * case["seq"]
        return {"bytes": n * (4 + 8 + (1 if case["prompt"] else 0)), "flops": 0}
    if case["op"] == "attention":
        n, h, kh, d = case["batch"] * case["seq"], case["heads"], case["kv_heads"], case["head_dim"]
        pairs = _visible_pairs(case) * h
        size = n * (8 + 2 * d * (2 * h + 2 * kh)) + (0 if case["train"] else 4 * n * h)
        if case["train"]:
            size += n * 2 * d * (2 * h + 2 * kh)
        return {"bytes": size, "flops": pairs * d * (14 if case["train"] else 4)}
    if case["op"] == "rmsnorm":
        n, size = case["rows"] * case["cols"], 2 if case["dtype"] == BF16 else 4
        return {"bytes": n * size * (7 if case["train"] else 4), "flops": n * (16 if case["train"] else 5)}
    size = 2 if case["dtype"] == BF16 else 4
    each = [(math.prod(shape), size if typed else 4) for shape, typed in _gradient_shapes(case)]
    return {"bytes": sum(2 * n * s for n, s in each), "flops": sum(3 * n for n, _ in each)}


# ---------------------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The outputs of `run` from the operators' definitions in 64 bits."""
    state = prepare(case, seed)
    return {"spans": _exact_spans, "attention": _exact_attention, "rmsnorm": _exact_rmsnorm, "clip": _exact_clip}[case["op"]](state)


def _exact_spans(state):
    numbers = state["documents"].cpu().tolist()
    flags = None if state["flags"] is None else state["flags"].cpu().tolist()
    rows = []
    for b, row in enumerate(numbers):
        line, t, n = [], 0, len(row)
        while t < n:
            end = t
            while end + 1 < n and row[end + 1] == row[t]:
                end += 1
            seen = t
            while flags is not None and seen <= end and flags[b][seen]:
                seen += 1
            for i in range(t, end + 1):
                line.append([0, -1] if row[t] < 0 else [t, max(i, seen - 1) if state["causal"] else end])
            t = end + 1
        rows.append(line)
    return torch.tensor(rows, dtype=torch.int32)


def _exact_attention(state):
    b, s, h, kh, d = (state[n] for n in ("batch", "seq", "heads", "kv_heads", "head_dim"))
    if float(b) * h * s * s * d > 3.0e11:
        return None
    wide = lambda x, n: x.double().view(b, s, n, d)  # noqa: E731
    q, k, v = wide(state["q"], h), wide(state["k"], kh), wide(state["v"], kh)
    out, lse = torch.zeros(b, s, h, d, dtype=torch.float64, device="cuda"), torch.zeros(b, h, s, dtype=torch.float64, device="cuda")
    dq, dk, dv = torch.zeros_like(out), torch.zeros_like(k), torch.zeros_like(v)
    dout = wide(state["dout"], h) if state["train"] else None
    at = torch.arange(s, device="cuda")
    for n in range(b):
        seen = (at[None] >= state["spans"][n, :, :1]) & (at[None] <= state["spans"][n, :, 1:])
        for i in range(h):
            g = i // (h // kh)
            u = state["scale"] * (q[n, :, i] @ k[n, :, g].T)
            t = torch.tanh(u / state["cap"]) if state["cap"] > 0 else None
            x = u if t is None else state["cap"] * t
            if state["slopes"] is not None:
                x = x - state["slopes"][i].double() * (at[:, None] - at[None]).abs()
            x = torch.where(seen, x, torch.full_like(x, -math.inf))
            some = seen.any(1)
            total = torch.logsumexp(x, 1)
            total = torch.where(some, total, torch.zeros_like(total))
            p = torch.exp(x - total[:, None])
            lse[n, i] = total / math.log(2.0)
            out[n, :, i] = p @ v[n, :, g]
            if dout is not None:
                dv[n, :, g] += p.T @ dout[n, :, i]
                dp = dout[n, :, i] @ v[n, :, g].T
                ds = p * (dp - (p * dp).sum(1, keepdim=True))
                if t is not None:
                    ds = ds * (1.0 - t * t)
                dq[n, :, i] = state["scale"] * (ds @ k[n, :, g])
                dk[n, :, g] += state["scale"] * (ds.T @ q[n, :, i])
    out = out.view(b * s, h * d)
    if dout is None:
        return out, lse
    return out, dq.view(b * s, h * d), dk.view(b * s, kh * d), dv.view(b * s, kh * d)


def _exact_rmsnorm(state):
    h = (state["x"].double() + state["residual"].double()).to(state["x"].dtype).double()
    root = ((h ** 2).sum(1) / h.shape[1] + 1e-6) ** 0.5
    unit, gamma = h / root[:, None], state["gamma"].double()
    y = unit * gamma
    if not state["train"]:
        return y, h
    dy = state["dy"].double()
    part = dy * gamma
    dx = (part - unit * ((part * unit).sum(1) / h.shape[1])[:, None]) / root[:, None] + state["dsum"].double()
    return y, h, dx, (dy * unit).sum(0)


def _exact_clip(state):
    norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g in state["grads"]))
    scale = min(1.0, state["max_norm"] / norm)
    flat = [f.double() for f in state["flat"]]
    for g, c in zip(state["grads"], state["clipped_grads"]):
        at = next(i for i, f in enumerate(state["flat"]) if f.data_ptr() <= c.data_ptr() < f.data_ptr() + f.numel() * f.element_size())
        start = (c.data_ptr() - state["flat"][at].data_ptr()) // c.element_size()
        flat[at][start:start + g.numel()] = g.double().reshape(-1) * scale
    return [torch.tensor([norm], dtype=torch.float64)] + flat

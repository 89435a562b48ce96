"""
Three more operators of a recurrent language model, as its users call them: in front of its layers, in them, and behind its scores.

``delta``      a recurrent layer whose state is a matrix (:func:`returnn_amd.delta_rule.gated_delta_rule`), on projected queries, keys and values
``embedding``  scaled rows of a table (:func:`returnn_amd.embedding.embed`), with the table's gradient
``beam``       a step of beam search: the best continuations of all hypotheses (:func:`returnn_amd.beam_search.beam_select`) and the
               states that go with them (:func:`returnn_amd.beam_search.reorder_states`)

Sequences are right-padded where ``ragged``: lengths spread evenly over [T/2, T] in an order of the seed's; they lie on the GPU.
With ``own`` false everything is computed from elementary torch operations in float32, rounded once at the end.
"""

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # a step of a decoder in beam search (beam 12), once per label: the layer's state goes through memory
        {"name": "delta_step", "kind": "delta", "T": 1, "B": 12, "key_heads": 8, "heads": 8, "dk": 128, "dv": 128, "dtype": "bf16", "ragged": False, "direction": 1, "train": False},
        # one long utterance or prompt by itself: few heads, all parallelism is in time and columns
        {"name": "delta_prompt", "kind": "delta", "T": 4000, "B": 1, "key_heads": 8, "heads": 8, "dk": 128, "dv": 128, "dtype": "bf16", "ragged": False, "direction": 1, "train": False},
        # a training step of a layer of a speech encoder's size, ragged
        {"name": "delta_train", "kind": "delta", "T": 1000, "B": 32, "key_heads": 8, "heads": 8, "dk": 128, "dv": 128, "dtype": "bf16", "ragged": True, "direction": 1, "train": True},
        # training on long documents, two at a time, two value heads to each head of queries and keys
        {"name": "delta_train_long_shared", "kind": "delta", "T": 8192, "B": 2, "key_heads": 4, "heads": 8, "dk": 64, "dv": 128, "dtype": "bf16", "ragged": True, "direction": 1, "train": True},
        # odd sizes everywhere, float32, backward in time
        {"name": "delta_train_odd", "kind": "delta", "T": 333, "B": 11, "key_heads": 5, "heads": 5, "dk": 50, "dv": 71, "dtype": "f32", "ragged": True, "direction": -1, "train": True},
        # the tokens of a search step
        {"name": "embedding_step", "kind": "embedding", "T": 1, "B": 12, "V": 32000, "D": 1024, "dtype": "bf16", "ragged": False, "train": False},
        # training of a language model
        {"name": "embedding_train", "kind": "embedding", "T": 64, "B": 64, "V": 32000, "D": 1024, "dtype": "bf16", "ragged": True, "train": True},
        # training in float32, an odd vocabulary and an odd width
        {"name": "embedding_train_odd", "kind": "embedding", "T": 333, "B": 11, "V": 10007, "D": 501, "dtype": "f32", "ragged": True, "train": True},
        # a large batch on a large vocabulary
        {"name": "embedding_train_large", "kind": "embedding", "T": 1000, "B": 32, "V": 131072, "D": 1024, "dtype": "bf16", "ragged": True, "train": True},
        # one search, two layers of 1024 channels
        {"name": "beam_step", "kind": "beam", "B": 1, "beam": 12, "V": 32000, "dtype": "f32", "states": 2, "width": 1024, "ended": False},
        # a batch of searches, an odd vocabulary, some hypotheses at their end
        {"name": "beam_batch_odd", "kind": "beam", "B": 16, "beam": 5, "V": 10007, "dtype": "bf16", "states": 6, "width": 500, "ended": True},
        # many searches on a large vocabulary, states that are matrices (two layers of 4 heads, 128 x 128)
        {"name": "beam_large", "kind": "beam", "B": 32, "beam": 8, "V": 131072, "dtype": "f32", "states": 2, "width": 65536, "ended": True},
    ]  # fmt: skip


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Widths: multiples of 64 or of 16 as most configurations have them, and any others."""
    n = _log_int(rng, lo, hi)
    unit = rng.choice((64, 16, 1, 1))
    return max(lo, n // unit * unit)


def _drawn(rng):
    kind = rng.choice(("delta", "delta", "embedding", "beam"))
    case = {"kind": kind, "dtype": rng.choice(("f32", "bf16"))}
    if kind == "delta":
        T = rng.choice((1, _log_int(rng, 2, 8192), _log_int(rng, 2, 8192), _log_int(rng, 2, 8192)))
        key_heads = _log_int(rng, 1, 16)
        case.update(T=T, B=_log_int(rng, 1, 64), key_heads=key_heads, heads=key_heads * rng.choice((1, 1, 2, 4)), dk=_width(rng, 16, 128), dv=_width(rng, 16, 256),
                    ragged=T > 1 and rng.random() < 0.6, direction=rng.choice((1, 1, -1)), train=T > 1 and rng.random() < 0.6)  # fmt: skip
    elif kind == "embedding":
        case.update(T=_log_int(rng, 1, 1000), B=_log_int(rng, 1, 256), V=_width(rng, 64, 131072), D=_width(rng, 32, 4096), ragged=rng.random() < 0.5, train=rng.random() < 0.7)
    else:
        beam, V = rng.randint(1, 32), _width(rng, 64, 131072)
        case.update(B=_log_int(rng, 1, 64), beam=beam, V=V, states=rng.randint(1, 8), width=_width(rng, 32, 65536), ended=rng.random() < 0.5)
    return case


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        for what in ("bytes", "flops"):
            most[c["kind"], what] = max(most.get((c["kind"], what), 0.0), w[what])
    while True:
        case = _drawn(rng)
        w = work(case)
        if all(w[what] <= most[case["kind"], what] for what in ("bytes", "flops")):
            return case


def _lengths(T, B):
    """B lengths spread evenly over [T/2, T], the longest first."""
    return [max(1, T - (j * (T // 2)) // max(1, B - 1)) for j in range(B)]


def _normal(shape, std, dtype, gen):
    return (torch.randn(shape, device="cuda", generator=gen) * std).to(dtype)


def _unit(shape, dtype, gen):
    v = torch.randn(shape, device="cuda", generator=gen)
    return (v / v.square().sum(dim=-1, keepdim=True).sqrt()).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    act = _DTYPES[case["dtype"]]
    B = case["B"]
    state = {"case": case, "lens": None}
    if case.get("ragged"):
        order = torch.randperm(B, generator=torch.Generator().manual_seed(seed))
        state["lens"] = torch.tensor(_lengths(case["T"], B), dtype=torch.int64)[order].cuda()
    if case["kind"] == "delta":
        T, Hk, H, dk, dv, train = case["T"], case["key_heads"], case["heads"], case["dk"], case["dv"], case["train"]
        lead = (B,) if T == 1 else (T, B)  # one step comes without a time axis
        state["q"], state["k"] = _unit(lead + (Hk, dk), act, gen).requires_grad_(train), _unit(lead + (Hk, dk), act, gen).requires_grad_(train)
        state["v"] = _normal(lead + (H, dv), 1.0, act, gen).requires_grad_(train)
        # decays of most frames near 1, of some far below; write strengths anywhere between 0 and 1
        state["g"] = (-torch.nn.functional.softplus(_normal(lead + (H,), 2.0, torch.float32, gen) - 3.0)).requires_grad_(train)
        state["b"] = torch.sigmoid(_normal(lead + (H,), 1.5, torch.float32, gen)).requires_grad_(train)
        state["s0"] = _normal((B, H, dk, dv), 0.1, torch.float32, gen).requires_grad_(train)
        if train:
            state["dy"] = _normal(lead + (H, dv), 1.0 / math.sqrt(T * B), act, gen)
            state["ds"] = _normal((B, H, dk, dv), 1.0 / math.sqrt(T * B * dk), torch.float32, gen)
    elif case["kind"] == "embedding":
        T, V, D, train = case["T"], case["V"], case["D"], case["train"]
        state["weight"] = _normal((V, D), 1.0 / math.sqrt(D), act, gen).requires_grad_(train)
        # frequent tokens and rare ones, as in a text: token number r about 1 / (r + 3) of the time, in an order of the seed's
        u = torch.rand((T, B), device="cuda", generator=gen, dtype=torch.float64)
        rank = (3.0 * torch.exp(u * math.log((V + 3.0) / 3.0)) - 3.0).to(torch.int64).clamp(max=V - 1)
        tokens = torch.randperm(V, device="cuda", generator=gen)[rank]
        if state["lens"] is not None:  # frames past the end have no token
            tokens = torch.where(torch.arange(T, device="cuda")[:, None] < state["lens"][None, :], tokens, -1)
        state["tokens"], state["scale"] = tokens, math.sqrt(D)
        if train:
            state["dy"] = _normal((T, B, D), 1.0 / math.sqrt(T * B), act, gen)
    else:
        K, V = case["beam"], case["V"]
        logits = torch.randn((B, K, V), device="cuda", generator=gen) * 2.5
        state["scores"] = torch.log_softmax(logits, dim=-1).to(act)
        state["totals"] = -5.0 * torch.rand((B, K), device="cuda", generator=gen)
        state["ended"] = (torch.rand((B, K), device="cuda", generator=gen) < 0.2) if case["ended"] else None
        state["end"] = V // 3 if case["ended"] else None
        state["states"] = [_normal((B, K, case["width"]), 1.0, torch.float32, gen) for _ in range(case["states"])]
    return state


def run(state):
    with torch.enable_grad():
        return _run_own(state) if own else _run_plain(state)


_DELTA_INPUTS = ("q", "k", "v", "g", "b", "s0")


def _run_own(state):
    case = state["case"]
    if case["kind"] == "delta":
        from returnn_amd.delta_rule import gated_delta_rule

        inputs = [state[name] for name in _DELTA_INPUTS]
        y, s = gated_delta_rule(*inputs[:5], state=inputs[5], seq_lens=state["lens"], direction=case["direction"])
        if not case["train"]:
            return y, s
        return (y.detach(), s.detach()) + torch.autograd.grad((y, s), inputs, (state["dy"], state["ds"]))
    if case["kind"] == "embedding":
        from returnn_amd.embedding import embed

        y = embed(state["tokens"], state["weight"], scale=state["scale"])
        if not case["train"]:
            return y
        return (y.detach(),) + torch.autograd.grad(y, state["weight"], state["dy"])
    from returnn_amd.beam_search import beam_select, reorder_states

    step = beam_select(state["scores"], state["totals"], case["beam"], ended=state["ended"], end_token=state["end"])
    return step.totals, step.sources, step.tokens, reorder_states(state["states"], step.sources)


# ---- the plain forms ----
def _inverse(a):
    """(1 + a)^-1 of strictly lower triangular [...,C,C], row by row."""
    C = a.shape[-1]
    one = torch.eye(C, dtype=a.dtype, device=a.device).expand(a.shape)
    rows = [one[..., :1, :]]
    for i in range(1, C):
        rows.append(one[..., i : i + 1, :] - a[..., i : i + 1, :i] @ torch.cat(rows, dim=-2))
    return torch.cat(rows, dim=-2)


def _plain_delta_forward(case, lens, q, k, v, g, b, s):
    """In chunks of up to 64 frames, all of them at once but for the state."""
    H, T = case["heads"], v.shape[0]
    each = H // case["key_heads"]
    q, k = q.repeat_interleave(each, dim=2), k.repeat_interleave(each, dim=2)
    if lens is not None:
        inside = torch.arange(T, device=v.device)[:, None, None] < lens[None, :, None]
        g, b = torch.where(inside, g, 0.0), torch.where(inside, b, 0.0)
    C = min(T, 64)
    pad = -T % C

    def chunks(t):  # [T,B,H,...] -> [chunks,B,H,C,...]
        t = t.flip(0) if case["direction"] < 0 else t
        t = torch.cat((t, t.new_zeros((pad,) + t.shape[1:]))) if pad else t
        return t.unflatten(0, (-1, C)).movedim(1, 3)

    q, k, v, g, b = chunks(q * q.shape[-1] ** -0.5), chunks(k), chunks(v), chunks(g), chunks(b)[..., None]
    total = g.cumsum(dim=-1)
    c = torch.exp(total)[..., None]
    row = torch.arange(C, device=v.device)
    lower = row[:, None] >= row[None, :]
    between = torch.exp(torch.where(lower, total[..., :, None] - total[..., None, :], -math.inf))
    kt = k.transpose(-1, -2)
    p = (q @ kt) * between
    t = _inverse(b * (k @ kt) * between * (row[:, None] > row[None, :]))
    left, right = t @ (b * v), t @ (b * c * k)
    q, kt, c_end = q * c, kt * torch.exp(total[..., -1:] - total)[..., None, :], c[..., -1:, :]
    out = []
    for j in range(v.shape[0]):
        u = left[j] - right[j] @ s
        out.append(q[j] @ s + p[j] @ u)
        s = c_end[j] * s + kt[j] @ u
    y = torch.stack(out).movedim(3, 1).flatten(0, 1)[:T]
    y = y.flip(0) if case["direction"] < 0 else y
    return (y if lens is None else torch.where(inside[..., None], y, 0.0)), s


def _plain_delta(state):
    case = state["case"]
    inputs = [state[name].detach() for name in _DELTA_INPUTS]
    single = case["T"] == 1
    x = [t.float().requires_grad_(case["train"]) for t in inputs]
    with torch.set_grad_enabled(case["train"]):
        y, s = _plain_delta_forward(case, state["lens"], *((t[None] for t in x[:5]) if single else x[:5]), x[5])
    grads = []
    if case["train"]:
        grads = [d.to(t.dtype) for d, t in zip(torch.autograd.grad((y, s), x, (state["dy"].float(), state["ds"])), inputs)]
    y = y.detach().to(state["v"].dtype)
    return (y[0] if single else y, s.detach()) + tuple(grads)


def _plain_embedding(state):
    tokens, weight = state["tokens"], state["weight"].detach()
    has = tokens >= 0
    rows = weight[tokens.clamp(min=0)].float() * state["scale"]
    y = torch.where(has[..., None], rows, 0.0).to(weight.dtype)
    if not state["case"]["train"]:
        return y
    V, D = weight.shape
    dw = torch.zeros((V + 1, D), device=weight.device)  # (the last row of what has no token)
    dw.index_add_(0, torch.where(has, tokens, V).flatten(), state["dy"].float().flatten(0, 1) * state["scale"])
    return y, dw[:V].to(weight.dtype)


def _plain_beam(state):
    scores, totals, beam = state["scores"].float(), state["totals"], state["case"]["beam"]
    V = scores.shape[-1]
    if state["ended"] is not None:  # what has ended goes on with its end and nothing else, at no cost
        only = torch.where(torch.arange(V, device=scores.device) == state["end"], 0.0, -math.inf)
        scores = torch.where(state["ended"][..., None], only, scores)
    joint = (totals[..., None] + scores).flatten(1)
    # whole numbers in the order of the sums, the lower index first among equal ones: no two of a search are alike
    bits = joint.view(torch.int32).to(torch.int64)
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    best = torch.topk(order * 2**31 + (2**31 - 1 - torch.arange(joint.shape[-1], device=joint.device)), beam, dim=-1).values
    at = 2**31 - 1 - best % 2**31
    sources = torch.div(at, V, rounding_mode="floor")
    search = torch.arange(scores.shape[0], device=scores.device)[:, None]
    return joint.gather(1, at), sources, at % V, [s[search, sources] for s in state["states"]]


def _run_plain(state):
    with torch.no_grad():
        return {"delta": _plain_delta, "embedding": _plain_embedding, "beam": _plain_beam}[state["case"]["kind"]](state)


# ---- the definitions in 64 bits ----
def _exact_delta(state):
    case = state["case"]
    q, k, v, g, b, s = (state[name].detach().double() for name in _DELTA_INPUTS)
    if case["T"] == 1:
        q, k, v, g, b = (t.unsqueeze(0) for t in (q, k, v, g, b))
    T, B, H, dv = v.shape
    Hk, dk = q.shape[2:]
    shared = torch.arange(H, device=v.device) // (H // Hk)  # a head's queries and keys
    a, scale = torch.exp(g), 1.0 / math.sqrt(dk)
    lens = torch.full((B,), T, device=v.device) if state["lens"] is None else state["lens"]
    frames = list(range(T))[:: case["direction"]]

    def frame(t, s):
        """The state behind frame t, and what led to it: all of [B,H,...]."""
        kt = k[t][:, shared]
        kept = a[t][..., None, None] * s
        missing = v[t] - (kept * kt[..., None]).sum(dim=-2)
        return kept + kt[..., None] * (b[t][..., None] * missing)[..., None, :], kept, missing, kt

    y = torch.zeros_like(v)
    every = 64
    marks = []
    for n, t in enumerate(frames):
        if n % every == 0:
            marks.append(s)
        inside = (t < lens)[:, None, None]
        after = frame(t, s)[0]
        s = torch.where(inside[..., None], after, s)
        y[t] = torch.where(inside, scale * (after * q[t][:, shared][..., None]).sum(dim=-2), 0.0)
    out = (y[0] if case["T"] == 1 else y, s)
    if not case["train"]:
        return out
    dq, dk_, dv_, dg, db = (torch.zeros_like(x) for x in (q, k, v, g, b))
    d = state["ds"].double()
    dy = state["dy"].double()
    for m in reversed(range(len(marks))):
        span, s = frames[m * every : (m + 1) * every], marks[m]
        before = []
        for t in span:
            before.append(s)
            s = torch.where((t < lens)[:, None, None, None], frame(t, s)[0], s)
        for t in reversed(span):
            s = before.pop()
            after, kept, missing, kt = frame(t, s)
            inside = (t < lens)[:, None]
            e = scale * dy[t]
            into = d + q[t][:, shared][..., None] * e[..., None, :]  # of the state behind the frame
            du = (into * kt[..., None]).sum(dim=-2)
            dm = b[t][..., None] * du
            of_kept = into - kt[..., None] * dm[..., None, :]
            dkt = (into * (b[t][..., None] * missing)[..., None, :]).sum(dim=-1) - (kept * dm[..., None, :]).sum(dim=-1)
            dqt = (after * e[..., None, :]).sum(dim=-1)
            for total, part in ((dq, dqt), (dk_, dkt)):
                total[t] = torch.where(inside[..., None], part, 0.0).view(B, Hk, H // Hk, dk).sum(dim=2)
            dv_[t] = torch.where(inside[..., None], dm, 0.0)
            db[t] = torch.where(inside, (du * missing).sum(dim=-1), 0.0)
            dg[t] = torch.where(inside, (of_kept * kept).sum(dim=(-1, -2)), 0.0)
            d = torch.where(inside[..., None, None], a[t][..., None, None] * of_kept, d)
    return out + (dq, dk_, dv_, dg, db, d)


def _exact_embedding(state):
    weight, tokens, scale = state["weight"].detach().double(), state["tokens"].flatten(), state["scale"]
    given = torch.nonzero(tokens >= 0).flatten()
    rows = weight.new_zeros((tokens.numel(), weight.shape[1]))
    rows[given] = scale * weight[tokens[given]]
    y = rows.view(state["tokens"].shape + (-1,))
    if not state["case"]["train"]:
        return y
    # the errors in the order of their tokens, and sums over the runs of one token
    order = given[torch.sort(tokens[given], stable=True).indices]
    dw = torch.zeros_like(weight)
    found, counts = torch.unique_consecutive(tokens[order], return_counts=True)
    errors = state["dy"].flatten(0, 1).double()[order]
    dw[found] = scale * torch.segment_reduce(errors, "sum", lengths=counts, axis=0)
    return y, dw


def _exact_beam(state):
    case = state["case"]
    totals, sources, tokens = [], [], []
    for n in range(case["B"]):
        scores = state["scores"][n].double()
        if state["ended"] is not None:
            for j in torch.nonzero(state["ended"][n]).flatten().tolist():
                scores[j] = -math.inf
                scores[j, state["end"]] = 0.0
        joint = (state["totals"][n].double()[:, None] + scores).float().flatten()  # the sum is one of float32 by definition
        values, at = torch.sort(joint, descending=True, stable=True)
        totals.append(values[: case["beam"]].double())
        sources.append(at[: case["beam"]] // case["V"])
        tokens.append(at[: case["beam"]] % case["V"])
    sources = torch.stack(sources)
    states = [torch.stack([s[n].index_select(0, sources[n]) for n in range(case["B"])]).double() for s in state["states"]]
    return torch.stack(totals), sources, torch.stack(tokens), states


def exact(case, seed):
    if case["kind"] == "delta" and case["T"] * (4 if case["train"] else 1) * max(1.0, case["B"] * case["heads"] * case["dk"] * case["dv"] / 2**22) > 40000:
        return None
    state = prepare(case, seed)
    with torch.no_grad():
        return {"delta": _exact_delta, "embedding": _exact_embedding, "beam": _exact_beam}[case["kind"]](state)


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    B = case["B"]
    if case["kind"] == "beam":
        K, V, rows = case["beam"], case["V"], B * case["beam"]
        return {"bytes": float(e * rows * V) + rows * (8.0 * case["states"] * case["width"] + 24.0), "flops": 2.0 * rows * V}
    T = case["T"]
    rows = T * B
    valid = sum(_lengths(T, B)) if case.get("ragged") else rows  # frames that belong to a sequence: no others need be read
    if case["kind"] == "embedding":
        V, D = case["V"], case["D"]
        forward = e * float(D) * (valid + rows) + 8.0 * rows
        if not case["train"]:
            return {"bytes": forward, "flops": float(valid * D)}
        return {"bytes": forward + e * float(D) * (valid + V), "flops": 2.0 * valid * D}
    Hk, H, dk, dv = case["key_heads"], case["heads"], case["dk"], case["dv"]
    # queries, keys, values, decays and strengths of the valid frames and the state are read, the outputs and the new state written
    inputs, matrix = e * (2.0 * Hk * dk + H * dv) + 8.0 * H, 4.0 * B * H * dk * dv
    forward = valid * inputs + e * float(rows * H * dv) + 2.0 * matrix
    flops = 7.0 * valid * H * dk * dv  # decay, prediction, correction and output of a frame
    if not case["train"]:
        return {"bytes": forward, "flops": flops}
    # the errors of outputs and state; the errors of all inputs
    return {"bytes": forward + e * float(valid * H * dv) + rows * inputs + 2.0 * matrix, "flops": 22.0 / 7.0 * flops}

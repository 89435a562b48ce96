"""
The operators of a recurrent language model behind and between its matrix products, as its users call them: training
steps, scoring and search.

``recurrence``  a gated linear recurrence over time (:func:`returnn_amd.recurrence.gated_recurrence`), on gates projected before
``dropout``     dropout whose mask is computed from a counter (:func:`returnn_amd.dropout.dropout`), with its gradient
``scores``      log probabilities of given tokens, entropy and the best alternatives (:func:`returnn_amd.scoring.token_log_probs`)

Sequences are right-padded where ``ragged``: lengths spread evenly over [T/2, T] in an order of the seed's; they lie on the GPU.
With ``own`` false everything is computed from elementary torch operations in float32, rounded once at the end.
"""

import math

import numpy
import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one step of a recurrent decoder in beam search (beam 12): called once per label, all of it is latency
        {"name": "recurrence_step", "kind": "recurrence", "T": 1, "B": 12, "n": 1024, "dtype": "bf16", "ragged": False, "direction": 1, "train": False},
        # one long utterance recognised by itself: few channels, all parallelism is in time
        {"name": "recurrence_single_sequence", "kind": "recurrence", "T": 4000, "B": 1, "n": 1024, "dtype": "bf16", "ragged": False, "direction": 1, "train": False},
        # a middle-sized layer in float32, ragged batch, backward in time
        {"name": "recurrence_f32_reverse", "kind": "recurrence", "T": 500, "B": 64, "n": 512, "dtype": "f32", "ragged": True, "direction": -1, "train": False},
        # a training step of a layer of a speech encoder's size
        {"name": "recurrence_train", "kind": "recurrence", "T": 1000, "B": 32, "n": 1024, "dtype": "bf16", "ragged": True, "direction": 1, "train": True},
        # training on long documents, two at a time, a width that is no power of two
        {"name": "recurrence_train_long", "kind": "recurrence", "T": 16384, "B": 2, "n": 500, "dtype": "bf16", "ragged": True, "direction": 1, "train": True},
        # an odd width in an odd ragged batch, float32, backward in time
        {"name": "recurrence_train_odd", "kind": "recurrence", "T": 333, "B": 11, "n": 1001, "dtype": "f32", "ragged": True, "direction": -1, "train": True},
        # between two layers in training: dropout of a layer's output, added to the layer's input
        {"name": "dropout_residual", "kind": "dropout", "T": 1000, "B": 32, "n": 1024, "dtype": "bf16", "drop_prob": 0.1, "residual": True, "same_over_time": False},
        # one mask for all frames of a sequence, on training chunks of 50 frames
        {"name": "dropout_same_over_time", "kind": "dropout", "T": 50, "B": 40, "n": 500, "dtype": "f32", "drop_prob": 0.3, "residual": False, "same_over_time": True},
        # a search step: the alternatives of every hypothesis of a beam, a tenth of the tokens not allowed
        {"name": "scores_beam", "kind": "scores", "T": 1, "B": 12, "V": 32000, "dtype": "bf16", "ragged": False, "given": False, "top_k": 12, "blocked": 0.1, "padded": False,
         "train": False},
        # one sampled token of a large vocabulary, reported with its alternatives and the entropy
        {"name": "scores_one_token", "kind": "scores", "T": 1, "B": 1, "V": 131072, "dtype": "f32", "ragged": False, "given": True, "top_k": 20, "blocked": 0.0, "padded": False,
         "train": False},
        # fine-tuning in float32 on ragged hypotheses with the alternatives reported, an odd vocabulary in a projection padded to a multiple of 64
        {"name": "scores_odd", "kind": "scores", "T": 37, "B": 21, "V": 10007, "dtype": "f32", "ragged": True, "given": True, "top_k": 5, "blocked": 0.0, "padded": True,
         "train": True},
        # training of a language model: log probabilities and entropy of all tokens of a batch, and the gradient of the logits
        {"name": "scores_train", "kind": "scores", "T": 64, "B": 64, "V": 32000, "dtype": "bf16", "ragged": True, "given": True, "top_k": 0, "blocked": 0.0, "padded": False,
         "train": True},
    ]  # fmt: skip


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Widths: multiples of 64 or of 32 as most configurations have them, and any others."""
    n = _log_int(rng, lo, hi)
    unit = rng.choice((64, 32, 1, 1))
    return max(unit, n // unit * unit)


def _largest():
    works = [work(c) for c in listed()]
    return max(w["bytes"] for w in works), max(c["T"] * c["B"] * c.get("n", 0) for c in listed()), max(c["T"] * c["B"] * c.get("V", 0) for c in listed())


def draw(rng):
    kind = rng.choice(("recurrence", "recurrence", "dropout", "scores", "scores"))
    max_bytes, max_n, max_v = _largest()
    while True:
        case = {"kind": kind, "T": _log_int(rng, 1, 16384 if kind == "recurrence" else 1000), "B": _log_int(rng, 1, 256), "dtype": rng.choice(("f32", "bf16"))}
        if kind == "recurrence":
            case.update(n=_width(rng, 32, 4096), ragged=rng.random() < 0.7, direction=rng.choice((1, -1)), train=rng.random() < 0.6)
        elif kind == "dropout":
            case.update(n=_width(rng, 32, 4096), drop_prob=rng.choice((0.05, 0.1, 0.2, 0.3, 0.5)), residual=rng.random() < 0.5, same_over_time=rng.random() < 0.3)
        else:
            given = rng.random() < 0.7
            train = given and rng.random() < 0.5
            case.update(V=_width(rng, 64, 131072), ragged=given and rng.random() < 0.5, given=given, top_k=rng.choice((0, 0, 5)) if train else rng.randint(0 if given else 1, 20),
                        blocked=0.0 if given else rng.choice((0.0, 0.1, 0.5)), padded=rng.random() < 0.3, train=train)  # fmt: skip
        sizes = (case["T"], case["B"], case["T"] * case["B"], case.get("n", 0), 2 * case.get("n", 0), 4 * case.get("n", 0), case.get("V", 0), -(-case.get("V", 0) // 64) * 64)
        if 3072 in sizes:
            continue
        rows = case["T"] * case["B"]
        if work(case)["bytes"] <= max_bytes and rows * case.get("n", 0) <= max_n and rows * case.get("V", 0) <= max_v:
            return case


def _lengths(T, B):
    """B lengths spread evenly over [T/2, T], the longest first."""
    return [max(1, T - (j * (T // 2)) // max(1, B - 1)) for j in range(B)]


def _normal(shape, std, dtype, gen):
    return (torch.randn(shape, device="cuda", generator=gen) * std).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    act = _DTYPES[case["dtype"]]
    T, B = case["T"], case["B"]
    state = {"case": case, "lens": None}
    if case.get("ragged"):
        order = torch.randperm(B, generator=torch.Generator().manual_seed(seed))
        state["lens"] = torch.tensor(_lengths(T, B), dtype=torch.int64)[order].cuda()
    if case["kind"] == "recurrence":
        n, train = case["n"], case["train"]
        x = torch.randn((T, B, 4 * n), device="cuda", generator=gen)
        x[..., 2 * n : 3 * n] += 2.0  # forget gates that keep: what a layer learns that remembers
        x = x.to(act)
        state["x"] = (x[0] if T == 1 and not train else x).requires_grad_(train)  # one step comes without a time axis
        state["c0"] = _normal((B, n), 0.5, torch.float32, gen).requires_grad_(train)
        if train:
            state["dy"] = _normal((T, B, n), 1.0 / math.sqrt(T * B), act, gen)
            state["dc"] = _normal((B, n), 1.0 / math.sqrt(T * B), torch.float32, gen)
    elif case["kind"] == "dropout":
        n = case["n"]
        state["x"] = _normal((T, B, n), 1.0, act, gen).requires_grad_(True)
        state["residual"] = _normal((T, B, n), 1.0, act, gen).requires_grad_(True) if case["residual"] else None
        state["dy"] = _normal((T, B, n), 1.0 / math.sqrt(T * B), act, gen)
        state["seed"], state["offset"] = (0x9E3779B97F4A7C15 ^ (seed * 0x2545F491)) & (1 << 64) - 1, (seed & 0xFFFFFFFF) * 7 + 1
    else:
        V = case["V"]
        ld = -(-V // 64) * 64 if case["padded"] else V
        logits = torch.randn((T, B, ld), device="cuda", generator=gen) * 2.5
        if case["blocked"]:
            logits = logits.masked_fill(torch.rand((T, B, ld), device="cuda", generator=gen) < case["blocked"], -math.inf)
        state["logits"] = logits.to(act)[..., :V].requires_grad_(case["train"])
        state["targets"] = None
        if case["given"]:
            targets = torch.randint(0, V, (T, B), device="cuda", generator=gen)
            if state["lens"] is not None:  # frames past the end have no token
                targets = torch.where(torch.arange(T, device="cuda")[:, None] < state["lens"][None, :], targets, -1)
            state["targets"] = targets
        if case["train"]:
            state["d_log_probs"] = _normal((T, B), 1.0 / (T * B), torch.float32, gen) - 1.0 / (T * B)
            state["d_entropy"] = _normal((T, B), 0.1 / (T * B), torch.float32, gen)
    return state


def run(state):
    with torch.enable_grad():
        return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    case = state["case"]
    if case["kind"] == "recurrence":
        from returnn_amd.recurrence import gated_recurrence

        y, c = gated_recurrence(state["x"], state=state["c0"], seq_lens=state["lens"], direction=case["direction"])
        if not case["train"]:
            return y, c
        return (y.detach(), c.detach()) + torch.autograd.grad((y, c), (state["x"], state["c0"]), (state["dy"], state["dc"]))
    if case["kind"] == "dropout":
        from returnn_amd.dropout import dropout

        y = dropout(state["x"], case["drop_prob"], seed=state["seed"], offset=state["offset"], residual=state["residual"], same_over_time=case["same_over_time"])
        inputs = (state["x"],) if state["residual"] is None else (state["x"], state["residual"])
        return (y.detach(),) + torch.autograd.grad(y, inputs, state["dy"])
    from returnn_amd.scoring import token_log_probs

    s = token_log_probs(state["logits"], state["targets"], entropy=True, top_k=case["top_k"])
    out = [s.entropy.detach()]
    if case["given"]:
        out.append(s.log_probs.detach())
    if case["top_k"]:
        out += [s.top_log_probs, s.top_ids]
    if case["train"]:
        out += torch.autograd.grad((s.log_probs, s.entropy), (state["logits"],), (state["d_log_probs"], state["d_entropy"]))
    return out


# ---- the plain forms ----
def _valid(state, T, device):
    """[T,B,1]: which frames belong to a sequence."""
    if state["lens"] is None:
        return torch.ones((T, state["case"]["B"], 1), dtype=torch.bool, device=device)
    return (torch.arange(T, device=device)[:, None] < state["lens"][None, :])[..., None]


def _scan(a, s):
    """h_t = a_t h_{t-1} + s_t along the first axis, h_{-1} = 0: spans of doubled length joined."""
    span = 1
    while span < a.shape[0]:
        s = torch.cat((s[:span], s[span:] + a[span:] * s[:-span]))
        a = torch.cat((a[:span], a[span:] * a[:-span]))
        span *= 2
    return s


def _plain_recurrence(state):
    case = state["case"]
    x = state["x"].detach()
    single = x.dim() == 2
    x, c0 = (x[None] if single else x).float(), state["c0"].detach()
    valid = _valid(state, x.shape[0], x.device)
    back = case["direction"] < 0

    def turned(t):
        return t.flip(0) if back else t

    z, i, f, o = turned(x).chunk(4, dim=-1)
    valid = turned(valid)
    z, i, f, o = torch.tanh(z), torch.sigmoid(i), torch.sigmoid(f), torch.sigmoid(o)
    a = torch.where(valid, f, 1.0)
    s = torch.where(valid, i * z, 0.0)
    s[0] += a[0] * c0
    c = _scan(a, s)
    y = turned(torch.where(valid, o * c, 0.0)).to(state["x"].dtype)
    out = (y[0] if single else y, c[-1])
    if not case["train"]:
        return out
    dy = turned(state["dy"].float())
    g = torch.where(valid, dy * o, 0.0)
    g[-1] += state["dc"]
    later = torch.cat((a[1:], torch.ones_like(a[:1])))  # what the error of frame t+1 is multiplied with
    g = _scan(later.flip(0), g.flip(0)).flip(0)
    before = torch.cat((c0[None], c[:-1]))
    dx = torch.cat((g * i * (1 - z * z), g * z * i * (1 - i), g * before * f * (1 - f), dy * c * o * (1 - o)), dim=-1)
    return out + (turned(torch.where(valid, dx, 0.0)).to(state["x"].dtype), a[0] * g[0])


_PHILOX_M = (0xD2511F53, 0xCD9E8D57)
_PHILOX_W = (0x9E3779B9, 0xBB67AE85)


def _plain_dropout(state):
    case = state["case"]
    x, residual, dy = state["x"].detach(), state["residual"], state["dy"]
    shape = x.shape[1:] if case["same_over_time"] else x.shape
    count = math.prod(shape)
    low = 0xFFFFFFFF
    group = torch.arange((count + 7) // 8, dtype=torch.int64, device=x.device)
    offset = state["offset"]
    c = [group & low, group >> 32, torch.full_like(group, offset & low), torch.full_like(group, offset >> 32 & low)]
    key = [state["seed"] & low, state["seed"] >> 32 & low]
    for _ in range(10):
        p0, p1 = c[0] * _PHILOX_M[0], c[2] * _PHILOX_M[1]  # (64 bits, of which the sign is one)
        c = [(p1 >> 32 & low) ^ c[1] ^ key[0], p1 & low, (p0 >> 32 & low) ^ c[3] ^ key[1], p0 & low]
        key = [(k + w) & low for k, w in zip(key, _PHILOX_W)]
    draws = torch.stack([w >> shift & 0xFFFF for w in c for shift in (0, 16)], dim=-1).reshape(-1)[:count].view(shape)
    threshold = int(round(case["drop_prob"] * 65536))
    keep, scale = draws >= threshold, 65536.0 / (65536 - threshold)
    y = torch.where(keep, x.float() * scale, 0.0)
    if residual is not None:
        y = y + residual.detach().float()
    dx = torch.where(keep, dy.float() * scale, 0.0).to(x.dtype)
    return (y.to(x.dtype), dx) if residual is None else (y.to(x.dtype), dx, dy)


def _plain_scores(state):
    case = state["case"]
    logits, targets = state["logits"].detach(), state["targets"]
    x = logits.float()
    m = x.amax(dim=-1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(dim=-1, keepdim=True)
    lse = m + torch.log(total)
    p = e / total
    allowed = x > -math.inf
    logp = x - lse
    entropy = -torch.where(allowed, p * logp, 0.0).sum(dim=-1)
    has = torch.ones(x.shape[:-1], dtype=torch.bool, device=x.device) if targets is None else targets >= 0
    out = [torch.where(has, entropy, 0.0)]
    if case["given"]:
        at = targets.clamp(min=0)[..., None]
        out.append(torch.where(has, logp.gather(-1, at)[..., 0], 0.0))
    if case["top_k"]:
        # whole numbers in the order of the logits, the lower index first among equal ones: no two of a row are alike
        bits = x.view(torch.int32).to(torch.int64)
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        best = torch.topk(order * 2**31 + (2**31 - 1 - torch.arange(x.shape[-1], device=x.device)), case["top_k"], dim=-1).values
        ids = 2**31 - 1 - best % 2**31
        out += [torch.where(has[..., None], logp.gather(-1, ids), -math.inf), torch.where(has[..., None], ids, -1)]
    if case["train"]:
        d_log_probs, d_entropy = state["d_log_probs"][..., None], state["d_entropy"][..., None]
        d = -p * (d_log_probs + d_entropy * torch.where(allowed, logp + entropy[..., None], 0.0))
        d.scatter_add_(-1, at, d_log_probs)
        out.append(torch.where(has[..., None], d, 0.0).to(logits.dtype))
    return out


def _run_plain(state):
    with torch.no_grad():
        return {"recurrence": _plain_recurrence, "dropout": _plain_dropout, "scores": _plain_scores}[state["case"]["kind"]](state)


# ---- the definitions in 64 bits ----
def _exact_recurrence(state):
    case = state["case"]
    x = state["x"].detach().double()
    single = x.dim() == 2
    if single:
        x = x[None]
    T, B, n = x.shape[0], case["B"], case["n"]
    lens = torch.full((B,), T, device=x.device) if state["lens"] is None else state["lens"]
    frames = list(range(T)) if case["direction"] > 0 else list(range(T - 1, -1, -1))
    c = state["c0"].detach().double()
    y = torch.zeros((T, B, n), dtype=torch.float64, device=x.device)
    states = []
    for t in frames:
        z, i, f, o = x[t].view(B, 4, n).unbind(1)
        inside = (t < lens)[:, None]
        states.append(c)
        c = torch.where(inside, torch.tanh(z) / (1 + torch.exp(-i)) + c / (1 + torch.exp(-f)), c)
        y[t] = torch.where(inside, c / (1 + torch.exp(-o)), 0.0)
    out = (y[0] if single else y, c)
    if not case["train"]:
        return out
    dx = torch.zeros_like(x)
    g = state["dc"].double()
    after = c
    for t in reversed(frames):
        z, i, f, o = x[t].view(B, 4, n).unbind(1)
        inside = (t < lens)[:, None]
        z, i, f, o = torch.tanh(z), 1 / (1 + torch.exp(-i)), 1 / (1 + torch.exp(-f)), 1 / (1 + torch.exp(-o))
        before, dy = states.pop(), state["dy"][t].double()
        total = g + dy * o
        parts = torch.stack((total * i / torch.cosh(x[t].view(B, 4, n)[:, 0]) ** 2, total * z * i * (1 - i), total * before * f * (1 - f), dy * after * o * (1 - o)), dim=1)
        dx[t] = torch.where(inside, parts.reshape(B, 4 * n), 0.0)
        g = torch.where(inside, total * f, g)
        after = before
    return out + (dx, g)


def _exact_dropout(state):
    case = state["case"]
    shape = state["x"].shape[1:] if case["same_over_time"] else state["x"].shape
    count = int(numpy.prod(shape))
    half = numpy.uint64(32)
    groups = numpy.arange((count + 7) // 8, dtype=numpy.uint64)
    c0, c1 = groups.astype(numpy.uint32), (groups >> half).astype(numpy.uint32)
    c2, c3 = (numpy.full_like(c0, state["offset"] >> s & 0xFFFFFFFF) for s in (0, 32))
    for r in range(10):
        k0, k1 = (numpy.uint32(((state["seed"] >> 32 * j) + r * w) & 0xFFFFFFFF) for j, w in enumerate((0x9E3779B9, 0xBB67AE85)))
        a = c0.astype(numpy.uint64) * numpy.uint64(0xD2511F53)
        b = c2.astype(numpy.uint64) * numpy.uint64(0xCD9E8D57)
        c0, c1, c2, c3 = (b >> half).astype(numpy.uint32) ^ c1 ^ k0, b.astype(numpy.uint32), (a >> half).astype(numpy.uint32) ^ c3 ^ k1, a.astype(numpy.uint32)
    draws = numpy.stack((c0, c1, c2, c3), axis=-1).astype("<u4").view("<u2").reshape(-1)[:count]
    dropped = int(round(case["drop_prob"] * 65536))
    factor = torch.from_numpy((draws >= dropped) * (65536.0 / (65536 - dropped))).view(shape).to(state["x"].device)
    y = state["x"].detach().double() * factor
    dx = state["dy"].double() * factor
    if state["residual"] is None:
        return y, dx
    return y + state["residual"].detach().double(), dx, state["dy"].double()


def _exact_scores(state):
    case = state["case"]
    rows = state["logits"].detach().reshape(-1, case["V"])
    lead = state["logits"].shape[:-1]
    targets = None if state["targets"] is None else state["targets"].reshape(-1).cpu().tolist()
    entropy, given, top, ids, grads = [], [], [], [], []
    for r in range(rows.shape[0]):
        x = rows[r].double()
        if targets is not None and targets[r] < 0:
            x = torch.zeros_like(x)
        logp = torch.log_softmax(x, dim=0)
        p = torch.exp(logp)
        h = torch.special.entr(p).sum()
        token = 0 if targets is None else targets[r]
        skip = token < 0
        entropy.append(0 * h if skip else h)
        if targets is not None:
            given.append(0 * h if skip else logp[token])
        if case["top_k"]:
            values, order = torch.sort(x, descending=True, stable=True)
            k = case["top_k"]
            top.append(torch.full_like(values[:k], -math.inf) if skip else logp[order[:k]])
            ids.append(torch.full_like(order[:k], -1) if skip else order[:k])
        if case["train"]:
            a, b = state["d_log_probs"].reshape(-1)[r].double(), state["d_entropy"].reshape(-1)[r].double()
            d = -a * p - b * (p * logp.clamp(min=-1e4) + p * h)
            d[token] += a
            grads.append(torch.zeros_like(d) if skip else d)
    out = [torch.stack(entropy).view(lead)]
    if targets is not None:
        out.append(torch.stack(given).view(lead))
    if case["top_k"]:
        out += [torch.stack(top).view(lead + (-1,)), torch.stack(ids).view(lead + (-1,))]
    if case["train"]:
        out.append(torch.stack(grads).view(state["logits"].shape))
    return out


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"recurrence": _exact_recurrence, "dropout": _exact_dropout, "scores": _exact_scores}[case["kind"]](state)


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    T, B = case["T"], case["B"]
    rows = T * B
    valid = sum(_lengths(T, B)) if case.get("ragged") else rows  # frames that belong to a sequence: no others need be read
    if case["kind"] == "recurrence":
        n = case["n"]
        # the gates of the valid frames and the state are read, the outputs and the new state written
        forward = e * (4.0 * valid * n + rows * n) + 8.0 * B * n
        if not case["train"]:
            return {"bytes": forward, "flops": 20.0 * valid * n}
        # the gates once more, the errors of outputs and state; the errors of all gates and of the state before
        return {"bytes": forward + e * (5.0 * valid * n + 4.0 * rows * n) + 12.0 * B * n, "flops": 60.0 * valid * n}
    if case["kind"] == "dropout":
        n = case["n"]
        # forward and gradient: one read and one write each, and the residual's read
        return {"bytes": float(e * rows * n * (5 if case["residual"] else 4)), "flops": (5.0 if case["residual"] else 4.0) * rows * n}
    V, k = case["V"], case["top_k"]
    forward = float(e * valid * V) + rows * (16.0 + 12.0 * k)
    if not case["train"]:
        return {"bytes": forward, "flops": 6.0 * valid * V}
    return {"bytes": forward + e * (valid * V + rows * V) + 16.0 * rows, "flops": 13.0 * valid * V}

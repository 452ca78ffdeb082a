"""What is measured of the training tail: the output head's softmax cross entropy
(`ops.linear_cross_entropy`, `ops.linear_cross_entropy_grad`) and the global
gradient norm with clipping (`ops.grad_norm`, `ops.clip_grads`).

A case's "op" is one of
  loss    hidden states [m, k] and the head's weight [v, k] in, the loss and
          each row's log-sum-exp out;
  train   the same and the gradients of the loss: dh [m, k] and dw [v, k];
  norm    the L2 norm over a list of gradients;
  clip    the norm, and the gradients scaled to at most `max_norm` of it.

`run` with `own` false computes the plain form (fp32 torch operations, sums of
squares in 64 bits, one rounding at the end); with `own` true it calls the
framework. `exact` evaluates the definitions in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
IGNORE = -100
F16_SCALE = 1024.0  # the loss scale of fp16 gradients
EPS = 1e-6  # added to the norm before dividing, as training loops do


# ---- cases -----------------------------------------------------------------------


def _loss(name, op, m, k, v, dtype, *, reduction="mean", ignored=0.0, scale=1.0):
    c = {"op": op, "m": m, "k": k, "v": v, "dtype": dtype, "reduction": reduction, "ignored": ignored,
         "scale": scale}
    return {"name": name, **c} if name else c


def _grads(name, op, hidden, inter, layers, vocab, dtype, *, mixed=False, max_norm=1.0):
    c = {"op": op, "hidden": hidden, "inter": inter, "layers": layers, "vocab": vocab, "dtype": dtype,
         "mixed": mixed, "max_norm": max_norm}
    return {"name": name, **c} if name else c


def listed():
    return [
        # scoring one token of a generation against the whole vocabulary: the weight is read once
        _loss("loss_token_bf16", "loss", 1, 4096, 128256, "bf16", reduction="none"),
        # a small model with an odd vocabulary and a ragged batch with padding: launch latency counts
        _loss("loss_small_f16", "loss", 37, 512, 32001, "f16", ignored=0.2),
        # evaluation of a 2048-token sequence (perplexity)
        _loss("loss_eval_bf16", "loss", 2048, 4096, 128256, "bf16"),
        # fine-tuning on short sequences: few rows, so reading and writing the weight bounds it
        _loss("train_short_bf16", "train", 64, 2048, 32000, "bf16", reduction="sum"),
        # a mid-sized model in fp16 with loss scaling, an odd vocabulary and padded rows
        _loss("train_odd_f16", "train", 1001, 1024, 50257, "f16", ignored=0.1, scale=8192.0),
        # a training step's output head: 4096 tokens, hidden 4096, the 128256-word vocabulary
        _loss("train_step_bf16", "train", 4096, 4096, 128256, "bf16", ignored=0.02),
        # one small block in fp32: launch latency
        _grads("norm_block_f32", "norm", 256, 688, 1, 0, "f32"),
        # a pipeline stage of four layers, 4096 x 14336 (0.87e9 gradients)
        _grads("norm_stage_bf16", "norm", 4096, 14336, 4, 0, "bf16"),
        # a small block clipped every step
        _grads("clip_block_bf16", "clip", 512, 1376, 1, 0, "bf16", max_norm=0.5),
        # odd sizes, an odd vocabulary, fp32 norm weights beside 16-bit matrices
        _grads("clip_odd_mixed", "clip", 515, 1387, 6, 32001, "bf16", mixed=True),
        # many tensors: 24 layers and an embedding, 217 tensors
        _grads("clip_many_f16", "clip", 1024, 4096, 24, 32000, "f16", max_norm=F16_SCALE),
        # the pipeline stage again, clipped
        _grads("clip_stage_bf16", "clip", 4096, 14336, 4, 0, "bf16"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["loss", "loss", "train", "train", "norm", "clip", "clip"])
    if op in ("loss", "train"):
        while True:
            m, k, v = _log_uniform(rng, 1, 4096), 8 * _log_uniform(rng, 8, 512), _log_uniform(rng, 500, 131072)
            if m * k * v <= 4096 * 4096 * 128256:
                break
        dtype = rng.choice(["bf16", "f16"])
        return _loss(None, op, m, k, v, dtype, reduction=rng.choice(["none", "sum", "mean"]),
                     ignored=rng.choice([0.0, 0.1, 0.5]) if m > 1 else 0.0,
                     scale=F16_SCALE if dtype == "f16" else 1.0)
    while True:
        hidden, layers = _log_uniform(rng, 64, 4096), _log_uniform(rng, 1, 32)
        inter, vocab = int(hidden * rng.uniform(2, 4)), rng.choice([0, _log_uniform(rng, 500, 131072)])
        dtype = rng.choice(["bf16", "f16", "f32"])
        c = _grads(None, op, hidden, inter, layers, vocab, dtype, mixed=rng.choice([True, False]),
                   max_norm=rng.choice([0.1, 1.0, 1e6]) * (F16_SCALE if dtype == "f16" else 1.0))
        if sum(n * b for n, b in _sizes(c)) <= 1_750_000_000:
            return c


# ---- inputs ----------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _head_inputs(case, seed):
    """Hidden states as a final norm leaves them (unit variance), a head weight
    whose logits have a spread of about 1.3, and targets that are from
    unlikely to almost certain: each row is moved along its target's weight.
    A share `ignored` of the rows carries the ignored index (the prompt's
    tokens and the padding of a batch)."""
    g = _gen(seed)
    m, k, v, dt = case["m"], case["k"], case["v"], DTYPES[case["dtype"]]
    h = torch.randn(m, k, device="cuda", generator=g)
    w = torch.empty(v, k, device="cuda", dtype=dt)
    for i in range(0, v, 16384):
        n = min(16384, v - i)
        w[i:i + n] = (torch.randn(n, k, device="cuda", generator=g) * (1.3 / math.sqrt(k))).to(dt)
    targets = torch.randint(0, v, (m,), device="cuda", generator=g)
    wt = w[targets].float()
    pull = 12.0 * torch.rand(m, 1, device="cuda", generator=g)
    h = (h + pull * wt / wt.norm(dim=1, keepdim=True)).to(dt)
    if case["ignored"]:
        drop = torch.rand(m, device="cuda", generator=g) < case["ignored"]
        drop[0] = False
        targets = torch.where(drop, torch.full_like(targets, IGNORE), targets)
    if case["reduction"] == "none":
        dloss = case["scale"] * (0.5 + torch.rand(m, device="cuda", generator=g))
    else:
        dloss = torch.full((1,), case["scale"], device="cuda")
    return h, w, targets, dloss


def _sizes(case):
    """(elements, bytes each) of the gradients of a stack of layers: the four
    attention matrices (a quarter as many key and value heads), the three of
    the gated MLP, two norm weights, and the embedding if there is one."""
    e = 4 if case["dtype"] == "f32" else 2
    en = 4 if case["mixed"] else e
    hd, it, kv = case["hidden"], case["inter"], max(1, case["hidden"] // 4)
    one = [(hd * hd, e), (kv * hd, e), (kv * hd, e), (hd * hd, e), (it * hd, e), (it * hd, e), (hd * it, e),
           (hd, en), (hd, en)]
    return one * case["layers"] + ([(case["vocab"] * hd, e)] if case["vocab"] else [])


def _shapes(case):
    hd, it, kv = case["hidden"], case["inter"], max(1, case["hidden"] // 4)
    dt = DTYPES[case["dtype"]]
    dn = torch.float32 if case["mixed"] else dt
    one = [((hd, hd), dt), ((kv, hd), dt), ((kv, hd), dt), ((hd, hd), dt), ((it, hd), dt), ((it, hd), dt),
           ((hd, it), dt), ((hd,), dn), ((hd,), dn)]
    return one * case["layers"] + ([((case["vocab"], hd), dt)] if case["vocab"] else [])


def _grad_inputs(case, seed):
    """Gradients with another magnitude for each tensor (3e-4 to 3e-3), times
    the loss scale that fp16 training carries."""
    g = _gen(seed)
    out = []
    for i, (shape, dt) in enumerate(_shapes(case)):
        mag = 3e-4 * 10 ** ((i * 7 % 11) / 11) * (F16_SCALE if case["dtype"] == "f16" else 1.0)
        out.append(torch.randn(shape, device="cuda", generator=g, dtype=dt).mul_(mag))
    return out


def _flat(case, dtype=None):
    """One zero-filled buffer for each type of the case's gradients, with a view
    of it for each tensor at a 256-byte boundary: the buckets in which training
    loops hold the gradients that they reduce and clip together."""
    bufs, views, at = {}, [], {}
    spans = []
    for shape, dt in _shapes(case):
        n = math.prod(shape)
        spans.append((dt, at.get(dt, 0), n, shape))
        at[dt] = at.get(dt, 0) + (n + 127) // 128 * 128
    for dt, n in at.items():
        bufs[str(dt).removeprefix("torch.")] = torch.zeros(n, dtype=dtype or dt, device="cuda")
    for dt, start, n, shape in spans:
        views.append(bufs[str(dt).removeprefix("torch.")][start:start + n].view(shape))
    return bufs, views


def prepare(case, seed):
    if case["op"] in ("loss", "train"):
        h, w, targets, dloss = _head_inputs(case, seed)
        return {"case": case, "h": h, "w": w, "targets": targets, "dloss": dloss}
    grads = _grad_inputs(case, seed)
    state = {"case": case, "grads": grads, "flat": None, "out": None}
    if case["op"] == "clip":
        # clipped into buffers of their own, so that a pass can be repeated on the same gradients
        state["flat"], state["out"] = _flat(case)
    if own:
        from enzyme_b200 import ops

        state["list"] = ops.GradList(grads, out=state["out"])  # a training loop keeps it with its buffers
    return state


# ---- one pass --------------------------------------------------------------------


def _reduce(loss, valid, reduction):
    if reduction == "none":
        return loss
    return loss.sum() if reduction == "sum" else loss.sum() / valid.sum()


def _row_grad(dloss, valid, reduction):
    if reduction == "mean":
        dloss = dloss / valid.sum()
    return torch.where(valid, dloss.expand(valid.shape), torch.zeros((), dtype=dloss.dtype, device=dloss.device))


def _plain_head(s):
    case, h, w, targets = s["case"], s["h"], s["w"], s["targets"]
    hf, wf = h.float(), w.float()
    logits = hf @ wf.T
    valid = targets != IGNORE
    rows = torch.arange(case["m"], device=h.device)
    t = torch.where(valid, targets, torch.zeros_like(targets))
    at = logits[rows, t]
    # the sum over the other words, and the target's logit beside it in 64
    # bits: an almost certain target's loss is far below the log-sum-exp
    logits[rows, t] = torch.where(valid, -math.inf, at)
    top = logits.max(dim=1, keepdim=True).values
    rest = top.squeeze(1).double() + torch.log(torch.exp(logits - top).sum(dim=1)).double()
    each = torch.where(valid, torch.logaddexp(rest - at, torch.zeros_like(rest)), 0.0)
    lse = torch.where(valid, at + each, rest).float()
    each = each.float()
    out = {"loss": _reduce(each, valid, case["reduction"]), "lse": lse}
    if case["op"] == "train":
        g = _row_grad(s["dloss"], valid, case["reduction"])
        d = torch.exp(logits - lse[:, None])
        d[rows, t] = torch.where(valid, torch.expm1(-each), d[rows, t])
        d *= g[:, None]
        out["dh"] = (d @ wf).to(h.dtype)
        out["dw"] = (d.T @ hf).to(w.dtype)
    return out


def _own_head(s):
    from enzyme_b200 import ops

    case = s["case"]
    loss, stats = ops.linear_cross_entropy(s["h"], s["w"], s["targets"], ignore_index=IGNORE,
                                           reduction=case["reduction"])
    out = {"loss": loss, "lse": stats[0]}
    if case["op"] == "train":
        out["dh"], out["dw"] = ops.linear_cross_entropy_grad(
            s["h"], s["w"], s["targets"], stats, s["dloss"], ignore_index=IGNORE, reduction=case["reduction"])
    return out


def _plain_grads(s):
    case, grads = s["case"], s["grads"]
    total = torch.zeros((), dtype=torch.float64, device=grads[0].device)
    for t in grads:
        f = t.float()
        total += (f * f).sum(dtype=torch.float64)
    norm = total.sqrt().float()
    if case["op"] == "norm":
        return {"norm": norm}
    scale = torch.clamp(case["max_norm"] / (norm + EPS), max=1.0)
    for t, o in zip(grads, s["out"]):
        o.copy_(t.float() * scale)
    return {"norm": norm, **s["flat"]}


def _own_grads(s):
    from enzyme_b200 import ops

    if s["case"]["op"] == "norm":
        return {"norm": ops.grad_norm(s["list"])}
    _, norm = ops.clip_grads(s["list"], s["case"]["max_norm"], eps=EPS)
    return {"norm": norm, **s["flat"]}


def run(state):
    if state["case"]["op"] in ("loss", "train"):
        return _own_head(state) if own else _plain_head(state)
    return _own_grads(state) if own else _plain_grads(state)


# ---- what a pass cannot do without -------------------------------------------------


def work(case):
    if case["op"] in ("loss", "train"):
        m, k, v = case["m"], case["k"], case["v"]
        flops = 2.0 * m * k * v
        nbytes = 2 * (m * k + v * k) + 8 * m + 4 * m + (4 * m if case["reduction"] == "none" else 4)
        if case["op"] == "train":
            flops *= 3
            nbytes += 2 * (m * k + v * k)
        return {"bytes": nbytes, "flops": flops}
    n = sum(c for c, _ in _sizes(case))
    nbytes = sum(c * b for c, b in _sizes(case))
    if case["op"] == "norm":
        return {"bytes": nbytes + 4, "flops": 2.0 * n}
    return {"bytes": 2 * nbytes + 4, "flops": 3.0 * n}


# ---- the definition in 64 bits -----------------------------------------------------


def exact(case, seed):
    if case["op"] in ("loss", "train"):
        h, w, targets, dloss = _head_inputs(case, seed)
        h, m = h.double(), case["m"]
        keep = targets >= 0
        at = targets.clamp(min=0)
        # a first walk over the vocabulary for the log-sum-exp, a second one for the gradient
        step = 16384
        rest = torch.full((m,), -math.inf, dtype=torch.float64, device=h.device)
        own_logit = (h * w[at].double()).sum(dim=1)
        for i in range(0, case["v"], step):
            z = h @ w[i:i + step].double().T
            z[(at[:, None] == torch.arange(i, i + z.shape[1], device=h.device)) & keep[:, None]] = -math.inf
            rest = torch.logaddexp(rest, torch.logsumexp(z, dim=1))
        lse = torch.where(keep, torch.logaddexp(rest, own_logit), rest)
        loss = torch.where(keep, torch.logaddexp(rest - own_logit, torch.zeros_like(rest)), 0.0)
        count = keep.double().sum()
        total = {"none": loss, "sum": loss.sum(), "mean": loss.sum() / count}[case["reduction"]]
        out = {"loss": total, "lse": lse}
        if case["op"] == "train":
            g = dloss.double().expand(m) / (count if case["reduction"] == "mean" else 1.0)
            g = torch.where(keep, g, 0.0)
            dh = torch.zeros_like(h)
            dw = torch.empty(case["v"], case["k"], dtype=torch.float64, device=h.device)
            for i in range(0, case["v"], step):
                wi = w[i:i + step].double()
                hot = at[:, None] == torch.arange(i, i + wi.shape[0], device=h.device)
                d = torch.exp(h @ wi.T - lse[:, None])
                d = g[:, None] * torch.where(hot, torch.expm1(-loss)[:, None], d)
                dh += d @ wi
                dw[i:i + step] = d.T @ h
            out["dh"], out["dw"] = dh, dw
        return out
    grads = _grad_inputs(case, seed)
    norm = torch.stack([torch.linalg.vector_norm(t.double()) for t in grads]).square().sum().sqrt()
    if case["op"] == "norm":
        return {"norm": norm}
    scale = min(1.0, case["max_norm"] / (float(norm) + EPS))
    flat, views = _flat(case, torch.float64)
    for t, o in zip(grads, views):
        o.copy_(t.double() * scale)
    return {"norm": norm, **flat}

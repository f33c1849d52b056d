"""Timed cases of the vocabulary operators: log probabilities of given tokens, and distillation from top logits.

Both work on a matrix of logits ``[rows, vocabulary]`` in float32, bfloat16 or float16, whose rows may be longer in
memory than the vocabulary (``pad``):

``score``        log probability of one given token a row, the row's entropy, and its ``top`` most likely tokens
``score_grad``   gradient of those outputs with respect to the logits
``distill``      Kullback-Leibler divergence from a teacher known by its ``top`` largest logits, with the gradient
                 where ``grad`` is set
``distill_grad`` that gradient alone, from the statistics which an earlier forward call saved

``own`` selects the framework's kernels; otherwise ``run`` evaluates the formulas with elementary torch operations.
"""
import math

import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_IGNORE = -100


def _case(name, op, rows, vocab, dtype, **more):
    case = {"name": name, "op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "pad": 0, "top": 0,
            "entropy": False, "temperature": 1.0, "ignored": 0.0, "masked": 0.0, "ragged": False, "grad": False,
            "reduction": "mean"}
    case.update(more)
    return case


def listed():
    return [
        # one token of one sequence is scored while it is generated: latency
        _case("score-1x32000-f32", "score", 1, 32000, "float32", entropy=True),
        # a decoding batch that reports the twenty most likely alternatives of each new token
        _case("score-16x128256-bf16-top20", "score", 16, 128256, "bfloat16", top=20, temperature=0.8),
        # scoring of short answers, the vocabulary padded in memory, under a grammar that bans half of the tokens
        _case("score-509x50257-f16-top5", "score", 509, 50257, "float16", pad=47, top=5, masked=0.5, entropy=True),
        # per-token terms of a policy loss over a padded batch of rollouts
        _case("score-8192x50257-f32", "score", 8192, 50257, "float32", entropy=True, temperature=0.7, ignored=0.2),
        # perplexity of long documents
        _case("score-4096x128256-bf16", "score", 4096, 128256, "bfloat16", entropy=True),
        # a teacher's pass over a training batch that keeps its 64 largest logits
        _case("score-2048x151936-f32-top64", "score", 2048, 151936, "float32", top=64),
        # backward pass of the policy loss: gradients of the log probability and of the entropy bonus
        _case("score-grad-4096x128256-bf16", "score_grad", 4096, 128256, "bfloat16", entropy=True, ignored=0.1),
        # backward pass through reported alternatives as well
        _case("score-grad-601x32003-f32-top16", "score_grad", 601, 32003, "float32", top=16, temperature=1.3),
        # a classifier distilled on a small batch: latency
        _case("distill-8x1000-f32-top5", "distill", 8, 1000, "float32", top=5, temperature=2.0, grad=True),
        # a training step's loss and gradient
        _case("distill-4096x128256-bf16-top64", "distill", 4096, 128256, "bfloat16", top=64, grad=True),
        # the same where the teacher kept as many logits as it needed, on an odd vocabulary
        _case("distill-1021x50257-f32-top100", "distill", 1021, 50257, "float32", top=100, temperature=2.0, ragged=True,
              ignored=0.1, grad=True, reduction="none"),
        # the backward pass by itself, as the tape of a model runs it
        _case("distill-grad-2048x151936-f16-top32", "distill_grad", 2048, 151936, "float16", top=32, reduction="sum"),
    ]


def draw(rng):
    op = rng.choice(["score", "score", "score_grad", "distill", "distill", "distill_grad"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    vocab = int(round(math.exp(rng.uniform(math.log(1000), math.log(200000)))))
    most = min(8192, (260 if dtype == "float32" else 400) * 1000 * 1000 // vocab)
    rows = int(round(math.exp(rng.uniform(0.0, math.log(most)))))
    more = {"pad": rng.choice([0, 0, rng.randrange(1, 64), (-vocab) % 64]),
            "temperature": rng.choice([1.0, 1.0, round(rng.uniform(0.5, 3.0), 2)]),
            "ignored": rng.choice([0.0, 0.0, round(rng.uniform(0.05, 0.5), 2)])}
    if op in ("score", "score_grad"):
        more["top"] = rng.choice([0, rng.randrange(1, 21), rng.randrange(21, 129)])
        more["entropy"] = rng.random() < 0.5
        more["masked"] = rng.choice([0.0, 0.0, round(rng.uniform(0.1, 0.9), 2)])
    else:
        more["top"] = rng.randrange(1, 129)
        more["ragged"] = rng.random() < 0.5
        more["grad"] = rng.random() < 0.7
        more["reduction"] = rng.choice(["mean", "sum", "none"])
    return _case(None, op, rows, vocab, dtype, **more)


# ---------------------------------------------------------------------- inputs
def _inputs(case, seed):
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev).manual_seed(seed * 7919 + 17)
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    dtype = _TYPES[case["dtype"]]
    scores = case["op"] in ("score", "score_grad")
    wide = torch.randn(rows, vocab + case["pad"], generator=gen, device=dev)
    wide.mul_(2.5)                                            # spread of a language model's logits
    every = torch.arange(rows, device=dev)
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device=dev)
    # the wanted token is usually a likely one
    wide[every, tokens] += 12.0 * torch.rand(rows, generator=gen, device=dev)
    if case["masked"]:
        banned = torch.rand(rows, vocab, generator=gen, device=dev) < case["masked"]
        banned[every, tokens] = False
        wide[:, :vocab].masked_fill_(banned, -math.inf)
        del banned
    left_out = torch.randperm(rows, generator=gen, device=dev)[:int(rows * case["ignored"])]
    s = {"logits": wide.to(dtype)[:, :vocab]}
    if scores:
        s["tokens"] = tokens.index_fill(0, left_out, _IGNORE)
        if case["op"] == "score_grad":
            s["d_log_probs"] = torch.randn(rows, generator=gen, device=dev)
            if case["entropy"]:
                s["d_entropy"] = 0.01 + 0.01 * torch.rand(rows, generator=gen, device=dev)
            if top:
                s["d_top"] = torch.randn(rows, top, generator=gen, device=dev)
    else:
        noise = torch.randn(rows, vocab, generator=gen, device=dev)
        values, index = torch.topk(wide[:, :vocab] + noise, top, dim=1)
        del noise
        if case["ragged"]:                                    # later entries missing, by row
            kept = torch.randint(1, top + 1, (rows, 1), generator=gen, device=dev)
            index[torch.arange(top, device=dev) >= kept] = -1
        index[left_out] = -1
        s["teacher_indices"], s["teacher_logits"] = index.to(torch.int32), values
        if case["op"] == "distill_grad" or case["reduction"] == "none":
            s["upstream_rows"] = 0.5 + torch.rand(rows, generator=gen, device=dev)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        from minitensor_b200.backend import get_backend
        s["backend"] = be = get_backend(0)
        if case["op"] == "score_grad":
            s["saved"] = be.token_log_probs(s["logits"], s["tokens"], temperature=case["temperature"], top=case["top"],
                                            entropy=case["entropy"], ignore_index=_IGNORE)
        elif case["op"] == "distill_grad":
            s["saved"] = torch.empty(case["rows"], 2, dtype=torch.float32, device=s["logits"].device)
            be.distillation_loss(s["logits"], s["teacher_indices"], s["teacher_logits"], reduction=case["reduction"],
                                 temperature=case["temperature"], want_grad=False, stats=s["saved"])
    elif case["op"] == "score_grad":
        s["saved"] = _plain_score(s)
    return s


def run(state):
    return _run_own(state) if "backend" in state else _run_plain(state)


# ---------------------------------------------------------------------- the framework's calls
def _run_own(s):
    case, be = s["case"], s["backend"]
    if case["op"] == "score":
        out = be.token_log_probs(s["logits"], s["tokens"], temperature=case["temperature"], top=case["top"],
                                 entropy=case["entropy"], ignore_index=_IGNORE)
        return [out.log_probs, out.entropy, out.top_log_probs, out.top_indices]
    if case["op"] == "score_grad":
        saved = s["saved"]
        return be.token_log_probs_bwd(s["logits"], s["tokens"], saved.stats, d_log_probs=s["d_log_probs"],
                                      entropy=saved.entropy, d_entropy=s.get("d_entropy"),
                                      top_indices=saved.top_indices, d_top=s.get("d_top"),
                                      temperature=case["temperature"], ignore_index=_IGNORE)
    if case["op"] == "distill":
        loss, grad = be.distillation_loss(s["logits"], s["teacher_indices"], s["teacher_logits"],
                                          temperature=case["temperature"], reduction=case["reduction"],
                                          upstream_rows=s.get("upstream_rows"), want_grad=case["grad"])
        return [loss, grad]
    return be.distillation_loss_bwd(s["logits"], s["teacher_indices"], s["teacher_logits"], s["saved"],
                                    temperature=case["temperature"], reduction=case["reduction"],
                                    upstream_rows=s["upstream_rows"])


# ---------------------------------------------------------------------- plain form
def _log_softmax(logits, temperature):
    """Logarithm of the softmax in 32 bits; a row whose logits are all -inf has -inf everywhere."""
    z = logits.float() / temperature
    peak = z.amax(dim=1, keepdim=True)
    peak = torch.where(peak == -math.inf, torch.zeros_like(peak), peak)
    z = z - peak
    total = z.exp().sum(dim=1, keepdim=True)
    return torch.where(total == 0, torch.full_like(z[:, :1], -math.inf), z - total.log())


def _plain_score(s):
    case = s["case"]
    logits, tokens = s["logits"], s["tokens"]
    lp = _log_softmax(logits, case["temperature"])
    live = tokens != _IGNORE
    log_probs = torch.where(live, lp.gather(1, tokens.clamp(min=0)[:, None])[:, 0], torch.zeros_like(lp[:, 0]))
    entropy = top_lp = top_idx = None
    if case["entropy"]:
        p = lp.exp()
        entropy = -torch.where(p == 0, p, p * lp).sum(dim=1)
        del p
        entropy = torch.where(live, entropy, torch.zeros_like(entropy))
    if case["top"]:
        # value in the high half of a 64-bit key, complement of the index in the low half: ties go to the lowest index
        bits = (logits.float() + 0.0).view(torch.int32).long()
        bits = torch.where(bits < 0, -2147483648 - bits, bits)
        key = bits * 4294967296 + (4294967295 - torch.arange(logits.shape[1], device=logits.device))
        best = torch.topk(key, case["top"], dim=1).values
        idx = 4294967295 - (best & 4294967295)
        top_lp = torch.where(live[:, None], lp.gather(1, idx), torch.full_like(lp[:, :1], -math.inf))
        top_idx = torch.where(live[:, None], idx, torch.full_like(idx[:, :1], -1)).to(torch.int32)
    return [log_probs, entropy, top_lp, top_idx]


def _teacher(s):
    """The teacher's distribution over the entries it kept (zero where an entry is missing) and its logarithm."""
    index = s["teacher_indices"].long()
    z = s["teacher_logits"].float() / s["case"]["temperature"]
    lq = _log_softmax(torch.where(index < 0, torch.full_like(z, -math.inf), z), 1.0)
    return index, lq.exp(), lq


def _run_plain(s):
    case = s["case"]
    logits, temperature = s["logits"], case["temperature"]
    if case["op"] == "score":
        return _plain_score(s)
    lp = _log_softmax(logits, temperature)
    if case["op"] == "score_grad":
        _, entropy, _, top_idx = s["saved"]
        live = s["tokens"] != _IGNORE
        up = torch.where(live, s["d_log_probs"], torch.zeros_like(s["d_log_probs"]))
        mass = up
        p = lp.exp()
        grad = torch.zeros_like(lp)
        if case["top"]:
            d_top = torch.where(live[:, None], s["d_top"], torch.zeros_like(s["d_top"]))
            grad.scatter_add_(1, top_idx.long().clamp(min=0), d_top)
            mass = mass + d_top.sum(dim=1)
        grad.scatter_add_(1, s["tokens"].clamp(min=0)[:, None], up[:, None])
        grad -= p * mass[:, None]
        if case["entropy"]:
            slope = torch.where(p == 0, p, p * (lp + entropy[:, None]))
            grad -= slope * torch.where(live, s["d_entropy"], torch.zeros_like(s["d_entropy"]))[:, None]
        return (grad / temperature).to(logits.dtype)
    index, q, lq = _teacher(s)
    rows = logits.shape[0]
    share = 1.0 / rows if case["reduction"] == "mean" else 1.0
    terms = torch.where(q == 0, q, q * (lq - lp.gather(1, index.clamp(min=0))))
    loss = terms.sum(dim=1) * temperature ** 2
    if case["reduction"] != "none":
        loss = (loss.double().sum() * share).float().reshape(1)
    if case["op"] == "distill" and not case["grad"]:
        return [loss, None]
    grad = lp.exp() * q.sum(dim=1, keepdim=True)
    grad.scatter_add_(1, index.clamp(min=0), -q)
    scale = share * temperature
    if "upstream_rows" in s:
        grad *= s["upstream_rows"][:, None] * scale
    else:
        grad *= scale
    grad = grad.to(logits.dtype)
    return grad if case["op"] == "distill_grad" else [loss, grad]


# ---------------------------------------------------------------------- 64-bit values
def exact(case, seed):
    """Outputs of ``run`` from the definitions in 64 bits, a few rows at a time."""
    s = _inputs(case, seed)
    rows, vocab = case["rows"], case["vocab"]
    step = max(1, 50_000_000 // vocab)
    scores = case["op"] in ("score", "score_grad")
    part = _exact_score if scores else _exact_distill
    pieces = [part(case, {k: v[i:i + step] for k, v in s.items()}) for i in range(0, rows, step)]
    joined = [None if p[0] is None else torch.cat(p) for p in zip(*pieces)]
    if case["op"] == "score":
        return joined[:4]
    if case["op"] == "score_grad":
        return joined[4]
    loss, grad = joined
    if case["reduction"] == "mean":
        loss, grad = loss.mean().reshape(1), (None if grad is None else grad.div_(rows))
    elif case["reduction"] == "sum":
        loss = loss.sum().reshape(1)
    return grad if case["op"] == "distill_grad" else [loss, grad]


def _exact_probs(case, logits):
    x = logits.double() / case["temperature"]
    weight = torch.exp(x - x.max(dim=1, keepdim=True).values)
    total = weight.sum(dim=1, keepdim=True)
    return weight / total, x - x.max(dim=1, keepdim=True).values - torch.log(total)


def _exact_score(case, s):
    p, lp = _exact_probs(case, s["logits"])
    n = p.shape[0]
    every = torch.arange(n, device=p.device)
    dead = s["tokens"] == _IGNORE
    tokens = s["tokens"].masked_fill(dead, 0)
    log_probs = lp[every, tokens].masked_fill(dead, 0.0)
    entropy = top_lp = top_idx = grad = None
    h = -torch.special.xlogy(p, p).sum(dim=1)
    if case["entropy"]:
        entropy = h.masked_fill(dead, 0.0)
    if case["top"]:
        order = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True).indices[:, :case["top"]]
        top_lp = lp.gather(1, order).masked_fill(dead[:, None], -math.inf)
        top_idx = order.to(torch.int32).masked_fill(dead[:, None], -1)
    if case["op"] == "score_grad":
        # derivative of each output by the row's logits: one-hot minus p, and -p (log p + entropy)
        grad = -p * s["d_log_probs"].double()[:, None]
        grad[every, tokens] += s["d_log_probs"].double()
        if case["top"]:
            d_top = s["d_top"].double()
            grad -= p * d_top.sum(dim=1, keepdim=True)
            for j in range(case["top"]):
                grad[every, order[:, j]] += d_top[:, j]
        if case["entropy"]:
            grad -= s["d_entropy"].double()[:, None] * (torch.special.xlogy(p, p) + p * h[:, None])
        grad = (grad / case["temperature"]).masked_fill(dead[:, None], 0.0)
    return log_probs, entropy, top_lp, top_idx, grad


def _exact_distill(case, s):
    t = case["temperature"]
    p, lp = _exact_probs(case, s["logits"])
    index = s["teacher_indices"].long()
    there = index >= 0
    v = s["teacher_logits"].double() / t
    v = torch.exp(v - v.max(dim=1, keepdim=True).values) * there
    mass = v.sum(dim=1, keepdim=True)
    q = v / torch.where(mass > 0, mass, torch.ones_like(mass))
    at = index.masked_fill(~there, 0)
    cross = (q * lp.gather(1, at)).sum(dim=1)
    loss = t * t * (torch.special.xlogy(q, q).sum(dim=1) - cross)
    if case["op"] == "distill" and not case["grad"]:
        return loss, None
    grad = p * (mass > 0)
    every = torch.arange(p.shape[0], device=p.device)
    for j in range(index.shape[1]):
        grad[every, at[:, j]] -= q[:, j]
    grad *= t
    if "upstream_rows" in s:
        grad *= s["upstream_rows"].double()[:, None]
    return loss, grad


# ---------------------------------------------------------------------- work
def work(case):
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    size = 4 if case["dtype"] == "float32" else 2
    live = rows - int(rows * case["ignored"])
    logits = live * vocab * size                              # rows that are left out need no look at their logits
    grads = rows * vocab * size
    if case["op"] == "score":
        moved = logits + rows * (8 + 4 + 4 * case["entropy"] + 8 * top)
        flops = live * vocab * (4 + 2 * case["entropy"])
    elif case["op"] == "score_grad":
        moved = logits + grads + rows * (8 + 4 + 8 + 8 * case["entropy"] + 8 * top)
        flops = live * vocab * (4 + 4 * case["entropy"])
    elif case["op"] == "distill":
        moved = logits + (grads if case["grad"] else 0) + rows * (8 * top + (8 if case["reduction"] == "none" else 0))
        flops = live * vocab * (8 if case["grad"] else 4)
    else:
        moved = logits + grads + rows * (8 * top + 12)
        flops = live * vocab * 4
    return {"bytes": moved, "flops": flops}

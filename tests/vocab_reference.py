"""64-bit definitions of the vocabulary operators, for their tests (CPU or GPU tensors)."""
import math

import torch

U = 2.0 ** -24  # half a unit in the last place of an f32, relative


def softmax64(logits, temperature):
    """(p, log p) of ``logits / temperature``; rows of -inf alone have p = 0."""
    x = logits.double() / temperature
    m = x.max(dim=1, keepdim=True).values
    empty = (logits == -math.inf).all(dim=1, keepdim=True)
    d = x - torch.where(empty, torch.zeros_like(m), m)
    lp = d - torch.exp(d).sum(dim=1, keepdim=True).log()
    lp = torch.where(empty, torch.full_like(lp, -math.inf), lp)
    return lp.exp(), lp


def entropy64(p, lp):
    return -torch.where(p == 0, torch.zeros_like(p), p * lp).sum(dim=1)


def order64(logits, top):
    """Indices of the ``top`` largest logits: ties to the lower index, -0 = +0, NaN with -inf."""
    x = logits.double() + 0.0
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    return torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]


def score_grad64(logits, tokens, temperature, d_log_probs=None, d_entropy=None, top_indices=None, d_top=None,
                 ignore_index=None):
    p, lp = softmax64(logits, temperature)
    rows, vocab = logits.shape
    every = torch.arange(rows, device=logits.device)
    g = torch.zeros_like(p)
    live = torch.ones(rows, dtype=torch.bool, device=logits.device)
    if tokens is not None and ignore_index is not None:
        live = tokens != ignore_index
    if d_log_probs is not None:
        g -= p * d_log_probs.double()[:, None]
        g[every, tokens.long().clamp(min=0)] += d_log_probs.double()
    if d_top is not None:
        for k in range(d_top.shape[1]):
            j = top_indices[:, k].long()
            w = torch.where(j >= 0, d_top[:, k].double(), torch.zeros_like(d_top[:, k].double()))
            g -= p * w[:, None]
            g[every, j.clamp(min=0)] += w
    if d_entropy is not None:
        slope = torch.where(p == 0, torch.zeros_like(p), p * (lp + entropy64(p, lp)[:, None]))
        g -= slope * d_entropy.double()[:, None]
    return torch.where(live[:, None], g / temperature, torch.zeros_like(g))


def teacher64(indices, values, temperature):
    there = indices >= 0
    v = torch.where(there, values.double() / temperature, torch.full_like(values, -math.inf, dtype=torch.float64))
    m = v.max(dim=1, keepdim=True).values if v.shape[1] else torch.full((v.shape[0], 1), -math.inf, dtype=torch.float64, device=v.device)
    none = m == -math.inf
    e = torch.exp(v - torch.where(none, torch.zeros_like(m), m))
    s = e.sum(dim=1, keepdim=True)
    return torch.where(none, torch.zeros_like(e), e / torch.where(none, torch.ones_like(s), s))


def distill64(logits, indices, values, temperature):
    """(row losses, gradient of their plain sum)."""
    p, lp = softmax64(logits, temperature)
    q = teacher64(indices, values, temperature)
    at = indices.long().clamp(min=0)
    lq = torch.where(q > 0, q, torch.ones_like(q)).log()
    terms = torch.where(q > 0, q * (lq - lp.gather(1, at)), torch.zeros_like(q))
    g = p * (q.sum(dim=1, keepdim=True) > 0)
    every = torch.arange(p.shape[0], device=p.device)
    for k in range(indices.shape[1]):
        g[every, at[:, k]] -= q[:, k]
    return terms.sum(dim=1) * temperature ** 2, g * temperature


def sum_error(vocab):
    """Bound on the relative error of S = sum 2^(c d): every term carries the rounding of d, c and their product (3 U |d| / T,
    whose mean under p is at most ln(vocab) plus the entropy's deficit, 3 U ln(vocab) in all up to a factor of 2) and the
    2^-22 of the power of two; a thread adds a chain of vocab / 128 terms at most, blocks and clusters 16 more levels,
    each with a factor that has its own 2^-22."""
    return U * (6 * math.log(vocab + 1) + 4 + vocab / 128 + 1 + 16 * 6)


def log_prob_tolerance(lp, vocab):
    """lp = d / T - ln S: three roundings of d / T, where |d / T| <= |lp| + ln S <= |lp| + ln(vocab); ln S adds the
    relative error of S and its own rounding; one more for the difference."""
    big = lp.abs() + math.log(vocab + 1)
    return U * (3 * big + 2 * math.log(vocab + 1) + lp.abs()) + sum_error(vocab)


def entropy_tolerance(h, vocab):
    """H = ln S - U / (S T): both terms carry the relative errors of their sums; |U| / (S T) <= H <= ln(vocab)."""
    return sum_error(vocab) * (1 + 2 * math.log(vocab + 1)) + 8 * U * (h.abs() + 1)


def grad_tolerance(ref, dtype, vocab, dense, p, lp):
    """``dense``: bound on |a| + |b log p| per row, the factors of p.  p = 2^(c d - log2 S): relative error 4 U (|log p| + ln S) from
    the exponent, the error of S, and 2^-22; p |log p| <= 1/e keeps the first term finite where p underflows.  The sum
    with the sparse entry and the factors round a few times in f32, then once to the type, whose subnormals round
    absolutely."""
    plp = torch.where(p > 0, p * lp.abs(), torch.zeros_like(p))
    rel = sum_error(vocab) + U * (4 * math.log(vocab + 1) + 16)
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * half * 2
    weights = (ref.abs() + dense * p)  # a sparse entry's weight is at most the result plus the dense part
    return dense * (p * rel + 8 * U * plp) + 8 * U * weights + half * ref.abs() * (1 + 1e-3) + tiny + 2.0 ** -126 * dense

"""Token log probabilities, entropy, top alternatives and distillation on the device, against their 64-bit definitions."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import vocab_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
# (rows, vocabulary, extra columns in memory): one token and one class, odd sizes, parts of a vector, several blocks a row
SHAPES = [(1, 1, 0), (1, 2, 1), (3, 7, 0), (5, 8, 8), (9, 127, 3), (4, 1000, 0), (33, 4099, 13), (2, 32003, 61), (301, 6007, 1),
          (700, 515, 0), (1, 200001, 7), (320, 20001, 2), (300, 40009, 3), (298, 70001, 0), (1500, 515, 1)]


def logits_for(rows, vocab, pad, dtype, seed, spread=2.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    wide = torch.randn(rows, vocab + pad, generator=gen, device="cuda") * spread
    return wide.to(dtype)[:, :vocab]


def close(got, want, tol):
    # a value beyond the result's type is an infinity there: the lowest f32 over a temperature of 0.5 is -6.8e38, and
    # round to nearest takes everything above max + half its last place (relative eps / 4) to infinity
    most = torch.finfo(got.dtype).max * (1 + torch.finfo(got.dtype).eps / 4)
    want = torch.where(want.double().abs() > most, want.double() * math.inf, want.double())
    got = got.double()
    assert got.shape == want.shape
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    err = torch.where(same, torch.zeros_like(want), (got - want).abs())
    assert not torch.isnan(err).any(), "NaN or infinity on one side only"
    worst = (err - tol).max().item() if err.numel() else -1.0
    assert worst <= 0, f"off by up to {err.max().item():.3e}, {worst:.3e} above the tolerance"


def check_scores(be, x, tokens, temperature, top, ignore_index=None):
    rows, vocab = x.shape
    got = be.token_log_probs(x, tokens, temperature=temperature, top=top, entropy=True, ignore_index=ignore_index)
    be.sync()
    p, lp = ref.softmax64(x, temperature)
    live = tokens != ignore_index if ignore_index is not None else torch.ones_like(tokens, dtype=torch.bool)
    zero = torch.zeros(rows, dtype=torch.float64, device=x.device)
    want = torch.where(live, lp.gather(1, tokens.long().clamp(min=0)[:, None])[:, 0], zero)
    close(got.log_probs, want, ref.log_prob_tolerance(want, vocab))
    h = torch.where(live, ref.entropy64(p, lp), zero)
    close(got.entropy, h, ref.entropy_tolerance(h, vocab))
    if top:
        order = torch.where(live[:, None], ref.order64(x, top), torch.full((1, 1), -1, device=x.device))
        assert torch.equal(got.top_indices.long(), order)
        want = torch.where(live[:, None], lp.gather(1, order.clamp(min=0)), torch.full_like(lp[:, :1], -math.inf))
        close(got.top_log_probs, want, ref.log_prob_tolerance(want, vocab))
    return got


# ------------------------------------------------------------------ forward
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,pad", SHAPES)
@pytest.mark.parametrize("top,temperature", [(0, 1.0), (1, 0.7), (20, 1.0), (256, 2.5)])
def test_scores_against_the_definition(be, dtype, rows, vocab, pad, top, temperature):
    x = logits_for(rows, vocab, pad, dtype, rows + vocab)
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(vocab))
    check_scores(be, x, tokens, temperature, min(top, vocab))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(6, 37), (6, 5003), (400, 5003), (6, 40009), (1500, 333)])
def test_masked_and_empty_rows(be, dtype, rows, vocab):
    x = logits_for(rows, vocab, 0, dtype, 5)
    lowest = torch.finfo(dtype).min
    x[0] = -math.inf                         # a mask that leaves nothing
    x[1] = lowest                            # the same, written with the type's lowest value: uniform
    x[2, 1:] = -math.inf                     # one token left
    x[3, ::2] = -math.inf
    x[4, ::3] = lowest
    tokens = torch.zeros(rows, dtype=torch.int64, device="cuda")
    got = check_scores(be, x, tokens, 1.0, 16)
    assert got.log_probs[0].item() == -math.inf and got.entropy[0].item() == 0.0
    assert got.top_indices[0].tolist() == list(range(16))
    assert got.log_probs[2].item() == 0.0 and got.entropy[2].item() == 0.0
    check_scores(be, x, tokens, 0.5, 16)


@pytest.mark.parametrize("dtype", TYPES)
def test_nan_and_infinite_rows(be, dtype):
    rows, vocab = 5, 3001
    x = logits_for(rows, vocab, 0, dtype, 6)
    x[0, 17] = math.nan
    x[1, 2999] = math.inf
    x[2] = -math.inf
    x[2, 5] = math.nan
    x[3] = math.nan
    tokens = torch.tensor([3, 4, 5, 6, 7], device="cuda")
    got = be.token_log_probs(x, tokens, top=4, entropy=True)
    be.sync()
    assert torch.isnan(got.log_probs[:4]).all() and torch.isnan(got.entropy[:4]).all() and torch.isnan(got.top_log_probs[:4]).all()
    assert torch.equal(got.top_indices.long(), ref.order64(x, 4))
    check_scores(be, x[4:], tokens[4:], 1.0, 4)
    grad = be.token_log_probs_bwd(x, tokens, got.stats, d_log_probs=torch.ones(rows, device="cuda"), entropy=got.entropy,
                                  d_entropy=torch.ones(rows, device="cuda"))
    be.sync()
    assert torch.isnan(grad[:4]).all() and torch.isfinite(grad[4]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [300, 4096, 50257, 200000])
@pytest.mark.parametrize("rows", [3, 310])
def test_ties_and_orders(be, dtype, vocab, rows):
    """Ties go to the lower index whatever threads meet them; sorted rows and rows whose large entries all belong to a few
    threads (vector index modulo the block) take the selection's longer ways."""
    rows = min(rows, 3 * 2 ** 24 // vocab) if rows > 3 else rows
    j = torch.arange(vocab, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    patterns = [torch.zeros(vocab, device="cuda"),
                torch.where(j % 2 == 0, 0.0, -0.0),
                j.float() / vocab * 8 - 4,
                4 - j.float() / vocab * 8,
                torch.randint(0, 3, (vocab,), generator=gen, device="cuda").float(),
                torch.where(j >= vocab - 40, 1.0, 0.0),
                -((j // 4) % 512).float() * 0.01 + torch.rand(vocab, generator=gen, device="cuda") * 1e-3,
                -((j // 8) % 512).float() * 0.01 + torch.rand(vocab, generator=gen, device="cuda") * 1e-3,
                -((j // 8) % 128).float() * 0.01]
    x = torch.stack([patterns[r % len(patterns)] for r in range(max(rows, len(patterns)))]).to(dtype)
    tokens = torch.zeros(x.shape[0], dtype=torch.int32, device="cuda")
    for top in (1, 64, 256):
        check_scores(be, x, tokens, 1.0, top)


@pytest.mark.parametrize("dtype", TYPES)
def test_ignored_rows_and_no_tokens(be, dtype):
    x = logits_for(11, 2050, 6, dtype, 9)
    tokens = torch.arange(11, device="cuda", dtype=torch.int32)
    tokens[[0, 5, 10]] = -100
    x[5] = math.nan                                  # not looked at
    check_scores(be, x[[0, 1, 2, 10]], tokens[[0, 1, 2, 10]], 1.0, 3, ignore_index=-100)
    got = be.token_log_probs(x, tokens, top=3, entropy=True, ignore_index=-100)
    assert got.log_probs[5].item() == 0.0 and got.top_indices[5].tolist() == [-1] * 3
    none = be.token_log_probs(x[:5], None, top=3)
    be.sync()
    assert none.log_probs is None and none.entropy is None
    assert torch.equal(none.top_indices.long(), ref.order64(x[:5], 3))


def test_token_outside_the_vocabulary_is_reported_once(be):
    x = logits_for(4, 100, 0, torch.float32, 2)
    for bad in (100, -1, 2 ** 40):
        got = be.token_log_probs(x, torch.tensor([1, bad, 2, 3], device="cuda"), top=2)
        with pytest.raises(IndexError):
            be.sync()
        be.sync()
        assert torch.isnan(got.log_probs[1]) and torch.isfinite(got.log_probs[[0, 2, 3]]).all()


# ------------------------------------------------------------------ gradient of the scores
def check_score_grad(be, x, tokens, temperature, top, ignore_index=None, seed=0):
    rows, vocab = x.shape
    gen = torch.Generator(device="cuda").manual_seed(seed)
    fwd = be.token_log_probs(x, tokens, temperature=temperature, top=top, entropy=True, ignore_index=ignore_index)
    up = {"d_log_probs": torch.randn(rows, generator=gen, device="cuda"),
          "d_entropy": torch.randn(rows, generator=gen, device="cuda")}
    if top:
        up["d_top"] = torch.randn(rows, top, generator=gen, device="cuda")
    p, lp = ref.softmax64(x, temperature)
    for names in (["d_log_probs"], ["d_entropy"], list(up)) + ((["d_top"],) if top else ()):
        some = {k: up[k] for k in names}
        got = be.token_log_probs_bwd(x, tokens, fwd.stats, entropy=fwd.entropy, top_indices=fwd.top_indices,
                                     temperature=temperature, ignore_index=ignore_index, **some)
        be.sync()
        assert got.dtype == x.dtype and got.shape == x.shape
        want = ref.score_grad64(x, tokens, temperature, top_indices=fwd.top_indices, ignore_index=ignore_index, **some)
        dense = sum(v.double().abs().reshape(rows, -1).sum(1) for k, v in some.items() if k != "d_entropy")
        dense = torch.as_tensor(dense, device=x.device, dtype=torch.float64).expand(rows)[:, None]
        if "d_entropy" in some:
            size = torch.where(p > 0, lp.abs(), torch.zeros_like(lp)) + math.log(vocab + 1)
            # the entropy itself comes from the forward call, to within its own tolerance
            off = ref.entropy_tolerance(ref.entropy64(p, lp), vocab)[:, None]
            dense = dense + some["d_entropy"].double().abs()[:, None] * size
            extra = some["d_entropy"].double().abs()[:, None] * off * p / temperature
        else:
            extra = 0.0
        close(got, want, ref.grad_tolerance(want, x.dtype, vocab, dense / temperature, p, lp) + extra)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,pad", SHAPES)
@pytest.mark.parametrize("top,temperature", [(0, 1.0), (5, 0.7)])
def test_score_gradient(be, dtype, rows, vocab, pad, top, temperature):
    x = logits_for(rows, vocab, pad, dtype, rows * 3 + vocab)
    if vocab > 20:
        x[:, 3:7] = -math.inf
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(7))
    ignore = -100 if rows > 2 else None
    if ignore:
        tokens[1] = ignore
    check_score_grad(be, x, tokens, temperature, min(top, vocab), ignore)


@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_of_rows_without_a_distribution(be, dtype):
    x = logits_for(4, 1003, 0, dtype, 3)
    x[0] = -math.inf
    x[1] = torch.finfo(dtype).min
    x[2, 1:] = -math.inf
    check_score_grad(be, x, torch.tensor([2, 3, 0, 4], device="cuda"), 1.0, 3)


def test_score_gradient_against_differences(be):
    """Central differences of the kernel's own forward pass, along random directions, in f32: the forward error over the
    step (2 e / h) plus the curvature term (third derivatives of these functions are below 8 per unit direction: h^2 * 8)."""
    rows, vocab, h = 6, 411, 0.05
    x = logits_for(rows, vocab, 0, torch.float32, 21, spread=1.0)
    tokens = torch.arange(rows, device="cuda")
    w = torch.randn(rows, device="cuda")
    fwd = be.token_log_probs(x, tokens, temperature=1.3, top=4, entropy=True)
    wt = torch.randn(rows, 4, device="cuda")
    grad = be.token_log_probs_bwd(x, tokens, fwd.stats, d_log_probs=w, entropy=fwd.entropy, d_entropy=-w, top_indices=fwd.top_indices,
                                  d_top=wt, temperature=1.3)
    gen = torch.Generator(device="cuda").manual_seed(4)
    for _ in range(5):
        v = torch.randn(rows, vocab, generator=gen, device="cuda")
        v /= v.norm(dim=1, keepdim=True)

        def value(y):
            o = be.token_log_probs(y, tokens, temperature=1.3, top=4, entropy=True)
            _, lp = ref.softmax64(y, 1.3)   # the alternatives at the indices of the base point
            at = torch.log_softmax(y / 1.3, 1).gather(1, fwd.top_indices.long())
            return (w * o.log_probs - w * o.entropy + (wt * at).sum(1)).double()
        slope = (value(x + h * v) - value(x - h * v)) / (2 * h)
        want = (grad.double() * v.double()).sum(1)
        size = 2 * w.abs().double() + wt.abs().double().sum(1)
        tol = size * (8 * h * h + (ref.sum_error(vocab) + 20 * ref.U) * 16 / h)
        close(want, slope, tol)


# ------------------------------------------------------------------ distillation
def teacher_for(rows, vocab, top, seed, index_dtype=torch.int32, value_dtype=torch.float32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    idx = torch.stack([torch.randperm(vocab, generator=gen, device="cuda")[:top] for _ in range(rows)]) if vocab >= top else \
        torch.randint(0, vocab, (rows, top), generator=gen, device="cuda")
    val = torch.randn(rows, top, generator=gen, device="cuda") * 2
    return idx.to(index_dtype), val.to(value_dtype)


def check_distill(be, x, idx, val, temperature):
    rows, vocab = x.shape
    want, grad64 = ref.distill64(x, idx, val, temperature)
    p, lp = ref.softmax64(x, temperature)
    q = ref.teacher64(idx, val, temperature)
    top = idx.shape[1]
    # per term q (log q - log p): roundings of both logarithms, then the sum over the entries
    at = torch.where((q > 0) & torch.isfinite(lp.gather(1, idx.long().clamp(min=0))), lp.gather(1, idx.long().clamp(min=0)).abs(), torch.zeros_like(q))
    lq = torch.where(q > 0, q, torch.ones_like(q)).log().abs()
    per = (q * ((at + lq + 2 * math.log(vocab + top + 1)) * 8 * ref.U + 2 * ref.sum_error(vocab) + (top + 32) * ref.U)).sum(1)
    big = (q * (at + lq)).sum(1)
    tol = temperature ** 2 * (per + big * (top / 512 + 24) * ref.U)
    rows_w = 0.5 + torch.rand(rows, device="cuda")
    for reduction in ("none", "mean", "sum"):
        stats = torch.empty(rows, 2, device="cuda")
        loss, grad = be.distillation_loss(x, idx, val, temperature=temperature, reduction=reduction, upstream=1.5,
                                          upstream_rows=rows_w, stats=stats)
        only, nothing = be.distillation_loss(x, idx, val, temperature=temperature, reduction=reduction, want_grad=False)
        again = be.distillation_loss_bwd(x, idx, val, stats, temperature=temperature, reduction=reduction, upstream=1.5,
                                         upstream_rows=rows_w)
        be.sync()
        assert nothing is None
        f = 1.0 / rows if reduction == "mean" else 1.0
        for got in (loss, only):   # the loss alone may be added up in another order: both are held to the definition
            if reduction == "none":
                close(got, want, tol)
            else:
                close(got, (want.sum() * f).reshape(1), (tol.sum() * f + ref.U * 2 * want.sum().abs() * f).reshape(1))
        scale = 1.5 * f * rows_w.double()[:, None]
        g = grad64 * scale
        # q carries the errors of its own softmax: as the dense part does, over `top` entries
        qs = torch.zeros_like(p).scatter_add_(1, idx.long().clamp(min=0), q)
        more = (qs * (top / 512 + 64 + 8 * math.log(top + 2)) * ref.U + torch.where(qs > 0, qs * 8 * ref.U * qs.clamp(min=1e-300).log().abs(), qs)) * scale * temperature
        tol_g = ref.grad_tolerance(g, x.dtype, vocab, scale * temperature, p, lp) + more
        close(grad, g, tol_g)
        close(again, g, tol_g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,pad", SHAPES)
@pytest.mark.parametrize("top,temperature", [(1, 1.0), (5, 2.0), (64, 0.8)])
def test_distillation(be, dtype, rows, vocab, pad, top, temperature):
    x = logits_for(rows, vocab, pad, dtype, rows + 5 * vocab)
    idx, val = teacher_for(rows, vocab, min(top, vocab), vocab)
    if rows > 2:
        idx[1] = -1                                            # a row without a teacher
        idx[2, idx.shape[1] // 2:] = -1
    check_distill(be, x, idx, val, temperature)


@pytest.mark.parametrize("index_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("value_dtype", TYPES)
def test_distillation_types_duplicates_and_extremes(be, index_dtype, value_dtype):
    rows, vocab, top = 9, 2003, 700
    x = logits_for(rows, vocab, 0, torch.float32, 8)
    idx, val = teacher_for(rows, vocab, top, 3, index_dtype, value_dtype)
    idx[0, 100:200] = idx[0, 0]                # the same index many times: its weights add up
    idx[1] = 7
    val[2, 5:] = -math.inf                     # teacher entries of no weight
    val[3] = -math.inf                         # none at all
    val[4] = torch.finfo(value_dtype).min      # all equal, at the type's lowest value
    x[5, idx[5, 0].long()] = -math.inf         # the student rules out what the teacher wants: infinite loss
    x[6] = -math.inf
    x[7] = torch.finfo(torch.float32).min
    check_distill(be, x, idx, val, 1.0)
    loss, _ = be.distillation_loss(x, idx, val, reduction="none")
    assert loss[3].item() == 0.0 and loss[5].item() == math.inf and loss[6].item() == math.inf


@pytest.mark.parametrize("dtype", TYPES)
def test_distillation_without_entries_and_with_the_most(be, dtype):
    x = logits_for(5, 4001, 0, dtype, 8)
    loss, grad = be.distillation_loss(x, torch.empty(5, 0, dtype=torch.int32, device="cuda"), torch.empty(5, 0, device="cuda"))
    assert loss.item() == 0.0 and not grad.any()
    idx, val = teacher_for(5, 4001, 1024, 2)
    check_distill(be, x, idx, val, 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(3, 40), (2000, 40), (2, 50257), (700, 2003)])
def test_distillation_of_the_lowest_logit_below_temperature_one(be, dtype, rows, vocab):
    """The teacher wants an entry that holds the type's lowest value: (v - m) / T is beyond f32, T times it is not."""
    x = logits_for(rows, vocab, 0, dtype, vocab)
    idx, val = teacher_for(rows, vocab, 7, vocab)
    x[0, idx[0, 2].long()] = torch.finfo(dtype).min
    if rows > 2:
        idx[2] = idx[2, 0].item()                              # all of a row's weight on that value
        x[2, idx[2, 0].long()] = torch.finfo(dtype).min
    check_distill(be, x, idx, val, 0.3)
    loss, _ = be.distillation_loss(x, idx, val, temperature=0.3, reduction="none")
    be.sync()
    assert torch.isfinite(loss).all()


def test_distillation_nan_teacher_and_bad_index(be):
    x = logits_for(4, 500, 0, torch.float32, 8)
    idx, val = teacher_for(4, 500, 6, 2)
    val[1, 3] = math.nan
    loss, grad = be.distillation_loss(x, idx, val, reduction="none")
    be.sync()
    assert torch.isnan(loss[1]) and torch.isnan(grad[1]).all() and torch.isfinite(grad[[0, 2, 3]]).all()
    val[1, 3] = 0.0
    for bad in (500, -2):
        idx[2, 0] = bad
        loss, grad = be.distillation_loss(x, idx, val, reduction="none")
        with pytest.raises(IndexError):
            be.sync()
        idx[2, 0] = -1
        same, _ = be.distillation_loss(x, idx, val, reduction="none")
        be.sync()
        assert torch.equal(loss, same)


def test_distillation_gradient_against_differences(be):
    """Central differences of the kernel's own loss: 2 e / h for the forward error, h^2 * 8 T^2 for the curvature."""
    rows, vocab, t, h = 5, 311, 1.7, 0.05
    x = logits_for(rows, vocab, 0, torch.float32, 12, spread=1.0)
    idx, val = teacher_for(rows, vocab, 9, 4)
    _, grad = be.distillation_loss(x, idx, val, temperature=t, reduction="none")
    gen = torch.Generator(device="cuda").manual_seed(4)
    for _ in range(5):
        v = torch.randn(rows, vocab, generator=gen, device="cuda")
        v /= v.norm(dim=1, keepdim=True)
        value = lambda y: be.distillation_loss(y, idx, val, temperature=t, reduction="none", want_grad=False)[0].double()
        slope = (value(x + h * v) - value(x - h * v)) / (2 * h)
        want = (grad.double() * v.double()).sum(1)
        tol = t * t * (8 * h * h + (ref.sum_error(vocab) + 20 * ref.U) * 16 / h)
        close(want, slope, torch.full_like(want, tol))


# ------------------------------------------------------------------ together, and how they are called
@pytest.mark.parametrize("dtype", TYPES)
def test_teacher_to_student(be, dtype):
    """A teacher's top logits, taken by one operator, are what the other one distils from; left-out rows stay left out."""
    teacher, student = logits_for(40, 5003, 0, dtype, 1), logits_for(40, 5003, 5, dtype, 2)
    tokens = torch.arange(40, device="cuda")
    tokens[::7] = -100
    top = be.token_log_probs(teacher, tokens, top=32, ignore_index=-100)
    check_distill(be, student, top.top_indices, top.top_log_probs, 1.5)
    loss, grad = be.distillation_loss(student, top.top_indices, top.top_log_probs, reduction="none")
    assert not loss[::7].any() and not grad[::7].any()
    same, _ = be.distillation_loss(teacher, top.top_indices, top.top_log_probs, reduction="none")
    mass = ref.softmax64(teacher, 1.0)[0].gather(1, top.top_indices.long().clamp(min=0)).sum(1)
    want = torch.where(tokens == -100, torch.zeros_like(mass), -mass.log())  # KL of the renormalised top against the whole
    close(same, want, ref.log_prob_tolerance(want, 5003) * 2)


def test_model_trains_through_both(be):
    """A dense layer's gradients through the distillation loss and through log probabilities, entropy and alternatives."""
    import minitensor_b200.nn as nn
    from minitensor_b200.tensor import Tensor
    rng = np.random.default_rng(0)
    b, s, d, v, k = 3, 5, 24, 301, 7
    layer = nn.DenseLayer(d, v, rng=rng)
    x = rng.standard_normal((b, s, d)).astype(np.float32)
    teacher = Tensor(rng.standard_normal((b, s, v)).astype(np.float32))
    tokens = rng.integers(0, v, (b, s))
    tokens[0, 0] = -1
    known = nn.token_log_probs(teacher, Tensor(tokens), top=k, ignore_index=-1)
    assert known.top_indices.shape == (b, s, k) and known.log_probs.shape == (b, s) and known.entropy is None
    coef = rng.standard_normal((b, s)).astype(np.float32)
    coef_top = rng.standard_normal((b, s, k)).astype(np.float32)

    w64 = torch.tensor(layer.weight.numpy(), dtype=torch.float64, requires_grad=True)
    b64 = torch.tensor(layer.bias.numpy(), dtype=torch.float64, requires_grad=True)
    logits = torch.tensor(x, dtype=torch.float64) @ w64.T + b64
    live = torch.tensor(tokens != -1)
    lp = torch.log_softmax(logits, -1)
    q_lp = torch.tensor(known.top_log_probs.numpy(), dtype=torch.float64)
    q = torch.where(live[..., None], torch.softmax(torch.where(live[..., None], q_lp, torch.zeros_like(q_lp)), -1), torch.zeros_like(q_lp))
    at = torch.tensor(known.top_indices.numpy()).long().clamp(min=0)
    t = 2.0
    lp_t = torch.log_softmax(logits / t, -1)
    q_t = torch.where(live[..., None], torch.softmax(torch.where(live[..., None], q_lp, torch.zeros_like(q_lp)) / t, -1), torch.zeros_like(q_lp))
    kl = t * t * (torch.special.xlogy(q_t, q_t) - q_t * lp_t.gather(-1, at)).sum(-1)

    cases = {"mean": kl.mean(), "sum": kl.sum(), "none": (kl * torch.tensor(coef, dtype=torch.float64)).sum()}
    for reduction, value in cases.items():
        layer.weight.zero_grad(), layer.bias.zero_grad()
        loss = nn.DistillationLoss(t, reduction)(layer(Tensor(x)), known.top_indices, known.top_log_probs)
        loss.backward(Tensor(coef) if reduction == "none" else None)
        gw, gb = torch.autograd.grad(value, [w64, b64], retain_graph=True)
        if reduction != "none":
            assert abs(loss.item() - value.item()) <= 1e-5 * (1 + abs(value.item()))
        np.testing.assert_allclose(layer.weight.grad.numpy(), gw.numpy(), rtol=0, atol=1e-4 * gw.abs().max().item())
        np.testing.assert_allclose(layer.bias.grad.numpy(), gb.numpy(), rtol=0, atol=1e-4 * gb.abs().max().item())

    # three outputs of one call, joined and separately
    h = -(lp.exp() * lp).sum(-1)
    tok = torch.tensor(np.maximum(tokens, 0))
    parts = {"log_probs": (lp.gather(-1, tok[..., None])[..., 0] * live * torch.tensor(coef)).sum(),
             "entropy": (h * live * torch.tensor(coef)).sum()}
    order = logits.topk(k, dim=-1).indices
    parts["top_log_probs"] = (lp.gather(-1, order) * live[..., None] * torch.tensor(coef_top)).sum()
    for names in (["log_probs"], ["entropy"], ["top_log_probs"], ["log_probs", "entropy", "top_log_probs"]):
        layer.weight.zero_grad(), layer.bias.zero_grad()
        out = nn.token_log_probs(layer(Tensor(x)), Tensor(tokens), top=k, entropy=True, ignore_index=-1)
        assert np.array_equal(out.top_indices.numpy()[tokens != -1], order.numpy()[tokens != -1])
        for n in names:  # gradients of several backward calls add up in the leaves
            getattr(out, n).backward(Tensor(coef_top if n == "top_log_probs" else coef))
        gw, gb = torch.autograd.grad(sum(parts[n] for n in names), [w64, b64], retain_graph=True)
        np.testing.assert_allclose(layer.weight.grad.numpy(), gw.numpy(), rtol=0, atol=1e-4 * gw.abs().max().item())
        np.testing.assert_allclose(layer.bias.grad.numpy(), gb.numpy(), rtol=0, atol=1e-4 * gb.abs().max().item())
    # one scalar of two of the outputs: their gradients meet in one backward pass over the logits
    layer.weight.zero_grad()
    before = be.launches
    out = nn.token_log_probs(layer(Tensor(x)), Tensor(tokens), top=k, entropy=True, ignore_index=-1)
    (out.log_probs + out.entropy).backward(Tensor(coef))
    assert be.launches > before
    gw, = torch.autograd.grad(parts["log_probs"] + parts["entropy"], [w64], retain_graph=True)
    np.testing.assert_allclose(layer.weight.grad.numpy(), gw.numpy(), rtol=0, atol=1e-4 * gw.abs().max().item())
    with pytest.raises(IndexError):
        nn.token_log_probs(teacher, Tensor(np.full((b, s), v)))


@pytest.mark.parametrize("dtype", TYPES)
def test_other_stream_and_repeated_calls(be, dtype):
    x = logits_for(64, 20011, 0, dtype, 4)
    idx, val = teacher_for(64, 20011, 33, 4)
    tokens = torch.arange(64, device="cuda")
    torch.cuda.synchronize()
    first = be.token_log_probs(x, tokens, top=30, entropy=True)
    loss, grad = be.distillation_loss(x, idx, val)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = be.token_log_probs(x, tokens, top=30, entropy=True)
        loss2, grad2 = be.distillation_loss(x, idx, val)
        be.sync()
    for a, b in zip(list(first) + [loss, grad], list(again) + [loss2, grad2]):
        assert torch.equal(a, b)


def test_captured_graphs_replay_on_new_inputs(be):
    """Two captured graphs, run on two streams at once: the calls share no scratch memory."""
    xs = [logits_for(48, 9001, 0, torch.bfloat16, 30 + i) for i in range(2)]
    idx, val = teacher_for(48, 9001, 20, 4)
    tokens = torch.arange(48, device="cuda")
    state = []
    for x in xs:
        be.token_log_probs(x, tokens, top=10, entropy=True)
        be.distillation_loss(x, idx, val)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = be.token_log_probs(x, tokens, top=10, entropy=True)
            grad = be.token_log_probs_bwd(x, tokens, out.stats, d_log_probs=out.log_probs, entropy=out.entropy, d_entropy=out.entropy,
                                          top_indices=out.top_indices, d_top=out.top_log_probs)
            loss = be.distillation_loss(x, idx, val)
        state.append((graph, list(out) + [grad] + list(loss)))
    streams = [torch.cuda.Stream() for _ in xs]
    for round_ in range(3):
        for i, x in enumerate(xs):
            x.copy_(logits_for(48, 9001, 0, torch.bfloat16, 50 + 2 * round_ + i))
        torch.cuda.synchronize()
        for (graph, _), s in zip(state, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for x, (_, got) in zip(xs, state):
            out = be.token_log_probs(x, tokens, top=10, entropy=True)
            grad = be.token_log_probs_bwd(x, tokens, out.stats, d_log_probs=out.log_probs, entropy=out.entropy, d_entropy=out.entropy,
                                          top_indices=out.top_indices, d_top=out.top_log_probs)
            want = list(out) + [grad] + list(be.distillation_loss(x, idx, val))
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [5, 1001, 4099])
def test_c_entry_keeps_to_its_rows(be, dtype, vocab):
    """Logits and gradient that start at different offsets within 16 bytes, with columns between the rows: only the
    vocabulary's columns of the gradient are written."""
    from minitensor_b200 import _lib
    from minitensor_b200.backend import _LOGIT_DTYPES
    rows, ld, top = 6, vocab + 9, 4
    size = torch.empty(0, dtype=dtype).element_size()
    idx, val = teacher_for(rows, vocab, top, 4)
    for off_x, off_g in [(0, 0), (1, 0), (0, 3), (3, 1), (5, 5)]:
        flat = torch.randn(16 + rows * ld, device="cuda").to(dtype)
        x = flat[off_x:off_x + rows * ld].view(rows, ld)[:, :vocab]
        out = torch.full((16 + rows * ld,), 77.0, dtype=dtype, device="cuda")
        stats, row_loss, loss = (torch.empty(n, device="cuda") for n in (2 * rows, rows, 1))
        torch.cuda.synchronize()
        be._bind_stream()
        args = [be._h, _LOGIT_DTYPES[dtype], rows, vocab, x.data_ptr(), ld, top, idx.data_ptr(), _lib.I32, val.data_ptr(), _lib.F32, 1.0,
                1, 1.0, None]
        _lib.check(be.lib.mtb200_distill(*args, row_loss.data_ptr(), loss.data_ptr(), stats.data_ptr(), out.data_ptr() + off_g * size))
        be.sync()
        _, want = be.distillation_loss(x, idx, val)
        view = out[off_g:off_g + rows * ld].view(rows, ld)
        assert torch.equal(view[:, :vocab], want)
        kept = torch.cat([out[:off_g], view[:, vocab:].reshape(-1), out[off_g + rows * ld:]])
        assert (kept == 77.0).all()
        out.fill_(77.0)
        _lib.check(be.lib.mtb200_distill_bwd(*args, stats.data_ptr(), out.data_ptr() + off_g * size))
        be.sync()
        assert torch.equal(view[:, :vocab], want)
        kept = torch.cat([out[:off_g], view[:, vocab:].reshape(-1), out[off_g + rows * ld:]])
        assert (kept == 77.0).all()


def test_offsets_beyond_32_bits(be):
    """Rows behind element 2^31 of the matrix, in a matrix that is mostly row padding."""
    rows, vocab, ld = 5, 70001, 2 ** 29 + 8
    flat = torch.zeros((rows - 1) * ld + vocab, dtype=torch.bfloat16, device="cuda")
    x = flat.as_strided((rows, vocab), (ld, 1))
    x.copy_(logits_for(rows, vocab, 0, torch.bfloat16, 6))
    tokens = torch.arange(rows, device="cuda")
    # against the definitions, not bit by bit against a dense copy: a row's offset within 16 bytes decides which thread
    # adds which elements, and 70001 columns start every row of a dense copy at another offset
    check_scores(be, x, tokens, 1.0, 9)
    check_score_grad(be, x, tokens, 1.0, 9)
    idx, val = teacher_for(rows, vocab, 9, 6)
    check_distill(be, x, idx, val, 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(2, 2500001), (200, 600011)])
def test_very_long_rows(be, dtype, rows, vocab):
    """Rows of many rounds per thread: the selection's spans cover several rounds each."""
    x = logits_for(rows, vocab, 0, dtype, vocab)
    x[0, ::2] = -math.inf
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) | 1
    tokens = tokens.clamp(max=vocab - 1)
    for top in (20, 256):
        got = be.token_log_probs(x, tokens, top=top, entropy=True)
        be.sync()
        for i in range(0, rows, 40):   # some rows at a time: the 64-bit definition takes 8 bytes an element and more
            part = slice(i, min(rows, i + 2))
            p, lp = ref.softmax64(x[part], 1.0)
            want = lp.gather(1, tokens[part, None])[:, 0]
            close(got.log_probs[part], want, ref.log_prob_tolerance(want, vocab))
            h = ref.entropy64(p, lp)
            close(got.entropy[part], h, ref.entropy_tolerance(h, vocab))
            assert torch.equal(got.top_indices[part].long(), ref.order64(x[part], top))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(200, 257), (200, 1000), (170, 2048), (300, 33000), (1300, 300)])
def test_nearly_all_entries_wanted(be, dtype, rows, vocab):
    """Many alternatives of short rows: more wanted than there are threads' shares, and candidates by the thousand."""
    x = logits_for(rows, vocab, 0, dtype, 17)
    x[3] = 1.0
    x[4, 5:] = -math.inf
    tokens = torch.zeros(rows, dtype=torch.int64, device="cuda")
    for top in (21, 65, 128, 129, 256):
        check_scores(be, x, tokens, 1.0, top)


def test_two_backends_and_backward_after_other_calls(be):
    """Statistics belong to the caller: another handle, and other calls in between, change nothing."""
    from minitensor_b200.backend import Backend
    other = Backend(0)
    x, y = logits_for(30, 9001, 0, torch.float32, 1), logits_for(30, 9001, 0, torch.float32, 2)
    tokens = torch.arange(30, device="cuda")
    fwd = be.token_log_probs(x, tokens, top=5, entropy=True)
    d = torch.ones(30, device="cuda")
    first = be.token_log_probs_bwd(x, tokens, fwd.stats, d_log_probs=d, entropy=fwd.entropy, d_entropy=d)
    other.token_log_probs(y, tokens, top=5, entropy=True)
    be.token_log_probs(y, tokens, top=7)
    second = other.token_log_probs_bwd(x, tokens, fwd.stats, d_log_probs=d, entropy=fwd.entropy, d_entropy=d)
    other.sync()
    be.sync()
    assert torch.equal(first, second)
    other.close()


def test_refusals_on_the_device(be):
    x = logits_for(4, 50, 0, torch.float32, 1)
    tokens = torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="backend on"):
        be.token_log_probs(x.cpu(), tokens)
    with pytest.raises(ValueError, match="backend on"):
        be.token_log_probs(x, tokens.cpu())
    for t in (0.0, -1.0, math.nan, math.inf, 1e-45, 1e30):
        with pytest.raises(ValueError, match="temperature"):
            be.token_log_probs(x, tokens, temperature=t)
    big = logits_for(2, 1000, 0, torch.float32, 1)
    with pytest.raises(ValueError, match="top"):
        be.token_log_probs(big, None, top=257)
    with pytest.raises(ValueError, match="entries"):
        be.distillation_loss(big, torch.zeros(2, 1025, dtype=torch.int32, device="cuda"), torch.zeros(2, 1025, device="cuda"))
    from minitensor_b200 import _lib
    be._bind_stream()
    stats = torch.empty(8, device="cuda")
    rc = be.lib.mtb200_token_log_probs_bwd(be._h, 0, 4, 50, x.data_ptr(), 50, tokens.data_ptr(), _lib.I64, 0, 0, 1.0, stats.data_ptr(),
                                           stats.data_ptr(), None, None, 0, None, None, x.data_ptr())
    assert rc == _lib.ERR_INVALID and "in place" in _lib.last_error()
    rc = be.lib.mtb200_token_log_probs(be._h, 0, 4, 40, x.data_ptr() + 2, 50, None, 0, 0, 0, 1.0, 0, None, None, None, None, stats.data_ptr())
    assert rc == _lib.ERR_INVALID and "misaligned" in _lib.last_error()
    rc = be.lib.mtb200_token_log_probs(be._h, 1, 4, 40, x.data_ptr(), 50, None, 0, 0, 0, 1.0, 0, None, None, None, None, stats.data_ptr())
    assert rc == _lib.ERR_UNSUPPORTED
    empty = be.token_log_probs(x[:0], tokens[:0], top=2, entropy=True)
    assert empty.log_probs.shape == (0,) and empty.top_indices.shape == (0, 2)
    loss, grad = be.distillation_loss(x[:0], torch.zeros(0, 3, dtype=torch.int32, device="cuda"), torch.zeros(0, 3, device="cuda"), reduction="sum")
    be.sync()
    assert loss.item() == 0.0 and grad.shape == (0, 50)


_RISING_TOPS = """
import sys, torch
sys.path[:0] = [{root!r}, {tests!r}]
import vocab_reference as ref
from test_vocab_ops_gpu import check_scores, close, logits_for
from minitensor_b200.backend import get_backend
be = get_backend(0)
for dtype in (torch.float32, torch.bfloat16, torch.float16):
    x = logits_for(9, 128256 if dtype != torch.float32 else 50257, 0, dtype, 13)
    tokens = torch.arange(9, device="cuda")
    _, lp = ref.softmax64(x, 1.0)
    for top in range(130, 144):
        check_scores(be, x, tokens, 1.0, top)
        got = be.token_log_probs(x, tokens, top=top)
        be.sync()
        order = ref.order64(x, top)
        assert torch.equal(got.top_indices.long(), order)
        want = lp.gather(1, order)
        close(got.top_log_probs, want, ref.log_prob_tolerance(want, x.shape[1]))
"""


def test_more_alternatives_from_call_to_call_in_a_new_process():
    """Few long rows are cut into eight parts, whose lists of alternatives lie in shared memory beside the scratch of the
    selection: with rising `top` the sum passes the size that a launch may have without asking.  What a process has asked
    for stays granted, so the calls come in a process of their own."""
    import os
    import subprocess
    import sys
    from conftest import ROOT
    script = _RISING_TOPS.format(root=ROOT, tests=os.path.join(ROOT, "tests"))
    run = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert run.returncode == 0, run.stderr[-2000:]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,seq,vocab", [(6, 5, 1003), (160, 3, 515), (3, 4, 50257), (400, 2, 9001)])
def test_gradients_of_the_last_positions(be, dtype, rows, seq, vocab):
    """Logits whose rows lie further apart than they are long; their gradient takes the room of its own rows."""
    x = logits_for(rows * seq, vocab, 0, dtype, 31).view(rows, seq, vocab)[:, -1]
    tokens = torch.arange(rows, device="cuda") % vocab
    check_scores(be, x, tokens, 1.0, 5)
    check_score_grad(be, x, tokens, 0.9, 5)
    idx, val = teacher_for(rows, vocab, 11, 6)
    check_distill(be, x, idx, val, 1.5)
    _, grad = be.distillation_loss(x, idx, val)
    assert grad.untyped_storage().nbytes() <= (rows * (vocab + 8) + 8) * grad.element_size()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [5, 1001, 20011])
def test_c_entries_with_two_row_strides(be, dtype, vocab):
    """Logits and gradient with row strides that differ by whole vectors or by single elements, either one the longer:
    only the vocabulary's columns of the gradient are written, with the values that a dense gradient gets."""
    from minitensor_b200 import _lib
    from minitensor_b200.backend import _LOGIT_DTYPES
    rows, top = 7, 4
    code, unit = _LOGIT_DTYPES[dtype], 16 // torch.empty(0, dtype=dtype).element_size()
    idx, val = teacher_for(rows, vocab, top, 4)
    tokens = torch.arange(rows, device="cuda") % vocab
    d = torch.randn(rows, device="cuda")
    for ld, ldg in [(vocab, vocab), (vocab + 3, vocab), (vocab, vocab + 5), (vocab + 4 * unit, vocab), (vocab, vocab + 2 * unit)]:
        x = torch.randn(rows * ld, device="cuda").to(dtype).view(rows, ld)[:, :vocab]
        fwd = be.token_log_probs(x, tokens, entropy=True)
        want_s = be.token_log_probs_bwd(x, tokens, fwd.stats, d_log_probs=d, entropy=fwd.entropy, d_entropy=d)
        row_loss, loss, stats = torch.empty(rows, device="cuda"), torch.empty(1, device="cuda"), torch.empty(rows, 2, device="cuda")
        _, want_d = be.distillation_loss(x, idx, val, stats=stats)
        want_b = be.distillation_loss_bwd(x, idx, val, stats)
        out = torch.empty(rows * ldg + 16, dtype=dtype, device="cuda")
        be._bind_stream()

        def kept(want):
            be.sync()
            rest = out[:rows * ldg].view(rows, ldg)
            assert torch.equal(rest[:, :vocab], want)
            assert (rest[:, vocab:] == 77.0).all() and (out[rows * ldg:] == 77.0).all()
            out.fill_(77.0)
        out.fill_(77.0)
        _lib.check(be.lib.mtb200_token_log_probs_bwd_ex(
            be._h, code, rows, vocab, x.data_ptr(), ld, tokens.data_ptr(), _lib.I64, 0, 0, 1.0, fwd.stats.data_ptr(), d.data_ptr(),
            fwd.entropy.data_ptr(), d.data_ptr(), 0, None, None, out.data_ptr(), ldg))
        kept(want_s)
        args = [be._h, code, rows, vocab, x.data_ptr(), ld, top, idx.data_ptr(), _lib.I32, val.data_ptr(), _lib.F32, 1.0, 1, 1.0, None]
        _lib.check(be.lib.mtb200_distill_ex(*args, row_loss.data_ptr(), loss.data_ptr(), stats.data_ptr(), out.data_ptr(), ldg))
        kept(want_d)
        _lib.check(be.lib.mtb200_distill_bwd_ex(*args, stats.data_ptr(), out.data_ptr(), ldg))
        kept(want_b)
        for call in (lambda: be.lib.mtb200_distill_bwd_ex(*args, stats.data_ptr(), out.data_ptr(), vocab - 1),
                     lambda: be.lib.mtb200_distill_ex(*args, row_loss.data_ptr(), loss.data_ptr(), None, out.data_ptr(), vocab - 1),
                     lambda: be.lib.mtb200_token_log_probs_bwd_ex(
                         be._h, code, rows, vocab, x.data_ptr(), ld, None, _lib.I32, 0, 0, 1.0, stats.data_ptr(), None, None, None, 0,
                         None, None, out.data_ptr(), vocab - 1)):
            assert call() == _lib.ERR_INVALID and "row stride" in _lib.last_error()


def test_gradients_beyond_32_bits(be):
    """Gradients whose rows lie behind element 2^31, by the C entries with one row stride for both matrices."""
    from minitensor_b200 import _lib
    rows, vocab, ld, top = 5, 20001, 2 ** 29 + 8, 9
    size = (rows - 1) * ld + vocab
    x, out = (torch.zeros(size, dtype=torch.bfloat16, device="cuda").as_strided((rows, vocab), (ld, 1)) for _ in range(2))
    x.copy_(logits_for(rows, vocab, 0, torch.bfloat16, 6))
    idx, val = teacher_for(rows, vocab, top, 6)
    tokens = torch.arange(rows, device="cuda")
    d = torch.randn(rows, device="cuda")
    fwd = be.token_log_probs(x, tokens)
    want_s = be.token_log_probs_bwd(x, tokens, fwd.stats, d_log_probs=d)
    row_loss, loss, stats = torch.empty(rows, device="cuda"), torch.empty(1, device="cuda"), torch.empty(rows, 2, device="cuda")
    _, want_d = be.distillation_loss(x, idx, val, stats=stats)
    want_b = be.distillation_loss_bwd(x, idx, val, stats)
    be._bind_stream()
    _lib.check(be.lib.mtb200_token_log_probs_bwd(
        be._h, _lib.BF16, rows, vocab, x.data_ptr(), ld, tokens.data_ptr(), _lib.I64, 0, 0, 1.0, fwd.stats.data_ptr(), d.data_ptr(), None,
        None, 0, None, None, out.data_ptr()))
    be.sync()
    assert torch.equal(out, want_s)
    args = [be._h, _lib.BF16, rows, vocab, x.data_ptr(), ld, top, idx.data_ptr(), _lib.I32, val.data_ptr(), _lib.F32, 1.0, 1, 1.0, None]
    for want, call in ((want_d, lambda: be.lib.mtb200_distill(*args, row_loss.data_ptr(), loss.data_ptr(), stats.data_ptr(), out.data_ptr())),
                       (want_b, lambda: be.lib.mtb200_distill_bwd(*args, stats.data_ptr(), out.data_ptr()))):
        out.zero_()
        _lib.check(call())
        be.sync()
        assert torch.equal(out, want)


def test_an_expired_wait_is_not_laid_on_the_products(be):
    """The distillation step waits for messages between blocks and reports as the tensor kernels do; the message names
    the role, and no kernel that it cannot know."""
    from minitensor_b200._lib import Mtb200Error, check
    be.sync()
    check(be.lib.mtb200_selftest_wait_expiry(be._h, 1000))
    with pytest.raises(Mtb200Error, match="role 15, site 1") as err:
        be.sync()
    assert "GEMM" not in str(err.value)
    be.sync()


# ------------------------------------------------------------------ special rows of long vocabularies
def distill_bounds(x, idx, val, temperature):
    """(row losses, gradient of their sum, tolerance of the losses, tolerance of the gradient but for its final rounding) in
    64 bits.

    With q = 2^(c dv) / S_q: the exponent carries the roundings of dv, c and their product, 3 U |dv / T| where |dv / T| is at
    most |ln q| + ln(entries); the power of two 4 U and the division 2 U.  S_q has the mean of that over q, at most
    3 U * 2 ln(entries + 1) + 4 U, and no more than 44 additions on the way of any term (8 a thread, 5 + 5 by shuffles, 16
    warps, a few to spare).  A term of the loss is q times a bracket of ln q - ln p, in whose pieces no number is larger than
    |ln q| + |ln p| + 2 ln(entries) + 2 ln(vocabulary): 8 roundings of that, the errors of q, ln S_q and ln S, and 44
    additions.  Weights with the same index are added one after the other: one U of their sum for each."""
    rows, vocab = x.shape
    top = idx.shape[1]
    U = ref.U
    loss, grad = ref.distill64(x, idx, val, temperature)
    _, lp = ref.softmax64(x, temperature)
    q = ref.teacher64(idx, val, temperature)
    at = idx.long().clamp(min=0)
    lpk = lp.gather(1, at)
    lpk = torch.where((q > 0) & torch.isfinite(lpk), lpk.abs(), torch.zeros_like(q))
    lqk = torch.where(q > 0, q, torch.ones_like(q)).log().abs()
    e_q = U * (6 * math.log(top + 1) + 48)
    rel_q = U * (3 * (lqk + math.log(top + 1)) + 8) + e_q
    size = lqk + lpk + 2 * math.log(top + 1) + 2 * math.log(vocab + 1)
    tol = temperature ** 2 * (q * (size * (52 * U + rel_q) + e_q + ref.sum_error(vocab))).sum(1)
    count = torch.zeros_like(grad).scatter_add_(1, at, (idx >= 0).double())
    mass = torch.zeros_like(grad).scatter_add_(1, at, q)
    more = torch.zeros_like(grad).scatter_add_(1, at, q * (rel_q + 2 * U)) + count * U * mass
    return loss, grad, tol, more * temperature


def check_special_distill(be, x, idx, val, temperature, nan_rows=()):
    rows, vocab = x.shape
    good = torch.tensor([r not in nan_rows for r in range(rows)], device="cuda")
    want, grad64, tol, more = distill_bounds(x[good], idx[good], val[good], temperature)
    p, lp = ref.softmax64(x[good], temperature)
    weights = 0.5 + torch.rand(rows, device="cuda")
    for reduction in ("none", "mean", "sum"):
        if nan_rows and reduction != "none":
            continue
        kw = dict(temperature=temperature, reduction=reduction)
        stats = torch.empty(rows, 2, device="cuda")
        loss, grad = be.distillation_loss(x, idx, val, upstream=0.5, upstream_rows=weights, stats=stats, **kw)
        only, _ = be.distillation_loss(x, idx, val, want_grad=False, **kw)
        again = be.distillation_loss_bwd(x, idx, val, stats, upstream=0.5, upstream_rows=weights, **kw)
        be.sync()
        f = 1.0 / rows if reduction == "mean" else 1.0
        for got in (loss, only):
            if reduction == "none":
                assert torch.isnan(got[~good]).all()
                close(got[good], want, tol)
            else:
                close(got, (want.sum() * f).reshape(1), (tol.sum() * f + ref.U * 2 * want.sum().abs() * f).reshape(1))
        scale = 0.5 * f * weights[good].double()[:, None]
        for got in (grad, again):
            assert torch.isnan(got[~good]).all()
            close(got[good], grad64 * scale,
                  ref.grad_tolerance(grad64 * scale, x.dtype, vocab, scale * temperature, p, lp) + more * scale)


# 8 blocks a row and one block a row for the step with the gradient; up to 480 entries and more
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(13, 50257), (160, 20011)])
@pytest.mark.parametrize("top", [31, 64, 480, 481, 1024])
def test_distillation_of_long_rows_duplicates_and_extremes(be, dtype, rows, vocab, top):
    x = logits_for(rows, vocab, 0, dtype, top)
    idx, val = teacher_for(rows, vocab, top, 11)
    idx[0, -1] = idx[0, 0]                             # the same index first and last
    idx[1, 3:27] = idx[1, 3].item()                    # many times in a row
    idx[2] = vocab - 1                                 # all entries the same
    val[3, 5:] = -math.inf                             # entries of no weight
    val[4] = -math.inf                                 # no weight at all
    val[5] = torch.finfo(torch.float32).min
    idx[6, :-1] = -1                                   # only the last entry
    idx[7, ::2] = idx[7, 1].item()
    x[8] = torch.finfo(dtype).min                      # a uniform student
    x[9, ::2] = -math.inf                              # masked, but not where the teacher looks
    idx[9] = idx[9] | 1
    check_special_distill(be, x, idx.clamp(max=vocab - 1), val, 1.0)
    check_special_distill(be, x, idx.clamp(max=vocab - 1), val, 2.5)
    x[10, idx[10, 0].long()] = -math.inf               # the student rules out what the teacher wants: infinite loss
    x[11] = -math.inf                                  # or everything
    check_special_distill(be, x, idx.clamp(max=vocab - 1), val, 1.0)
    loss, _ = be.distillation_loss(x, idx.clamp(max=vocab - 1), val, reduction="none")
    be.sync()
    assert loss[4].item() == 0.0 and loss[10].item() == math.inf and loss[11].item() == math.inf


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(13, 50257), (160, 20011)])
@pytest.mark.parametrize("top", [5, 100, 480, 481, 1024])
def test_distillation_of_long_rows_nan_and_bad_indices(be, dtype, rows, vocab, top):
    x = logits_for(rows, vocab, 0, dtype, top)
    idx, val = teacher_for(rows, vocab, top, 12)
    val[0, top - 1] = math.nan
    val[1, 0] = math.inf
    x[2, vocab - 1] = math.nan
    x[3, vocab // 2] = math.inf
    val[4] = math.nan
    val[5, 1] = math.nan                               # of an entry that is missing: nobody looks at it
    idx[5, 1] = -1
    check_special_distill(be, x, idx, val, 1.0, nan_rows=(0, 1, 2, 3, 4))
    for bad in (vocab, -2):
        idx[6, top // 2] = bad
        loss, grad = be.distillation_loss(x, idx, val, reduction="none")
        with pytest.raises(IndexError):
            be.sync()
        idx[6, top // 2] = -1
        same, same_grad = be.distillation_loss(x, idx, val, reduction="none")
        be.sync()
        assert torch.equal(loss[5:], same[5:]) and torch.equal(grad[5:], same_grad[5:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(1500, 515), (40, 6007), (13, 50257)])
def test_score_gradient_where_the_token_is_an_alternative(be, dtype, rows, vocab):
    """One index in the list twice: the gradients of both outputs meet in one place of the row."""
    x = logits_for(rows, vocab, 0, dtype, 41)
    check_score_grad(be, x, x.float().argmax(1), 1.0, 9)


def test_captured_long_rows_replay_on_new_inputs(be):
    """Calls whose rows are cut into clusters of blocks, and with shared memory that has to be asked for."""
    x = logits_for(16, 50257, 0, torch.float32, 30)
    tokens = torch.arange(16, device="cuda")
    few, many = teacher_for(16, 50257, 64, 4), teacher_for(16, 50257, 700, 4)

    def calls():
        out = be.token_log_probs(x, tokens, top=200, entropy=True)
        grad = be.token_log_probs_bwd(x, tokens, out.stats, d_log_probs=out.log_probs, entropy=out.entropy, d_entropy=out.entropy,
                                      top_indices=out.top_indices, d_top=out.top_log_probs)
        return list(out) + [grad] + list(be.distillation_loss(x, *few)) + list(be.distillation_loss(x, *many, reduction="none"))
    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls()
    for round_ in range(3):
        x.copy_(logits_for(16, 50257, 0, torch.float32, 50 + round_))
        graph.replay()
        torch.cuda.synchronize()
        want = calls()
        be.sync()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_outputs_of_one_call_share_one_backward_pass(be, monkeypatch):
    """Gradients of two and three outputs that meet in one scalar: the logits are gone through once."""
    import minitensor_b200.nn as nn
    from minitensor_b200.tensor import Tensor
    passes = []
    inner = be.token_log_probs_bwd
    monkeypatch.setattr(be, "token_log_probs_bwd", lambda *a, **k: passes.append(sorted(n for n in k if k[n] is not None)) or inner(*a, **k))
    rng = np.random.default_rng(1)
    tokens = Tensor(rng.integers(0, 50, (3, 4)))
    x = Tensor(rng.standard_normal((3, 4, 50)).astype(np.float32), requires_grad=True)
    out = nn.token_log_probs(x, tokens, top=5, entropy=True)
    (out.log_probs + out.entropy).sum().backward()
    assert len(passes) == 1 and "d_log_probs" in passes[0] and "d_entropy" in passes[0] and "d_top" not in passes[0]
    out = nn.token_log_probs(x, tokens, top=5, entropy=True)
    (out.log_probs.sum() + out.entropy.sum() + out.top_log_probs.sum()).backward()
    assert len(passes) == 2 and all(n in passes[1] for n in ("d_log_probs", "d_entropy", "d_top"))
    out = nn.token_log_probs(x, tokens, top=5, entropy=True)
    out.top_log_probs.sum().backward()
    assert len(passes) == 3 and "d_top" in passes[2] and "d_log_probs" not in passes[2] and "d_entropy" not in passes[2]


def test_two_threads_with_a_backend_each(be):
    """Handles share nothing but the record of granted shared memory: calls from two threads at once, on two streams."""
    import threading
    from minitensor_b200.backend import Backend
    idx, val = teacher_for(16, 50257, 90, 5)
    tokens = torch.arange(16, device="cuda")
    xs = [logits_for(16, 50257, 0, torch.bfloat16, 70 + i) for i in range(2)]

    def calls(b, x, top):
        out = b.token_log_probs(x, tokens, top=top, entropy=True)
        grad = b.token_log_probs_bwd(x, tokens, out.stats, d_log_probs=out.log_probs, top_indices=out.top_indices, d_top=out.top_log_probs)
        return list(out) + [grad] + list(b.distillation_loss(x, idx, val))
    want = [[calls(be, x, top) for top in range(100, 160, 3)] for x in xs]
    be.sync()
    others = [Backend(0) for _ in xs]
    got, failed = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                got[i] = [calls(others[i], xs[i], top) for top in range(100, 160, 3)]
                others[i].sync()
        except Exception as e:  # reported below, in the test's own thread
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for a, b in zip(g, w):
            assert all(torch.equal(p, q) for p, q in zip(a, b) if p is not None)
    for b in others:
        b.close()

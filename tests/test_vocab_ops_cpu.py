"""Argument checks of the vocabulary operators (no device needed: every refusal comes before the library is called), and
their 64-bit test definitions against independent ones."""
import math

import pytest
import torch

import vocab_reference as ref


@pytest.fixture()
def host_be():
    """A backend object without a handle, on CPU tensors: calls get as far as the argument checks."""
    from minitensor_b200 import build, _lib
    from minitensor_b200.backend import Backend
    build.build()
    be = object.__new__(Backend)
    be.lib, be.device, be._h, be.launches = _lib.load(), torch.device("cpu"), None, 0
    be._bind_stream = lambda: None
    return be


X = torch.zeros(4, 50)
TOK = torch.zeros(4, dtype=torch.int64)
IDX, VAL = torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4, 3)


@pytest.mark.parametrize("call,error", [
    (lambda be: be.token_log_probs(X.double(), TOK), TypeError),
    (lambda be: be.token_log_probs(X.int(), TOK), TypeError),
    (lambda be: be.token_log_probs(X[0], TOK), ValueError),
    (lambda be: be.token_log_probs(X.T, torch.zeros(50, dtype=torch.int64)), ValueError),
    (lambda be: be.token_log_probs(X[:, ::2], TOK), ValueError),
    (lambda be: be.token_log_probs(X[:1].expand(4, 50), TOK), ValueError),
    (lambda be: be.token_log_probs(X, TOK[:3]), ValueError),
    (lambda be: be.token_log_probs(X, TOK.float()), TypeError),
    (lambda be: be.token_log_probs(X, TOK.short()), TypeError),
    (lambda be: be.token_log_probs(X, TOK, top=51), ValueError),
    (lambda be: be.token_log_probs(X, TOK, top=-1), ValueError),
    (lambda be: be.token_log_probs_bwd(X, TOK, torch.zeros(4)), ValueError),
    (lambda be: be.token_log_probs_bwd(X, TOK, torch.zeros(4, 2).double()), TypeError),
    (lambda be: be.token_log_probs_bwd(X, None, torch.zeros(4, 2), d_log_probs=torch.zeros(4)), ValueError),
    (lambda be: be.token_log_probs_bwd(X, TOK, torch.zeros(4, 2), d_entropy=torch.zeros(4)), ValueError),
    (lambda be: be.token_log_probs_bwd(X, TOK, torch.zeros(4, 2), d_top=VAL), ValueError),
    (lambda be: be.token_log_probs_bwd(X, TOK, torch.zeros(4, 2), d_top=VAL, top_indices=IDX[:, :2]), ValueError),
    (lambda be: be.token_log_probs_bwd(X, TOK, torch.zeros(4, 2), d_log_probs=torch.zeros(4).half()), TypeError),
    (lambda be: be.distillation_loss(X, IDX, VAL, reduction="average"), ValueError),
    (lambda be: be.distillation_loss(X, IDX[0], VAL[0]), ValueError),
    (lambda be: be.distillation_loss(X, IDX, VAL[:, :2]), ValueError),
    (lambda be: be.distillation_loss(X, VAL, VAL), TypeError),
    (lambda be: be.distillation_loss(X, IDX, VAL.double()), TypeError),
    (lambda be: be.distillation_loss(X, IDX, VAL, upstream_rows=torch.zeros(3)), ValueError),
    (lambda be: be.distillation_loss(X, IDX, VAL, stats=torch.zeros(4, 3)), ValueError),
    (lambda be: be.distillation_loss_bwd(X, IDX, VAL, torch.zeros(2, 2)), ValueError),
])
def test_refused_arguments(host_be, call, error):
    with pytest.raises(error):
        call(host_be)


def test_tensors_of_another_device_are_refused(host_be):
    host_be.device = torch.device("cuda", 0)
    with pytest.raises(ValueError, match="backend on"):
        host_be.token_log_probs(X, TOK)


def test_null_handle_is_refused(host_be):
    with pytest.raises(ValueError, match="null handle|CUDA tensors"):
        host_be.token_log_probs(X, None)


def test_gradient_buffers_follow_the_logits():
    from minitensor_b200.backend import Backend
    base = torch.zeros(1 + 5 * 24)
    for x in (base[:100].view(5, 20), base[1:101].view(5, 20), base[1:].view(5, 24)[:, :20], base[1:].view(5, 24)[:, 3:20]):
        g = Backend._grad_like(x, x.shape[0], x.shape[1], x.stride(0))
        assert g.shape == x.shape and g.stride() == x.stride() and (g.data_ptr() ^ x.data_ptr()) & 15 == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,seq,vocab", [(4, 300, 50), (7, 33, 1), (3, 3, 77), (5, 2, 24)])
def test_gradient_buffers_of_slices_are_no_larger_than_their_rows(dtype, rows, seq, vocab):
    """The last position of every sequence: the gradient holds these rows, not the whole of what they were taken from, and
    every row starts at its logits' offset within 16 bytes."""
    from minitensor_b200.backend import Backend
    for off in (0, 1):
        x = torch.zeros(rows * seq * vocab + off, dtype=dtype)[off:].view(rows, seq, vocab)[:, -1]
        g = Backend._grad_like(x, rows, vocab, x.stride(0))
        size, unit = g.element_size(), 16 // g.element_size()
        assert g.shape == x.shape and g.dtype == dtype and g.stride(1) == 1 and g.stride(0) >= vocab
        assert g.untyped_storage().nbytes() <= (rows * (vocab + unit) + unit) * size
        assert all((g[r].data_ptr() - x[r].data_ptr()) % 16 == 0 for r in range(rows))


def test_nn_refusals_come_before_the_device():
    import minitensor_b200.nn as nn
    from minitensor_b200.tensor import Tensor
    t = lambda x: Tensor(None, _buf=x)
    with pytest.raises(TypeError):
        nn.token_log_probs(t(X.double()), t(TOK))
    with pytest.raises(TypeError):
        nn.token_log_probs(t(X), t(TOK.float()))
    with pytest.raises(ValueError):
        nn.token_log_probs(t(X), t(TOK[:3]))
    with pytest.raises(ValueError):
        nn.distillation_loss(t(X), t(IDX), t(VAL), reduction="average")
    with pytest.raises(ValueError):
        nn.DistillationLoss(reduction="average")
    with pytest.raises(ValueError):
        nn.distillation_loss(t(X), t(IDX[:3]), t(VAL[:3]))
    with pytest.raises(TypeError):
        nn.distillation_loss(t(X), t(VAL), t(VAL))
    with pytest.raises(TypeError):
        nn.distillation_loss(t(X), t(IDX), t(VAL.double()))


def test_definitions_against_autograd():
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(5, 40, generator=gen, dtype=torch.float64, requires_grad=True)
    tokens = torch.tensor([3, 1, -100, 39, 0])
    live = tokens != -100
    t = 1.4
    lp = torch.log_softmax(x / t, 1)
    idx = ref.order64(x.detach(), 6)
    assert torch.equal(idx, x.topk(6).indices)
    d1, d2, d3 = torch.randn(5, generator=gen), torch.randn(5, generator=gen), torch.randn(5, 6, generator=gen)
    value = ((lp.gather(1, tokens.clamp(min=0)[:, None])[:, 0] * d1 - (lp.exp() * lp).sum(1) * d2 + (lp.gather(1, idx) * d3).sum(1)) * live).sum()
    got = ref.score_grad64(x.detach(), tokens, t, d1, d2, idx, d3, ignore_index=-100)
    assert torch.allclose(got, torch.autograd.grad(value, x)[0], atol=1e-12)
    val = torch.randn(5, 6, generator=gen)
    idx = idx.clone()
    idx[1] = -1
    idx[2, 3:] = -1
    q = torch.softmax(torch.where(idx >= 0, val.double() / t, torch.full_like(val, -1e30, dtype=torch.float64)), 1) * (idx >= 0)
    kl = t * t * (torch.special.xlogy(q, q) - q * torch.log_softmax(x / t, 1).gather(1, idx.clamp(min=0))).sum(1)
    loss, grad = ref.distill64(x.detach(), idx, val, t)
    assert torch.allclose(loss, kl, atol=1e-12) and loss[1] == 0
    assert torch.allclose(grad, torch.autograd.grad(kl.sum(), x)[0], atol=1e-12)
    empty = torch.full((1, 4), -math.inf)
    p, lp = ref.softmax64(empty, 1.0)
    assert not p.any() and (lp == -math.inf).all()

"""The dense operators at the ends of what their documentation allows.

Where a test's vectors hold small whole numbers, every product and every partial sum is a whole number below 2^24: exact in fp32
in any order, whether a sum is rounded or cut.  What remains of the error is what comes after the products."""
import numpy as np
import pytest
import torch

import apoe

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


@pytest.mark.parametrize("rows", [60, 200])
@pytest.mark.parametrize("scale", [1.407, -1.407, 1.44, 0.36, 0.9])
def test_gradients_of_logits_of_thousands(rows, scale):
    """Probabilities of logits from 50 000 to 85 000 (whole products, so exact): 2^-24 of such a logit is up to 5e-3 of each
    probability, ten times f16's rounding.  Column 63 of a gradient is the sum of the probabilities
    of the documents that are no row's target."""
    docs, dim = 300, 64
    g = gen(91)
    few = abs(scale) < 0.5                            # the same logits from larger products
    q = torch.full((rows, dim), 32.0, device=DEV)
    d = torch.full((docs, dim), 116.0 if few else 29.0, device=DEV)
    q[:, 62] = torch.randint(1, 4, (rows,), generator=g, device=DEV).float()
    d[:, 62] = torch.randint(0, 6, (docs,), generator=g, device=DEV).float()
    q[:, 63], d[:, 63] = 0.0, (torch.arange(docs, device=DEV) >= 20).float()
    t = torch.randint(0, 20, (rows,), generator=g, device=DEV).to(torch.int32)
    q, d = q.half(), d.half()
    exact = q.double() @ d.double().t()
    assert float(exact.max()) < 2 ** 24 and torch.equal(exact, exact.round())
    l = float(np.float32(scale)) * exact
    loss, lse = apoe.softmax_loss_forward(q, d, t, scale)
    want_lse = torch.logsumexp(l, 1)
    assert float((lse.double() - want_lse).abs().max()) <= 2.0 ** -23 * float(want_lse.abs().max()) + 2e-6
    at = l.gather(1, t.long()[:, None])
    others = torch.logsumexp(l.scatter(1, t.long()[:, None], -torch.inf) - at, 1)
    assert float((loss.double() - torch.nn.functional.softplus(others, threshold=60.0)).abs().max()) <= 2e-5
    dq, dd = apoe.softmax_loss_backward(q, d, t, loss, lse, torch.ones(rows, device=DEV), scale)
    # from lse as it is given; of each G: one rounding to f16, the exponent's fused product and sum (|exponent| below 64: 2^-18)
    # and exp2 (2^-21); the fp32 sum of at most 300 terms; the result's rounding
    p = torch.exp(l - lse.double()[:, None])[:, 20:]
    tol = 2 * U[torch.float16] + 2.0 ** -18 + 2.0 ** -21 + 300 * 2.0 ** -23
    s = float(np.float32(scale))
    want = s * p.sum(1)
    assert float(((dq[:, 63].double() - want) / want).abs().max()) <= tol
    want = s * 32.0 * p.sum(0)                        # column 0 of the queries is 32 throughout
    assert float(((dd[20:, 0].double() - want) / want).abs().max()) <= tol


def plain_rows(q, d, t, scale):
    l = float(np.float32(scale)) * (q.double() @ d.double().t())
    at = l.gather(1, t.long()[:, None])
    others = torch.logsumexp(l.scatter(1, t.long()[:, None], -torch.inf), 1)
    return l, torch.nn.functional.softplus(others - at[:, 0], threshold=60.0), torch.logsumexp(l, 1)


@pytest.mark.parametrize("rows", [40, 200])
@pytest.mark.parametrize("size", [2.0 ** 52, 2.0 ** 60])
def test_loss_of_logits_beyond_1e30(rows, size):
    """bf16 holds them, and fp32 their logits: rows whose documents are all far below zero have a loss like any other."""
    g = gen(92)
    q = (torch.rand(rows, 64, generator=g, device=DEV) + 0.5).bfloat16() * size
    d = -(torch.rand(300, 64, generator=g, device=DEV) + 0.5).bfloat16() * size
    t = torch.randint(0, 300, (rows,), generator=g, device=DEV).to(torch.int32)
    l, want_loss, want_lse = plain_rows(q, d, t, 1.0)
    assert float(l.max()) < -1e30 and float(l.min()) > -3e38
    loss, lse = apoe.softmax_loss_forward(q, d, t, 1.0)
    tol = float(l.abs().max()) * (64 + 8) * 2.0 ** -23           # 64 terms of one sign, and the roundings of the join
    assert float((loss.double() - want_loss).abs().max()) <= tol
    assert float((lse.double() - want_lse).abs().max()) <= tol
    assert float(want_loss.max()) > 100 * tol


@pytest.mark.parametrize("rows", [40, 200])
def test_ordinary_logits_from_a_tiny_scale(rows):
    """Products near 1e34 and a scale near 1e-34: the logits are ordinary."""
    g = gen(93)
    q = torch.randn(rows, 64, generator=g, device=DEV).bfloat16() * 2.0 ** 56
    d = torch.randn(300, 64, generator=g, device=DEV).bfloat16() * 2.0 ** 56
    t = torch.randint(0, 300, (rows,), generator=g, device=DEV).to(torch.int32)
    scale = 2.0 ** -113
    l, want_loss, want_lse = plain_rows(q, d, t, scale)
    assert 1.0 < float(l.abs().max()) < 100.0
    loss, lse = apoe.softmax_loss_forward(q, d, t, scale)
    most = float((q.double().abs() @ d.double().abs().t()).max()) * scale
    tol = 2 * most * (64 + 4) * 2.0 ** -23 + 1e-6
    assert float((loss.double() - want_loss).abs().max()) <= tol
    assert float((lse.double() - want_lse).abs().max()) <= tol + 2.0 ** -22 * float(want_lse.abs().max())


@pytest.mark.parametrize("rows", [40, 200])
@pytest.mark.parametrize("size", [2.0 ** 14, 2.0 ** 20, 2.0 ** 58])
def test_loss_of_large_logits_of_both_signs(rows, size):
    """Logits from 1e9 to 1e37 either way: a rounded maximum of them would be off by more than an exponential bears."""
    g = gen(94)
    q = torch.randn(rows, 64, generator=g, device=DEV).bfloat16() * size
    d = torch.randn(300, 64, generator=g, device=DEV).bfloat16() * size
    t = torch.randint(0, 300, (rows,), generator=g, device=DEV).to(torch.int32)
    for scale in (0.75, -1.3):
        l, want_loss, want_lse = plain_rows(q, d, t, scale)
        assert float(l.abs().max()) > 5 * size ** 2
        loss, lse = apoe.softmax_loss_forward(q, d, t, scale)
        tol = float((q.double().abs() @ d.double().abs().t()).max()) * abs(scale) * (64 + 8) * 2.0 ** -23
        assert float((loss.double() - want_loss).abs().max()) <= 2 * tol
        assert float((lse.double() - want_lse).abs().max()) <= 2 * tol
        assert float(want_loss.max()) > 100 * tol

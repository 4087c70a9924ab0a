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


def whole(rows, cols, g, dtype, share):
    """-1, 0 and 1, so few of them that sums stay small."""
    x = torch.randint(-1, 2, (rows, cols), generator=g, device=DEV).to(dtype)
    return x * (torch.rand(rows, cols, generator=g, device=DEV) < share).to(dtype)


@pytest.mark.parametrize("m,n,dim", [(3, 70, 1536), (150, 333, 1537), (300, 500, 4096), (5, 40, 16400), (140, 90, 65536 + 128 * 5 + 7), (2, 9, 1 << 20), (130, 33, 1 << 20)])
def test_scores_of_long_rows(m, n, dim):
    """Many groups of scale bytes, each block with a scale of its own; the scores are whole numbers below 2^24, so equal."""
    g = gen(dim + m)
    ld = (dim + 15) // 16 * 16
    blocks = -(-dim // 128)
    qa = torch.zeros(m, ld, device=DEV).to(torch.float8_e4m3fn)[:, :dim]
    qb = torch.zeros(n, ld, device=DEV).to(torch.float8_e4m3fn)[:, :dim]
    a, b = (whole(r, dim, g, torch.float32, min(1.0, 30.0 / dim ** 0.5)) for r in (m, n))
    qa.copy_(a), qb.copy_(b)
    sa, sb = (torch.randint(127, 131, (r, blocks), generator=g, device=DEV).to(torch.uint8) for r in (m, n))
    va, vb = (x.double() * torch.exp2(s.double() - 127.0).repeat_interleave(128, 1)[:, :dim] for x, s in ((a, sa), (b, sb)))
    assert float((va.abs() @ vb.abs().t()).max()) < 2 ** 20
    assert torch.equal(apoe.scaled_scores(qa, sa, qb, sb).double(), va @ vb.t())
    apoe.dense_check_status()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,docs,dim", [(32, 256, 1536), (130, 300, 1544), (200, 700, 4096), (20, 100, 8200), (129, 200, 65536), (4, 90, 65536)])
def test_loss_and_gradients_of_long_rows(rows, docs, dim, dtype):
    """Whole logits, so of the loss only the join's errors remain, and of the gradients the roundings of G and of the result."""
    g = gen(dim + rows)
    ld = (dim + 7) // 8 * 8
    q, d = (torch.zeros(r, ld, dtype=dtype, device=DEV)[:, :dim] for r in (rows, docs))
    share = min(1.0, 3.0 / dim ** 0.5)
    q.copy_(whole(rows, dim, g, dtype, share)), d.copy_(whole(docs, dim, g, dtype, share))
    t = torch.randint(0, docs, (rows,), generator=g, device=DEV).to(torch.int32)
    t[rows // 2] = -1
    scale, live = 0.5, t >= 0
    l, want_loss, want_lse = plain_rows(q, d, t.clamp(min=0), scale)
    assert float(l.abs().max()) < 64
    loss, lse = apoe.softmax_loss_forward(q, d, t, scale)
    assert float((loss.double() - want_loss)[live].abs().max()) <= 64 * 2.0 ** -22 + 1e-6      # roundings at the size of a logit
    assert float((lse.double() - want_lse)[live].abs().max()) <= 64 * 2.0 ** -22 + 1e-6
    grad = torch.rand(rows, generator=g, device=DEV) + 0.5
    dq, dd = apoe.softmax_loss_backward(q, d, t, loss, lse, grad, scale)
    apoe.dense_check_status()
    p = torch.exp(l - want_lse[:, None])
    p[torch.arange(rows, device=DEV), t.clamp(min=0).long()] = torch.expm1(-want_loss)
    p *= torch.where(live, grad.double(), 0.0)[:, None]
    u = U[dtype]
    # each G: a rounding, and its exponential's error (lse and the exponent, 2^-17 at |logit| 64); sums of at most 700 terms
    near = u + 2.0 ** -17 + 2.0 ** -19 + 700 * 2.0 ** -23
    small = 2.0 ** -25 if dtype == torch.float16 else 0.0                                       # f16's smallest step, halved
    for got, want, mass, other in ((dq, scale * (p @ d.double()), scale * (p.abs() @ d.double().abs()), d),
                                   (dd, scale * (p.t() @ q.double()), scale * (p.abs().t() @ q.double().abs()), q)):
        low = small + small * 2.0 ** -13 * 1.5 * scale * other.double().abs().sum(0, keepdim=True)   # G at 2^14: steps of 2^-24
        assert bool(((got.double() - want).abs() <= mass * near * (1 + u) + u * want.abs() + low).all())
    assert not dq[rows // 2].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gradients_of_certain_and_hopeless_rows(dtype):
    """Losses from 1e-12 to 100 in one batch, every element of both gradients against its own bound: a rounding of each G, its
    exponential's and the loss's relative error, the result's rounding; f16 holds G in steps of 2^-24 where the batch's largest
    is near 2^14."""
    dim, docs, scale = 64, 300, 50.0
    g = gen(13)
    d = torch.randn(docs, dim, generator=g, device=DEV)
    d = d / d.norm(dim=1, keepdim=True)
    t = torch.arange(64, device=DEV, dtype=torch.int32)
    q, d = torch.cat([d[:32], -d[32:64]]).to(dtype), d.to(dtype)
    loss, lse = apoe.softmax_loss_forward(q, d, t, scale)
    l, want_loss, want_lse = plain_rows(q, d, t, scale)
    assert float(want_loss.min()) < 1e-9 and float(want_loss.max()) > 50
    dq, dd = apoe.softmax_loss_backward(q, d, t, loss, lse, torch.ones(64, device=DEV), scale)
    p = torch.exp(l - want_lse[:, None])
    p[torch.arange(64, device=DEV), t.long()] = torch.expm1(-want_loss)
    most = float((q.double().abs() @ d.double().abs().t()).max()) * scale
    eps = 4 * most * (dim + 4) * 2.0 ** -23 + 4e-6           # two logits and lse in every exponent, the loss's in the target's
    u = U[dtype]
    small = 2.0 ** -25 if dtype == torch.float16 else 0.0
    for got, want, mass, other in ((dq, scale * (p @ d.double()), scale * (p.abs() @ d.double().abs()), d),
                                   (dd, scale * (p.t() @ q.double()), scale * (p.abs().t() @ q.double().abs()), q)):
        low = small + small * 2.0 ** -13 * scale * other.double().abs().sum(0, keepdim=True)
        assert bool(((got.double() - want).abs() <= mass * (u + eps + 300 * 2.0 ** -23) * (1 + u) + u * want.abs() + low).all())

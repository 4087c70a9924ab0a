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

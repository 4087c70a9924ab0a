"""Dense operators that follow each other without a pause: each kernel may start while the one before it is still writing what
it reads (scale bytes, the gradients' factor, targets).  Buffers are used over and over with other contents."""
import pytest
import torch

import apoe

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("m,n,dim", [(1, 60, 1024), (40, 900, 640), (300, 2000, 200), (1000, 4000, 1024)])
def test_rows_quantised_just_before_are_scored_with_their_own_scales(m, n, dim):
    g = torch.Generator(device=DEV).manual_seed(m + n)
    rounds, blocks, ld = 12, -(-dim // 128), (dim + 15) // 16 * 16
    sources = [tuple(torch.randn(r, dim, generator=g, device=DEV) * 2.0 ** (5 * (i % 4) - 7) for r in (m, n)) for i in range(rounds)]
    out = torch.empty(rounds, m, n, device=DEV)
    q = [torch.empty(r, ld, dtype=torch.uint8, device=DEV) for r in (m, n)]
    s = [torch.empty(r, blocks, dtype=torch.uint8, device=DEV) for r in (m, n)]
    rows = [apoe.ScaledRows(r, q[k].data_ptr(), ld, s[k].data_ptr(), blocks) for k, r in enumerate((m, n))]

    def run(i, pause):
        for k, r in enumerate((m, n)):
            apoe._check(apoe.lib().ap_quantize_rows_device(0, r, dim, 0, sources[i][k].data_ptr(), dim, q[k].data_ptr(), ld, s[k].data_ptr(), blocks, stream()))
            pause()
        apoe._check(apoe.lib().ap_scaled_scores_device(0, dim, rows[0], rows[1], 1.0, 0, out[i].data_ptr(), n, stream()))
        pause()

    for i in range(rounds):
        run(i, torch.cuda.synchronize)
    want = out.clone()
    assert len({float(x.abs().max()) for x in want}) == rounds
    for _ in range(20):
        out.zero_()
        for i in range(rounds):
            run(i, lambda: None)
        assert torch.equal(out, want)


@pytest.mark.parametrize("rows,docs,dim", [(20, 300, 128), (300, 900, 256), (1200, 3000, 128)])
def test_gradients_of_one_call_take_their_own_factor(rows, docs, dim):
    """Calls whose gradients differ in size by many powers of two, back to back: the factor of G is written just before the kernel
    that reads it starts, in the workspace that the call before has used."""
    g = torch.Generator(device=DEV).manual_seed(rows)
    q, d = ((torch.randn(r, dim, generator=g, device=DEV) * 0.3).bfloat16() for r in (rows, docs))
    targets = [torch.randint(0, docs, (rows,), generator=g, device=DEV).to(torch.int32) for _ in range(8)]
    grads = [torch.rand(rows, generator=g, device=DEV) * 2.0 ** (9 * i - 40) for i in range(8)]

    def step(i, pause):
        loss, lse = apoe.softmax_loss_forward(q, d, targets[i], 2.0)
        pause()
        out = (loss, lse, *apoe.softmax_loss_backward(q, d, targets[i], loss, lse, grads[i], 2.0))
        pause()
        return out

    want = [step(i, torch.cuda.synchronize) for i in range(8)]
    for _ in range(10):
        got = [step(i, lambda: None) for i in range(8)]
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    apoe.dense_check_status()

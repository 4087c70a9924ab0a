"""Dense operators that follow each other without a pause: each kernel may start while the one before it is still writing what
it reads (scale bytes, the gradients' factor, targets).  Buffers are used over and over with other contents.  And the first
calls of a process inside a capture."""
import os
import subprocess
import sys

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


FIRST = """
import sys
sys.path.insert(0, sys.argv[1])
import torch, apoe
g = torch.Generator(device="cuda").manual_seed(1)
q, d = (torch.randn(n, 128, generator=g, device="cuda").half() for n in (200, 500))
t = torch.randint(0, 500, (200,), generator=g, device="cuda").to(torch.int32)
grad = torch.full((200,), 0.5, device="cuda")
def step():
    loss, lse = apoe.softmax_loss_forward(q, d, t, 0.1)
    dq, dd = apoe.softmax_loss_backward(q, d, t, loss, lse, grad, 0.1)
    q8, sq = apoe.quantize_rows(q)
    d8, sd = apoe.quantize_rows(d)
    return loss, lse, dq, dd, sq, sd, apoe.scaled_scores(q8, sq, d8, sd)
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    held = step()
for x in held: x.zero_()
graph.replay()
torch.cuda.synchronize()
got = [x.clone() for x in held]
assert all(torch.equal(a, b) for a, b in zip(got, step()))
apoe.dense_check_status()
print("same")
"""


def test_first_calls_of_a_process_may_be_captured():
    """Nothing has to have run before: a process whose first dense calls are made inside a capture."""
    r = subprocess.run([sys.executable, "-c", FIRST, os.path.dirname(apoe.__file__)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stderr[-2000:]

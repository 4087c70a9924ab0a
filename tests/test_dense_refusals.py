"""What the dense operators refuse, on the host and before any device work (no GPU needed)."""
import ctypes as C

import pytest
import torch

import apoe

F16, BF16, F32 = 1, 2, 0
GOOD = 1 << 12       # an aligned address that is never read


@pytest.fixture(scope="module")
def L():
    import build as apoe_build
    apoe_build.build()
    return apoe.lib()


def refused(code, text, rc):
    assert rc == code, rc
    assert text in apoe.lib().ap_last_error().decode(), apoe.lib().ap_last_error()


def test_quantize_refuses(L):
    def call(rows=4, dim=256, kind=F32, src=GOOD, ld=256, q=GOOD, ldq=256, s=GOOD, lds=2):
        return L.ap_quantize_rows_device(0, rows, dim, kind, src, ld, q, ldq, s, lds, None)
    refused(1, "type 3", call(kind=3))
    refused(1, "0 values", call(dim=0))
    refused(1, "null", call(src=None))
    refused(1, "null", call(q=None))
    refused(1, "null", call(s=None))
    refused(1, "stride", call(ld=255))
    refused(1, "stride", call(ldq=255))
    refused(1, "stride", call(lds=1))
    refused(1, "aligned", call(src=GOOD + 2))
    assert call(rows=0) == 0


def test_scores_refuse(L):
    def call(m=4, n=4, dim=256, qa=GOOD, lda=256, sa=GOOD, lsa=2, kind=F32, out=GOOD, ldo=4, qb=GOOD, ldb=256):
        a, b = apoe.ScaledRows(m, qa, lda, sa, lsa), apoe.ScaledRows(n, qb, ldb, GOOD, 2)
        return L.ap_scaled_scores_device(0, dim, a, b, 1.0, kind, out, ldo, None)
    refused(1, "null", L.ap_scaled_scores_device(0, 256, None, None, 1.0, F32, GOOD, 4, None))
    refused(1, "output type", call(kind=7))
    refused(1, "0 values", call(dim=0))
    refused(1, "null", call(qa=None))
    refused(1, "null", call(sa=None))
    refused(1, "null", call(out=None))
    refused(1, "stride", call(lda=240))
    refused(1, "stride", call(lsa=1))
    refused(1, "stride", call(ldo=3))
    refused(1, "16-byte", call(qa=GOOD + 8))
    refused(1, "16-byte", call(ldb=264))
    refused(1, "aligned to its type", call(out=GOOD + 2))
    refused(4, "2^30", call(m=(1 << 30) + 1))
    refused(4, "in one call", call(m=1 << 30, n=1 << 30, ldo=1 << 30))
    assert call(m=0) == 0 and call(n=0) == 0


def test_loss_refuses(L):
    size = C.c_size_t(0)
    def forward(rows=8, docs=64, dim=64, kind=BF16, q=GOOD, ldq=64, d=GOOD, ldd=64, t=GOOD, scale=1.0, loss=GOOD, ws=GOOD, nbytes=1 << 40):
        return L.ap_softmax_loss_forward_device(0, rows, docs, dim, kind, q, ldq, d, ldd, t, scale, loss, GOOD, ws, nbytes, None)
    def backward(rows=8, docs=64, dim=64, kind=BF16, q=GOOD, grad=GOOD, gq=GOOD, ldgq=64, gd=GOOD, ldgd=64, scale=1.0, ws=GOOD):
        return L.ap_softmax_loss_backward_device(0, rows, docs, dim, kind, q, 64, GOOD, 64, GOOD, scale, GOOD, GOOD, grad, gq, ldgq, gd, ldgd, ws,
                                                 1 << 40, None)
    for call in (forward, backward):
        refused(1, "f16 or bf16", call(kind=F32))
        refused(1, "none may be 0", call(rows=0))
        refused(1, "none may be 0", call(docs=0))
        refused(1, "none may be 0", call(dim=0))
        refused(1, "null", call(q=None))
        refused(1, "null", call(ws=None))
        refused(1, "stride", call(dim=65))
        refused(1, "16-byte", call(q=GOOD + 2))
        refused(1, "finite", call(scale=float("nan")))
        refused(1, "finite", call(scale=float("inf")))
        refused(4, "2^20", call(rows=(1 << 20) + 1))
    refused(1, "16-byte", forward(ldq=68))
    refused(1, "null", forward(t=None))
    refused(1, "null", forward(loss=None))
    refused(1, "bytes", forward(nbytes=16))
    refused(1, "256-byte", forward(ws=GOOD + 16))
    refused(1, "null", backward(grad=None))
    refused(1, "null", backward(gd=None))
    refused(1, "stride", backward(ldgq=63))
    refused(1, "8-byte", backward(gq=GOOD + 2))
    refused(1, "none may be 0", L.ap_softmax_loss_workspace(0, 0, 4, 4, 0, size))
    refused(1, "null", L.ap_softmax_loss_workspace(0, 4, 4, 4, 0, None))
    assert L.ap_softmax_loss_workspace(0, 4, 4, 4, 0, size) == 0 and size.value > 0


def test_wait_probe_refuses_long_waits(L):
    refused(1, "4096", L.ap_debug_dense_wait_timeout(0, 4097, None))


def test_python_layer_refuses_what_is_not_on_the_device():
    x = torch.zeros(4, 64)
    for call in (lambda: apoe.quantize_rows(x), lambda: apoe.quantize_rows(x.double()),
                 lambda: apoe.softmax_loss_forward(x.half(), x.half(), torch.zeros(4, dtype=torch.int32)),
                 lambda: apoe.scaled_scores(x, x, x, x)):
        with pytest.raises(apoe.ApoeError) as e:
            call()
        assert e.value.code == 1

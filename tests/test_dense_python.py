"""What the Python layer of the dense operators settles before any device work (no GPU needed)."""
import warnings

import pytest
import torch

import apoe


class Matrix:
    """As much of a CUDA matrix as the argument checks look at."""
    is_cuda = True
    requires_grad = False

    def __init__(self, rows, cols, dtype):
        self.shape, self.dtype, self.device = (rows, cols), dtype, torch.device("cuda", 0)

    def stride(self):
        return self.shape[1], 1

    def dim(self):
        return 2

    def get_device(self):
        return 0


@pytest.mark.parametrize("rows", [1 << 32, (1 << 32) + 5, 1 << 40])
def test_counts_beyond_32_bits_are_refused(rows):
    """The library takes 32-bit counts: 2^32 + 5 rows must not become 5."""
    e4m3, half = torch.float8_e4m3fn, torch.float16
    few, scale, targets = Matrix(3, 16, e4m3), Matrix(3, 1, torch.uint8), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: apoe.quantize_rows(Matrix(rows, 16, torch.float32)),
                 lambda: apoe.scaled_scores(Matrix(rows, 16, e4m3), scale, few, scale),
                 lambda: apoe.scaled_scores(few, scale, Matrix(rows, 16, e4m3), scale),
                 lambda: apoe.softmax_loss_forward(Matrix(rows, 16, half), Matrix(3, 16, half), targets),
                 lambda: apoe.softmax_loss_forward(Matrix(3, 16, half), Matrix(rows, 16, half), targets),
                 lambda: apoe.softmax_loss_forward(Matrix(3, rows, half), Matrix(3, rows, half), targets)):
        with pytest.raises(apoe.ApoeError) as e:
            call()
        assert e.value.code == 4 and "2^32" in str(e.value)


def test_a_loss_that_records_no_gradients_says_so():
    """The loss takes no part in autograd: inputs that require gradients would lose them silently where it is one term of a sum."""
    targets = torch.zeros(4, dtype=torch.int32)
    plain, wants = torch.zeros(4, 64).half(), torch.zeros(4, 64).half().requires_grad_()

    def call(queries, docs):
        with pytest.raises(apoe.ApoeError):            # host tensors: the call itself is refused
            apoe.softmax_loss_forward(queries, docs, targets)

    for pair in ((wants, plain), (plain, wants), (wants, wants)):
        with pytest.warns(UserWarning, match="softmax_loss_backward"):
            call(*pair)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        call(plain, plain)
        call(wants.detach(), wants.detach())
        with torch.no_grad():
            call(wants, wants)

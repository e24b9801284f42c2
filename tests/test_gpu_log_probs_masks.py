"""Log probabilities of rows that are masked with large finite values, or stand far from 0, against the plain 64-bit form.

The bounds are those of test_gpu_log_probs.check: the exponents are of x - M, so that neither a mask nor a row's offset is in them."""
import pytest
import torch

from test_gpu_log_probs import BF16, F16, F32, check

pytestmark = pytest.mark.gpu


def rows(vocab, dtype, low):
    """Rows of ordinary logits with masks of ``low`` in front, behind, everywhere, nearly everywhere, by whole batches of a warp and at every other entry."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(8, vocab, device="cuda", generator=g) * 3
    at = torch.arange(vocab, device="cuda")
    kept = torch.stack([at >= vocab // 2, at < vocab // 3, at < 0, at == vocab - 1, at == 0, at // 512 % 2 == 1, at % 2 == 1, at >= 0])
    return torch.where(kept, x, torch.full_like(x, low)).to(dtype)


@pytest.mark.parametrize("vocab", [33, 5000, 50257, 128256])
@pytest.mark.parametrize("dtype,low", [(F32, torch.finfo(F32).min), (BF16, torch.finfo(BF16).min), (F16, torch.finfo(F16).min), (F32, -2.5e38), (F32, -1e38), (F32, -1e30), (F32, -1e10), (BF16, -1e30),
                                       (BF16, -1e9), (F32, -1e6)])
def test_finite_masks(pkg, vocab, dtype, low):
    x = rows(vocab, dtype, low)
    check(pkg, x, torch.tensor([vocab - 1, 0, 5, vocab - 1, 0, 7, 1, 3], device="cuda").int(), 20)
    check(pkg, x, torch.full((8,), vocab // 2 + 1, device="cuda").int(), 0)


@pytest.mark.parametrize("offset", [30.0, -100.0, 1000.0, -1e4, 1e6, 1e8, 3e38, -3e38])
def test_rows_far_from_zero(pkg, offset):
    """The logits' own FP32 or BF16 values are the input: at 1e8 a row has few different ones, at 3e38 one."""
    for dtype in (F32, BF16):
        g = torch.Generator(device="cuda").manual_seed(3)
        x = (torch.randn(5, 40000, device="cuda", generator=g) * 2.5 + offset).to(dtype)
        check(pkg, x, torch.arange(5, device="cuda").int() * 777, 20)
        check(pkg, torch.full((2, 9000), offset, device="cuda").to(dtype), torch.tensor([0, 8999], device="cuda").int(), 4)


def test_both_ends_of_the_range(pkg):
    """Differences that pass FP32's range count as none: the largest entry has everything."""
    big = torch.finfo(F32).max
    x = torch.full((2, 3000), -big, device="cuda")
    x[0, 1234] = big
    x[1, 5], x[1, 6] = big, 0.5 * big
    lp, h, ids, values = pkg.log_probs(x, torch.tensor([1234, 5], device="cuda").int(), 2)
    assert (lp == 0).all() and (h == 0).all() and ids.tolist() == [[1234, 0], [5, 6]]
    assert (values[:, 0] == 0).all() and values[0, 1] == -float("inf") and values[1, 1] == -0.5 * big

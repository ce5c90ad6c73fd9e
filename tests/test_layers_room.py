"""CPU checks of the room that the loss over a vocabulary asks for: half a GB of what stands for its logits, whatever their number."""

import ctypes

import pytest

from selective_attention_b200 import _lib

SIZES = [(1, 1 << 24), (128, 1 << 24), (300, 1 << 24), (4096, 1 << 20), (16384, 50304), (131072, 50304), (262144, 50304), (1 << 20, 50304), (65536, 128000),
         (41000, 4097), (1 << 20, 300), (1 << 24, 257), (1 << 24, 1), (1 << 24, 1 << 24)]


def _loss(tokens, vocab, width, dtype, reduction=2):
    p = _lib.LinearLoss()
    for name, value in dict(struct_bytes=ctypes.sizeof(p), product=dtype, x_dtype=dtype, weight_dtype=dtype, reduction=reduction, tokens=tokens, vocab=vocab,
                            width=width, ignore_index=-100, x=256, x_stride=width, weight=256, weight_stride=width, targets=256, lse=256, count=256, loss=256,
                            dloss=256, dx=256, dweight=256, dx_sums=256, dweight_sums=256).items():
        setattr(p, name, value)
    return p


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("tokens,vocab", SIZES)
def test_the_loss_takes_half_a_gigabyte_for_its_logits(tokens, vocab, dtype):
    lib, width = _lib.load(), 8
    p = _loss(tokens, vocab, width, dtype)
    # beside the logits: copies of both operands (three parts of fp32), sums of both gradients, the targets in order and their gradients' parts, a
    # dozen numbers a token, and what of a product's last tiles is cut among the clusters
    parts = 6 if dtype == 0 else 2
    beside = (tokens + vocab) * width * (parts + 4) + tokens * (8 + 48 + 2 * width * 4 // 4) + 4 * vocab + 2 * 74 * 256 * 256 * 4 + (1 << 20)
    assert 0 < lib.sa_linear_loss_forward_bytes(ctypes.byref(p)) <= (512 << 20) + beside
    assert 0 < lib.sa_linear_loss_backward_bytes(ctypes.byref(p)) <= (512 << 20) + beside
    if lib.sa_linear_loss_prefers_train(ctypes.byref(p)):
        # and half tiles' sums, a 16th or, of three parts, a 48th
        assert 0 < lib.sa_linear_loss_train_bytes(ctypes.byref(p)) <= (512 << 20) * 17 // 16 + beside


def test_tables_of_which_few_tokens_exponentials_fit_are_computed_again():
    """Sums of a table's gradient over runs of few tokens would cost more than the product that they save."""
    lib = _lib.load()
    prefers = lambda *a: lib.sa_linear_loss_prefers_train(ctypes.byref(_loss(*a)))  # noqa: E731
    assert prefers(16384, 50304, 1024, 1) == 1 and prefers(16384, 128000, 1024, 1) == 1 and prefers(2048, 50304, 768, 1) == 1
    assert prefers(16384, 1 << 20, 1024, 1) == 0 and prefers(4096, 1 << 21, 64, 1) == 0 and prefers(512, 1 << 24, 8, 0) == 0

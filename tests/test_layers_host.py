"""CPU checks of layer norm, the embedding and the loss: the C entries refuse bad arguments before any launch, the Python calls name
what is wrong."""

import ctypes

import pytest
import torch

from selective_attention_b200 import _lib, layers

OK_NORM = dict(x_dtype=0, branch_dtype=0, y_dtype=0, weight_dtype=0, width=64, rows=4, eps=1e-5, x=256, x_stride=64, y=256)
OK_EMBEDDING = dict(weight_dtype=0, y_dtype=0, tokens=4, vocab=9, width=64, scale=1.0, idx=256, weight=256, weight_stride=64, y=256)
OK_LOSS = dict(product=1, x_dtype=1, weight_dtype=1, reduction=2, tokens=4, vocab=9, width=64, ignore_index=-100, x=256, x_stride=64, weight=256,
               weight_stride=64, targets=256, lse=256, count=256, loss=256, workspace=256, workspace_bytes=1 << 40)


def _of(struct, ok, **changes):
    p = struct()
    p.struct_bytes = ctypes.sizeof(struct)
    for name, value in {**ok, **changes}.items():
        setattr(p, name, value)
    return ctypes.byref(p)


def test_structs_match_the_header_layout():
    assert ctypes.sizeof(_lib.Norm) == 200 and _lib.Norm.x.offset == 40 and _lib.Norm.stream.offset == 192
    assert ctypes.sizeof(_lib.Embedding) == 112 and _lib.Embedding.idx.offset == 32
    assert ctypes.sizeof(_lib.LinearLoss) == 168 and _lib.LinearLoss.ignore_index.offset == 32 and _lib.LinearLoss.targets.offset == 72


@pytest.mark.parametrize("status,changes", [
    (1, dict(struct_bytes=8)), (1, dict(x_dtype=3)), (1, dict(y_dtype=-1)), (1, dict(width=0)), (1, dict(rows=0)), (1, dict(eps=-1.0)),
    (1, dict(eps=float("nan"))), (1, dict(x=None)), (1, dict(y=None)), (1, dict(branch=256)), (1, dict(sum=256)), (1, dict(x_stride=-1)),
    (2, dict(width=16385)), (3, dict(x=258)), (3, dict(weight=257)), (7, dict(rows=1 << 31))])
def test_norm_forward_refuses(status, changes):
    assert _lib.load().sa_norm_forward(_of(_lib.Norm, OK_NORM, **changes)) == status


def test_norm_backward_refuses():
    lib, ok = _lib.load(), {**OK_NORM, "dy": 256, "dy_stride": 64, "dx": 256, "stats": 256}
    for status, changes in ((1, dict(dy=None)), (1, dict(dx=None)), (1, dict(stats=None)), (1, dict(dweight=256)), (3, dict(dx=257)),
                            (4, dict(weight=256, dweight=256, workspace=256, workspace_bytes=255)), (1, dict(weight=256, dweight=256)),
                            (3, dict(dbias=256, workspace=264, workspace_bytes=1 << 30))):
        assert lib.sa_norm_backward(_of(_lib.Norm, ok, **changes)) == status, changes
    assert lib.sa_norm_backward_bytes(_of(_lib.Norm, ok)) == 0
    assert lib.sa_norm_backward_bytes(_of(_lib.Norm, ok, dweight=256)) >= 64 * 4
    assert lib.sa_norm_backward_bytes(_of(_lib.Norm, ok, struct_bytes=0)) == 0


@pytest.mark.parametrize("status,changes", [
    (1, dict(struct_bytes=8)), (1, dict(weight_dtype=5)), (1, dict(tokens=0)), (1, dict(vocab=0)), (1, dict(width=-1)), (1, dict(idx=None)),
    (1, dict(weight=None)), (1, dict(y=None)), (1, dict(weight_stride=-64)), (3, dict(idx=260)), (3, dict(weight=257)), (7, dict(width=(1 << 20) + 1))])
def test_embedding_forward_refuses(status, changes):
    assert _lib.load().sa_embedding_forward(_of(_lib.Embedding, OK_EMBEDDING, **changes)) == status


def test_embedding_backward_refuses():
    lib, ok = _lib.load(), {**OK_EMBEDDING, "dy": 256, "dy_stride": 64, "dweight": 256, "workspace": 256, "workspace_bytes": 1 << 20}
    for status, changes in ((1, dict(dy=None)), (1, dict(dweight=None)), (1, dict(workspace=None)), (3, dict(workspace=8)), (4, dict(workspace_bytes=100))):
        assert lib.sa_embedding_backward(_of(_lib.Embedding, ok, **changes)) == status, changes
    assert lib.sa_embedding_backward_bytes(_of(_lib.Embedding, ok)) >= 4 * 8 + 10 * 4 + 2 * 64 * 4


@pytest.mark.parametrize("status,changes", [
    (1, dict(struct_bytes=8)), (1, dict(product=3)), (1, dict(reduction=3)), (1, dict(tokens=0)), (1, dict(vocab=0)), (1, dict(width=0)),
    (1, dict(x=None)), (1, dict(targets=None)), (1, dict(lse=None)), (1, dict(count=None)), (1, dict(loss=None)), (1, dict(workspace=None)),
    (2, dict(product=0)), (3, dict(x=257)), (3, dict(targets=260)), (3, dict(workspace=128)), (4, dict(workspace_bytes=16)), (7, dict(tokens=1 << 25)),
    (7, dict(width=(1 << 16) + 1))])
def test_loss_forward_refuses(status, changes):
    assert _lib.load().sa_linear_loss_forward(_of(_lib.LinearLoss, OK_LOSS, **changes)) == status


def test_loss_backward_refuses():
    lib, ok = _lib.load(), {**OK_LOSS, "dloss": 256, "dx": 256}
    for status, changes in ((1, dict(dloss=None)), (1, dict(dx=None)), (3, dict(dx=257)), (4, dict(workspace_bytes=16))):
        assert lib.sa_linear_loss_backward(_of(_lib.LinearLoss, ok, **changes)) == status, changes
    assert lib.sa_linear_loss_backward_bytes(_of(_lib.LinearLoss, ok, struct_bytes=0)) == 0


def test_loss_with_its_gradients_refuses():
    lib, ok = _lib.load(), {**OK_LOSS, "dx_sums": 256, "dweight_sums": 256, "dloss": 256, "dx": 256}
    for status, changes in ((2, dict(reduction=0)), (2, dict(product=2)), (1, dict(dx_sums=None, dweight_sums=None)), (3, dict(dx_sums=258)), (1, dict(loss=None)),
                            (1, dict(count=None)), (4, dict(workspace_bytes=16)), (1, dict(targets=None))):
        assert lib.sa_linear_loss_train(_of(_lib.LinearLoss, ok, **changes)) == status, changes
    for status, changes in ((2, dict(reduction=0)), (1, dict(dloss=None)), (1, dict(dx=None)), (1, dict(dx_sums=None)), (1, dict(dweight=256, dweight_sums=None)),
                            (3, dict(dx=257))):
        assert lib.sa_linear_loss_scale(_of(_lib.LinearLoss, ok, **changes)) == status, changes
    large = {**ok, "tokens": 16384, "vocab": 50304, "width": 1024, "x_stride": 1024, "weight_stride": 1024}
    assert lib.sa_linear_loss_prefers_train(_of(_lib.LinearLoss, large)) == 1
    for changes in (dict(tokens=64), dict(reduction=0), dict(product=2, x_dtype=2, weight_dtype=2), dict(struct_bytes=0)):
        assert lib.sa_linear_loss_prefers_train(_of(_lib.LinearLoss, large, **changes)) == 0, changes


def test_the_loss_takes_less_room_than_its_logits():
    """At 16,384 tokens of 50,304 words the logits are 1.6 GB in 16 bits."""
    lib, big = _lib.load(), {**OK_LOSS, "tokens": 16384, "vocab": 50304, "width": 1024, "x_stride": 1024, "weight_stride": 1024, "dx": 256, "dweight": 256, "dx_sums": 256, "dweight_sums": 256}
    assert 0 < lib.sa_linear_loss_train_bytes(_of(_lib.LinearLoss, big)) < 800e6
    assert 0 < lib.sa_linear_loss_forward_bytes(_of(_lib.LinearLoss, big)) < 120e6
    assert 0 < lib.sa_linear_loss_backward_bytes(_of(_lib.LinearLoss, big)) < 700e6


def test_calls_on_cpu_tensors_are_refused():
    x, w, t = torch.randn(4, 32), torch.randn(9, 32), torch.zeros(4, dtype=torch.long)
    for call in (lambda: layers.layer_norm(x), lambda: layers.add_layer_norm(x, x), lambda: layers.embedding(t, w), lambda: layers.linear_cross_entropy(x, w, t)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="reduction"):
        layers.linear_cross_entropy(x, w, t, reduction="max")

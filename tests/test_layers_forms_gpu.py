"""Layer norm, the embedding and the loss over a vocabulary where torch, a mask or a size asks something unusual of them."""

import pytest
import torch

from selective_attention_b200 import layers

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _calls():
    """Every call by itself: what it takes that may have a derivative, and the call of these."""
    x, branch, w = (torch.randn(4, 32, device="cuda") for _ in range(3))
    p, b = torch.ones(32, device="cuda"), torch.zeros(32, device="cuda")
    t = torch.tensor([0, 1, 2, 3], device="cuda")
    return {
        "layer_norm": ([x, p, b], layers.layer_norm), "add_layer_norm": ([x, branch, p, b], layers.add_layer_norm),
        "embedding": ([w], lambda a: layers.embedding(t, a)), "linear_cross_entropy": ([x, w], lambda a, c: layers.linear_cross_entropy(a, c, t)),
        "linear_cross_entropy of each": ([x, w], lambda a, c: layers.linear_cross_entropy(a, c, t, reduction="none")),
    }


@pytest.mark.parametrize("name", ["layer_norm", "add_layer_norm", "embedding", "linear_cross_entropy", "linear_cross_entropy of each"])
def test_tangents_and_batches_of_a_transform_are_refused(name):
    """Dropped, a tangent would read as a derivative of zero."""
    inputs, call = _calls()[name]
    want = call(*inputs)
    for i in range(len(inputs)):
        for wants in (False, True):
            args = [a.clone().requires_grad_(wants) for a in inputs]
            with torch.autograd.forward_ad.dual_level():
                args[i] = torch.autograd.forward_ad.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(*args)
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                    call(*args)
                again = call(*inputs)                       # others are taken as ever
                assert all(torch.equal(a, b) for a, b in zip(again if isinstance(again, tuple) else [again], want if isinstance(want, tuple) else [want]))
        with pytest.raises(RuntimeError):
            torch.func.jvp(lambda a: call(*inputs[:i], a, *inputs[i + 1:]), (inputs[i],), (torch.ones_like(inputs[i]),))
        with pytest.raises(RuntimeError):
            torch.func.vmap(lambda a: call(*inputs[:i], a, *inputs[i + 1:]))(inputs[i][None])

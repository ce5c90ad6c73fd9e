"""The decoder with its embedding, norms and loss by the library's kernels where targets are ignored and modules have hooks."""

import pytest
import torch

from selective_attention_b200 import decoder

pytestmark = pytest.mark.gpu


def _pair(**kw):
    torch.manual_seed(1)
    plain = decoder.SelectiveDecoder(vocab_size=97, n_layers=2, d_model=128, n_heads=2, loss_chunk=128, **kw).cuda()
    own = decoder.SelectiveDecoder(vocab_size=97, n_layers=2, d_model=128, n_heads=2, own_layers=True, **kw).cuda()
    own.load_state_dict(plain.state_dict())
    idx, targets = (t.cuda() for t in decoder.synthetic_batch(2, 130, 97, 96, torch.Generator("cpu").manual_seed(2)))
    return plain, own, idx, targets


def _run(model, idx, targets):
    model.zero_grad()
    loss = model(idx, targets)
    loss.backward()
    return float(loss.detach()), {n: p.grad.clone() for n, p in model.named_parameters()}


def test_hooks_of_blocks_run():
    _, own, idx, targets = _pair()
    want, wanted = _run(own, idx, targets)
    seen = []
    for i, block in enumerate(own.h):
        block.register_forward_pre_hook(lambda module, args, i=i: seen.append(("before", i, args[0].shape)))
        block.register_forward_hook(lambda module, args, out, i=i: seen.append(("behind", i, out[0].shape)))
    loss, grads = _run(own, idx, targets)
    assert seen == [(when, i, (2, 130, 128)) for i in range(2) for when in ("before", "behind")]
    assert abs(loss - want) <= 1e-6 * want
    for name, grad in grads.items():                        # the attention's sums are not in a fixed order
        assert float((grad - wanted[name]).norm()) <= 1e-4 * float(wanted[name].norm()), name
    own.h[0].register_forward_hook(lambda module, args, out: (out[0], 0 * out[1]))       # what a hook returns is what goes on
    assert abs(_run(own, idx, targets)[0] - want) > 1e-4 * want


@pytest.mark.parametrize("name", ["wte", "ln_f", "h.0.ln_1", "h.1.ln_2"])
@pytest.mark.parametrize("kind", ["register_forward_pre_hook", "register_forward_hook", "register_full_backward_hook", "register_full_backward_pre_hook"])
def test_hooks_of_what_is_not_called_are_refused(name, kind):
    plain, own, idx, targets = _pair()
    getattr(plain.get_submodule(name), kind)(lambda *args: None)
    plain(idx, targets)
    handle = getattr(own.get_submodule(name), kind)(lambda *args: None)
    with pytest.raises(RuntimeError, match="hooks would not run"):
        own(idx, targets)
    handle.remove()
    assert torch.isfinite(own(idx, targets))


@pytest.mark.parametrize("ignored", [1, 100, 260])
def test_ignored_targets_weigh_the_same_either_way(ignored):
    plain, own, idx, targets = _pair()
    targets.view(-1)[:ignored] = -100
    want, wanted = _run(plain, idx, targets)
    loss, grads = _run(own, idx, targets)
    assert abs(loss - want) <= 1e-5 * want                  # fp32 on both sides
    for name, grad in grads.items():
        assert float((grad - wanted[name]).norm()) <= 2e-4 * float(wanted[name].norm()), name

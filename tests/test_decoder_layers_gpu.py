"""The decoder with its embedding, norms and loss by the library's kernels, against the one with torch's operators: the same loss and
gradients up to roundings."""

import pytest
import torch

from selective_attention_b200 import decoder

pytestmark = pytest.mark.gpu


def _pair(**kw):
    torch.manual_seed(1)
    plain = decoder.SelectiveDecoder(**kw).cuda()
    own = decoder.SelectiveDecoder(own_layers=True, **kw).cuda()
    own.load_state_dict(plain.state_dict())
    return plain, own


def _run(model, idx, tgt, autocast):
    model.zero_grad()
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
        loss = model(idx, tgt)
    loss.backward()
    return loss.detach(), {n: p.grad.float() for n, p in model.named_parameters()}


@pytest.mark.parametrize("layers", [0, 1, 3])
def test_decoder_with_own_layers_equals_the_plain_one(layers):
    plain, own = _pair(vocab_size=97, n_layers=layers, d_model=128, n_heads=2, loss_chunk=128)
    gen = torch.Generator("cpu").manual_seed(2)
    idx, tgt = (t.cuda() for t in decoder.synthetic_batch(2, 300, 97, 96, gen))
    loss, grads = _run(own, idx, tgt, False)
    want, wanted = _run(plain, idx, tgt, False)
    assert abs(float(loss) - float(want)) < 1e-5 * float(want)
    for name, grad in grads.items():                       # fp32 on both sides
        assert grad.shape == wanted[name].shape and float((grad - wanted[name]).norm() / wanted[name].norm()) < 2e-4, name
    loss, grads = _run(own, idx, tgt, True)
    assert loss.dtype == torch.float32 and abs(float(loss) - float(want)) < 2e-2
    for name, grad in grads.items():                       # bf16 products
        assert float((grad - wanted[name]).norm() / wanted[name].norm()) < 5e-2, name


def test_an_accumulated_step_and_a_replayed_one():
    _, own = _pair(vocab_size=320, n_layers=2, d_model=128, n_heads=2)
    gen = torch.Generator("cpu").manual_seed(3)
    idx, tgt = (t.cuda() for t in decoder.synthetic_batch(2, 130, 320, 0, gen))
    _, once = _run(own, idx, tgt, True)
    own.zero_grad()
    for _ in range(2):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            own(idx, tgt).backward()
    for name, p in own.named_parameters():                 # the attention's sums are not in a fixed order
        assert float((p.grad.float() - 2 * once[name]).norm() / once[name].norm()) < 2e-2, name
    own.zero_grad(set_to_none=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    params = list(own.parameters())

    def step():
        with torch.autocast("cuda", dtype=torch.bfloat16, cache_enabled=False):
            loss = own(idx, tgt)
        return loss.detach(), torch.autograd.grad(loss, params)

    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grads = step()
    idx2, tgt2 = (t.cuda() for t in decoder.synthetic_batch(2, 130, 320, 0, gen))
    idx.copy_(idx2)
    tgt.copy_(tgt2)
    graph.replay()
    want, wanted = step()
    assert abs(float(loss) - float(want)) < 1e-3
    for a, b in zip(grads, wanted):
        assert float((a.float() - b.float()).norm() / b.float().norm()) < 2e-2

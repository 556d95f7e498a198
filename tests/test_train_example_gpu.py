"""The masked-MSA training example: the loss falls, and one step's gradients are those of the same
model in float32 torch operations.

Tolerance of the gradients: two chains of 16-bit operations (embedding, projections, attention,
output, head: about ten roundings of 2^-9 relative and the attention's own, below 1e-2 relative
2-norm) against float32 from the same 16-bit weights: 3e-2 relative 2-norm a parameter.
"""
import importlib.util
import math
import os

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


def example():
    path = os.path.join(ROOT, 'examples', 'train_masked_msa.py')
    spec = importlib.util.spec_from_file_location('train_masked_msa', path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def plain_loss(model, ex, msa, labels):
    """The model's loss in float32, without the library."""
    half = lambda p: p.to(model.dtype).float()
    N, S = msa.shape
    C, H = model.project.shape[0], model.heads
    x = half(model.tokens[msa.long()] * math.sqrt(C))
    at = torch.arange(S, device=msa.device)
    offsets = (at[None] - at[:, None]).clamp(-ex.FAR, ex.FAR) + ex.FAR
    bias = half(model.offsets[offsets]).permute(2, 0, 1)
    q, k, v, gate = (x @ half(model.project)).view(N, S, 4, H, C // H).permute(2, 0, 3, 1, 4)
    p = (q @ k.transpose(-1, -2) * (C // H) ** -.5 + bias).softmax(-1)
    y = (p @ v) * torch.sigmoid(gate + half(model.gate_bias)[None, :, None])
    x = x + y.permute(0, 2, 1, 3).reshape(N, S, C) @ half(model.out)
    logits = x @ half(model.head).t() + half(model.head_bias)
    return torch.nn.functional.cross_entropy(logits.view(-1, ex.CLASSES), labels.view(-1).long(),
                                             ignore_index=-1)


def test_gradients_of_a_step(cuda_device):
    ex = example()
    torch.manual_seed(1)
    model = ex.Model()
    g = torch.Generator(device='cuda').manual_seed(1)
    msa, labels = ex.masked_msa(9, 40, g)
    params = list(model.parameters())
    loss = model(msa, labels)
    got = torch.autograd.grad(loss, params)
    plain = plain_loss(model, ex, msa, labels)
    want = torch.autograd.grad(plain, params)
    assert abs(loss.item() - plain.item()) < 2e-2 * plain.item()
    for (name, _), a, b in zip(model.named_parameters(), got, want):
        off = float((a - b).norm() / b.norm())
        assert off < 3e-2, '%s: %.3g' % (name, off)
    assert ex.b200.device_status() == 0


def test_loss_falls_and_norm_is_that_of_the_gradients(cuda_device):
    ex = example()
    history = ex.train(steps=30, seqs=32, res=64)
    losses = [a for a, _ in history]
    assert abs(losses[0] - math.log(ex.CLASSES)) < .5  # an untrained head
    assert losses[-1] < .7 * losses[0] and all(math.isfinite(n) for _, n in history)

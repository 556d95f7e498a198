"""Masked-MSA training on the B200 kernels: a row-attention block between an embedding and a head.

  python examples/train_masked_msa.py [--steps 100] [--seqs 64] [--res 128]

Synthetic sequences, each with a residue of its own at most positions, are masked at 15 % of their
positions, and the model learns to fill them in from the rest of the sequence:

  tokens -> embed (b200.embed, scaled) -> q, k, v, gate (torch.matmul)
         -> gated row attention with a bias from embedded residue offsets
            (b200.volta_mma_gated / volta_mma_gated_bwd, b200.embed / embed_bwd)
         -> residual -> cross entropy of the 23 classes at the masked positions
            (b200.linear_xent / linear_xent_bwd)
  gradients -> clipped by their global norm (b200.clip_grad_norm) -> Adam on float32 weights

The library's operators join torch's autograd through the small Functions below.
"""
import argparse
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, 'colabfold-legacy-kernels_b200', 'src'))

from colabfold_legacy_kernels import b200  # noqa: E402

CLASSES, MASK, FAR = 23, 22, 32  # 20 residues, unknown, gap, mask; offsets clipped at +-32


class Embed(torch.autograd.Function):
    """Rows of a float32 table in the compute type."""

    @staticmethod
    def forward(ctx, ids, table, scale, dtype):
        ctx.ids, ctx.rows, ctx.scale = ids, table.shape[0], scale
        return b200.embed(ids, table, scale=scale, out_dtype=dtype)

    @staticmethod
    def backward(ctx, dout):
        return None, b200.embed_bwd(ctx.ids, dout.contiguous(), ctx.rows, scale=ctx.scale), None, None


class GatedAttention(torch.autograd.Function):
    """Row attention with a shared pair bias and a sigmoid gate."""

    @staticmethod
    def forward(ctx, q, k, v, gate, gate_bias, bias, kmask):
        ctx.scale = q.shape[-1] ** -0.5
        y, lse = b200.volta_mma_gated(q, k, v, gate, gate_bias, bias, kmask, scale=ctx.scale)
        ctx.save_for_backward(q, k, v, gate, gate_bias, bias, kmask, y, lse)
        return y

    @staticmethod
    def backward(ctx, dy):
        saved = ctx.saved_tensors
        dq, dk, dv, dgate, dgate_bias, dbias = b200.volta_mma_gated_bwd(
            *saved[:7], saved[7], dy.contiguous(), saved[8], scale=ctx.scale)
        return (dq, dk, dv, dgate, dgate_bias.to(saved[4].dtype), dbias.to(saved[5].dtype), None)


class LinearXent(torch.autograd.Function):
    """Loss a position of the classes x w^T + bias."""

    @staticmethod
    def forward(ctx, x, w, bias, labels):
        loss, lse = b200.linear_xent(x, w, labels, bias)
        ctx.save_for_backward(x, w, bias, labels, lse)
        return loss

    @staticmethod
    def backward(ctx, dloss):
        x, w, bias, labels, lse = ctx.saved_tensors
        dx, dw, db = b200.linear_xent_bwd(x, w, labels, lse, dloss.contiguous(), bias)
        return dx, dw, db, None


class Model(torch.nn.Module):
    def __init__(self, channels=128, heads=4, dtype=torch.bfloat16):
        super().__init__()
        self.heads, self.dtype = heads, dtype
        normal = lambda *s, std: torch.nn.Parameter(torch.randn(*s, device='cuda') * std)
        self.tokens = normal(CLASSES, channels, std=1 / math.sqrt(channels))
        self.offsets = normal(2 * FAR + 1, heads, std=.1)
        self.project = normal(channels, 4 * channels, std=1 / math.sqrt(channels))
        self.gate_bias = normal(heads, channels // heads, std=.1)
        self.out = normal(channels, channels, std=1 / math.sqrt(channels))
        self.head, self.head_bias = normal(CLASSES, channels, std=.02), normal(CLASSES, std=.01)

    def forward(self, msa, labels):
        N, S = msa.shape
        C, H, half = self.project.shape[0], self.heads, lambda p: p.to(self.dtype)
        x = Embed.apply(msa, self.tokens, math.sqrt(C), self.dtype)
        at = torch.arange(S, device=msa.device, dtype=torch.int32)
        offsets = (at[None] - at[:, None]).clamp(-FAR, FAR) + FAR
        bias = Embed.apply(offsets, self.offsets, 1.0, self.dtype).permute(2, 0, 1).contiguous()
        q, k, v, gate = (x @ half(self.project)).view(N, S, 4, H, C // H).permute(2, 0, 3, 1, 4)
        kmask = torch.ones(N, S, dtype=torch.uint8, device=msa.device)
        y = GatedAttention.apply(q.contiguous(), k.contiguous(), v.contiguous(), gate.contiguous(),
                                 half(self.gate_bias), bias, kmask)
        x = x + y.permute(0, 2, 1, 3).reshape(N, S, C) @ half(self.out)
        loss = LinearXent.apply(x, half(self.head), half(self.head_bias), labels)
        return loss.sum() / (labels >= 0).sum()


def masked_msa(seqs, res, generator):
    """Sequences of one residue with three tenths of the positions changed; (masked tokens, labels),
    labels -1 where nothing is masked."""
    rand = lambda: torch.rand(seqs, res, generator=generator, device='cuda')
    own = torch.randint(0, 20, (seqs, 1), generator=generator, device='cuda')
    other = torch.randint(0, 20, (seqs, res), generator=generator, device='cuda')
    msa = torch.where(rand() < .7, own, other)
    masked = rand() < .15
    return (torch.where(masked, MASK, msa).int(), torch.where(masked, msa, -1).int())


def train(steps=100, seqs=64, res=128, lr=3e-3, max_norm=1.0, seed=0):
    """[(loss, gradient norm)] of the steps."""
    torch.manual_seed(seed)
    generator = torch.Generator(device='cuda').manual_seed(seed)
    model = Model()
    params = list(model.parameters())
    adam = torch.optim.Adam(params, lr=lr)
    history = []
    for _ in range(steps):
        adam.zero_grad()
        loss = model(*masked_msa(seqs, res, generator))
        loss.backward()
        norm = b200.clip_grad_norm([p.grad for p in params], max_norm)
        adam.step()
        history.append((loss.detach(), norm))
    return [(float(a), float(b)) for a, b in history]


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument('--steps', type=int, default=100)
    ap.add_argument('--seqs', type=int, default=64)
    ap.add_argument('--res', type=int, default=128)
    a = ap.parse_args()
    for i, (loss, norm) in enumerate(train(a.steps, a.seqs, a.res)):
        print('step %3d  loss %.4f  gradient norm %.4f' % (i, loss, norm))


if __name__ == '__main__':
    main()

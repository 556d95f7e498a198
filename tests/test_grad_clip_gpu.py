"""The global gradient norm and clipping on the B200 against the float64 restatement.

Tolerances. The sum of squares is float64: sums of up to 2^24 terms within 2^-29 relative. norm:
its rounding to float32, 2^-24 (2^-23 with the square root's and the scale's). Outputs: the factor
takes three float32 roundings after the norm (sum with eps, quotient, product with scale) and the
element's product one: 6 2^-24 relative, then the 16-bit rounding (u, or 2^-25 absolute below
float16's normal range; bf16 has float32's).
"""
import numpy as np
import pytest
import torch

from oracle import tokens as ot
from oracle.numerics import round_to

pytestmark = pytest.mark.gpu

TD = {'f16': torch.float16, 'bf16': torch.bfloat16, 'f32': torch.float32}
U = {'f16': 2.0 ** -11, 'bf16': 2.0 ** -8, 'f32': 0.0}


def b200():
    from colabfold_legacy_kernels import b200 as m
    return m


def make(sizes, kinds, d, amp=1.0, seed=0, offset=0):
    """Host values and tensors; `offset` elements into their storage (any alignment)."""
    rng = np.random.default_rng(seed + sum(sizes))
    host = [round_to(rng.standard_normal(n) * amp, k) for n, k in zip(sizes, kinds)]
    out = []
    for i, (a, k) in enumerate(zip(host, kinds)):
        o = (offset * (i + 1)) % 9
        buf = torch.zeros(len(a) + o, dtype=TD[k], device=d)
        buf[o:] = torch.tensor(np.asarray(a, np.float32), device=d).to(TD[k])
        out.append(buf[o:])
    return host, out


def close(host, norm, outs, max_norm, scale, kinds, eps=1e-6):
    wn, wo = ot.clip(host, max_norm, scale, eps)
    assert abs(norm.item() - wn) <= 2.0 ** -23 * wn
    for got, want, k in zip(outs, wo, kinds):
        g = got.double().cpu().numpy()
        tol = (6 * 2.0 ** -24 + U[k]) * np.abs(want) + (2.0 ** -25 if k == 'f16' else 1e-44)
        assert (np.abs(g - want) <= tol).all()


SIZES = [[1], [7, 0, 8, 9], [4095, 16384, 16385, 3], [100003], [33] * 50,
         [1, 2, 3, 5, 8, 13, 21, 34, 1000, 70000]]


@pytest.mark.parametrize('offset', [0, 1, 4])
@pytest.mark.parametrize('kinds', [['f32'], ['bf16'], ['f16'], ['f32', 'bf16', 'f16']])
@pytest.mark.parametrize('sizes', SIZES, ids=lambda s: '%dx%d' % (len(s), max(s)))
def test_clip(sizes, kinds, offset, cuda_device):
    m = b200()
    kinds = [kinds[i % len(kinds)] for i in range(len(sizes))]
    for max_norm, scale in ((.5, 1.0), (.25, 1 / 64.), (1e9, 1.0)):
        host, grads = make(sizes, kinds, cuda_device, offset=offset)
        # into buffers of their own at other alignments, the gradients left alone
        outs = [torch.zeros(g.numel() + 1, dtype=g.dtype, device=g.device)[1:] for g in grads]
        norm = m.clip_grad_norm(grads, max_norm, scale=scale, out=outs)
        close(host, norm, outs, max_norm, scale, kinds)
        assert all(np.array_equal(g.double().cpu().numpy(), a) for g, a in zip(grads, host))
        # the same bits in place
        n2 = m.clip_grad_norm(grads, max_norm, scale=scale)
        assert torch.equal(n2, norm) and all(torch.equal(a, b) for a, b in zip(grads, outs))
        # into float32
        host, grads = make(sizes, kinds, cuda_device, offset=offset)
        wide = [torch.zeros(g.numel(), device=g.device) for g in grads]
        n3 = m.clip_grad_norm(grads, max_norm, scale=scale, out=wide)
        assert torch.equal(n3, norm)
        close(host, n3, wide, max_norm, scale, ['f32'] * len(sizes))


def test_more_tensors_than_a_launch_takes(cuda_device):
    sizes = [1 + i % 37 for i in range(2500)]
    kinds = [('f32', 'bf16')[i % 2] for i in range(2500)]
    host, grads = make(sizes, kinds, cuda_device)
    norm = b200().clip_grad_norm(grads, 1.0)
    close(host, norm, grads, 1.0, 1.0, kinds)


def test_sum_of_squares_and_shards(cuda_device):
    m = b200()
    host, grads = make([5000, 31, 70001], ['f32'] * 3, cuda_device)
    total = sum(float((a * a).sum()) for a in host)
    got = m.grad_sumsq(grads)
    assert got.dtype == torch.float64 and abs(got.item() - total) <= 2.0 ** -29 * total
    # two shards clipped by their common sum, as two ranks would
    parts = m.grad_sumsq(grads[:1]) + m.grad_sumsq(grads[1:])
    norms = [m.clip_grad_norm(p, .5, sumsq=parts) for p in (grads[:1], grads[1:])]
    assert torch.equal(norms[0], norms[1])
    close(host, norms[0], grads, .5, 1.0, ['f32'] * 3)


def test_range_and_values_that_are_not_finite(cuda_device):
    m = b200()
    for amp in (1e25, 1e-30):  # squares beyond float32's range
        for kind in ('f32', 'bf16'):
            host, grads = make([1000, 40], [kind] * 2, cuda_device, amp=amp)
            norm = m.clip_grad_norm(grads, amp, eps=0.0)
            close(host, norm, grads, amp, 1.0, [kind] * 2, eps=0.0)
    _, grads = make([10, 10], ['f32', 'f16'], cuda_device)
    grads[1][3] = float('inf')
    norm = m.clip_grad_norm(grads, 1.0)
    assert torch.isinf(norm) and (grads[0] == 0).all() and torch.isnan(grads[1][3])
    _, grads = make([10, 10], ['f32', 'f16'], cuda_device)
    grads[0][3] = float('nan')
    norm = m.clip_grad_norm(grads, 1.0)
    assert torch.isnan(norm) and all(torch.isnan(g).all() for g in grads)
    assert (m.clip_grad_norm([torch.zeros(5, device=cuda_device)], 1.0) == 0)
    assert (m.clip_grad_norm([], 1.0) == 0)
    zeros = [torch.ones(5, device=cuda_device)]
    m.clip_grad_norm(zeros, 0.0)
    assert (zeros[0] == 0).all()


def test_past_32_bits(cuda_device):
    """One tensor of more than 2^31 elements (bf16, 4.3 GB), its last ones counted and scaled."""
    n = 2 ** 31 + 12345
    g = torch.zeros(n, dtype=torch.bfloat16, device=cuda_device)
    g[-3:] = 4.0
    g[5] = 1.0
    norm = b200().clip_grad_norm([g], 3.5, eps=0.0)
    assert norm.item() == 7.0 and (g[-3:] == 2.0).all() and g[5] == .5 and (g[-99:-3] == 0).all()


def test_another_stream(cuda_device):
    host, grads = make([70001, 9], ['f32', 'bf16'], cuda_device)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        norm = b200().clip_grad_norm(grads, .5)
    s.synchronize()
    close(host, norm, grads, .5, 1.0, ['f32', 'bf16'])


def test_refusals(cuda_device):
    m, d = b200(), cuda_device
    g = torch.ones(4, 4, device=d)
    for bad in (lambda: m.clip_grad_norm([g.t()[:, 1:]], 1.0), lambda: m.clip_grad_norm([g.int()], 1.0),
                lambda: m.clip_grad_norm([g.cpu()], 1.0), lambda: m.clip_grad_norm([g], -1.0),
                lambda: m.clip_grad_norm([g], float('nan')),
                lambda: m.clip_grad_norm([g], 1.0, scale=0.0),
                lambda: m.clip_grad_norm([g], 1.0, eps=-1.0),
                lambda: m.clip_grad_norm([g], 1.0, out=[]),
                lambda: m.clip_grad_norm([g], 1.0, out=[g[0]]),
                lambda: m.clip_grad_norm([g], 1.0, out=[g.half()]),
                lambda: m.clip_grad_norm([g], 1.0, sumsq=g[0, :1]),
                lambda: m.grad_sumsq([g.double()])):
        with pytest.raises(ValueError):
            bad()
    assert (g == 1).all()


def test_sum_of_squares_of_few_elements(cuda_device):
    """The squares of 16 bytes of float32 are added in float32: three roundings, 3 2^-24 relative; of 16-bit
    types they are exact and added in three; all else is float64 (2^-50 here)."""
    m = b200()
    rng = np.random.default_rng(2)
    for kind in ('f32', 'bf16', 'f16'):
        for n in (4, 8, 12, 40, 9):
            for _ in range(40):
                a = round_to(rng.uniform(.5, 2, n), kind)
                t = torch.tensor(np.asarray(a, np.float32), device=cuda_device).to(TD[kind])
                want = float((a.astype(np.float64) ** 2).sum())
                assert abs(m.grad_sumsq([t]).item() - want) <= (3 * 2.0 ** -24 + 2.0 ** -50) * want


def test_autograd_sees_what_was_written(cuda_device):
    """Tensors that a call writes count as changed in place; those it only reads do not."""
    m = b200()
    p = torch.randn(64, device=cuda_device, requires_grad=True)
    y = p * 2
    z = (y * y).sum()  # y is saved
    m.grad_sumsq([y.detach()])
    wide = torch.empty(64, device=cuda_device)
    v, o = y._version, wide._version
    m.clip_grad_norm([y.detach()], .5, out=[wide])
    assert y._version == v and wide._version > o
    m.clip_grad_norm([y.detach()], .5)
    assert y._version > v
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        z.backward()
    with torch.inference_mode():
        t = torch.ones(8, device=cuda_device)
    m.clip_grad_norm([t], .5)  # has no version
    assert abs(t.norm().item() - .5) < 1e-5

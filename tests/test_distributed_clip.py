"""Gradients sharded over CPU ranks (gloo, world size 2) are clipped by the norm of all of them: the
sums of squares are all-reduced. The per-rank arithmetic is the CPU restatement here."""
import datetime
import os

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from colabfold_legacy_kernels import distributed as cd
from oracle import tokens as ot
from test_distributed import _free_port


def _grads():
    rng = np.random.default_rng(0)
    return [torch.tensor(rng.standard_normal(n)) for n in (5, 1, 40, 17)]


def _sumsq(grads):
    return torch.tensor([sum(float((g * g).sum()) for g in grads)], dtype=torch.float64)


def _clip(grads, max_norm, *, sumsq, scale=1.0):
    norm = scale * float(sumsq.sqrt())
    for g in grads:
        g *= scale * min(1.0, max_norm / (norm + 1e-6))
    return norm


def _rank_main(rank, world, port, results):
    os.environ.update(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port))
    dist.init_process_group('gloo', rank=rank, world_size=world,
                            timeout=datetime.timedelta(seconds=60))
    try:
        mine = _grads()[2 * rank:2 * rank + 2]
        norm = cd.clip_grad_norm(mine, .5, sumsq=_sumsq, clip=_clip, scale=.25)
        results[rank] = (norm, [g.numpy() for g in mine])
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize('world', [1, 2])
def test_sharded_norm(world):
    want_norm, want = ot.clip([g.numpy() for g in _grads()], .5, scale=.25)
    if world == 1:
        grads = _grads()
        results = {0: (cd.clip_grad_norm(grads, .5, sumsq=_sumsq, clip=_clip, scale=.25),
                       [g.numpy() for g in grads])}
    else:
        results = mp.get_context('spawn').Manager().dict()
        mp.start_processes(_rank_main, args=(world, _free_port(), results), nprocs=world,
                           join=True, start_method='spawn')
    got = [g for rank in range(world) for g in results[rank][1]]
    assert all(abs(results[r][0] - want_norm) < 1e-12 for r in range(world))
    for a, b in zip(got, want):
        np.testing.assert_allclose(a, b, atol=1e-12)

"""Embedding lookup and its gradient on the B200 against the float64 restatement.

Tolerances. Lookup: one float32 product and one rounding, so equal bits to the same two steps in
numpy. Gradient: a row's sum of n float32 terms in any order is within n 2^-24 times the sum of
their magnitudes, and the scaling adds two roundings: (n + 2) 2^-24 scale sum |dout|.
"""
import numpy as np
import pytest
import torch

from oracle import tokens as ot
from oracle.numerics import round_to

pytestmark = pytest.mark.gpu

TD = {'f16': torch.float16, 'bf16': torch.bfloat16, 'f32': torch.float32}
IDS = {32: torch.int32, 64: torch.int64}


def b200():
    from colabfold_legacy_kernels import b200 as m
    return m


def make_ids(rng, T, V, kind):
    if kind == 'one':  # a single row takes every token
        return np.full(T, V // 2)
    if kind == 'none':
        return np.full(T, -1)
    ids = rng.integers(0, max(V, 1), T) if kind == 'uniform' else (
        V * rng.random(T) ** 6).astype(np.int64)
    return np.where(rng.random(T) < .1, rng.choice([-100, -1, V, 2 ** 31 - 1], T), ids)


def dev(a, dt, d):
    return torch.tensor(np.asarray(a, np.float32), device=d).to(TD[dt])


SIZES = [(1, 1, 8), (1, 23, 256), (7, 5, 1), (33, 2, 129), (300, 21, 12), (1000, 65, 128),
         (1025, 257, 24), (2049, 1000, 40), (4000, 513, 6)]


@pytest.mark.parametrize('bits', [32, 64])
@pytest.mark.parametrize('dt,out', [('f16', 'f16'), ('bf16', 'bf16'), ('f32', 'f32'),
                                    ('f32', 'bf16'), ('f32', 'f16')])
@pytest.mark.parametrize('T,V,C', SIZES)
def test_embed(T, V, C, dt, out, bits, cuda_device):
    rng = np.random.default_rng(T + V + C)
    ids, table = make_ids(rng, T, V, 'uniform'), round_to(rng.standard_normal((V, C)), dt)
    scale = np.float32(np.sqrt(C) * 1.1)
    got = b200().embed(torch.tensor(ids, device=cuda_device).to(IDS[bits]),
                       dev(table, dt, cuda_device), scale=float(scale), out_dtype=TD[out])
    assert got.shape == (T, C) and got.dtype == TD[out]
    ok = (ids >= 0) & (ids < V)
    want = np.where(ok[:, None], table.astype(np.float32)[np.where(ok, ids, 0)] * scale,
                    np.float32(0))
    assert torch.equal(got.cpu(), torch.tensor(want).to(TD[out]))


def test_embed_keeps_shape_and_unaligned_tables(cuda_device):
    rng = np.random.default_rng(3)
    table = dev(rng.standard_normal(8 * 16 + 1), 'bf16', cuda_device)[1:].view(8, 16)
    ids = torch.tensor(rng.integers(0, 8, (3, 5, 2)), device=cuda_device)
    assert table.data_ptr() % 16 and torch.equal(b200().embed(ids, table), table[ids])
    assert b200().embed(ids[:0], table).shape == (0, 5, 2, 16)
    assert (b200().embed(ids, table[:0]) == 0).all()  # no row at all


def grad_close(ids, dout, V, scale, got, C):
    want = ot.embed_bwd(ids, dout, V, scale)
    n = ot.embed_bwd(ids, np.ones((len(ids), 1)), V, 1.0)
    bound = (n + 2) * 2.0 ** -24 * ot.embed_bwd(ids, np.abs(dout), V, abs(scale))
    got = got.cpu().numpy().astype(np.float64)
    assert got.shape == (V, C) and (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize('kind', ['uniform', 'skewed', 'one', 'none'])
@pytest.mark.parametrize('dt', ['f16', 'bf16', 'f32'])
@pytest.mark.parametrize('T,V,C', SIZES)
def test_embed_bwd(T, V, C, dt, kind, cuda_device):
    rng = np.random.default_rng(T + V + C)
    ids, dout = make_ids(rng, T, V, kind), round_to(rng.standard_normal((T, C)), dt)
    got = b200().embed_bwd(torch.tensor(ids, device=cuda_device).to(IDS[32 + 32 * (T % 2)]),
                           dev(dout, dt, cuda_device), V, scale=1.5)
    grad_close(ids, dout, V, 1.5, got, C)


@pytest.mark.parametrize('T,V,C', [(70001, 65, 16), (20000, 300001, 8), (5000, 2 ** 21 + 3, 4),
                                   (30011, 50001, 264), (131072, 23, 256)])
def test_embed_bwd_many(T, V, C, cuda_device):
    rng = np.random.default_rng(T)
    for kind in ('skewed', 'uniform'):
        ids = make_ids(rng, T, V, kind)
        dout = round_to(rng.standard_normal((T, C)), 'bf16')
        tids = torch.tensor(ids, device=cuda_device).int()
        tdout = dev(dout, 'bf16', cuda_device)
        got = b200().embed_bwd(tids, tdout, V)
        grad_close(ids, dout, V, 1.0, got, C)
        assert torch.equal(got, b200().embed_bwd(tids, tdout, V))  # the same bits


@pytest.mark.parametrize('T,V,C', [(40000, 2000, 128), (40000, 2000, 130), (6400, 3201, 128),
                                   (6400, 3200, 128)])
@pytest.mark.parametrize('kind', ['one', 'few', 'uniform'])
def test_embed_bwd_rows_without_a_token_get_zeros(T, V, C, kind, cuda_device):
    """Few tokens' rows of many: every other row has to be written all the same."""
    rng = np.random.default_rng(V)
    ids = make_ids(rng, T, V, 'one' if kind == 'one' else 'uniform')
    if kind == 'few':
        ids = np.where((ids >= 0) & (ids < V), ids // 97 * 97, ids)
    dout = round_to(rng.standard_normal((T, C)), 'bf16')
    # memory that held something else before
    torch.full((V, C), 7.0, device=cuda_device)
    got = b200().embed_bwd(torch.tensor(ids, device=cuda_device).int(),
                           dev(dout, 'bf16', cuda_device), V, scale=0.5)
    grad_close(ids, dout, V, 0.5, got, C)


def test_embed_bwd_ignores_rows_without_a_token(cuda_device):
    dout = torch.full((4, 8), float('nan'), device=cuda_device)
    dout[1] = 2.0
    ids = torch.tensor([-1, 2, 7, 3], device=cuda_device)
    got = b200().embed_bwd(ids, dout, 3, scale=0.5)
    assert (got[:2] == 0).all() and (got[2] == 1.0).all()
    assert (b200().embed_bwd(ids[:0], dout[:0], 3) == 0).all()
    # the gradient of the lookup: a step in the table moves sum(out * dout) by the product
    rng = np.random.default_rng(0)
    table = torch.tensor(rng.integers(-8, 8, (3, 8)) / 4., device=cuda_device).float()
    step = torch.tensor(rng.integers(-8, 8, (3, 8)) / 4., device=cuda_device).float()
    dout = torch.tensor(rng.integers(-8, 8, (4, 8)) / 4., device=cuda_device).float()
    diff = ((b200().embed(ids, table + step) - b200().embed(ids, table)) * dout).double().sum()
    assert diff == (b200().embed_bwd(ids, dout, 3) * step).double().sum()  # exact in binary


def test_embed_on_another_stream(cuda_device):
    rng = np.random.default_rng(5)
    s = torch.cuda.Stream()
    ids = torch.tensor(rng.integers(0, 50, 3000), device=cuda_device)
    dout = dev(rng.standard_normal((3000, 32)), 'f32', cuda_device)
    want = b200().embed_bwd(ids, dout, 50)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = b200().embed_bwd(ids, dout, 50)
    s.synchronize()
    assert torch.equal(got, want)


def test_refusals(cuda_device):
    m, d = b200(), cuda_device
    ids, table = torch.zeros(4, dtype=torch.int32, device=d), torch.zeros(3, 8, device=d)
    dout = torch.zeros(4, 8, device=d)
    for bad in (lambda: m.embed(ids.float(), table), lambda: m.embed(ids, table.double()),
                lambda: m.embed(ids, table[0]), lambda: m.embed(ids, table.t()),
                lambda: m.embed(ids, table.half(), out_dtype=torch.float32),
                lambda: m.embed(ids, table, out=dout[:2]), lambda: m.embed(ids.cpu(), table),
                lambda: m.embed_bwd(ids, dout[:3], 3), lambda: m.embed_bwd(ids, dout, -1),
                lambda: m.embed_bwd(ids, dout, 2 ** 31),
                lambda: m.embed_bwd(ids.short(), dout, 3),
                lambda: m.embed_bwd(ids, dout.double(), 3)):
        with pytest.raises(ValueError):
            bad()


def test_embed_bwd_of_tokens_near_2_to_31(cuda_device):
    """The last chunk of the sorted list ends less than a chunk's length below 2^31."""
    T = 2 ** 31 - 1200
    dout = torch.zeros(T, 1, dtype=torch.float16, device=cuda_device)
    ids = torch.zeros(T, dtype=torch.int32, device=cuda_device)
    ids[[3, T // 2, T - 2]] = torch.tensor([1, 2, 1], dtype=torch.int32, device=cuda_device)
    dout[[0, 3, T // 2, T - 2, T - 1]] = torch.tensor([1., 2, 4, 8, 16], device=cuda_device).half()[:, None]
    got = b200().embed_bwd(ids, dout, 3)
    assert got[:, 0].tolist() == [17.0, 10.0, 4.0]
    del dout, ids
    torch.cuda.empty_cache()  # 47 GB with the workspace


def test_embed_bwd_of_rows_near_2_to_31(cuda_device):
    V = 2 ** 31 - 2
    torch.full((V, 1), 7.0, device=cuda_device)  # memory that held something else before
    ids = torch.tensor([V - 1, 0, V, V - 1, V - 40000], device=cuda_device)
    dout = torch.tensor([1., 2, 4, 8, 16], device=cuda_device)[:, None]
    got = b200().embed_bwd(ids, dout, V)[:, 0]
    assert got[[0, V - 40000, V - 1]].tolist() == [2.0, 16.0, 9.0]
    assert int(torch.count_nonzero(got)) == 3
    del got
    torch.cuda.empty_cache()


@pytest.mark.parametrize('C', [128 * 65535, 128 * 65535 + 8, 8500001])
def test_embed_bwd_of_more_slabs_than_a_grid_has_rows(C, cuda_device):
    dout = torch.randn(3, C, device=cuda_device)
    ids = torch.tensor([1, -1, 1], device=cuda_device)
    got = b200().embed_bwd(ids, dout, 2, scale=2.0)
    assert torch.equal(got[1], 2.0 * (dout[0] + dout[2])) and (got[0] == 0).all()


@pytest.mark.parametrize('C', [2 ** 31 - 8, 2 ** 31 - 21])
def test_channels_near_2_to_31(C, cuda_device):
    m = b200()
    table = torch.empty(1, C, dtype=torch.float16, device=cuda_device).uniform_(-1, 1)
    ids = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    assert torch.equal(m.embed(ids, table), table)
    got = m.embed_bwd(ids + 1, table, 2)  # the table as a gradient of one token
    assert int(torch.count_nonzero(got[0])) == 0 and torch.equal(got[1], table[0].float())
    del got, table
    torch.cuda.empty_cache()


def test_embed_into_a_tensor_counts_as_a_change_of_it(cuda_device):
    out = torch.zeros(4, 8, device=cuda_device)
    v = out._version
    b200().embed(torch.zeros(4, dtype=torch.int32, device=cuda_device), out[:1].clone(), out=out)
    assert out._version > v

"""Linear softmax cross entropy and its gradients on the B200 against the float64 restatement.

Tolerances, from the arithmetic (u = 2^-8 in bf16, 2^-11 in f16, the types' unit roundoff):
  * a logit is a float32 sum of C exact products: off by at most e = (C + 1) 2^-23 max sum |x w|
    (2^-23 a step, as for an accumulation that truncates), plus the bias's rounding in it;
  * loss: two logits' errors, and the log2-domain sum's: exponentials within 2^-22, sums of at most
    a few hundred sequential terms, a product with log2 e each way: 2 e + 2^-16 (1 + |lse| + |loss|)
    stays above all of them;
  * g: softmax within 2 e + 2^-16 (1 + |lse|) relative (the exponent's absolute error), rounded to
    16 bits (u relative, and where float16 goes below its normal range 2^-25 of its scaled unit, at
    most 2^-38 of the largest |dloss|);
  * dx, dw, dbias: those errors through the sums, the float32 accumulation (K 2^-23 of the sum of
    magnitudes) and the final rounding (u relative, 2^-25 absolute in float16).
"""
import numpy as np
import pytest
import torch

from oracle import tokens as ot
from oracle.numerics import round_to

pytestmark = pytest.mark.gpu

TD = {'f16': torch.float16, 'bf16': torch.bfloat16}
U = {'f16': 2.0 ** -11, 'bf16': 2.0 ** -8}


def b200():
    from colabfold_legacy_kernels import b200 as m
    return m


def problem(T, V, C, dt, *, bias=True, labelled=.8, amp=2.0, seed=0):
    rng = np.random.default_rng(seed + T + 3 * V + 7 * C)
    x = round_to(rng.standard_normal((T, C)), dt)
    w = round_to(rng.standard_normal((V, C)) * amp / np.sqrt(C), dt)
    b = round_to(rng.standard_normal(V), dt) if bias else None
    labels = np.where(rng.random(T) < labelled, rng.integers(0, V, T),
                      rng.choice([-100, -1, V, 2 ** 31 - 1], T))
    dloss = (.5 + rng.random(T)).astype(np.float32) / max(T, 1)
    return x, w, b, labels, dloss


def dev(a, dt, d):
    return None if a is None else torch.tensor(np.asarray(a, np.float32), device=d).to(TD[dt])


def run(x, w, b, labels, dloss, dt, d, bits=32):
    m = b200()
    tx, tw, tb = dev(x, dt, d), dev(w, dt, d), dev(b, dt, d)
    tl = torch.tensor(labels, device=d).to(torch.int32 if bits == 32 else torch.int64)
    td = torch.tensor(np.asarray(dloss, np.float32), device=d)
    loss, lse = m.linear_xent(tx, tw, tl, tb)
    grads = m.linear_xent_bwd(tx, tw, tl, lse, td, tb)
    again = m.linear_xent_bwd(tx, tw, tl, lse, td, tb)
    assert m.device_status() == 0
    for a, c in zip(grads, again):
        # the same bits, those of NaN among them
        assert (a is None and c is None) or torch.equal(a.view(torch.int16), c.view(torch.int16))
    f = lambda t: None if t is None else t.double().cpu().numpy()
    return [f(t) for t in (loss, lse, *grads)]


def bounds(x, w, b, labels, dloss, dt):
    """(loss, lse, dx, dw, dbias) of the restatement and how far each may be off."""
    u = U[dt]
    loss, lse = ot.linear_xent(x, w, labels, b)
    dx, dw, db, g, rows = ot.linear_xent_bwd(x, w, labels, dloss, b)
    C, V, n = x.shape[1], w.shape[0], len(rows)
    with np.errstate(invalid='ignore', over='ignore'):
        finite = np.zeros(V) if b is None else np.where(np.isfinite(b) & (np.abs(b) < 1e30), b, 0)
        e = (C + 1) * 2.0 ** -23 * (np.abs(x[rows]) @ np.abs(w).T).max(initial=0.0) + \
            2.0 ** -22 * np.abs(finite).max(initial=0.0)
    size = np.where(np.isfinite(lse), np.abs(lse), 0)
    tol_loss = 2 * e + 2.0 ** -16 * (1 + size + np.where(np.isfinite(loss), np.abs(loss), 0))
    dl = np.abs(dloss[rows]).astype(np.float64)
    rel = 2 * e + 2.0 ** -16 * (1 + size[rows])
    one = np.zeros_like(g)
    one[np.arange(n), labels[rows]] = dl
    p = np.abs(g + np.where(one > 0, dloss[rows, None], 0))
    small = 2.0 ** -38 * dl.max(initial=0.0) if dt == 'f16' else 0.0
    dg = rel[:, None] * p + u * np.abs(g) + small
    low = 2.0 ** -25 if dt == 'f16' else 0.0
    aw, ax, ag = np.abs(w), np.abs(x[rows]), np.abs(g)
    tol_dx = np.zeros(x.shape)
    tol_dx[rows] = dg @ aw + V * 2.0 ** -23 * (ag @ aw)
    tol_dw = dg.T @ ax + n * 2.0 ** -23 * (ag.T @ ax)
    tol_db = dg.sum(0) + n * 2.0 ** -23 * ag.sum(0)
    fin = lambda want, t: t + u * (np.abs(want) + t) + low
    return ((loss, tol_loss), (lse, tol_loss * ot.LOG2E), (dx, fin(dx, tol_dx)),
            (dw, fin(dw, tol_dw)), (db, fin(db, tol_db)))


def close(got, want):
    for name, a, (b, tol) in zip(('loss', 'lse', 'dx', 'dw', 'dbias'), got, want):
        if a is None:
            continue
        same = (a == b)  # infinities among them
        with np.errstate(invalid='ignore'):
            off = np.where(same, 0, np.abs(a - b) / np.maximum(tol, 1e-300))
        assert a.shape == b.shape and (off <= 1).all(), \
            '%s: %.3g times the tolerance' % (name, np.nanmax(off))


@pytest.mark.parametrize('dt', ['bf16', 'f16'])
@pytest.mark.parametrize('T,V,C', [
    (1, 1, 8), (1, 23, 256), (1, 1000, 64), (3, 2, 8), (5, 64, 128), (64, 23, 24), (127, 50, 384),
    (128, 128, 128), (129, 129, 136), (255, 21, 72), (256, 256, 256), (257, 257, 264),
    (300, 513, 64), (513, 64, 520), (700, 1000, 40), (1100, 300, 16), (1025, 22, 256),
    (20000, 23, 256), (19500, 70, 128), (300, 100, 200), (300, 40, 392)])
def test_linear_xent(T, V, C, dt, cuda_device):
    for bias in (True, False):
        p = problem(T, V, C, dt, bias=bias)
        close(run(*p, dt, cuda_device, bits=32 if bias else 64), bounds(*p, dt))


@pytest.mark.parametrize('dt', ['bf16', 'f16'])
@pytest.mark.parametrize('labelled', [0.0, 0.02, 0.15, 1.0])
@pytest.mark.parametrize('T,V,C', [(1, 23, 64), (600, 23, 64), (2500, 300, 32), (900, 600, 24)])
def test_labelled_shares(T, V, C, labelled, dt, cuda_device):
    x, w, b, labels, dloss = problem(T, V, C, dt, labelled=labelled)
    # rows without a label hold anything
    x = x.copy()
    x[(labels < 0) | (labels >= V)] = np.nan
    dloss = np.where((labels < 0) | (labels >= V), np.float32(np.nan), dloss)
    got = run(x, w, b, labels, dloss, dt, cuda_device)
    assert all(np.isfinite(a).all() for a in (got[0], *got[2:]))
    close(got, bounds(x, w, b, labels, dloss, dt))


@pytest.mark.parametrize('dt', ['bf16', 'f16'])
@pytest.mark.parametrize('V', [23, 300, 700])
def test_masked_classes(V, dt, cuda_device):
    """Classes masked by a bias of -inf or of the type's lowest value, up to all of them."""
    x, w, b, labels, dloss = problem(150, V, 32, dt)
    lowest = float(torch.finfo(TD[dt]).min)
    for value in (-np.inf, lowest):
        b2 = b.copy()
        b2[::2] = value
        b2[: V // 2] = value  # whole tiles among them
        keep = np.where((labels >= 0) & (labels < V), V - 2 + V % 2, labels)
        got = run(x, w, b2, keep, dloss, dt, cuda_device)
        close(got, bounds(x, w, b2, keep, dloss, dt))
    got = run(x, w, np.full(V, -np.inf), labels, dloss, dt, cuda_device)
    assert (got[0] == 0).all() and (got[1] == -np.inf).all()
    assert all((a == 0).all() for a in got[2:])


@pytest.mark.parametrize('dt', ['bf16', 'f16'])
def test_masked_classes_of_few_tokens(dt, cuda_device):
    x, w, b, labels, dloss = problem(33, 900, 40, dt)
    b[:700] = float(torch.finfo(TD[dt]).min)
    b[100:300] = -np.inf
    keep = np.where((labels >= 0) & (labels < 900), 700 + labels % 200, labels)
    close(run(x, w, b, keep, dloss, dt, cuda_device), bounds(x, w, b, keep, dloss, dt))
    got = run(x, w, np.full(900, -np.inf), labels, dloss, dt, cuda_device)
    assert (got[0] == 0).all() and (got[1] == -np.inf).all()
    assert all((a == 0).all() for a in got[2:])


@pytest.mark.parametrize('V', [23, 513])
def test_label_of_a_masked_class_and_nan(V, cuda_device):
    x, w, b, _, dloss = problem(40, V, 32, 'bf16')
    labels = np.arange(40) % V
    b[3] = -np.inf
    x[7] = np.nan
    got = run(x, w, b, labels, dloss, 'bf16', cuda_device)
    assert got[0][3] == np.inf and np.isnan(got[0][7]) and np.isnan(got[2][7]).all()
    rest = [i for i in range(40) if labels[i] != 3 and i != 7]
    assert np.isfinite(got[0][rest]).all() and np.isfinite(got[2][rest]).all()
    # the row's own gradient: softmax(l) - onehot with the softmax zero at the masked class
    close([got[2][rest]], [bounds(x[rest], w, b, labels[rest], dloss[rest], 'bf16')[2]])


@pytest.mark.parametrize('dt', ['bf16', 'f16'])
def test_confident_and_flat_rows(dt, cuda_device):
    for amp in (40.0, 0.0):
        p = problem(300, 400, 64, dt, amp=amp)
        close(run(*p, dt, cuda_device), bounds(*p, dt))


def test_gradients_are_the_losses_differences(cuda_device):
    """Central differences of the kernels' own losses, with steps that 16 bits hold exactly. The
    losses' float32 errors (below 2e-6 each) over the step and the third-order term (the square of
    the logits' steps, at most 0.02, times |sum g|) stay below 1 % of the products here."""
    rng = np.random.default_rng(4)
    m, d = b200(), cuda_device
    for T, V, C in ((64, 23, 64), (48, 300, 64)):
        h = 1 / 16.
        x = rng.integers(-48, 48, (T, C)) / 16.
        w = rng.integers(-48, 48, (V, C)) / 512.
        labels = torch.tensor(rng.integers(0, V, T), device=d)
        sx, sw = rng.choice([-1., 1.], (T, C)), rng.choice([-1., 1.], (V, C)) / 32
        tl = lambda a: dev(a, 'f16', d)
        dloss = torch.ones(T, device=d)
        loss, lse = m.linear_xent(tl(x), tl(w), labels)
        dx, dw, _ = m.linear_xent_bwd(tl(x), tl(w), labels, lse, dloss)
        total = lambda a, b: m.linear_xent(tl(a), tl(b), labels)[0].double().sum().item()
        fx = (total(x + h * sx, w) - total(x - h * sx, w)) / (2 * h)
        fw = (total(x, w + h * sw) - total(x, w - h * sw)) / (2 * h)
        px = (dx.double().cpu().numpy() * sx)
        pw = (dw.double().cpu().numpy() * sw)
        assert abs(fx - px.sum()) < .01 * np.sqrt((px ** 2).sum()) + .01 * abs(px.sum())
        assert abs(fw - pw.sum()) < .01 * np.sqrt((pw ** 2).sum()) + .01 * abs(pw.sum())


def reference64(x, w, labels, dloss, bias):
    """The definition in float64 on the GPU, for sizes numpy is slow at."""
    x, w = x.double(), w.double()
    ok = (labels >= 0) & (labels < w.shape[0])
    y = torch.where(ok, labels.long(), 0)
    x = torch.where(ok[:, None], x, 0)
    logits = x @ w.t() + (0 if bias is None else bias.double())
    z = torch.logsumexp(logits, 1)
    loss = torch.where(ok, z - logits.gather(1, y[:, None])[:, 0], 0)
    g = torch.exp(logits - z[:, None])
    g.scatter_add_(1, y[:, None], -torch.ones_like(loss)[:, None])
    g *= torch.where(ok, dloss.double(), 0)[:, None]
    return loss, torch.where(ok, z * ot.LOG2E, -np.inf), g @ w, g.t() @ x, g.sum(0)


@pytest.mark.parametrize('T,V,C,dt,labelled', [
    (5000, 70001, 64, 'bf16', .9),   # classes in several pieces
    (2100, 140003, 40, 'f16', 1.0),
    (300000, 23, 64, 'bf16', .15), (200001, 64, 128, 'f16', .9), (50003, 100, 256, 'bf16', 1.0),
    (20001, 129, 72, 'bf16', .5), (700001, 23, 16, 'f16', .3), (9, 33000, 1032, 'f16', 1.0)])
def test_large(T, V, C, dt, labelled, cuda_device):
    """Relative 2-norms against float64: the inputs' products in 16 bits leave u / sqrt(3) or so in
    g and the same again in the outputs; 2 u bounds their sum with room for the float32 sums."""
    g = torch.Generator(device=cuda_device).manual_seed(T)
    r = lambda *s: torch.randn(*s, generator=g, device=cuda_device)
    x, w, b = r(T, C).to(TD[dt]), (2 * r(V, C) / C ** .5).to(TD[dt]), r(V).to(TD[dt])
    labels = torch.randint(0, V, (T,), generator=g, device=cuda_device)
    labels = torch.where(torch.rand(T, generator=g, device=cuda_device) < labelled, labels, -100)
    dloss = torch.rand(T, generator=g, device=cuda_device)
    m = b200()
    loss, lse = m.linear_xent(x, w, labels, b)
    got = (loss, lse, *m.linear_xent_bwd(x, w, labels, lse, dloss, b))
    want = reference64(x, w, labels, dloss, b)
    assert m.device_status() == 0
    for name, a, c, tol in zip(('loss', 'lse', 'dx', 'dw', 'dbias'), got, want,
                               (2e-6, 2e-6, 2 * U[dt], 2 * U[dt], 2 * U[dt])):
        fine = torch.isfinite(c)
        assert torch.equal(torch.isfinite(a), fine), name
        off = (a.double() - c)[fine].norm() / c[fine].norm()
        assert off < tol, '%s: %.3g' % (name, off)


def test_many_rows_of_many_classes(cuda_device):
    """Statistics in several launches of rows; sampled rows against float64."""
    T, V, C = 66000, 70001, 16
    g = torch.Generator(device=cuda_device).manual_seed(0)
    x = torch.randn(T, C, generator=g, device=cuda_device).bfloat16()
    w = torch.randn(V, C, generator=g, device=cuda_device).bfloat16()
    labels = torch.randint(-V // 9, V, (T,), generator=g, device=cuda_device)
    loss, lse = b200().linear_xent(x, w, labels)
    some = torch.cat([torch.arange(8, device=cuda_device),
                      torch.randint(0, T, (200,), generator=g, device=cuda_device),
                      torch.arange(T - 8, T, device=cuda_device)])
    want = reference64(x[some], w, labels[some], torch.ones(len(some), device=cuda_device), None)
    fine = torch.isfinite(want[1])
    assert torch.equal(torch.isfinite(lse[some]), fine)
    assert ((loss[some] - want[0]).norm() / want[0].norm()) < 2e-6
    assert ((lse[some] - want[1])[fine].norm() / want[1][fine].norm()) < 2e-6
    assert b200().device_status() == 0


def test_another_stream_and_no_tokens(cuda_device):
    m, d = b200(), cuda_device
    x, w, b, labels, dloss = problem(200, 300, 64, 'bf16')
    tx, tw, tb = (dev(a, 'bf16', d) for a in (x, w, b))
    tl, td = torch.tensor(labels, device=d), torch.tensor(dloss, device=d)
    want = m.linear_xent(tx, tw, tl, tb)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = m.linear_xent(tx, tw, tl, tb)
        grads = m.linear_xent_bwd(tx, tw, tl, got[1], td, tb)
    s.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    want = m.linear_xent_bwd(tx, tw, tl, want[1], td, tb)
    assert all(torch.equal(a, c) for a, c in zip(grads, want))
    loss, lse = m.linear_xent(tx[:0], tw, tl[:0], tb)
    dx, dw, db = m.linear_xent_bwd(tx[:0], tw, tl[:0], lse, td[:0], tb)
    assert loss.shape == (0,) and dx.shape == (0, 64) and (dw == 0).all() and (db == 0).all()
    # leading dimensions
    l2, _ = m.linear_xent(tx.view(10, 20, 64), tw, tl.view(10, 20), tb)
    assert torch.equal(l2.view(-1), got[0])


def test_refusals(cuda_device):
    m, d = b200(), cuda_device
    x, w = torch.zeros(4, 16, device=d).half(), torch.zeros(5, 16, device=d).half()
    lab, f = torch.zeros(4, dtype=torch.int32, device=d), torch.zeros(4, device=d)
    for bad in (lambda: m.linear_xent(x.float(), w.float(), lab),
                lambda: m.linear_xent(x, w.bfloat16(), lab), lambda: m.linear_xent(x[:3], w, lab),
                lambda: m.linear_xent(x[:, :8], w[:, :8], lab),  # not contiguous
                lambda: m.linear_xent(x[:, :12].contiguous(), w[:, :12].contiguous(), lab),
                lambda: m.linear_xent(x, w[:0], lab), lambda: m.linear_xent(x, w, lab.float()),
                lambda: m.linear_xent(x, w, lab, w[0]), lambda: m.linear_xent(x.cpu(), w, lab),
                lambda: m.linear_xent(torch.zeros(65, device=d).half()[1:].view(4, 16), w, lab),
                lambda: m.linear_xent_bwd(x, w, lab, f[:3], f),
                lambda: m.linear_xent_bwd(x, w, lab, f.double(), f),
                lambda: m.linear_xent_bwd(x, w, lab, f, f.half())):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize('dt', ['bf16', 'f16'])
@pytest.mark.parametrize('labelled', [.6, .8, .95])
@pytest.mark.parametrize('T,V,C', [(900, 23, 64), (900, 64, 128), (40000, 64, 128), (900, 128, 128),
                                   (900, 100, 64), (900, 23, 256), (21000, 64, 200)])
def test_rows_without_a_label_that_are_not_finite(T, V, C, labelled, dt, cuda_device):
    """In rounds that take whole blocks of tokens too: rows without a label, and their dloss, reach no
    result."""
    for bias in (True, False):
        x, w, b, labels, dloss = problem(T, V, C, dt, bias=bias, labelled=labelled)
        x, out = x.copy(), np.nonzero((labels < 0) | (labels >= V))[0]
        x[out[0::4]] = np.nan
        x[out[1::4]] = np.inf
        x[out[2::4]] = -np.inf
        x[out[3::4], 5] = np.inf  # one channel
        dloss[out] = np.nan
        got = run(x, w, b, labels, dloss, dt, cuda_device)
        assert all(np.isfinite(a).all() for a in (got[0], *got[2:]) if a is not None)
        close(got, bounds(x, w, b, labels, dloss, dt))


def test_few_tokens_of_classes_near_2_to_31(cuda_device):
    """Zero weights but the last class's; the tolerance is that of the losses above."""
    V, m = 2 ** 31 - 1100, b200()
    w = torch.zeros(V, 8, dtype=torch.bfloat16, device=cuda_device)
    w[-1] = 1.0
    x = torch.ones(2, 8, dtype=torch.bfloat16, device=cuda_device)
    labels = torch.tensor([V - 1, 0], device=cuda_device)
    loss, lse = m.linear_xent(x, w, labels)
    z = np.log(V - 1 + np.exp(8.0))
    assert m.device_status() == 0
    assert (np.abs(loss.cpu().numpy() - [z - 8, z]) < 2.0 ** -16 * (1 + 2 * z)).all()
    assert (np.abs(lse.cpu().numpy() - z * ot.LOG2E) < 2.0 ** -16 * (1 + z) * ot.LOG2E).all()
    del w
    torch.cuda.empty_cache()


@pytest.mark.parametrize('T,V', [(40, 23), (40, 513), (200, 700)])
def test_class_that_is_nan(T, V, cuda_device):
    """Every row's softmax is NaN then, and with it every gradient."""
    x, w, b, labels, dloss = problem(T, V, 32, 'bf16')
    w[7] = np.nan
    got = run(x, w, b, labels, dloss, 'bf16', cuda_device)
    rows = (labels >= 0) & (labels < V)
    assert np.isnan(got[0][rows]).all() and np.isnan(got[1][rows]).all()
    assert np.isnan(got[2][rows]).all() and (got[2][~rows] == 0).all()
    assert np.isnan(got[3]).all() and np.isnan(got[4]).all()


@pytest.mark.parametrize('dt', ['bf16', 'f16'])
@pytest.mark.parametrize('T,V', [(200, 23), (200, 100), (33, 900), (200, 700), (20000, 23)])
def test_loss_of_large_logits(T, V, dt, cuda_device):
    """Rows of exact logits (a product each): `top` at class a, top - d at class b, 0 elsewhere. What the
    size of the logits leaves in the loss is one rounding of top - label; the sum's at most 100
    additions (2^-24 each), the exponentials and the logarithm (2^-22 each) stay below 2^-17."""
    rng = np.random.default_rng(T + V)
    C = 64
    w = np.zeros((V, C))
    w[np.arange(min(V, C)), np.arange(min(V, C))] = 1.0
    top = round_to(rng.uniform(20, 2000, T), dt)
    low = round_to(np.maximum(top - rng.choice([0, .5, 2, 20, 300], T), 0), dt)
    a = rng.integers(0, min(V, C), T)
    b = (a + 1 + rng.integers(0, min(V, C) - 1, T)) % min(V, C)
    x = np.zeros((T, C))
    x[np.arange(T), a], x[np.arange(T), b] = top, low
    m = b200()
    for labels in (a, b):
        want, lse = ot.linear_xent(x, w, labels)
        got, got_lse = m.linear_xent(dev(x, dt, cuda_device), dev(w, dt, cuda_device),
                                     torch.tensor(labels, device=cuda_device))
        got, got_lse = got.double().cpu().numpy(), got_lse.double().cpu().numpy()
        assert (got >= 0).all()
        assert (np.abs(got - want) <= 2.0 ** -17 + 2.0 ** -22 * want).all(), np.abs(got - want).max()
        assert (np.abs(got_lse - lse) <= 2.0 ** -16 + 2.0 ** -22 * np.abs(lse)).all()


@pytest.mark.parametrize('T,V', [(150, 23), (33, 900), (150, 300), (150, 700)])
def test_every_class_at_bf16s_lowest_value(T, V, cuda_device):
    """Logits below -2.3e38 leave float32 in the log2 domain: they count as -inf, in both directions."""
    x, w, b, labels, dloss = problem(T, V, 32, 'bf16')
    lowest = float(torch.finfo(torch.bfloat16).min)
    got = run(x, w, np.full(V, lowest), labels, dloss, 'bf16', cuda_device)
    assert (got[0] == 0).all() and (got[1] == -np.inf).all()
    assert all((a == 0).all() for a in got[2:])
    # one class above it takes every row
    b = np.full(V, lowest)
    b[V - 2] = 1.0
    keep = np.where((labels >= 0) & (labels < V), V - 2, labels)
    close(run(x, w, b, keep, dloss, 'bf16', cuda_device), bounds(x, w, b, keep, dloss, 'bf16'))

"""The token-training entry points refuse invalid arguments before any CUDA call (no GPU needed), and
their workspace sizes."""
import ctypes

import pytest

from test_capi import lib

Z, I64, F32 = ctypes.c_void_p(0), ctypes.c_int64, ctypes.c_float
P = ctypes.c_void_p(256)  # an aligned address that is never read


def call(name, *args):
    l = lib()
    l.cflk_last_error.restype = ctypes.c_char_p
    rc = getattr(l, name)(*args)
    return rc, l.cflk_last_error().decode()


def size(name, *args):
    n = ctypes.c_size_t(7)
    rc, msg = call(name, *[I64(a) for a in args], ctypes.byref(n))
    return rc, n.value, msg


def embed(dt=2, out=2, i64=0, ids=P, table=P, dst=P, T=4, V=5, C=8):
    return call('cflk_embed', Z, dt, out, i64, ids, table, dst, I64(T), I64(V), I64(C), F32(1))


@pytest.mark.parametrize('bad', [dict(dt=3), dict(dt=0), dict(dt=0, out=1), dict(out=7),
                                 dict(i64=2), dict(T=-1), dict(V=-1), dict(C=-1), dict(C=1 << 31),
                                 dict(T=1 << 62), dict(V=1 << 62), dict(ids=Z), dict(table=Z),
                                 dict(dst=Z)])
def test_embed_refuses(bad):
    rc, msg = embed(**bad)
    assert rc == 1 and msg.startswith('embed: ')


def test_embed_without_work_launches_nothing():
    assert embed(T=0, ids=Z, dst=Z)[0] == 0 and embed(C=0, dst=Z)[0] == 0


def embed_bwd(dt=0, i64=0, ids=P, dout=P, out=P, T=4, V=5, C=8, ws=P, n=1 << 40):
    return call('cflk_embed_bwd', Z, dt, i64, ids, dout, out, I64(T), I64(V), I64(C), F32(1), ws,
                ctypes.c_size_t(n))


@pytest.mark.parametrize('bad', [dict(dt=3), dict(i64=2), dict(T=-1), dict(V=1 << 31),
                                 dict(T=1 << 31), dict(T=1 << 62), dict(ids=Z), dict(dout=Z),
                                 dict(out=Z), dict(ws=Z), dict(n=16),
                                 dict(ws=ctypes.c_void_p(8))])
def test_embed_bwd_refuses(bad):
    rc, msg = embed_bwd(**bad)
    assert rc == 1 and msg.startswith('embed_bwd: ')


def test_embed_bwd_sizes():
    name = 'cflk_embed_bwd_workspace_size'
    assert size(name, 0, 5, 8)[:2] == (0, 0) and size(name, 5, 0, 8)[:2] == (0, 0)
    rc, n, _ = size(name, 1000, 50, 64)
    assert rc == 0 and n >= 4 * 4 * 1000  # keys and tokens, twice
    assert size(name, -1, 5, 8)[0] == 1 and size(name, 1 << 31, 5, 8)[0] == 1
    assert embed_bwd(V=0, out=Z)[0] == 0


def xent(dt=1, l64=0, x=P, w=P, b=Z, lab=P, loss=P, lse=P, T=4, V=5, C=8, ws=P, n=1 << 40):
    return call('cflk_linear_xent', Z, dt, l64, x, w, b, lab, loss, lse, I64(T), I64(V), I64(C),
                ws, ctypes.c_size_t(n))


def xent_bwd(dt=1, l64=0, x=P, w=P, b=Z, lab=P, lse=P, dl=P, dx=P, dw=P, db=Z, T=4, V=5, C=8,
             ws=P, n=1 << 40):
    return call('cflk_linear_xent_bwd', Z, dt, l64, x, w, b, lab, lse, dl, dx, dw, db, I64(T),
                I64(V), I64(C), ws, ctypes.c_size_t(n))


BAD = [dict(dt=2), dict(l64=2), dict(T=-1), dict(V=0), dict(C=0), dict(C=12), dict(T=1 << 31),
       dict(V=1 << 31), dict(x=Z), dict(w=Z), dict(lab=Z), dict(lse=Z), dict(ws=Z, V=500), dict(n=16, V=500),
       dict(ws=ctypes.c_void_p(16), V=500), dict(x=ctypes.c_void_p(8)), dict(w=ctypes.c_void_p(8))]


@pytest.mark.parametrize('bad', BAD + [dict(loss=Z)])
def test_xent_refuses(bad):
    rc, msg = xent(**bad)
    assert rc == 1 and msg.startswith('linear_xent: ')


@pytest.mark.parametrize('bad', BAD + [dict(dl=Z), dict(dx=Z), dict(dw=Z), dict(b=P), dict(db=P),
                                       dict(dx=ctypes.c_void_p(2)), dict(dw=ctypes.c_void_p(2))])
def test_xent_bwd_refuses(bad):
    rc, msg = xent_bwd(**bad)
    assert rc == 1 and msg.startswith('linear_xent_bwd: ')


def test_xent_sizes():
    assert xent(T=0, x=Z, loss=Z)[0] == 0
    for name in ('cflk_linear_xent_workspace_size', 'cflk_linear_xent_bwd_workspace_size'):
        assert size(name, 0, 5, 8)[:2] == (0, 0)
        assert size(name, 4, 5, 12)[0] == 1 and size(name, 4, 0, 8)[0] == 1
        assert size(name, 1 << 31, 5, 8)[0] == 1 and size(name, 5, 5, 1 << 40)[0] == 1
        # bounded: neither keeps the logits of a large vocabulary (here 26 GB in 16 bits)
        rc, n, _ = size(name, 65536, 200000, 512)
        assert rc == 0 and n < 3 << 30


def arrays(ptrs, numel, types):
    n = len(ptrs)
    return ((ctypes.c_void_p * n)(*ptrs), (ctypes.c_int64 * n)(*numel), (ctypes.c_int * n)(*types))


def clip(ptrs=(256, 512), numel=(3, 4), types=(2, 1), outs=(256, 512), otypes=(2, 1), max_norm=1.,
         eps=0., scale=1., n=None, ws=P, nb=1 << 20, sumsq=Z):
    p, m, t = arrays(ptrs, numel, types)
    o, _, ot = arrays(outs, numel, otypes)
    return call('cflk_grad_clip', Z, I64(len(ptrs) if n is None else n), p, o, m, t, ot, sumsq,
                F32(max_norm), F32(eps), F32(scale), Z, ws, ctypes.c_size_t(nb))


@pytest.mark.parametrize('bad', [dict(n=-1), dict(numel=(3, -1)), dict(numel=(1 << 44, 1)),
                                 dict(types=(2, 3)), dict(otypes=(1, 1)), dict(otypes=(2, 0)),
                                 dict(ptrs=(None, 512)), dict(ptrs=(258, 512)),
                                 dict(ptrs=(256, 513)), dict(outs=(256, None)),
                                 dict(outs=(257, 512)), dict(max_norm=-1.),
                                 dict(max_norm=float('nan')), dict(eps=-1.), dict(scale=0.),
                                 dict(scale=-1.), dict(ws=Z), dict(nb=8),
                                 dict(ws=ctypes.c_void_p(4))])
def test_clip_refuses(bad):
    rc, msg = clip(**bad)
    assert rc == 1 and msg.startswith('grad_')


def test_sumsq_refuses():
    p, m, t = arrays((256,), (3,), (2,))
    f = lambda n, out, ws, nb: call('cflk_grad_sumsq', Z, I64(n), p, m, t, out, ws,
                                    ctypes.c_size_t(nb))
    for args in ((-1, P, P, 1 << 20), (1, Z, P, 1 << 20), (1, P, Z, 1 << 20), (1, P, P, 8)):
        assert f(*args)[0] == 1
    assert size('cflk_grad_workspace_size', -1)[0] == 1
    # more tensors than a launch takes need a sum a launch
    assert size('cflk_grad_workspace_size', 10000)[1] > size('cflk_grad_workspace_size', 1)[1]


def test_tensor_table_reads_lists_and_refuses_what_is_no_gradient():
    """The host helper of the torch binding, on the CPU: what it refuses, and an empty list."""
    import importlib.util
    import os

    import torch

    import colabfold_legacy_kernels as clk
    path = os.path.join(os.path.dirname(clk.library_path('attention', 100)), '_cflk_table.so')
    spec = importlib.util.spec_from_file_location('_cflk_table', path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    table = module.tensor_table
    assert table([]) == (b'', b'', b'', -1) and table(()) == (b'', b'', b'', -1)
    t = torch.zeros(4, 6)
    for bad, why in ((t.t(), 'contiguous'), (t.double(), 'float16'), (t, 'CUDA'), (3, 'tensors'),
                     (None, 'tensors'), (t.to_sparse(), 'contiguous'), (t[0].int(), 'float16'),
                     (t.to('meta'), 'CUDA')):
        with pytest.raises(ValueError, match=why):
            table([bad])
    with pytest.raises(TypeError):
        table(7)


def test_gradients_refuse_more_elements_than_their_workspace_counts_launches_for():
    """A launch takes 900 tensors and below 2^31 chunks of 2^14 elements; a launch more would write past
    the workspace."""
    for n, one in ((4, 1 << 43), (900, 40 << 30)):
        # (without a workspace, so that no call can get to a launch)
        rc, msg = clip((256,) * n, (one,) * n, (2,) * n, (256,) * n, (2,) * n, ws=Z)
        assert rc == 1 and msg.startswith('grad_clip: ') and '2^45' in msg, (rc, msg)
        p, m, t = arrays((256,) * n, (one,) * n, (2,) * n)
        rc, msg = call('cflk_grad_sumsq', Z, I64(n), p, m, t, P, Z, ctypes.c_size_t(1 << 20))
        assert rc == 1 and msg.startswith('grad_norm: ') and '2^45' in msg, (rc, msg)


def test_helper_counts_writes():
    """What marks the tensors that a call wrote as changed, on the CPU."""
    import torch

    from colabfold_legacy_kernels import b200
    mark = b200._helper('grad_clip').mark_written
    a, b = torch.zeros(3), torch.zeros(0)
    with torch.inference_mode():
        c = torch.zeros(2)  # has no version
    before = a._version, b._version
    mark([a, b, c, a[1:]])  # a view shares its base's
    assert (a._version, b._version) == (before[0] + 2, before[1] + 1)
    mark([])
    with pytest.raises(ValueError, match='tensors'):
        mark([a, 3])
    with pytest.raises(TypeError):
        mark(7)


@pytest.mark.parametrize('bad', [dict(types=(1, 1), otypes=(2, 1)),  # widened onto itself
                                 dict(outs=(260, 512)), dict(ptrs=(260, 512), outs=(256, 512)),
                                 dict(ptrs=(256, 512), numel=(3, 4), outs=(256, 508))])
def test_clip_refuses_an_output_that_overlaps_its_gradient(bad):
    # (without a workspace, so that no call can get to a launch)
    rc, msg = clip(**bad, ws=Z)
    assert rc == 1 and 'overlaps' in msg


@pytest.mark.parametrize('good', [dict(), dict(outs=(268, 528)), dict(ptrs=(268, 528)),
                                  dict(types=(1, 1), otypes=(2, 1), outs=(264, 520)),
                                  dict(types=(1, 1), otypes=(2, 1), ptrs=(268, 528))])
def test_clip_takes_an_output_in_place_or_beside_its_gradient(good):
    rc, msg = clip(**good, ws=Z)
    assert rc == 1 and 'workspace' in msg

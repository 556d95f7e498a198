"""float64 restatements of the token-training operators: embedding lookup and its gradient, the
softmax cross entropy of a linear layer and its gradients, the global gradient norm and clipping.

These operators have no counterpart in the reference; the definitions are those of
include/cflk_b200.h.
"""
import numpy as np

LOG2E = 1.0 / np.log(2.0)
F32_MAX = float(np.finfo(np.float32).max)


def embed(ids, table, scale):
    """scale * table[ids]; zeros for an id outside [0, V)."""
    ids = np.asarray(ids)
    table = np.asarray(table, np.float64)
    ok = (ids >= 0) & (ids < len(table))
    out = np.zeros(ids.shape + (table.shape[1],))
    out[ok] = table[ids[ok]] * scale
    return out


def embed_bwd(ids, dout, rows, scale):
    """The scaled sum of dout over the tokens of each row, one token after the other."""
    ids = np.asarray(ids).reshape(-1)
    dout = np.asarray(dout, np.float64).reshape(len(ids), -1)
    out = np.zeros((rows, dout.shape[1]))
    ok = (ids >= 0) & (ids < rows)
    np.add.at(out, ids[ok], dout[ok])
    return out * scale


def _labelled(x, w, labels, bias):
    labels = np.asarray(labels)
    rows = np.nonzero((labels >= 0) & (labels < len(w)))[0]
    with np.errstate(invalid='ignore'):
        logits = np.asarray(x, np.float64)[rows] @ np.asarray(w, np.float64).T
        if bias is not None:
            logits = logits + np.asarray(bias, np.float64)
    top = logits.max(1, initial=-np.inf)
    # rows with a class left: their lse is float32 in the log2 domain
    left = ~(top * LOG2E < -F32_MAX)
    return rows[left], labels[rows[left]], logits[left], top[left]


def linear_xent(x, w, labels, bias=None):
    """(loss, lse in the log2 domain): 0 and -inf for a row without a label or a class left."""
    rows, lab, logits, top = _labelled(x, w, labels, bias)
    loss, lse = np.zeros(len(labels)), np.full(len(labels), -np.inf)
    total = np.log(np.exp(logits - top[:, None]).sum(1))
    lse[rows] = (top + total) * LOG2E
    loss[rows] = (top - logits[np.arange(len(rows)), lab]) + total
    return loss, lse


def linear_xent_bwd(x, w, labels, dloss, bias=None):
    """(dx, dw, dbias, g, rows): g [len(rows), V] is the logits' gradient of the rows that have
    one."""
    rows, lab, logits, top = _labelled(x, w, labels, bias)
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    g = np.exp(logits - top[:, None])
    g /= g.sum(1, keepdims=True)
    g[np.arange(len(rows)), lab] -= 1.0
    g *= np.asarray(dloss, np.float64)[rows, None]
    dx = np.zeros(x.shape)
    dx[rows] = g @ w
    return dx, g.T @ x[rows], g.sum(0), g, rows


def clip(grads, max_norm, scale=1.0, eps=1e-6):
    """(norm, the clipped gradients)."""
    grads = [np.asarray(a, np.float64) for a in grads]
    norm = scale * np.sqrt(sum(float((a * a).sum()) for a in grads))
    by = scale * min(1.0, max_norm / (norm + eps))
    return norm, [a * by for a in grads]

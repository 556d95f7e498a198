"""The token-training operators as workloads: embedding lookup and its gradient, the linear softmax cross entropy and its
gradients, and the global gradient norm with clipping.

`own` false: plain float32 torch operations; true: colabfold_legacy_kernels.b200. A case's sizes are T tokens, V table rows or
classes, C channels; `labelled` is the share of tokens that carry a label, `kind` how ids are distributed.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {'f16': torch.float16, 'bf16': torch.bfloat16, 'f32': torch.float32}


def listed():
    return [
        # one sequence's residues into channels: latency
        {'name': 'embed sequence', 'op': 'embed', 'dtype': 'bf16', 'T': 384, 'V': 23, 'C': 256,
         'kind': 'uniform'},
        # the clipped residue offsets of a 768-residue pair representation
        {'name': 'embed pair offsets', 'op': 'embed', 'dtype': 'bf16', 'T': 768 * 768, 'V': 65,
         'C': 128, 'kind': 'offsets'},
        # ... and the gradient of their table: few rows, each the sum of thousands of tokens
        {'name': 'embed_bwd pair offsets', 'op': 'embed_bwd', 'dtype': 'bf16', 'T': 768 * 768,
         'V': 65, 'C': 128, 'kind': 'offsets'},
        # a vocabulary's table: most rows without a token, a few with hundreds
        {'name': 'embed_bwd vocabulary', 'op': 'embed_bwd', 'dtype': 'f16', 'T': 16384, 'V': 50001,
         'C': 1024, 'kind': 'skewed'},
        # scoring a few tokens: one pass over the weights
        {'name': 'xent few tokens', 'op': 'xent', 'dtype': 'bf16', 'T': 4, 'V': 32000, 'C': 1024,
         'bias': False, 'labelled': 1.0},
        # the masked-MSA head of a 512 x 512 MSA: 15 % of the positions carry a label
        {'name': 'xent masked msa', 'op': 'xent_train', 'dtype': 'bf16', 'T': 512 * 512, 'V': 23,
         'C': 256, 'bias': True, 'labelled': 0.15},
        # a distance head over the pairs of 768 residues, some without coordinates
        {'name': 'xent distances', 'op': 'xent_train', 'dtype': 'f16', 'T': 768 * 768, 'V': 64,
         'C': 128, 'bias': True, 'labelled': 0.9},
        # token models: an ordinary step at odd sizes, and a large one
        {'name': 'xent vocabulary', 'op': 'xent_train', 'dtype': 'bf16', 'T': 4095, 'V': 32001,
         'C': 512, 'bias': False, 'labelled': 0.95},
        {'name': 'xent large vocabulary', 'op': 'xent_train', 'dtype': 'bf16', 'T': 8192,
         'V': 100003, 'C': 2048, 'bias': False, 'labelled': 1.0},
        # one block's gradients: latency
        {'name': 'clip block', 'op': 'clip', 'tensors': 16, 'elements': 300000, 'half': 0.0,
         'widen': False},
        # a whole pair-stack model: a few hundred ragged tensors, 16-bit ones among them
        {'name': 'clip model', 'op': 'clip', 'tensors': 384, 'elements': 93000000, 'half': 0.5,
         'widen': False},
        # 16-bit gradients clipped into the float32 buffers of an optimizer
        {'name': 'clip widened', 'op': 'clip', 'tensors': 60, 'elements': 300000000, 'half': 1.0,
         'widen': True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['embed', 'embed_bwd', 'xent', 'xent_train', 'head', 'clip'])
    dtype = rng.choice(['f16', 'bf16'])
    if op in ('embed', 'embed_bwd'):
        C = _log(rng, 8, 2048)
        C = C - C % 8 if rng.random() < 0.8 else C
        V = min(_log(rng, 2, 100000), 60000000 // C)
        T = min(_log(rng, 1, 600000), 75000000 // C)
        return {'op': op, 'dtype': dtype if rng.random() < 0.8 else 'f32', 'T': T, 'V': V, 'C': C,
                'kind': rng.choice(['uniform', 'skewed'])}
    if op == 'clip':
        n = _log(rng, 1, 300)
        return {'op': op, 'tensors': n, 'elements': max(n, _log(rng, 1000, 250000000)),
                'half': round(rng.choice([0.0, 1.0, rng.random()]), 3),
                'widen': rng.random() < 0.3}
    if op == 'head':  # a head of few classes over many positions
        V, C, T = _log(rng, 2, 256), 8 * _log(rng, 4, 48), _log(rng, 1000, 500000)
    else:
        V, C, T = _log(rng, 300, 100000), 8 * _log(rng, 8, 256), _log(rng, 1, 8192)
    if op == 'xent':
        T = _log(rng, 1, 4096)
    return {'op': 'xent' if op == 'xent' else 'xent_train', 'dtype': dtype, 'T': T, 'V': V, 'C': C,
            'bias': rng.random() < 0.5, 'labelled': round(rng.choice([1.0, rng.random()]), 3)}


def _ids(case, g):
    T, V = case['T'], case['V']
    if case['kind'] == 'offsets':
        n, far = math.isqrt(T), (V - 1) // 2
        # residues renumbered from a random start, with a chain break somewhere
        at = torch.arange(n, device='cuda')
        cut = torch.randint(1, n, (1,), generator=g, device='cuda')
        at = at + 200 * (at >= cut)
        return (at[None] - at[:, None]).clamp(-far, far).add(far).reshape(-1).int()
    u = torch.rand(T, generator=g, device='cuda')
    ids = (V * (u if case['kind'] == 'uniform' else u ** 4)).long().clamp(max=V - 1)
    # positions without a token
    return torch.where(torch.rand(T, generator=g, device='cuda') < 0.02, -1, ids).int()


def _tensors(case, g):
    """Ragged gradients as views of one buffer a type, as a bucketed all-reduce leaves them."""
    n, total = case['tensors'], case['elements']
    share = torch.rand(n, generator=torch.Generator().manual_seed(n * 7919 + total)) ** 4 + 1e-4
    sizes = (share / share.sum() * (total - n)).long().add(1).tolist()
    halves = int(round(case['half'] * n))
    groups = [('f32', sizes[halves:]), ('bf16', sizes[:halves])]
    state = {'flat': {}, 'flat_out': {}, 'grads': [], 'outs': []}
    for kind, part in groups:
        if not part:
            continue
        # every tensor starts on a 16-byte boundary
        starts, at = [], 0
        for s in part:
            starts.append(at)
            at += -(-s // 8) * 8
        x = torch.zeros(at, dtype=DTYPES[kind], device='cuda')
        x.normal_(0, 1e-3, generator=g)
        o = torch.zeros(at, dtype=torch.float32 if case['widen'] else x.dtype, device='cuda')
        state['flat'][kind], state['flat_out'][kind] = x, o
        state['grads'] += [x[b:b + s] for b, s in zip(starts, part)]
        state['outs'] += [o[b:b + s] for b, s in zip(starts, part)]
    # clipped to a tenth, after a loss scale of 256 is taken out
    state['scale'] = 1.0 / 256
    state['max_norm'] = 0.1 * 1e-3 * math.sqrt(total) / 256
    return state


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    op = case['op']
    if op == 'clip':
        return {'op': op, **_tensors(case, g)}
    T, V, C, dt = case['T'], case['V'], case['C'], DTYPES[case['dtype']]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device='cuda').mul_(std).to(dt)

    if op == 'embed':
        return {'op': op, 'ids': _ids(case, g), 'table': normal(V, C, std=0.02),
                'scale': math.sqrt(C)}
    if op == 'embed_bwd':
        return {'op': op, 'ids': _ids(case, g), 'dout': normal(T, C), 'rows': V,
                'scale': math.sqrt(C)}
    state = {'op': op, 'x': normal(T, C), 'w': normal(V, C, std=2.0 / math.sqrt(C)),
             'bias': normal(V, std=0.5) if case['bias'] else None}
    labels = (V * torch.rand(T, generator=g, device='cuda') ** 2).long().clamp(max=V - 1)
    labelled = torch.rand(T, generator=g, device='cuda') < case['labelled']
    labelled[torch.randint(0, T, (1,), generator=g, device='cuda')] = True
    state['labels'] = torch.where(labelled, labels, -100).int()
    # the mean's gradient with weights a position, under a loss scale where the type asks for one
    loss_scale = 4096.0 if case['dtype'] == 'f16' else 1.0
    state['dloss'] = (0.5 + torch.rand(T, generator=g, device='cuda')) * min(
        64.0, loss_scale / max(1.0, T * case['labelled']))
    return state


def _library():
    here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = os.path.join(here, 'colabfold-legacy-kernels_b200', 'src')
    if src not in sys.path:
        sys.path.insert(0, src)
    from colabfold_legacy_kernels import b200
    return b200


def _run_own(s):
    b200, op = _library(), s['op']
    if op == 'embed':
        return b200.embed(s['ids'], s['table'], scale=s['scale'])
    if op == 'embed_bwd':
        return b200.embed_bwd(s['ids'], s['dout'], s['rows'], scale=s['scale'])
    if op == 'clip':
        norm = b200.clip_grad_norm(s['grads'], s['max_norm'], scale=s['scale'], out=s['outs'])
        return {'norm': norm, 'out': s['flat_out']}
    loss, lse = b200.linear_xent(s['x'], s['w'], s['labels'], s['bias'])
    if op == 'xent':
        return {'loss': loss, 'lse': lse}
    dx, dw, db = b200.linear_xent_bwd(s['x'], s['w'], s['labels'], lse, s['dloss'], s['bias'])
    return {'loss': loss, 'lse': lse, 'dx': dx, 'dw': dw, 'dbias': db}


def run(state):
    if own:
        return _run_own(state)
    s, op = state, state['op']
    if op == 'embed':
        ids, table = s['ids'].long(), s['table']
        ok = (ids >= 0) & (ids < table.shape[0])
        rows = table[torch.where(ok, ids, 0)].float() * s['scale']
        return torch.where(ok[:, None], rows, 0.0).to(table.dtype)
    if op == 'embed_bwd':
        ids, V = s['ids'].long(), s['rows']
        ok = (ids >= 0) & (ids < V)
        order = torch.where(ok, ids, V)  # what belongs to no row falls into one past the end
        out = torch.zeros(V + 1, s['dout'].shape[1], device=ids.device)
        return out.index_add_(0, order, s['dout'].float())[:V] * s['scale']
    if op == 'clip':
        total = torch.stack([t.float().square().sum() for t in s['grads']]).sum()
        norm = total.sqrt() * s['scale']
        by = (s['max_norm'] / (norm + 1e-6)).clamp(max=1.0) * s['scale']
        _ = [o.copy_(t.float() * by) for t, o in zip(s['grads'], s['outs'])]
        return {'norm': norm, 'out': s['flat_out']}
    V = s['w'].shape[0]
    labels = s['labels'].long()
    ok = (labels >= 0) & (labels < V)
    labels = torch.where(ok, labels, 0)[:, None]
    x, w = torch.where(ok[:, None], s['x'].float(), 0.0), s['w'].float()
    logits = x @ w.t()
    if s['bias'] is not None:
        logits += s['bias'].float()
    top = logits.amax(1, keepdim=True)
    at = logits.gather(1, labels)
    p = logits.sub_(top).exp_()
    total = p.sum(1, keepdim=True)
    lse = top + total.log()
    loss = torch.where(ok, (lse - at)[:, 0], 0.0)
    lse = torch.where(ok, lse[:, 0] * math.log2(math.e), -math.inf)
    if op == 'xent':
        return {'loss': loss, 'lse': lse}
    dloss = torch.where(ok, s['dloss'], 0.0)[:, None]
    grad = p.mul_(dloss / total).scatter_add_(1, labels, -dloss)
    dt = s['x'].dtype
    return {'loss': loss, 'lse': lse, 'dx': (grad @ w).to(dt), 'dw': (grad.t() @ x).to(dt),
            'dbias': None if s['bias'] is None else grad.sum(0).to(dt)}


def work(case):
    """What cannot be left out: every input that matters read once, every output written once, the products without a
    recomputation of the logits."""
    op = case['op']
    if op == 'clip':
        # the groups' sizes follow their shares on average
        size = 4 - 2 * case['half']
        return {'bytes': case['elements'] * (size + (4 if case['widen'] else size)),
                'flops': 3 * case['elements']}
    T, V, C, e = case['T'], case['V'], case['C'], 4 if case['dtype'] == 'f32' else 2
    if op == 'embed':
        return {'bytes': 4 * T + min(T, V) * C * e + T * C * e, 'flops': T * C}
    if op == 'embed_bwd':
        return {'bytes': 4 * T + T * C * e + V * C * 4, 'flops': T * C}
    n = max(1.0, T * case['labelled'])
    moved = 4 * T + n * C * e + V * C * e + 8 * T
    if op == 'xent':
        return {'bytes': moved, 'flops': 2 * n * C * V}
    # x is read and dx written, w read and dw written, the rows without a label written as zeros
    return {'bytes': moved + 4 * T + T * C * e + V * C * e, 'flops': 6 * n * C * V}


def exact(case, seed):
    """The definitions in float64."""
    s, op = prepare(case, seed), case['op']
    if op == 'embed':
        table = s['table'].double()
        table = torch.cat([table, torch.zeros_like(table[:1])])  # the last row: no token
        return torch.nn.functional.embedding(s['ids'].long().remainder(case['V'] + 1),
                                             table).mul_(s['scale'])
    if op == 'embed_bwd':
        # sums of the tokens in the order of their ids, as differences of running sums
        ids = s['ids'].long()
        dout = s['dout'].double()[ids >= 0]
        ids, order = ids[ids >= 0].sort(stable=True)
        ends = torch.bincount(ids, minlength=case['V']).cumsum(0)
        run_ = torch.cat([torch.zeros_like(dout[:1]), dout[order].cumsum(0)]) if len(ids) else (
            torch.zeros(1, case['C'], dtype=torch.float64, device='cuda'))
        return (run_[ends] - run_[torch.cat([ends.new_zeros(1), ends[:-1]])]) * s['scale']
    if op == 'clip':
        total = sum(float(t.double().square().sum()) for t in s['grads'])
        norm = math.sqrt(total) * s['scale']
        by = s['scale'] * min(1.0, s['max_norm'] / (norm + 1e-6))
        out = {}
        for kind, flat in s['flat'].items():
            mine = torch.zeros(flat.numel(), dtype=torch.float64, device='cuda')
            for t in s['grads']:
                if t.dtype == flat.dtype:
                    b = t.storage_offset()
                    mine[b:b + t.numel()] = t.double() * by
            out[kind] = mine
        return {'norm': torch.tensor(norm, dtype=torch.float64), 'out': out}
    V = case['V']
    rows = (s['labels'] >= 0).nonzero()[:, 0]
    labels = s['labels'][rows].long()
    x, w = s['x'].double(), s['w'].double()
    dx, loss = torch.zeros_like(x), torch.zeros(len(x), dtype=torch.float64, device='cuda')
    lse = torch.full_like(loss, -math.inf)
    dw, db = torch.zeros_like(w), torch.zeros(V, dtype=torch.float64, device='cuda')
    step = max(1, (1 << 28) // V)
    for at in range(0, len(rows), step):
        r, y = rows[at:at + step], labels[at:at + step]
        logits = x[r] @ w.t()
        if s['bias'] is not None:
            logits += s['bias'].double()
        z = torch.logsumexp(logits, 1)
        loss[r] = torch.nn.functional.cross_entropy(logits, y, reduction='none')
        lse[r] = z / math.log(2.0)
        if op == 'xent':
            continue
        grad = (logits - z[:, None]).exp_()
        grad[torch.arange(len(r), device='cuda'), y] -= 1.0
        grad *= s['dloss'][r, None].double()
        dx[r] = grad @ w
        dw += grad.t() @ x[r]
        db += grad.sum(0)
    if op == 'xent':
        return {'loss': loss, 'lse': lse}
    return {'loss': loss, 'lse': lse, 'dx': dx, 'dw': dw,
            'dbias': None if s['bias'] is None else db}

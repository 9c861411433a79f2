"""Cases of the class-head operators: layer normalisation, the matrix product with its epilogue, and the log
probabilities of given labels.

Every operator is here in its plain form (elementary torch operations in 32 bits, rounded once at the end), as the
call a user makes of the package (`own`), and, apart from both, by its definition in 64 bits (`exact`).
"""
import math

import torch

own = False

DEVICE = 'cuda'
TYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
EPS = 1e-5


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # one region's feature vector normalised while serving: latency is all there is
        {'name': 'norm_one_row', 'op': 'norm', 'rows': 1, 'D': 1024, 'type': 'bf16', 'train': False},
        # the features of SSD300's 8732 default boxes, batch of 8, an odd width, training in single precision
        {'name': 'norm_ssd_odd_train', 'op': 'norm', 'rows': 69856, 'D': 257, 'type': 'fp32', 'train': True},
        # a wide head over RetinaNet-800's 120087 anchors, two images, training
        {'name': 'norm_wide_train', 'op': 'norm', 'rows': 240174, 'D': 1024, 'type': 'bf16', 'train': True},
        # one layer of a head's tower for four regions: the weight is all that is read
        {'name': 'linear_four_rows', 'op': 'linear', 'M': 4, 'K': 4096, 'N': 4096, 'type': 'bf16', 'act': 'silu',
         'bias': True, 'residual': True, 'out': 'same', 'train': False},
        # scores of RetinaNet's 81 classes for the anchors of one 800-pixel image, in single precision
        {'name': 'linear_scores_fp32', 'op': 'linear', 'M': 120087, 'K': 256, 'N': 81, 'type': 'fp32', 'act': 'sigmoid',
         'bias': True, 'residual': False, 'out': 'same', 'train': False},
        # one training step of a large tower layer
        {'name': 'linear_tower_train', 'op': 'linear', 'M': 16384, 'K': 4096, 'N': 4096, 'type': 'bf16', 'act': 'gelu',
         'bias': True, 'residual': True, 'out': 'same', 'train': True},
        # SSD300's default boxes against 1203 classes: no size is a multiple of a tile
        {'name': 'linear_ragged_train', 'op': 'linear', 'M': 8732, 'K': 1000, 'N': 1203, 'type': 'fp16', 'act': 'relu',
         'bias': True, 'residual': False, 'out': 'same', 'train': True},
        # the last layer of RetinaNet's class head over four 800-pixel images: 81 columns, single-precision logits, training
        {'name': 'linear_classes_train', 'op': 'linear', 'M': 480348, 'K': 256, 'N': 81, 'type': 'bf16', 'act': 'none',
         'bias': True, 'residual': False, 'out': 'fp32', 'train': True},
        # one answer over a large vocabulary: its alternatives and its entropy
        {'name': 'logprob_one_row', 'op': 'logprob', 'rows': 1, 'C': 131072, 'type': 'bf16', 'top': 20, 'entropy': True,
         'masked': True, 'train': False},
        # confidence of every anchor of four 800-pixel images over RetinaNet's 81 classes, training
        {'name': 'logprob_anchors_train', 'op': 'logprob', 'rows': 480348, 'C': 81, 'type': 'fp32', 'top': 0, 'entropy': True,
         'masked': False, 'train': True},
        # many answers over an odd vocabulary with their five best alternatives
        {'name': 'logprob_top5', 'op': 'logprob', 'rows': 2048, 'C': 49999, 'type': 'fp16', 'top': 5, 'entropy': False,
         'masked': False, 'train': False},
        # a training batch over a large padded vocabulary: the loss and its gradient
        {'name': 'logprob_vocabulary_train', 'op': 'logprob', 'rows': 4096, 'C': 131071, 'type': 'bf16', 'top': 0, 'entropy': False,
         'masked': True, 'train': True},
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op, kind = rng.choice(['norm', 'linear', 'logprob']), rng.choice(['fp32', 'bf16', 'fp16'])
    train = rng.random() < 0.5
    if op == 'norm':
        D = _log(rng, 8, 8192)
        return {'op': op, 'rows': _log(rng, 1, max(1, min(240174, 240174 * 1024 // (2 * D)))), 'D': D, 'type': kind, 'train': train}
    if op == 'linear':
        K, N = _log(rng, 16, 4096), _log(rng, 16, 4096)
        if rng.random() < 0.5:
            K, N = -(-K // 8) * 8, -(-N // 8) * 8
        act = rng.choice(['none', 'relu', 'gelu', 'silu', 'sigmoid'])
        most = min(16384 * 4096 * 4096 // (K * N), 480348, (1 << 28) // max(K, N))
        if kind == 'fp32':
            most //= 4
        return {'op': op, 'M': _log(rng, 1, max(1, most)), 'K': K, 'N': N, 'type': kind, 'act': act, 'bias': rng.random() < 0.7,
                'residual': rng.random() < 0.4, 'out': rng.choice(['same', 'same', 'fp32']), 'train': train}
    C = _log(rng, 2, 262144)
    top = rng.choice([0, 0, 1, 5, 20, 64])
    return {'op': op, 'rows': _log(rng, 1, max(1, min(480348, (1 << 28) // C))), 'C': C, 'type': kind, 'top': min(top, C),
            'entropy': rng.random() < 0.5, 'masked': rng.random() < 0.5, 'train': train}


# ------------------------------------------------------------------ inputs

def _sizes(case):
    if case['op'] == 'norm':
        return (case['rows'], case['D'])
    if case['op'] == 'linear':
        return (case['M'], case['N'])
    return (case['rows'], case['C'])


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    t = TYPES[case['type']]

    def normal(*shape, scale=1.0, shift=0.0, dtype=t):
        return (torch.randn(*shape, generator=g, device=DEVICE) * scale + shift).to(dtype)

    s = {'case': case}
    if case['op'] == 'norm':
        rows, D = case['rows'], case['D']
        # features of unlike scale and offset from row to row
        spread = torch.rand(rows, 1, generator=g, device=DEVICE) * 2 + 0.5
        offset = torch.randn(rows, 1, generator=g, device=DEVICE)
        s['x'] = torch.randn(rows, D, generator=g, device=DEVICE).mul_(spread).add_(offset).to(t)
        s['weight'], s['bias'] = normal(D, scale=0.2, shift=1.0), normal(D, scale=0.2)
        leaves = ['x', 'weight', 'bias']
    elif case['op'] == 'linear':
        M, K, N = case['M'], case['K'], case['N']
        s['x'], s['weight'] = normal(M, K), normal(N, K, scale=K ** -0.5)
        s['bias'] = normal(N, scale=0.5) if case['bias'] else None
        s['residual'] = normal(M, N, dtype=torch.float32 if case['out'] == 'fp32' else t) if case['residual'] else None
        leaves = ['x', 'weight'] + [k for k in ('bias', 'residual') if s[k] is not None]
    else:
        rows, C = case['rows'], case['C']
        x = torch.randn(rows, C, generator=g, device=DEVICE).mul_(2.0)
        valid = C - C // 32 if case['masked'] else C
        labels = torch.randint(0, valid, (rows,), generator=g, device=DEVICE)
        # a model that has learnt something: the label's logit stands out in most rows
        x.scatter_add_(1, labels[:, None], torch.rand(rows, 1, generator=g, device=DEVICE) * math.log(C + 1.0))
        if case['masked']:                                      # the vocabulary's padding is never an answer
            x[:, valid:] = float('-inf')
        if rows > 1:                                            # rows that do not take part carry the ignore label
            labels = torch.where(torch.rand(rows, generator=g, device=DEVICE) < 0.1, torch.full_like(labels, -1), labels)
        s['x'], s['labels'] = x.to(t), labels
        leaves = ['x']
    if case['train']:
        for k in leaves:
            s[k].requires_grad_()
        s['leaves'] = leaves
        if case['op'] == 'logprob':
            s['grad'] = normal(case['rows'], dtype=torch.float32)
            s['grad_entropy'] = normal(case['rows'], scale=0.1, dtype=torch.float32) if case['entropy'] else None
        else:
            out = torch.float32 if case.get('out') == 'fp32' else t
            s['grad'] = normal(*_sizes(case), dtype=out)
    return s


# ------------------------------------------------------------------ one pass

def run(s):
    case = s['case']
    if own:
        return _own(s, case)
    with torch.no_grad():
        return {'norm': _plain_norm, 'linear': _plain_linear, 'logprob': _plain_logprob}[case['op']](s, case)


def _own(s, case):
    from object_detection_amd import ops
    if case['op'] == 'logprob':
        r = ops.label_log_probs(s['x'], s['labels'], top_k=case['top'], entropy=case['entropy'])
        out = {'log_probs': r.log_probs}
        if case['entropy']:
            out['entropy'] = r.entropy
        if case['top']:
            out['top_log_probs'], out['top_ids'] = r.top_log_probs, r.top_ids
        if case['train']:
            heads, grads = [r.log_probs], [s['grad']]
            if case['entropy']:
                heads, grads = heads + [r.entropy], grads + [s['grad_entropy']]
            out['grad_x'] = torch.autograd.grad(heads, [s['x']], grads)[0]
        return {k: v.detach() for k, v in out.items()}
    if case['op'] == 'norm':
        y = ops.layer_norm(s['x'], s['weight'], s['bias'], EPS)
    else:
        y = ops.linear(s['x'], s['weight'], s['bias'], activation=case['act'], residual=s['residual'],
                       out_dtype=torch.float32 if case['out'] == 'fp32' else None)
    out = {'y': y.detach()}
    if case['train']:
        grads = torch.autograd.grad(y, [s[k] for k in s['leaves']], s['grad'])
        out.update({'grad_' + k: v for k, v in zip(s['leaves'], grads)})
    return out


def _plain_norm(s, case):
    x, w, b = s['x'].float(), s['weight'].float(), s['bias'].float()
    c = x - x.mean(1, keepdim=True)
    r = ((c * c).mean(1, keepdim=True) + EPS).rsqrt()
    h = c * r
    out = {'y': (h * w + b).to(s['x'].dtype)}
    if case['train']:
        g = s['grad'].float()
        gw = g * w
        gx = (gw - gw.mean(1, keepdim=True) - h * (gw * h).mean(1, keepdim=True)) * r
        out['grad_x'] = gx.to(s['x'].dtype)
        out['grad_weight'] = (g * h).sum(0).to(s['weight'].dtype)
        out['grad_bias'] = g.sum(0).to(s['bias'].dtype)
    return out


def _plain_act(z, act):
    """The activation of z and its derivative."""
    if act == 'relu':
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if act == 'sigmoid':
        p = 1 / (1 + (-z).exp())
        return p, p * (1 - p)
    if act == 'silu':
        p = 1 / (1 + (-z).exp())
        return z * p, p * (1 + z * (1 - p))
    if act == 'gelu':
        c = 0.5 * (1 + (z * 0.5 ** 0.5).erf())
        return z * c, c + z * (z * z * -0.5).exp() * (2 * math.pi) ** -0.5
    return z, None


def _plain_linear(s, case):
    x, w = s['x'].float(), s['weight'].float()
    z = x @ w.t()
    if s['bias'] is not None:
        z = z + s['bias'].float()
    y, d = _plain_act(z, case['act'])
    if s['residual'] is not None:
        y = y + s['residual'].float()
    out = {'y': y.to(torch.float32 if case['out'] == 'fp32' else s['x'].dtype)}
    if case['train']:
        g = s['grad'].float()
        dz = g if d is None else g * d
        out['grad_x'] = (dz @ w).to(s['x'].dtype)
        out['grad_weight'] = (dz.t() @ x).to(s['weight'].dtype)
        if s['bias'] is not None:
            out['grad_bias'] = dz.sum(0).to(s['bias'].dtype)
        if s['residual'] is not None:
            out['grad_residual'] = s['grad'].to(s['residual'].dtype)
    return out


def _plain_logprob(s, case):
    x, labels = s['x'].float(), s['labels']
    m = x.amax(1, keepdim=True)
    e = (x - m).exp()
    total = e.sum(1, keepdim=True)
    lp = (x - m) - total.log()
    part = labels >= 0
    at = labels.clamp(min=0)[:, None]
    out = {'log_probs': torch.where(part, lp.gather(1, at)[:, 0], torch.zeros_like(m[:, 0]))}
    if case['entropy'] or case['train']:
        p = e / total
    if case['entropy']:
        ent = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1)
        out['entropy'] = ent
    if case['top']:
        # the best first, the lower index first among equals: one whole number orders both
        bits = (x + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7fffffff) - 1, bits)
        key = order * 2 ** 32 + (2 ** 32 - 1 - torch.arange(x.shape[1], device=x.device))
        ids = key.topk(case['top'], dim=1).indices
        out['top_log_probs'], out['top_ids'] = lp.gather(1, ids), ids
    if case['train']:
        g = torch.where(part, s['grad'], torch.zeros_like(s['grad']))[:, None]
        gx = -g * p
        gx.scatter_add_(1, at, g)
        if case['entropy']:
            gx = gx - s['grad_entropy'][:, None] * torch.where(p > 0, p * (lp + ent[:, None]), torch.zeros_like(p))
        out['grad_x'] = gx.to(s['x'].dtype)
    return out


# ------------------------------------------------------------------ what one pass cannot do without

def work(case):
    size = 4 if case['type'] == 'fp32' else 2
    if case['op'] == 'norm':
        n = case['rows'] * case['D']
        return {'bytes': size * (n * (5 if case['train'] else 2) + case['D'] * (5 if case['train'] else 2)),
                'flops': n * (22 if case['train'] else 8)}
    if case['op'] == 'linear':
        M, K, N = case['M'], case['K'], case['N']
        o = 4 if case['out'] == 'fp32' else size
        forward = size * (M * K + N * K + (N if case['bias'] else 0)) + o * M * N * (2 if case['residual'] else 1)
        # the backward pass: the gradient read, those of x, the weight and the bias written; the residual's is the one read
        backward = o * M * N + size * (M * K + N * K + (N if case['bias'] else 0))
        return {'bytes': forward + (backward if case['train'] else 0), 'flops': 2 * M * N * K * (3 if case['train'] else 1)}
    n = case['rows'] * case['C']
    rows = case['rows'] * (8 + 4 + (4 if case['entropy'] else 0) + 12 * case['top'] + (8 if case['train'] else 0))
    return {'bytes': size * n * (3 if case['train'] else 1) + rows, 'flops': n * (12 if case['train'] else 5)}


# ------------------------------------------------------------------ by definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case['op'] == 'norm':
            return _exact_norm(s, case)
        if case['op'] == 'linear':
            return _exact_linear(s, case)
        return _exact_logprob(s, case)


def _exact_norm(s, case):
    x, w, b = s['x'].double(), s['weight'].double(), s['bias'].double()
    var, mean = torch.var_mean(x, dim=1, unbiased=False)
    sd = torch.sqrt(var + EPS)[:, None]
    h = torch.sub(x, mean[:, None]).div_(sd)
    out = {'y': torch.addcmul(b, h, w)}
    if case['train']:
        g = s['grad'].double()
        out['grad_weight'] = torch.einsum('rd,rd->d', g, h)
        out['grad_bias'] = g.sum(dim=0)
        # the projection of w * g off the vectors 1 and h, over the deviation
        u = g.mul(w)
        out['grad_x'] = (u - u.mean(dim=1)[:, None] - h * ((u * h).sum(dim=1) / case['D'])[:, None]) / sd
    return out


def _exact_linear(s, case):
    x, w = s['x'].double(), s['weight'].double()
    z = torch.mm(x, w.t().contiguous())
    if s['bias'] is not None:
        z += s['bias'].double()
    act = case['act']
    if act == 'relu':
        y, d = torch.relu(z), (z > 0).double()
    elif act == 'sigmoid':
        y = torch.sigmoid(z)
        d = y * torch.sigmoid(-z)
    elif act == 'silu':
        q = torch.sigmoid(z)
        y = z * q
        d = q + y * torch.sigmoid(-z)
    elif act == 'gelu':
        c = torch.special.ndtr(z)
        y, d = z * c, c + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
    else:
        y, d = z, None
    if s['residual'] is not None:
        y = y + s['residual'].double()
    out = {'y': y}
    if case['train']:
        dz = s['grad'].double()
        if d is not None:
            dz = dz * d
        out['grad_x'] = torch.mm(dz, w)
        out['grad_weight'] = torch.mm(dz.t().contiguous(), x)
        if s['bias'] is not None:
            out['grad_bias'] = dz.sum(dim=0)
        if s['residual'] is not None:
            out['grad_residual'] = s['grad'].double()
    return out


def _exact_logprob(s, case):
    x, labels = s['x'].double(), s['labels']
    lse = torch.logsumexp(x, dim=1)
    take = labels.ge(0)
    lab = torch.where(take, labels, 0)
    out = {'log_probs': torch.where(take, x.gather(1, lab[:, None]).squeeze(1) - lse, 0.0)}
    lp = x.sub_(lse[:, None]) if not case['top'] else x - lse[:, None]
    if case['top']:
        out['top_log_probs'] = torch.topk(x, case['top'], dim=1, sorted=True).values - lse[:, None]
        out['top_ids'] = None
    if case['entropy']:
        ent = torch.special.entr(lp.exp()).sum(dim=1)
        out['entropy'] = ent
    if case['train']:
        q = lp.exp()
        gx = q * -torch.where(take, s['grad'].double(), 0.0)[:, None]
        rows = torch.nonzero(take).squeeze(1)
        gx[rows, lab[rows]] += s['grad'].double()[rows]
        if case['entropy']:
            gx -= s['grad_entropy'].double()[:, None] * (q * ent[:, None] - torch.special.entr(q))
        out['grad_x'] = gx
    return out

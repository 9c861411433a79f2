"""Class-head operators (layer_norm, linear, label_log_probs) against their definitions in 64 bits.

Tolerances are derived, not fitted.  U[t] is the largest relative error of one rounding to type t (half a step, 2^-24 /
2^-8 / 2^-11); E = 2^-24.  A sum of n fp32 terms is off by at most n E times the sum of their magnitudes whatever its order;
a handful of elementary operations adds a few E more.  Every bound below is such a count times the magnitudes it applies to.
"""
import math

import pytest
import torch

import object_detection_amd as D
from object_detection_amd import _lib, ops

E = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}     # the smallest step


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=g) * scale + shift).to(dtype).to('cuda')


def close(got, want, tol, what=''):
    """Every element of got within tol of want (64 bits); infinities and NaN in the same places.  A value of twice the output
    type's largest or so (the difference of its two ends) rounds to infinity: from max + half a step, max * (1 + U), on."""
    top = torch.finfo(got.dtype).max * (1 + U[got.dtype])
    want = torch.where(want.abs() >= top, want.sign() * math.inf, want)
    got = got.detach().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if want.numel() == 0:
        return
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)), (what, 'finite places differ')
    assert torch.equal(torch.isnan(want), torch.isnan(got)), (what, 'NaN places differ')
    assert torch.equal(want[~fine & ~torch.isnan(want)], got[~fine & ~torch.isnan(want)]), (what, 'infinities differ')
    over = ((got - want).abs() - tol)[fine]
    assert over.numel() == 0 or float(over.max()) <= 0, (what, 'over the bound by', float(over.max()), 'bound there',
                                                         float(torch.as_tensor(tol).expand_as(want)[fine][over.argmax()]))


# ------------------------------------------------------------------ layer_norm

def norm_def(x, w, b, eps, g=None):
    """Values in 64 bits and the magnitudes the bounds are made of."""
    x = x.double()
    n = x.shape[-1]
    mean = x.mean(-1, keepdim=True)
    sd = ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    h = (x - mean) / sd
    wd = torch.ones_like(x[:1]) if w is None else w.double()
    bd = torch.zeros_like(x[:1]) if b is None else b.double()
    # h: the mean is off by at most (n + 2) E mean|x|, each difference by E |x - mean|, the deviation by (n + 8) E relative
    eh = ((n + 4) * E * x.abs().mean(-1, keepdim=True) + E * x.abs()) / sd * 2 + (n + 10) * E * h.abs()
    y = h * wd + bd
    out = {'y': (y, eh * wd.abs() + 2 * E * (h * wd).abs() + E * y.abs())}
    if g is not None:
        g = g.double()
        gw = g * wd
        a, c = gw.mean(-1, keepdim=True), (gw * h).mean(-1, keepdim=True)
        gx = (gw - a - h * c) / sd
        ec = (gw.abs() * eh).mean(-1, keepdim=True) + (n + 4) * E * (gw * h).abs().mean(-1, keepdim=True)
        ex = ((n + 8) * E * gw.abs().mean(-1, keepdim=True) + h.abs() * ec + eh * c.abs() + 4 * E * (gw.abs() + a.abs() + (h * c).abs())) / sd
        out['gx'] = (gx, ex + (n + 10) * E * gx.abs())
        rows = x.shape[0]
        out['gw'] = ((g * h).sum(0), (g.abs() * eh).sum(0) + (rows + 4) * E * (g * h).abs().sum(0))
        out['gb'] = (g.sum(0), (rows + 4) * E * g.abs().sum(0))
    return out


def check_norm(x, w, b, eps, g, seen=''):
    t = x.dtype
    leaves = [v.detach().requires_grad_() for v in (x, w, b) if v is not None]
    it = iter(leaves)
    xx, ww, bb = next(it), None if w is None else next(it), None if b is None else next(it)
    y = ops.layer_norm(xx, ww, bb, eps)
    assert y.dtype == t and y.shape == x.shape
    plain = ops.layer_norm(x, w, b, eps)
    assert torch.equal(plain.nan_to_num(), y.detach().nan_to_num())
    grads = torch.autograd.grad(y, leaves, g)
    again = torch.autograd.grad(ops.layer_norm(xx, ww, bb, eps), leaves, g)
    for u, v in zip(grads, again):
        assert torch.equal(u.nan_to_num(), v.nan_to_num())          # no atomics: the same bits every time
    n = x.shape[-1]
    want = norm_def(x.reshape(-1, n), w, b, eps, g.reshape(-1, n))
    got = {'y': y.reshape(-1, n), 'gx': grads[0].reshape(-1, n)}
    rest = list(grads[1:])
    if w is not None:
        got['gw'] = rest.pop(0)
    if b is not None:
        got['gb'] = rest.pop(0)
    for k, v in got.items():
        val, tol = want[k]
        close(v, val, tol + U[v.dtype] * (val.abs() + tol) + TINY[v.dtype], f'{seen} {k}')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('rows,n', [(1, 1), (3, 7), (2, 64), (5, 257), (64, 1000), (129, 256), (3, 2048), (2, 4100), (3, 8192),
                                    (2, 16385), (1, 70001), (1000, 96), (3000, 40), (700, 520)])
def test_layer_norm(dtype, rows, n):
    g = gen(rows * 1000 + n)
    x = randn(g, rows, n, dtype=dtype, scale=2.0, shift=0.7)
    w, b = randn(g, n, dtype=dtype, scale=0.3, shift=1.0), randn(g, n, dtype=dtype)
    gr = randn(g, rows, n, dtype=dtype)
    check_norm(x, w, b, 1e-5, gr, 'both')
    check_norm(x, None, None, 1e-3, gr, 'neither')
    check_norm(x, w.float(), None, 1e-5, gr, 'fp32 weight')
    check_norm(x, None, b.float(), 1e-5, gr, 'fp32 bias')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_layer_norm_layouts(dtype):
    g = gen(5)
    wide = randn(g, 6, 7, 83, dtype=dtype)
    w, b = randn(g, 70, dtype=dtype), randn(g, 70, dtype=dtype)
    gr = randn(g, 6, 7, 70, dtype=dtype)
    for x in (wide[..., :70], wide[..., 3:73], wide[:, ::2, 1:71], wide.transpose(0, 1)[..., 13:]):
        gx = gr[:, :x.shape[1]] if x.shape[0] == 6 else gr.transpose(0, 1)
        check_norm(x, w, b, 1e-5, gx)
    check_norm(wide[..., :70], w, b, 1e-5, gr[:1, :1, :1].expand(6, 7, 70), 'expanded gradient')
    check_norm(wide[0, 0, :70], w, b, 1e-5, gr[0, 0], 'one axis')
    strided = randn(g, 140, dtype=dtype)[::2]
    check_norm(wide[..., :70], strided, strided, 1e-5, gr, 'strided weight')


@pytest.mark.gpu
def test_layer_norm_no_rows():
    x = torch.zeros(0, 12, device='cuda', requires_grad=True)
    w = torch.ones(12, device='cuda', requires_grad=True)
    y = ops.layer_norm(x, w, w)
    gx, gw = torch.autograd.grad(y, [x, w], torch.zeros(0, 12, device='cuda'))
    assert y.shape == gx.shape == (0, 12) and torch.equal(gw, torch.zeros(12, device='cuda'))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_layer_norm_odd_rows(dtype):
    """A row without variance, one far from zero, one of large values, one with an infinity, one with NaN: each keeps to itself."""
    g = gen(6)
    n = 300
    x = randn(g, 6, n, dtype=dtype)
    x[1] = 3.0
    x[2] += 100
    x[3] *= 1000
    x[4, 17] = float('inf')
    x[5, 299] = float('nan')
    w, b = randn(g, n, dtype=dtype), randn(g, n, dtype=dtype)
    y = ops.layer_norm(x, w, b)
    val, tol = norm_def(x[:4], w, b, 1e-5)['y']
    close(y[:4], val, tol + U[dtype] * (val.abs() + tol) + TINY[dtype])
    assert torch.equal(y[1], b)                                       # no variance: h = 0 exactly
    assert torch.isnan(y[4:]).all()


# ------------------------------------------------------------------ linear

def act_def(z, act):
    if act == 'relu':
        return z.relu(), (z > 0).double(), 1.0, 0.0
    if act == 'sigmoid':
        p = z.sigmoid()
        return p, p * (1 - p), 0.25, 0.1
    if act == 'silu':
        p = z.sigmoid()
        return z * p, p + z * p * (1 - p), 1.1, 0.5
    if act == 'gelu':
        c = torch.special.ndtr(z)
        return z * c, c + z * (-z * z / 2).exp() / math.sqrt(2 * math.pi), 1.13, 0.8
    return z, torch.ones_like(z), 1.0, 0.0                             # value, slope, the most of |slope| and of |its change|


def check_linear(x, w, b, r, act, out_dtype, g, seen=''):
    t = x.dtype
    leaves = {k: v.detach().requires_grad_() for k, v in (('x', x), ('w', w), ('b', b), ('r', r)) if v is not None}
    y = ops.linear(leaves['x'], leaves['w'], leaves.get('b'), act, leaves.get('r'), out_dtype)
    assert y.dtype == (out_dtype or t) and y.shape == (*x.shape[:-1], w.shape[0])
    assert torch.equal(ops.linear(x, w, b, act, r, out_dtype), y.detach())
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), g)))
    again = torch.autograd.grad(ops.linear(leaves['x'], leaves['w'], leaves.get('b'), act, leaves.get('r'), out_dtype), list(leaves.values()), g)
    for u, v in zip(grads.values(), again):
        assert torch.equal(u, v)
    N, K = w.shape
    xd, wd = x.reshape(-1, K).double(), w.double()
    M = xd.shape[0]
    z = xd @ wd.t()
    ez = (K + 4) * E * (xd.abs() @ wd.abs().t())
    if b is not None:
        z = z + b.double()
        ez = ez + 2 * E * (z.abs() + b.double().abs())
    val, slope, most, bend = act_def(z, act)
    ey = most * ez + 16 * E * (val.abs() + z.abs() * (act not in ('none', 'relu')))
    if r is not None:
        val = val + r.reshape(-1, N).double()
        ey = ey + 2 * E * val.abs()
    close(y.reshape(-1, N), val, ey + U[y.dtype] * (val.abs() + ey) + TINY[y.dtype], f'{seen} y')
    gd = g.reshape(-1, N).double()
    dz = gd * slope
    # the slope is taken at z rounded to the type of x; relu's jumps where the sign of z is not certain
    es = 24 * E * (1 + z.abs()) * (act not in ('none', 'relu')) + (bend * (ez + U[t] * (z.abs() + ez)) if act not in ('none', 'relu') else 0.0)
    if act == 'relu':
        es = (z.abs() <= ez + TINY[t]).double()
    edz = gd.abs() * es + E * dz.abs()
    rounded = edz + (U[t] * (dz.abs() + edz) + TINY[t] if act != 'none' or (out_dtype or t) != t else 0.0)
    want = {'x': (dz @ wd, rounded @ wd.abs() + (N + 4) * E * ((dz.abs() + rounded) @ wd.abs())),
            'w': (dz.t() @ xd, rounded.t() @ xd.abs() + (M + 4) * E * ((dz.abs() + rounded).t() @ xd.abs()))}
    if b is not None:
        want['b'] = (dz.sum(0), edz.sum(0) + (M + 4) * E * (dz.abs() + edz).sum(0))
    if r is not None:
        want['r'] = (gd, torch.zeros_like(gd))
    for k, (v, tol) in want.items():
        got = grads[k].reshape(v.shape)
        assert got.dtype == leaves[k].dtype
        close(got, v, tol + U[got.dtype] * (v.abs() + tol) + TINY[got.dtype], f'{seen} grad {k}')


LINEAR_SIZES = [(1, 1, 1), (1, 1203, 1000), (1, 64, 4096), (3, 64, 33), (4, 1024, 512), (8, 200, 264), (16, 96, 640), (17, 81, 256),
                (33, 70, 2048), (65, 129, 70), (200, 257, 1000), (256, 256, 64), (300, 96, 64), (128, 128, 128), (513, 1000, 136),
                (700, 1, 50), (260, 3, 1), (1, 5, 20000), (5000, 81, 256), (40, 2500, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('M,N,K', LINEAR_SIZES)
def test_linear(dtype, M, N, K):
    g = gen(M + 7 * N + 13 * K)
    x, w = randn(g, M, K, dtype=dtype), randn(g, N, K, dtype=dtype, scale=K ** -0.5)
    b, r, gr = randn(g, N, dtype=dtype), randn(g, M, N, dtype=dtype), randn(g, M, N, dtype=dtype)
    check_linear(x, w, None, None, 'none', None, gr, 'plain')
    check_linear(x, w, b, r, 'gelu', None, gr, 'gelu')
    check_linear(x, w, b.float(), None, 'relu', None, gr, 'relu')
    check_linear(x, w, b, r.float(), 'silu', torch.float32, gr.float(), 'silu, fp32 out')
    check_linear(x, w, None, None, 'sigmoid', torch.float32, gr.float(), 'sigmoid, fp32 out')
    check_linear(x, w, b, None, 'none', torch.float32, gr.float(), 'fp32 out')


# many rows against few columns (whole weight on chip), and products that fill the chip with large tiles; each with rows that
# start at multiples of 16 bytes and without
@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('M,N,K', [(32768, 81, 256), (33001, 20, 37), (33001, 64, 300), (32769, 97, 61), (98304, 200, 24), (98311, 301, 31),
                                   (3584, 3712, 3600), (3600, 3700, 3650)])
def test_linear_large(dtype, M, N, K):
    g = torch.Generator(device='cuda').manual_seed(M + N + K)

    def rand(*shape, dtype=dtype, scale=1.0):
        return (torch.randn(*shape, generator=g, device='cuda') * scale).to(dtype)
    x, w, b, r, gr = rand(M, K), rand(N, K, scale=K ** -0.5), rand(N), rand(M, N), rand(M, N)
    check_linear(x, w, b, r, 'gelu', None, gr, 'gelu')
    check_linear(x, w, None, r.float(), 'relu', torch.float32, gr.float(), 'relu, fp32 out')
    check_linear(x, w, b, None, 'none', None, gr, 'plain')
    wide = torch.cat([rand(M, 3), x], 1)
    check_linear(wide[:, 3:], w, b, None, 'silu', None, gr, 'off alignment')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('M', [1, 5, 90])
def test_linear_layouts(dtype, M):
    """Row strides, starts off every alignment, transposed and expanded operands, leading axes."""
    g = gen(8)
    K, N = 72, 50
    wide = randn(g, 3, M, K + 11, dtype=dtype)
    ww = randn(g, N + 3, K + 5, dtype=dtype, scale=0.1)
    b, gr = randn(g, N, dtype=dtype), randn(g, 3, M, N, dtype=dtype)
    for x in (wide[..., :K], wide[..., 1:K + 1], wide[..., 8:K + 8], wide[..., 5:K + 5]):
        for w in (ww[:N, :K], ww[3:, 5:], ww[1:N + 1, 3:K + 3]):
            check_linear(x, w, b, gr, 'silu', None, gr)
    check_linear(wide.transpose(0, 1)[..., :K], ww[:N, :K], None, None, 'none', None, gr.transpose(0, 1), 'transposed')
    check_linear(wide[..., :K], ww.t().contiguous().t()[:N, :K], None, None, 'none', None, gr, 'weight by columns')
    check_linear(wide[..., :K], ww[:N, :K], b, None, 'none', None, gr[:1, :1, :1].expand(3, M, N), 'expanded gradient')
    check_linear(wide[0, 0, :K], ww[:N, :K], b, None, 'gelu', None, gr[0, 0], 'one axis')
    check_linear(wide[..., :K], ww[:N, :K], randn(g, 2 * N, dtype=dtype)[::2], gr[..., :1].expand(3, M, N), 'relu', None, gr, 'strided bias')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_linear_whole_values(dtype):
    """Whole numbers whose products and sums every type holds: the result is exact, so no element, column or split of the
    long axis is lost, doubled or misplaced; with more rows than one round of tiles and a long contraction."""
    g = gen(9)
    for M, N, K in ((1, 300, 4096), (7, 130, 1000), (64, 64, 64), (530, 270, 200), (3000, 19, 24), (2, 2, 9000), (1040, 512, 520), (33000, 24, 64), (98400, 300, 24),
                    (3600, 3700, 1000)):
        x = torch.randint(-1, 2, (M, K), generator=g).to(dtype).to('cuda').requires_grad_()
        w = (torch.randint(-1, 2, (N, K), generator=g) * (torch.rand(N, K, generator=g) < 100.0 / K)).to(dtype).to('cuda').requires_grad_()
        gr = (torch.randint(-1, 2, (M, N), generator=g) * (torch.rand(M, N, generator=g) < min(1.0, 100.0 / max(M, N)))).to(dtype).to('cuda')
        y = ops.linear(x, w)
        gx, gw = torch.autograd.grad(y, [x, w], gr)
        for got, want in ((y, x.double() @ w.double().t()), (gx, gr.double() @ w.double()), (gw, gr.double().t() @ x.double())):
            assert float(want.detach().abs().max()) <= 256 and torch.equal(got.detach().double(), want), (M, N, K)


@pytest.mark.gpu
@pytest.mark.parametrize('M,N,K', [(3, 20, 40), (70, 81, 256), (700, 203, 96), (5000, 81, 64), (3600, 3704, 3656)])
@pytest.mark.parametrize('act,out', [('none', torch.float32), ('gelu', torch.float32), ('relu', torch.float32), ('silu', torch.float16),
                                     ('sigmoid', torch.float32)])
def test_half_gradients_keep_their_range(M, N, K, act, out):
    """fp16 operands with gradients far below and far above fp16's range, up to 2^30 apart in one call: dz is brought into range by a power of two
    before it is rounded, so that beside the half step of every element only 2^-39 of the largest gradient is lost (the smallest
    step of fp16 is 2^-24, the largest gradient lies at 2^14 or above, half a step is 2^-25)."""
    g = torch.Generator(device='cuda').manual_seed(M + N + K)

    def rand(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device='cuda') * scale).to(dtype)
    x, w = rand(M, K, dtype=torch.float16), rand(N, K, scale=K ** -0.5, dtype=torch.float16)
    b = rand(N)
    wide = torch.exp2(torch.randint(-30, 1, (M, N), generator=g, device='cuda').float())
    grads = {'mean': rand(M, N, scale=2.0 ** -26), 'wide': rand(M, N) * wide, 'zero': torch.zeros(M, N, device='cuda')}
    if out == torch.float32:
        grads.update(large=rand(M, N, scale=2.0 ** 20), small=rand(M, N, scale=2.0 ** -100), wide_large=rand(M, N, scale=2.0 ** 18) * wide,
                     strided=rand(M, N + 5, scale=2.0 ** -26)[:, 3:N + 3])
    else:
        grads = {k: (v * 2.0 ** 14 if k == 'mean' else v).half() for k, v in grads.items()}
    bb = b.clone().requires_grad_()
    # gradients below fp16's range leave it again only through an output: x and the weight carry them up by powers of two
    for name, gr in grads.items():
        up = 2.0 ** {'large': -14, 'wide_large': -14, **({'mean': 10, 'small': 13, 'strided': 10} if act == 'none' else {})}.get(name, 0)
        xs, ws = [(v * up).half() for v in (x.float(), w.float())]
        leaves = [xs.requires_grad_(), ws.requires_grad_(), bb]
        y = ops.linear(leaves[0], leaves[1], bb, act, None, out)
        gx, gw, gb = torch.autograd.grad(y, leaves, gr)
        xd, wd, gd = xs.detach().double(), ws.detach().double(), gr.double()
        z = xd @ wd.t() + b.double()
        ez = (K + 4) * E * (xd.abs() @ wd.abs().t()) + 2 * E * (z.abs() + b.double().abs())
        _, slope, _, bend = act_def(z, act)
        dz = gd * slope
        es = 0.0
        if act == 'relu':
            es = (z.abs() <= ez + TINY[torch.float16]).double()
        elif act != 'none':
            es = 24 * E * (1 + z.abs()) + bend * (ez + U[torch.float16] * (z.abs() + ez) + TINY[torch.float16])
        edz = gd.abs() * es + E * dz.abs()
        rounded = edz + U[torch.float16] * (dz.abs() + edz) + 2.0 ** -39 * gd.abs().max()
        for got, want, tol, what in ((gx, dz @ wd, rounded @ wd.abs() + (N + 4) * E * ((dz.abs() + rounded) @ wd.abs()), 'x'),
                                     (gw, dz.t() @ xd, rounded.t() @ xd.abs() + (M + 4) * E * ((dz.abs() + rounded).t() @ xd.abs()), 'w'),
                                     (gb, dz.sum(0), edz.sum(0) + (M + 4) * E * (dz.abs() + edz).sum(0), 'b')):
            # 2^-126: fp32 sums of the smallest gradients may be flushed
            close(got, want, tol + U[got.dtype] * (want.abs() + tol) + TINY[got.dtype] + 2.0 ** -126, f'{name} {what}')
        if name in ('mean', 'large') and act == 'none':
            assert gx.any() and gw.any() and torch.isfinite(gx).all()


@pytest.mark.gpu
def test_half_gradients_beyond_numbers():
    """Infinities and NaN among the gradients stay in their row and column and leave the scale of the others alone."""
    g = gen(24)
    x, w = randn(g, 90, 64, dtype=torch.float16).requires_grad_(), randn(g, 50, 64, dtype=torch.float16).requires_grad_()
    gr = randn(g, 90, 50, scale=2.0 ** -10)
    clean = torch.autograd.grad(ops.linear(x, w, out_dtype=torch.float32), [x, w], gr.index_fill(0, torch.tensor([7, 30], device='cuda'), 0.0))
    for bad in (math.inf, -math.inf, math.nan):
        gr2 = gr.clone()
        gr2[7], gr2[30] = 0.0, 0.0
        gr2[7, 3], gr2[30, 3] = bad, bad
        gx, gw = torch.autograd.grad(ops.linear(x, w, out_dtype=torch.float32), [x, w], gr2)
        keep_m, keep_n = torch.ones(90, dtype=torch.bool), torch.ones(50, dtype=torch.bool)
        keep_m[[7, 30]], keep_n[3] = False, False
        assert not torch.isfinite(gx[~keep_m]).any() and torch.equal(gx[keep_m][:, :], clean[0][keep_m])
        assert not torch.isfinite(gw[3]).any() and torch.equal(gw[keep_n], clean[1][keep_n])


@pytest.mark.gpu
@pytest.mark.parametrize('M,N,K', [(2, 20, 8), (2, 20, 2048), (150, 40, 64), (150, 40, 2048), (40, 2000, 4096), (3600, 3700, 640)])
def test_half_relu_keeps_the_sign_of_small_sums(M, N, K):
    """Sums of 2^-28 and -2^-28, below half of fp16's smallest step: the slope of relu is 1 and 0 there, not 0 twice.  All of
    it in powers of two, so that the gradients are exact."""
    x, w = torch.zeros(M, K, dtype=torch.float16, device='cuda'), torch.zeros(N, K, dtype=torch.float16, device='cuda')
    x[:, K - 1] = 2.0 ** -14
    w[:, K - 1] = 2.0 ** -14
    w[1::2] *= -1
    gr = torch.zeros(M, N, dtype=torch.float16, device='cuda')
    gr[:2, :4] = 1.0
    for b in (None, torch.zeros(N, device='cuda')):
        for out in (None, torch.float32):
            leaves = [x.requires_grad_(), w.requires_grad_()]
            y = ops.linear(*leaves, b, 'relu', None, out)
            gx, gw = torch.autograd.grad(y, leaves, gr.to(out or torch.float16))
            want_x, want_w = torch.zeros_like(x), torch.zeros_like(w)
            want_x[:2, K - 1] = 2 * 2.0 ** -14
            want_w[0:4:2, K - 1] = 2 * 2.0 ** -14
            assert torch.equal(gx, want_x) and torch.equal(gw, want_w)
            if out:
                assert torch.equal(y.detach(), torch.where(torch.arange(N, device='cuda') % 2 == 0, 2.0 ** -28, 0.0).expand(M, N))


@pytest.mark.gpu
def test_linear_no_rows():
    x, w = torch.zeros(0, 6, device='cuda', requires_grad=True), torch.ones(4, 6, device='cuda', requires_grad=True)
    b = torch.ones(4, device='cuda', requires_grad=True)
    y = ops.linear(x, w, b, 'gelu')
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], torch.zeros(0, 4, device='cuda'))
    assert y.shape == (0, 4) and gx.shape == (0, 6) and not gw.any() and not gb.any()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('M', [2, 70])
def test_linear_values_beyond_numbers(dtype, M):
    """NaN and infinities stay in their row and column; activations have their limits at the ends."""
    g = gen(10)
    x, w = randn(g, M, 40, dtype=dtype), randn(g, 33, 40, dtype=dtype)
    clean = ops.linear(x, w)
    x2, w2 = x.clone(), w.clone()
    x2[0, 39] = float('nan')
    w2[32, 0] = float('inf')
    y = ops.linear(x2, w2)
    assert torch.isnan(y[0]).all() and torch.equal(y[1:, :32], clean[1:, :32]) and not torch.isfinite(y[1:, 32]).any()
    big = torch.tensor([[300.0], [-300.0]], dtype=dtype, device='cuda')
    one = torch.full((1, 1), 200.0, dtype=dtype, device='cuda')
    b = torch.zeros(1, dtype=dtype, device='cuda')
    for act, ends, slopes in (('sigmoid', (1, 0), (0, 0)), ('silu', (60000, 0), (1, 0)), ('gelu', (60000, 0), (1, 0)), ('relu', (60000, 0), (1, 0))):
        xx = b.detach().requires_grad_()
        y = ops.linear(big, one, xx, act, out_dtype=torch.float32)
        assert y.flatten().tolist() == pytest.approx(ends, abs=0, rel=2e-3), act
        for k in (0, 1):
            gr = torch.zeros(2, 1, device='cuda')
            gr[k] = 1
            assert float(torch.autograd.grad(y, xx, gr, retain_graph=True)[0]) == slopes[k], act
    # a pre-activation that overflows the type keeps its slope
    if dtype is torch.float16:
        xx = b.detach().requires_grad_()
        y = ops.linear(big, one * 10, xx, 'gelu', out_dtype=torch.float32)
        assert float(torch.autograd.grad(y, xx, torch.ones(2, 1, device='cuda'))[0]) == 1.0 and float(y.detach()[1]) == 0.0


# ------------------------------------------------------------------ label_log_probs

def rank_def(x):
    """Ids in descending order, NaN first, equal values by ascending id."""
    v = (x.double() + 0.0).nan_to_num(nan=math.inf, posinf=1e300, neginf=-1e300)
    return torch.sort(v, dim=1, descending=True, stable=True).indices


def check_logprob(x, labels, k, entropy, seed=0, seen=''):
    C = x.shape[-1]
    lead = x.shape[:-1]
    leaf = x.detach().requires_grad_()
    r = ops.label_log_probs(leaf, labels, k, entropy)
    q = ops.label_log_probs(x, labels, k, entropy)
    assert r.log_probs.shape == lead and r.log_probs.dtype == torch.float32
    assert torch.equal(q.log_probs.nan_to_num(), r.log_probs.detach().nan_to_num())
    xd, t = x.reshape(-1, C).double(), labels.reshape(-1).long()
    m = xd.amax(1, keepdim=True)
    ref = torch.where(m == -math.inf, torch.zeros_like(m), m)
    d = xd - ref
    e = d.exp()
    s = e.sum(1, keepdim=True)
    none = s == 0
    lp = torch.where(none, torch.full_like(d, -math.inf), d - s.log())
    p = torch.where(none, torch.zeros_like(e), e / s)
    part = (t >= 0) & (t < C)
    at = t.clamp(0, C - 1)[:, None]
    fin = torch.where(p > 0, d, torch.zeros_like(d)).nan_to_num()
    spread = (p * fin.abs()).sum(1, keepdim=True).nan_to_num()          # the mean distance from the largest logit
    # exp of a rounded distance is off by (4 + 2 |d|) E relative, the sum of C such terms by C E more
    es = (C + 8) * E + (4 + 2 * spread) * E
    elp = es + 4 * E * (1 + d.abs().nan_to_num(posinf=0, neginf=0) + lp.abs().nan_to_num(posinf=0, neginf=0))
    val = torch.where(part, lp.gather(1, at)[:, 0], torch.zeros_like(s[:, 0]))
    close(r.log_probs.reshape(-1), val, torch.where(part, elp.gather(1, at)[:, 0], torch.zeros_like(val)), f'{seen} log_probs')
    ent = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1, keepdim=True)
    ent = torch.where(torch.isnan(s), s, ent)
    eent = (2 * es + (C + 16) * E) * (1 + spread + ent.abs().nan_to_num()) + 8 * E * (p * fin * fin).sum(1, keepdim=True).nan_to_num()
    if entropy:
        close(r.entropy.reshape(-1), ent[:, 0], eent[:, 0], f'{seen} entropy')
    else:
        assert r.entropy is None
    if k:
        ids = rank_def(x.reshape(-1, C))[:, :k]
        assert r.top_ids.shape == (*lead, k) and torch.equal(r.top_ids.reshape(-1, k), ids), f'{seen} ids'
        assert not r.top_log_probs.requires_grad and torch.equal(q.top_ids, r.top_ids)
        close(r.top_log_probs.reshape(-1, k), lp.gather(1, ids), elp.gather(1, ids), f'{seen} top')
    else:
        assert r.top_ids is None and r.top_log_probs is None
    gen_ = gen(seed + 77)
    for with_lp in ((True, False) if entropy else (True,)):
        g = randn(gen_, *lead) if with_lp else None
        h = randn(gen_, *lead) if entropy else None
        outs = [o for o, v in ((r.log_probs, g), (r.entropy, h)) if v is not None]
        gx = torch.autograd.grad(outs, leaf, [v for v in (g, h) if v is not None], retain_graph=True)[0]
        assert gx.dtype == x.dtype and gx.shape == x.shape
        gd = torch.zeros_like(s) if g is None else torch.where(part[:, None], g.reshape(-1, 1).double(), torch.zeros_like(s))
        hd = torch.zeros_like(s) if h is None else h.reshape(-1, 1).double()
        hit = torch.zeros_like(p).scatter_(1, at, part[:, None].double())
        pl = torch.where(p > 0, p * (lp + ent), torch.zeros_like(p))
        want = gd * (torch.where(none, torch.zeros_like(hit), hit) - p) - hd * pl
        ep = p * (es + (6 + 2 * d.abs().nan_to_num(posinf=0, neginf=0)) * E)
        tol = gd.abs() * (ep + E * (hit + p)) + hd.abs() * (ep * (lp.abs().nan_to_num(posinf=0, neginf=0) + ent.abs()) + p * (elp + eent)) + 8 * E * want.abs()
        takes = (part[:, None] | (hd != 0)) if h is None else torch.ones_like(s, dtype=torch.bool)
        want, tol = torch.where(takes, want, torch.zeros_like(want)), tol.nan_to_num(0, 0, 0) + 2.0 ** -126
        close(gx.reshape(-1, C), want, tol + U[x.dtype] * (want.abs().nan_to_num() + tol) + TINY[x.dtype], f'{seen} grad')
    return r


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('rows,C', [(1, 1), (3, 2), (70, 21), (500, 81), (9, 128), (33, 129), (5, 256), (2, 511), (7, 1000), (4, 1024),
                                    (3, 2049), (2, 4097), (9, 10007), (1, 131072), (2, 200003), (700, 3000)])
def test_label_log_probs(dtype, rows, C):
    g = gen(rows + 31 * C)
    x = randn(g, rows, C, dtype=dtype, scale=2.0)
    labels = torch.randint(-1, C + 1, (rows,), generator=g).cuda()
    check_logprob(x, labels, 0, False, seen='labels only')
    check_logprob(x, labels, min(C, 5), True, seen='all')
    check_logprob(x, labels, min(C, 64), False, seen='64')
    check_logprob(x, labels, 1, True, seen='best')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('C', [1, 6, 81, 300, 2100, 9000, 70000])
def test_label_log_probs_odd_rows(dtype, C):
    """Masked classes, rows with one class left and with none, the type's lowest value as a mask, equal values, huge spreads,
    NaN, infinities; ascending and descending rows, which bring every element or only the first ones among the best."""
    g = gen(11 + C)
    x = randn(g, 14, C, dtype=dtype, scale=3.0)
    low = torch.finfo(dtype).min
    x[0, C // 2:] = -math.inf
    x[1] = -math.inf
    x[2] = -math.inf
    x[2, C - 1] = 0.5
    x[3, C // 3:] = low
    x[4] = low
    x[5] = 1.25
    x[6, 0], x[6, C - 1] = torch.finfo(dtype).max, low
    x[7] = torch.linspace(-20, 20, C).to(dtype).cuda()
    x[8] = torch.linspace(20, -20, C).to(dtype).cuda()
    x[9, C // 2] = math.nan
    x[10, C - 1] = math.inf
    x[11] = math.nan
    x[12] = torch.where(torch.arange(C) % 2 == 0, -0.0, 0.0).to(dtype).cuda()
    labels = torch.randint(0, C, (14,), generator=g).cuda()
    for k in sorted({0, 1, min(C, 7), min(C, 64)}):
        check_logprob(x, labels, k, True, seen=f'k={k}')
    # rows that do not take part have no gradient, whatever they hold
    leaf = x.detach().requires_grad_()
    none = torch.full_like(labels, -1)
    r = ops.label_log_probs(leaf, none)
    assert not r.log_probs.any() and not torch.autograd.grad(r.log_probs.sum(), leaf)[0].any()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('C', [21, 700, 5000])
def test_label_log_probs_layouts(dtype, C):
    g = gen(12)
    wide = randn(g, 4, 5, C + 13, dtype=dtype)
    labels = torch.randint(0, C, (4, 5), generator=g).cuda()
    check_logprob(wide[..., :C], labels, 3, True, seen='padded')
    check_logprob(wide[..., 7:C + 7], labels.int(), 3, True, seen='off alignment')
    check_logprob(wide.transpose(0, 1)[..., :C], labels.t(), 3, True, seen='transposed')
    check_logprob(wide[:, :, :C].permute(2, 0, 1).contiguous().permute(1, 2, 0), labels, 3, True, seen='by columns')
    check_logprob(wide[:1, :1, :C].expand(4, 5, C), labels, 3, True, seen='expanded')
    check_logprob(wide[0, 0, :C], labels[0, 0], 3, True, seen='one row')


@pytest.mark.gpu
def test_label_log_probs_no_rows():
    x = torch.zeros(0, 9, device='cuda', requires_grad=True)
    r = ops.label_log_probs(x, torch.zeros(0, dtype=torch.int64, device='cuda'), 2, True)
    assert r.log_probs.shape == r.entropy.shape == (0,) and r.top_ids.shape == (0, 2)
    assert torch.autograd.grad(r.log_probs.sum() + r.entropy.sum(), x)[0].shape == (0, 9)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('C', [5, 300, 5000])
def test_entropy_gradient_of_classes_that_cannot_be(dtype, C):
    """A large gradient of the entropy leaves classes of -inf and of the type's lowest value at 0: their probability is."""
    g = gen(25)
    x = randn(g, 3, C, dtype=dtype)
    x[:, 1], x[:, C - 1] = -math.inf, torch.finfo(dtype).min
    x.requires_grad_()
    r = ops.label_log_probs(x, torch.full((3,), -1, device='cuda'), entropy=True)
    small = torch.autograd.grad(r.entropy, x, torch.full((3,), 2.0 ** -10, device='cuda'), retain_graph=True)[0]
    for h in (2.0 ** 30, -2.0 ** 40):
        gx = torch.autograd.grad(r.entropy, x, torch.full((3,), h, device='cuda'), retain_graph=True)[0]
        assert not gx[:, [1, C - 1]].any() and not torch.isnan(gx).any()
        if dtype is torch.float32:                                      # powers of two: the same digits
            assert torch.equal(gx, small * (h * 2.0 ** 10))


# ------------------------------------------------------------------ all of them

@pytest.mark.gpu
def test_gradients_against_differences():
    """Directional differences of the forward passes themselves, in fp32 with a step of 2^-6: the forward values are off by
    at most 2^-18 of their size here and the cubic term by a few 2^-12, so 2^-9 of the derivative's scale covers both."""
    g = gen(13)
    x, w1, b1 = randn(g, 6, 40), randn(g, 40, scale=0.2, shift=1.0), randn(g, 40)
    w2, b2, r = randn(g, 30, 40, scale=0.2), randn(g, 30), randn(g, 6, 30)
    labels = torch.randint(0, 30, (6,), generator=g).cuda()
    c = randn(g, 6)

    def f(x, w1, b1, w2, b2, r):
        z = ops.label_log_probs(ops.linear(ops.layer_norm(x, w1, b1), w2, b2, 'gelu', r), labels, entropy=True)
        return (z.log_probs * c + z.entropy * c.flip(0)).double().sum()
    leaves = [v.requires_grad_() for v in (x, w1, b1, w2, b2, r)]
    grads = torch.autograd.grad(f(*leaves), leaves)
    for i, (v, gr) in enumerate(zip(leaves, grads)):
        step = randn(g, *v.shape)
        step = step / step.norm()
        with torch.no_grad():
            up, down = [[u + (s * 2.0 ** -6) * step if j == i else u for j, u in enumerate(leaves)] for s in (1, -1)]
            diff = float(f(*up) - f(*down)) * 2.0 ** 5
        assert abs(diff - float((gr * step).sum())) <= 2.0 ** -9 * (1 + float(gr.norm())), i


def head_def(features, tower, embeddings, bias):
    f = features
    for nw, nb, w, b in tower:
        h = (f - f.mean(-1, keepdim=True)) / (f.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt()
        f = ((h * nw + nb) @ w.t() + b).relu() + f
    return f @ embeddings.t() + bias


@pytest.mark.gpu
def test_head_logits_train_and_detect():
    """The chain as it is used: tower and class embeddings of a small RetinaNet head make the logits, the loss and the log
    probabilities of the labels run back through them, and detect takes the same logits."""
    g = gen(14)
    m = D.RetinaNet(20, [8, 4, 2, 1, 1])
    P, dim, B = m.pboxes.shape[0], 48, 2
    feats = randn(g, B, P, dim)
    tower = [(randn(g, dim, scale=0.1, shift=1.0), randn(g, dim, scale=0.1), randn(g, dim, dim, scale=dim ** -0.5), randn(g, dim, scale=0.1))
             for _ in range(2)]
    emb, bias = randn(g, m.nc, dim, scale=dim ** -0.5), randn(g, m.nc)
    leaves = [v.requires_grad_() for v in (feats, emb, bias, *[p for layer in tower for p in layer])]
    logits = m.head_logits(feats, emb, bias, tower)
    want = head_def(feats.double(), [[p.double() for p in layer] for layer in tower], emb.double(), bias.double())
    # fp32 throughout: two layers of 48-term sums, each within a few hundred E of its magnitudes
    close(logits, want.detach(), 4096 * E * (1 + want.detach().abs().amax()))
    locs = randn(g, B, P, 4, scale=0.1).requires_grad_()
    gt = [torch.tensor([[0.5, 0.5, 0.4, 0.4], [0.3, 0.3, 0.2, 0.3]]), torch.tensor([[0.6, 0.4, 0.5, 0.5]])]
    lab = [torch.tensor([3, 7]), torch.tensor([20])]
    loss = m.loss((locs, logits), gt, lab)['loss']
    _, target, _ = m.assign(gt, lab, feats.device)
    r = ops.label_log_probs(logits, target, top_k=3, entropy=True)
    grads = torch.autograd.grad(loss - r.log_probs.mean() + 0.1 * r.entropy.mean(), [*leaves, locs])
    assert all(torch.isfinite(v).all() for v in grads) and all(v.any() for v in grads)
    # the same gradient through the definition in 64 bits, from the same gradient at the logits
    leaf = logits.detach().requires_grad_()
    r2 = ops.label_log_probs(leaf, target, entropy=True)
    top = torch.autograd.grad(m.loss((locs.detach(), leaf), gt, lab)['loss'] - r2.log_probs.mean() + 0.1 * r2.entropy.mean(), leaf)[0]
    ref = torch.autograd.grad(want, leaves, top.double())
    for got, v in zip(grads, ref):
        assert float((got.double() - v).norm()) <= 2.0 ** -12 * float(v.norm())     # 48-term sums, P-row reductions of E each
    assert torch.equal(r.top_ids[..., 0], logits.detach().argmax(-1))
    ids, rows = m.detect((locs.detach(), logits.detach()), [{'image_id': i, 'height': 300, 'width': 400} for i in range(B)])
    assert ids.shape[0] == rows.shape[0] > 0
    with pytest.raises(ValueError):
        m.head_logits(feats, emb[:-1], bias)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_head_logits_train_on_a_mean_over_many_anchors(dtype):
    """The mean of the log probabilities over 120000 anchors of 81 classes: most of its gradients at the logits are near 1e-7.  Those
    of the features and the embeddings against the definition in 64 bits, from the same gradients at the logits: dz is off by half
    a step of the features' type (none in fp32) and, in fp16, by 2^-39 of the largest; then sums of n fp32 terms, rounded once."""
    g = torch.Generator(device='cuda').manual_seed(26)
    m = D.RetinaNet(80, [8, 4, 2, 1, 1])
    feats = torch.randn(4, 30000, 64, generator=g, device='cuda').to(dtype).requires_grad_()
    emb = (torch.randn(m.nc, 64, generator=g, device='cuda') / 8).to(dtype).requires_grad_()
    labels = torch.randint(0, m.nc, (4, 30000), generator=g, device='cuda')
    logits = m.head_logits(feats, emb)
    assert logits.shape == (4, 30000, 81) and logits.dtype == torch.float32
    top, gf, ge = torch.autograd.grad(ops.label_log_probs(logits, labels).log_probs.mean(), [logits, feats, emb])
    dz, fd, ed = top.double().reshape(-1, 81), feats.detach().double().reshape(-1, 64), emb.detach().double()
    off = (U[dtype] * dz.abs() + 2.0 ** -39 * dz.abs().max() if dtype != torch.float32 else torch.zeros_like(dz))
    for got, want, tol in ((gf.reshape(-1, 64), dz @ ed, off @ ed.abs() + 85 * E * ((dz.abs() + off) @ ed.abs())),
                           (ge, dz.t() @ fd, off.t() @ fd.abs() + 120004 * E * ((dz.abs() + off).t() @ fd.abs()))):
        close(got, want, tol + U[dtype] * (want.abs() + tol) + TINY[dtype])
    assert float((ge.double() - dz.t() @ fd).norm()) <= 4 * U[dtype] * float((dz.t() @ fd).norm()) + 120004 * E * float((dz.abs().t() @ fd.abs()).norm())


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_streams_and_graphs(dtype):
    """On a stream of its own, and captured (forward and backward) into graphs that are replayed with new inputs and eager
    calls between: every replay gives the eager result's bits.  Two graphs captured one after the other share nothing."""
    g = gen(15)

    def inputs(M):
        return {'x': randn(g, M, 96, dtype=dtype), 'nw': randn(g, 96, dtype=dtype), 'w': randn(g, 300, 96, dtype=dtype, scale=0.1),
                'b': randn(g, 300, dtype=dtype), 't': torch.randint(0, 300, (M,), generator=g).cuda(), 'g': randn(g, M)}

    def step(v):
        leaves = [v[k].detach().requires_grad_() for k in ('x', 'nw', 'w', 'b')]
        z = ops.linear(ops.layer_norm(leaves[0], leaves[1], leaves[1]), leaves[2], leaves[3], 'gelu')
        r = ops.label_log_probs(z, v['t'], 4, True)
        return [r.log_probs.detach(), r.entropy.detach(), r.top_log_probs, r.top_ids,
                *torch.autograd.grad([r.log_probs, r.entropy], leaves, [v['g'], v['g']])]

    for M in (1, 40, 700):
        sets = [inputs(M) for _ in range(3)]
        eager = [step(v) for v in sets]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step(sets[1])
        torch.cuda.current_stream().wait_stream(side)
        for a, b in zip(other, eager[1]):
            assert torch.equal(a, b)
        graphs = []
        for _ in range(2):
            held = {k: v.clone() for k, v in sets[0].items()}
            torch.cuda.synchronize()
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                outs = step(held)
            graphs.append((gr, held, outs))
        for turn in range(4):
            for n, (gr, held, outs) in enumerate(graphs):
                i = (turn + n) % 3
                for k in held:
                    held[k].copy_(sets[i][k])
                gr.replay()
            now = step(sets[turn % 3])
            torch.cuda.synchronize()
            for a, b in zip(now, eager[turn % 3]):
                assert torch.equal(a, b)
            for n, (gr, held, outs) in enumerate(graphs):
                for a, b in zip(outs, eager[(turn + n) % 3]):
                    assert torch.equal(a, b), (M, turn, n)
        del graphs


@pytest.mark.gpu
def test_two_streams_at_once():
    """Calls that overlap on two streams use workspaces of their own."""
    g = gen(16)
    x, w = randn(g, 20000, 64, dtype=torch.bfloat16), randn(g, 50, 64, dtype=torch.bfloat16)
    b, gr = randn(g, 50, dtype=torch.bfloat16), randn(g, 20000, 50, dtype=torch.bfloat16)

    def step(x):
        leaves = [v.detach().requires_grad_() for v in (x, w, b)]
        n = ops.layer_norm(leaves[0], w[0], w[1])
        return torch.autograd.grad(ops.linear(n, leaves[1], leaves[2], 'silu'), leaves, gr)
    xs = [x, x.flip(0).contiguous()]
    want = [step(v) for v in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(5):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(step(xs[k]))
    torch.cuda.synchronize()
    for k in (0, 1):
        for one in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(one, want[k]))


@pytest.mark.gpu
def test_two_threads_at_once():
    """Calls from two host threads, each on its own stream, with autograd: the results of the calls made alone."""
    import threading
    g = gen(19)
    w, b = randn(g, 300, 96), randn(g, 300)
    xs, labels = [randn(g, 500, 96) for _ in range(2)], torch.randint(0, 300, (500,), generator=g).cuda()

    def step(x):
        x = x.detach().requires_grad_()
        r = ops.label_log_probs(ops.linear(ops.layer_norm(x), w, b, 'gelu'), labels, 3, True)
        return [r.log_probs.detach(), r.top_ids, torch.autograd.grad(r.log_probs.sum() + r.entropy.sum(), x)[0]]
    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[k].append(step(xs[k]))
                torch.cuda.current_stream().synchronize()
        except Exception as e:                                          # a thread's exception would be lost otherwise
            errors.append(e)
    threads = [threading.Thread(target=work, args=(k,)) for k in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for k in (0, 1):
        assert len(got[k]) == 20
        for one in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(one, want[k]))


@pytest.mark.gpu
def test_no_memory_is_kept():
    """Repeated training steps hold no more memory than one (what earlier tests left may be freed meanwhile)."""
    g = gen(20)
    x, w = randn(g, 3000, 200).requires_grad_(), randn(g, 90, 200).requires_grad_()
    labels = torch.randint(0, 90, (3000,), generator=g).cuda()
    held = []
    for _ in range(6):
        r = ops.label_log_probs(ops.linear(ops.layer_norm(x), w, activation='silu'), labels, 2, True)
        torch.autograd.grad(r.log_probs.sum() + r.entropy.sum(), [x, w])
        del r
        held.append(torch.cuda.memory_allocated())
    assert held[-1] <= held[1]


@pytest.mark.gpu
def test_accumulated_gradients_and_changed_inputs():
    """.backward() twice adds up; an input changed in place between forward and backward is an error, not a wrong gradient."""
    g = gen(21)
    x, w, b = randn(g, 20, 64).requires_grad_(), randn(g, 30, 64).requires_grad_(), randn(g, 30).requires_grad_()
    n = randn(g, 64).requires_grad_()
    res = randn(g, 20, 30).requires_grad_()
    labels = torch.randint(0, 30, (20,), generator=g).cuda()

    def loss():
        r = ops.label_log_probs(ops.linear(ops.layer_norm(x, n, n), w, b, 'relu', res), labels, entropy=True)
        return r.log_probs.sum() + r.entropy.sum()
    once = torch.autograd.grad(loss(), [x, w, b, n, res])
    loss().backward()
    loss().backward()
    for leaf, v in zip((x, w, b, n, res), once):
        assert torch.equal(leaf.grad, v + v)
    for make in (lambda t: ops.layer_norm(t, n), lambda t: ops.linear(t, w), lambda t: ops.label_log_probs(t, labels).log_probs):
        t = (x * 1.0)
        y = make(t)
        t.add_(1)
        with pytest.raises(RuntimeError):
            y.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize('lead', [(), (5,), (2, 3), (2, 1, 3)], ids=str)
def test_outputs_changed_in_place(lead):
    """Outputs of any number of axes may be changed in place, and the gradient is that of the change made out of place."""
    g = gen(22)
    x, w, n = randn(g, *lead, 12), randn(g, 9, 12), randn(g, 12)
    labels = torch.randint(0, 12, lead, generator=g).cuda()
    gate = randn(g, *lead, 12) > 0

    def run(in_place):
        leaves = [v.detach().requires_grad_() for v in (x, w, n)]
        a = ops.layer_norm(leaves[0], leaves[2])
        a = a.masked_fill_(gate, 0.5) if in_place else a.masked_fill(gate, 0.5)
        b = ops.linear(a, leaves[1], activation='silu')
        b = torch.relu_(b) if in_place else torch.relu(b)
        r = ops.label_log_probs(leaves[0], labels, 2, True)
        assert not r.top_log_probs.requires_grad
        assert r.log_probs.shape == r.entropy.shape == lead and r.top_log_probs.shape == r.top_ids.shape == (*lead, 2)
        lp = r.log_probs.mul_(3.0) if in_place else r.log_probs * 3.0
        top = r.top_log_probs.neg_() if in_place else -r.top_log_probs
        loss = (b * b).sum() + lp.sum() + r.entropy.sum()
        return [b.detach(), lp.detach(), top, *torch.autograd.grad(loss, leaves)]
    for u, v in zip(run(True), run(False)):
        assert u.shape == v.shape and torch.equal(u, v)


@pytest.mark.gpu
@pytest.mark.parametrize('leaf', [False, True])
def test_forward_mode_is_refused(leaf):
    """Tangents are not carried through: a call with a dual tensor raises, also under no_grad and where no argument asks for a
    gradient, instead of returning a value without one."""
    import torch.autograd.forward_ad as fwAD
    g = gen(23)
    x, w, b, r = randn(g, 4, 8), randn(g, 6, 8), randn(g, 6), randn(g, 4, 6)
    n, labels = randn(g, 8), torch.zeros(4, dtype=torch.int64, device='cuda')
    calls = [(x, lambda t: ops.layer_norm(t, n, n)), (n, lambda t: ops.layer_norm(x, t, n)), (n, lambda t: ops.layer_norm(x, None, t)),
             (x, lambda t: ops.linear(t, w, b, 'gelu', r)), (w, lambda t: ops.linear(x, t, b, 'gelu', r)), (b, lambda t: ops.linear(x, w, t)),
             (r, lambda t: ops.linear(x, w, None, 'relu', t)), (x, lambda t: ops.label_log_probs(t, labels, 2, True))]
    with fwAD.dual_level():
        for v, call in calls:
            dual = fwAD.make_dual(v.detach().requires_grad_(leaf), torch.ones_like(v))
            with pytest.raises(NotImplementedError, match='forward-mode'):
                call(dual)
            with torch.no_grad(), pytest.raises(NotImplementedError, match='forward-mode'):
                call(dual)
        # an argument without a tangent is none: the call runs
        assert torch.equal(ops.layer_norm(x, n, n), ops.layer_norm(x, n, n))


@pytest.mark.gpu
def test_kernel_timing_names():
    """The per-kernel timer knows the calls by the names the header gives."""
    x, w = torch.randn(8, 16, device='cuda').requires_grad_(), torch.randn(4, 16, device='cuda').requires_grad_()
    ops.profile_reset()
    ops.profile_enable()
    try:
        r = ops.label_log_probs(ops.linear(ops.layer_norm(x), w), torch.zeros(8, dtype=torch.int64, device='cuda'))
        torch.autograd.grad(r.log_probs.sum(), [x, w])
        torch.cuda.synchronize()
        for name in ('layer_norm', 'linear', 'label_log_probs'):
            for way in ('forward', 'backward'):
                assert ops.profile_read(f'{name}_{way}')[1] == 1, (name, way)
    finally:
        ops.profile_enable(False)
        ops.profile_reset()


@pytest.mark.gpu
def test_rows_behind_the_last_are_left():
    """Outputs are written to their last element and not beyond: the C entry points into buffers with a guard behind."""
    L, st = _lib.lib(), torch.cuda.current_stream().cuda_stream
    g = gen(17)
    for dt, t in ((0, torch.float32), (1, torch.bfloat16), (2, torch.float16)):
        for M, N, K in ((1, 37, 50), (3, 129, 64), (130, 71, 65), (600, 81, 128)):
            x, w = randn(g, M, K, dtype=t), randn(g, N, K, dtype=t)
            gr = randn(g, M, N, dtype=t)
            def guarded(n, dtype=t):
                return torch.full((n + 64,), 7.0, dtype=dtype, device='cuda')
            y, pre, gx, gw, gb = guarded(M * N), guarded(M * N), guarded(M * K), guarded(N * K), guarded(N)
            nb = max(L.detbox_linear_workspace_bytes(dt, M, N, K), L.detbox_linear_backward_workspace_bytes(dt, 2, dt, M, N, K), 256)
            ws = torch.full((nb + 256,), 0xA5, dtype=torch.uint8, device='cuda')
            _lib.check(L.detbox_linear_forward(dt, 2, x.data_ptr(), K, w.data_ptr(), K, 0, None, None, 0, M, N, K, dt, y.data_ptr(),
                                               pre.data_ptr(), ws.data_ptr(), nb, st), 'forward')
            _lib.check(L.detbox_linear_backward(dt, 2, dt, gr.data_ptr(), N, pre.data_ptr(), x.data_ptr(), K, w.data_ptr(), K, M, N, K,
                                                gx.data_ptr(), gw.data_ptr(), dt, gb.data_ptr(), ws.data_ptr(), nb, st), 'backward')
            ny, stats = guarded(M * K), guarded(M * 2, torch.float32)
            nx, nw, nbias = guarded(M * K), guarded(K), guarded(K)
            _lib.check(L.detbox_layer_norm_forward(dt, x.data_ptr(), K, dt, None, None, M, K, 1e-5, ny.data_ptr(), stats.data_ptr(), st), 'norm')
            nn = L.detbox_layer_norm_backward_workspace_bytes(M, K)
            ws2 = torch.full((nn + 256,), 0xA5, dtype=torch.uint8, device='cuda')
            _lib.check(L.detbox_layer_norm_backward(dt, x.data_ptr(), K, x.data_ptr(), K, dt, None, stats.data_ptr(), M, K, nx.data_ptr(),
                                                    nw.data_ptr(), nbias.data_ptr(), ws2.data_ptr(), nn, st), 'norm backward')
            for v, n in ((y, M * N), (pre, M * N), (gx, M * K), (gw, N * K), (gb, N), (ny, M * K), (stats, 2 * M), (nx, M * K), (nw, K), (nbias, K)):
                assert (v[n:] == 7.0).all() and (v[:n] != 7.0).any()
            assert (ws[nb:] == 0xA5).all() and (ws2[nn:] == 0xA5).all()
        for rows, C, k in ((3, 81, 5), (2, 5000, 64), (1, 70000, 20)):
            x, lab = randn(g, rows, C, dtype=t), torch.zeros(rows, dtype=torch.int64, device='cuda')
            f = lambda n: torch.full((n + 64,), 7.0, device='cuda')                      # noqa: E731
            lp, ent, tv, stats = f(rows), f(rows), f(rows * k), f(rows * 2)
            ti = torch.full((rows * k + 64,), 7, dtype=torch.int64, device='cuda')
            gx = torch.full((rows * C + 64,), 7.0, dtype=t, device='cuda')
            nb = L.detbox_label_log_probs_workspace_bytes(rows, C, k)
            ws = torch.full((nb + 256,), 0xA5, dtype=torch.uint8, device='cuda')
            _lib.check(L.detbox_label_log_probs_forward(dt, x.data_ptr(), C, lab.data_ptr(), rows, C, k, lp.data_ptr(), ent.data_ptr(), tv.data_ptr(),
                                                        ti.data_ptr(), stats.data_ptr(), ws.data_ptr(), nb, st), 'log probs')
            _lib.check(L.detbox_label_log_probs_backward(dt, x.data_ptr(), C, lab.data_ptr(), rows, C, stats.data_ptr(), ent.data_ptr(),
                                                         lp.data_ptr(), ent.data_ptr(), gx.data_ptr(), st), 'log probs backward')
            for v, n in ((lp, rows), (ent, rows), (tv, rows * k), (ti, rows * k), (stats, rows * 2), (gx, rows * C)):
                assert (v[n:] == 7).all()
            assert (ws[nb:] == 0xA5).all()


@pytest.mark.gpu
def test_refusals():
    x, w = torch.zeros(4, 8, device='cuda'), torch.zeros(6, 8, device='cuda')
    lab = torch.zeros(4, dtype=torch.int64, device='cuda')
    h = x.half()
    for call in (lambda: ops.layer_norm(x.double()), lambda: ops.layer_norm(x, torch.zeros(7, device='cuda')),
                 lambda: ops.layer_norm(x, torch.zeros(8, device='cuda'), torch.zeros(8, device='cuda').half()),
                 lambda: ops.layer_norm(x[:, :0]), lambda: ops.layer_norm(x.int()), lambda: ops.layer_norm(torch.zeros((), device='cuda')),
                 lambda: ops.linear(x, w.half()), lambda: ops.linear(x, w[:, :7]), lambda: ops.linear(x, w[0]), lambda: ops.linear(x, w, activation='tanh'),
                 lambda: ops.linear(x, w, torch.zeros(5, device='cuda')), lambda: ops.linear(x, w, residual=torch.zeros(4, 5, device='cuda')),
                 lambda: ops.linear(x, w, residual=torch.zeros(4, 6, device='cuda').half()), lambda: ops.linear(x, w, out_dtype=torch.float16),
                 lambda: ops.linear(h, w.half(), residual=torch.zeros(4, 6, device='cuda').half(), out_dtype=torch.float32),
                 lambda: ops.linear(x, w[:0]), lambda: ops.linear(x[:, :0], w[:, :0]), lambda: ops.linear(x.double(), w.double()),
                 lambda: ops.label_log_probs(x, lab[:3]), lambda: ops.label_log_probs(x, lab.float()), lambda: ops.label_log_probs(x, lab, top_k=9),
                 lambda: ops.label_log_probs(x, lab, top_k=-1), lambda: ops.label_log_probs(x[:, :0], lab),
                 lambda: ops.label_log_probs(torch.zeros(4, 100, device='cuda'), lab, top_k=65), lambda: ops.label_log_probs(x, lab.cpu()),
                 lambda: ops.label_log_probs(x.long(), lab), lambda: ops.label_log_probs(x, lab.bool())):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ops.linear(x, w.cpu()), lambda: ops.layer_norm(x, torch.zeros(8))):
        with pytest.raises(_lib.DetboxError):
            call()
    # a second derivative is not there: refused, not wrong
    y = ops.layer_norm(x.requires_grad_())
    gx = torch.autograd.grad(y.square().sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gx.sum(), x)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Operands of more than 2^32 elements: the last rows give what the same rows give alone."""
    t = torch.bfloat16
    g = gen(18)

    def tail_of(rows, n, k):
        big = torch.zeros(rows, n, dtype=t, device='cuda')
        assert big.numel() > 2 ** 32
        big[-k:] = randn(g, k, n, dtype=t)
        return big.requires_grad_(), big[-k:].detach().clone().requires_grad_()
    k = 40
    # logits: 33000 rows of 131072
    x, small = tail_of(33000, 131072, k)
    labels = torch.randint(0, 131072, (33000,), generator=g).cuda()
    a, b = ops.label_log_probs(x, labels, 3, True), ops.label_log_probs(small, labels[-k:], 3, True)
    assert torch.equal(a.top_ids[-k:], b.top_ids)
    for u, v in ((a.log_probs[-k:], b.log_probs), (a.entropy[-k:], b.entropy)):
        assert torch.allclose(u, v, rtol=1e-5, atol=0)              # rows cut into pieces or not: the sums' order differs
    gr = randn(g, 33000)
    (gx,), (gs,) = torch.autograd.grad(a.log_probs, x, gr), torch.autograd.grad(b.log_probs, small, gr[-k:])
    assert float((gx[-k:].float() - gs.float()).norm()) <= 2.0 ** -8 * float(gs.float().norm())
    # rows of zeros: -g / C everywhere but at the label, whose g (1 - 1 / C) is of another size
    head = gx[:3].detach().float().scatter(1, labels[:3].clamp(min=0)[:, None], 0.0).abs().amax(1)
    assert torch.all(head <= gr[:3].abs() / 131072 * (1 + 2.0 ** -7))
    del x, gx, a
    # rows for a norm and a product: 1100000 of 4096
    x, small = tail_of(1100000, 4096, k)
    w, b = randn(g, 4096, dtype=t), randn(g, 4096, dtype=t)
    y, ys = ops.layer_norm(x, w, b), ops.layer_norm(small, w, b)
    assert torch.equal(y[-k:], ys)
    gr = torch.zeros_like(x)
    gr[-k:] = randn(g, k, 4096, dtype=t)
    gx, gs = torch.autograd.grad(y, x, gr)[0], torch.autograd.grad(ys, small, gr[-k:])[0]
    assert torch.equal(gx[-k:], gs) and not gx[:100].any()
    del y, gx, gr
    w = randn(g, 24, 4096, dtype=t, scale=1 / 64).requires_grad_()
    y, ys = ops.linear(x, w), ops.linear(small, w)
    # both are within one rounding of the same sums, taken in another order
    assert torch.allclose(y[-k:].float(), ys.float(), rtol=2.0 ** -7, atol=2.0 ** -10) and not y[:100].any()
    gr = torch.zeros_like(y)
    gr[-k:] = randn(g, k, 24, dtype=t)
    (gx, gw), (gs, gv) = torch.autograd.grad(y, [x, w], gr), torch.autograd.grad(ys, [small, w], gr[-k:])
    for u, v in ((gx[-k:], gs), (gw, gv)):
        assert torch.allclose(u.float(), v.float(), rtol=2.0 ** -7, atol=2.0 ** -8)


@pytest.mark.gpu
def test_columns_beyond_one_grid():
    """More columns than one grid of the column sums has threads for (2^27 sums of 32 threads each): with one row the sums are
    the row's own products, which are exact."""
    t = torch.bfloat16
    n = (1 << 26) + 37
    x = torch.zeros(1, n, dtype=t, device='cuda')
    x[0, ::2], x[0, n - 1] = 1.0, -1.0
    gr = (torch.arange(n, device='cuda') % 251).to(t)[None]
    w, b = torch.ones(n, dtype=t, device='cuda').requires_grad_(), torch.zeros(n, dtype=t, device='cuda').requires_grad_()
    y = ops.layer_norm(x, w, b)
    gw, gb = torch.autograd.grad(y, [w, b], gr)
    assert torch.equal(gb, gr[0])
    # the ends of the axis, each within one rounding of gradient times output (weight 1, bias 0: the output is h, rounded)
    for part in (slice(0, 4096), slice(n // 2, n // 2 + 4096), slice(n - 4096, n)):
        want = gr[0, part].double() * y.detach()[0, part].double()
        assert ((gw[part].double() - want).abs() <= 2.0 ** -7 * 1.01 * want.abs()).all()
    del x, gr, w, b, y, gw, gb
    n = (1 << 27) + 37
    w, x = torch.ones(n, 1, dtype=t, device='cuda'), torch.ones(1, 1, dtype=t, device='cuda')
    b = torch.zeros(n, dtype=t, device='cuda').requires_grad_()
    gr = (torch.arange(n, device='cuda') % 251).to(t)[None]
    assert torch.equal(torch.autograd.grad(ops.linear(x, w, b), b, gr)[0], gr[0])


@pytest.mark.gpu
def test_library_errors_are_the_packages():
    """A limit of the library arrives as DetboxError."""
    with pytest.raises(_lib.DetboxError, match='DETBOX_LINEAR_MAX_TILES'):
        ops.linear(torch.zeros(1 << 30, 1, dtype=torch.float16, device='cuda'), torch.zeros(1, 1, dtype=torch.float16, device='cuda'))


def test_refuse_without_a_device():
    x = torch.zeros(2, 3)
    for call in (lambda: ops.layer_norm(x), lambda: ops.linear(x, x), lambda: ops.label_log_probs(x, torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(_lib.DetboxError):
            call()


def test_c_entry_points_refuse():
    """Arguments are checked before any device work."""
    L = _lib.lib()
    p = 4096                                                            # a pointer that must never be followed
    inv, ws_err, unsup = -1, -2, -4
    assert L.detbox_layer_norm_forward(7, p, 8, 0, None, None, 2, 8, 1e-5, p, None, None) == inv
    assert L.detbox_layer_norm_forward(0, p, 7, 0, None, None, 2, 8, 1e-5, p, None, None) == inv
    assert L.detbox_layer_norm_forward(0, None, 8, 0, None, None, 2, 8, 1e-5, p, None, None) == inv
    assert L.detbox_layer_norm_forward(0, p, 8, 0, None, None, -1, 8, 1e-5, p, None, None) == inv
    assert L.detbox_layer_norm_forward(0, p, 8, 0, None, None, 2, 8, 1e-5, None, None, None) == inv
    assert L.detbox_layer_norm_forward(0, None, 8, 0, None, None, 0, 8, 1e-5, None, None, None) == 0
    need = L.detbox_layer_norm_backward_workspace_bytes(2, 8)
    assert need > 0
    assert L.detbox_layer_norm_backward(0, p, 8, p, 8, 0, None, p, 2, 8, p, p, p, None, 0, None) == ws_err
    assert L.detbox_layer_norm_backward(0, p, 8, p, 8, 0, None, p, 2, 8, p, p, p, p, need - 1, None) == ws_err
    assert L.detbox_layer_norm_backward(0, p, 8, p, 8, 0, None, p, 2, 8, p, p, p, p + 8, need, None) == ws_err
    assert L.detbox_layer_norm_backward(0, p, 7, p, 8, 0, None, p, 2, 8, p, None, None, None, 0, None) == inv
    assert L.detbox_linear_forward(3, 0, p, 8, p, 8, 0, None, None, 0, 2, 4, 8, 0, p, None, None, 0, None) == inv
    assert L.detbox_linear_forward(0, 5, p, 8, p, 8, 0, None, None, 0, 2, 4, 8, 0, p, None, None, 0, None) == inv
    assert L.detbox_linear_forward(0, 0, p, 7, p, 8, 0, None, None, 0, 2, 4, 8, 0, p, None, None, 0, None) == inv
    assert L.detbox_linear_forward(1, 0, p, 8, p, 8, 0, None, None, 0, 2, 4, 8, 2, p, None, None, 0, None) == inv
    assert L.detbox_linear_forward(0, 0, p, 8, p, 8, 0, None, p, 3, 2, 4, 8, 0, p, None, None, 0, None) == inv
    assert L.detbox_linear_forward(0, 0, p, 8, None, 8, 0, None, None, 0, 2, 4, 8, 0, p, None, None, 0, None) == inv
    assert L.detbox_linear_forward(0, 0, None, 8, None, 8, 0, None, None, 0, 0, 4, 8, 0, None, None, None, 0, None) == 0
    assert L.detbox_linear_forward(0, 0, p, 8, p, 8, 0, None, None, 0, 1 << 30, 4, 8, 0, p, None, None, 0, None) == unsup
    need = L.detbox_linear_workspace_bytes(1, 300, 4096, 4096)
    assert need >= 300 * 4096 * 4
    assert L.detbox_linear_forward(1, 0, p, 4096, p, 4096, 0, None, None, 0, 300, 4096, 4096, 1, p, None, p, need - 1, None) == ws_err
    need = L.detbox_label_log_probs_workspace_bytes(1, 100000, 4)
    assert need > 0
    assert L.detbox_label_log_probs_forward(0, p, 100000, p, 1, 100000, 4, p, None, p, p, None, p, need - 1, None) == ws_err
    need = L.detbox_linear_backward_workspace_bytes(1, 2, 1, 100, 40, 24)
    assert need >= 100 * 40 * 2
    assert L.detbox_linear_backward(1, 2, 1, p, 40, p, p, 24, p, 24, 100, 40, 24, p, p, 0, p, p, need - 1, None) == ws_err
    assert L.detbox_linear_backward(1, 2, 1, p, 40, None, p, 24, p, 24, 100, 40, 24, p, p, 0, p, p, need, None) == inv
    assert L.detbox_linear_backward(1, 2, 2, p, 40, p, p, 24, p, 24, 100, 40, 24, p, p, 0, p, p, need, None) == inv
    assert L.detbox_label_log_probs_forward(0, p, 8, p, 2, 8, 9, p, None, p, p, None, None, 0, None) == inv
    assert L.detbox_label_log_probs_forward(0, p, 80, p, 2, 80, 65, p, None, p, p, None, None, 0, None) == unsup
    assert L.detbox_label_log_probs_forward(0, p, 8, p, 2, 8, 1, p, None, None, p, None, None, 0, None) == inv
    assert L.detbox_label_log_probs_forward(0, p, 8, None, 2, 8, 0, p, None, None, None, None, None, 0, None) == inv
    assert L.detbox_label_log_probs_backward(0, p, 8, p, 2, 8, p, None, p, p, p, None) == inv
    assert L.detbox_label_log_probs_backward(0, p, 8, p, 2, 8, None, None, p, None, p, None) == inv

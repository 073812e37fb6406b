"""GPU: the operators of a trained output head — layer norm, cross entropy and distillation over the classes of a linear head —
against plain float64 formulas on identical inputs.

Tolerances are sums of the roundings that are made, derived before any run.  u = 2^-24 is float32's half step, eps/2 that of
the result's type.  A sum of n terms in float32, in any order, is off by at most (n - 1) u times the sum of the terms' sizes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'
U = 2.0 ** -24
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def half(t):
    return torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def close(got, want, tol, what):
    d = (got.double() - want).abs()
    bad = ~(d <= tol)
    assert not bool(bad.any()), f'{what}: off by {d[bad].max().item():.3e} where {(tol + 0 * want)[bad].min().item():.3e} is allowed ({int(bad.sum())} of {d.numel()})'


# ------------------------------------------------------------------------------------------------ layer norm
def norm64(x, w, b, eps, gy):
    x, gy = x.double(), gy.double()
    C = x.size(1)
    m = x.mean(1, keepdim=True)
    r = 1.0 / ((x - m).square().mean(1, keepdim=True) + eps).sqrt()
    h = (x - m) * r
    wd = w.double() if w is not None else torch.ones(C, dtype=torch.float64, device=x.device)
    bd = b.double() if b is not None else torch.zeros(C, dtype=torch.float64, device=x.device)
    gh = gy * wd
    gx = r * (gh - gh.mean(1, keepdim=True) - h * (gh * h).mean(1, keepdim=True))
    return dict(y=h * wd + bd, gx=gx, gw=(gy * h).sum(0), gb=gy.sum(0), h=h, r=r, gh=gh, wd=wd, bd=bd, x=x, gy=gy)


def check_norm(x, w, b, eps, gy, y, gx, gw, gb):
    """A row of C elements is added in chains of at most 16 per thread and at most 10 levels between the threads (256 for the rows
    beyond 512 threads, whose chains are C / 1024 long): k of them.  The mean is then off by at most k u mean|x|, r by (k + 4) u
    relative, and h by r (k u max|x| + 2 u |d|) + (k + 4) u |h| <= 2 k u (max|x| r + |h|)."""
    q = norm64(x, w, b, eps, gy)
    C, R = x.size(1), x.size(0)
    k = 32 if C <= 4096 else 32 + C / 512
    reach = 2 * k * U * (q['x'].abs().amax(1, keepdim=True) * q['r'] + q['h'].abs())           # of h
    close(y, q['y'], half(y.dtype) * q['y'].abs() * (1 + 1e-3) + (reach + 2 * U * q['h'].abs()) * q['wd'].abs() + 2 * U * q['bd'].abs(), 'y')
    if gx is not None:
        g1 = q['gh'].abs().mean(1, keepdim=True)
        hmax, ghmax = q['h'].abs().amax(1, keepdim=True), q['gh'].abs().amax(1, keepdim=True)
        rmax = reach.amax(1, keepdim=True)
        # r (gh - s1 - h s2): s1 off by k u mean|gh|, s2 by k u mean|gh h| + mean|gh| dh, h by dh; r and the last additions 8 u
        t = q['r'] * ((k + 8) * U * (g1 + q['gh'].abs() + hmax * hmax * g1) + 2 * rmax * hmax * g1 + rmax * g1) + (k + 4) * U * q['gx'].abs()
        close(gx, q['gx'], half(gx.dtype) * q['gx'].abs() * (1 + 1e-3) + t + 0 * ghmax, 'gx')
    # any order of R additions in chains: rows of a group, groups, partials — never more than R / 64 + 128 in a row
    n = R / 64 + 128
    if gw is not None:
        t = n * U * (q['gy'] * q['h']).abs().sum(0) + (q['gy'].abs() * reach).sum(0)
        close(gw, q['gw'], half(gw.dtype) * q['gw'].abs() * (1 + 1e-3) + t, 'gw')
    if gb is not None:
        close(gb, q['gb'], half(gb.dtype) * q['gb'].abs() * (1 + 1e-3) + n * U * q['gy'].abs().sum(0), 'gb')


# every group size of the kernels, odd widths, one row, more rows than workgroups
NORM = [(1, 1), (1, 8), (3, 7), (608, 128), (33, 31), (65, 65), (5, 255), (700, 257), (129, 513), (40, 1021), (9, 1025), (1030, 1024),
        (6, 2049), (7, 4095), (3, 8191), (2, 16385), (3, 40001), (20000, 24)]


@pytest.mark.parametrize('t', list(TYPES))
@pytest.mark.parametrize('R,C', NORM)
def test_layer_norm(R, C, t):
    from dig_amd import ops
    t = TYPES[t]
    g = gen(R * 31 + C)
    x = (randn(g, R, C) * 1.5 + 0.3).to(t).requires_grad_()
    w, b, gy = (1 + 0.2 * randn(g, C)).to(t).requires_grad_(), randn(g, C).to(t).requires_grad_(), randn(g, R, C).to(t)
    y = ops.layer_norm(x, w, b, 1e-5)
    assert y.dtype == t and y.shape == x.shape
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), gy)
    assert gx.dtype == gw.dtype == gb.dtype == t
    check_norm(x.detach(), w.detach(), b.detach(), 1e-5, gy, y.detach(), gx, gw, gb)


@pytest.mark.parametrize('t', ['bf16', 'f16'])
def test_layer_norm_float32_parameters_of_16_bit_rows(t):
    from dig_amd import ops
    t = TYPES[t]
    g = gen(5)
    x, gy = randn(g, 77, 320).to(t).requires_grad_(), randn(g, 77, 320).to(t)
    w, b = (1 + 0.2 * randn(g, 320)).requires_grad_(), randn(g, 320).requires_grad_()
    y = ops.layer_norm(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), gy)
    assert y.dtype == gx.dtype == t and gw.dtype == gb.dtype == torch.float32
    check_norm(x.detach(), w.detach(), b.detach(), 1e-5, gy, y.detach(), gx, gw, gb)


@pytest.mark.parametrize('have', ['none', 'w', 'b'])
def test_layer_norm_without_parameters(have):
    from dig_amd import ops
    g = gen(6)
    x, gy = randn(g, 50, 96).requires_grad_(), randn(g, 50, 96)
    w = (1 + 0.2 * randn(g, 96)).requires_grad_() if have == 'w' else None
    b = randn(g, 96).requires_grad_() if have == 'b' else None
    y = ops.layer_norm(x, w, b, eps=1e-6)
    leaves = [p for p in (x, w, b) if p is not None]
    gr = torch.autograd.grad(y, leaves, gy)
    d = lambda p: p.detach() if p is not None else None
    check_norm(d(x), d(w), d(b), 1e-6, gy, y.detach(), gr[0], gr[1] if have == 'w' else None, gr[1] if have == 'b' else None)


def test_layer_norm_strided_leading_dimensions_and_broadcast_gradient():
    from dig_amd import ops
    g = gen(7)
    wide = randn(g, 60, 50).to(torch.bfloat16)
    x = wide[:, 3:40]
    w = torch.ones(37, device=DEV, dtype=torch.bfloat16)
    y = ops.layer_norm(x, w)
    assert torch.equal(y, ops.layer_norm(x.contiguous(), w))
    assert torch.equal(ops.layer_norm(wide[::2, 1:38], w), ops.layer_norm(wide[::2, 1:38].contiguous(), w))
    x3 = randn(g, 4, 5, 37).requires_grad_()
    y3 = ops.layer_norm(x3)
    assert y3.shape == x3.shape and torch.equal(y3.reshape(20, 37), ops.layer_norm(x3.reshape(20, 37)))
    assert torch.equal(ops.layer_norm(x3.transpose(0, 1)), y3.transpose(0, 1))
    one = randn(g, 37)
    assert torch.equal(ops.layer_norm(one), ops.layer_norm(one[None])[0])
    assert torch.equal(ops.layer_norm(one.expand(6, 37)), ops.layer_norm(one.repeat(6, 1)))
    (a,) = torch.autograd.grad(ops.layer_norm(x3).sum(), x3)                       # a gradient of stride 0
    (b,) = torch.autograd.grad(ops.layer_norm(x3), x3, torch.ones_like(x3))
    assert torch.equal(a, b)


def test_layer_norm_constant_rows_empty_batches_and_what_is_no_number():
    from dig_amd import ops
    w, b = torch.full((64,), 2.0, device=DEV, requires_grad=True), torch.full((64,), 3.0, device=DEV, requires_grad=True)
    x = torch.full((5, 64), 7.0, device=DEV)
    assert torch.equal(ops.layer_norm(x, w, b), torch.full_like(x, 3.0))             # a row without variance: its bias
    e = torch.empty(0, 64, device=DEV, requires_grad=True)
    y = ops.layer_norm(e, w, b)
    gx, gw, gb = torch.autograd.grad(y, (e, w, b), torch.empty(0, 64, device=DEV))
    assert y.shape == gx.shape == (0, 64) and not gw.any() and not gb.any()
    x[2, 5] = float('nan')
    x[3, 6] = float('inf')
    y = ops.layer_norm(x, w, b)
    assert torch.isnan(y[2]).all() and torch.isnan(y[3]).all() and torch.equal(y[[0, 1, 4]], torch.full_like(y[:3], 3.0))


def test_layer_norm_large_offset_keeps_the_centred_variance():
    """mean 1000, deviation 1: a variance from the mean square would have lost 20 of its 24 bits"""
    from dig_amd import ops
    g = gen(8)
    x = randn(g, 64, 512) + 1000.0
    gy = randn(g, 64, 512)
    y = ops.layer_norm(x)
    check_norm(x, None, None, 1e-5, gy, y, None, None, None)


def test_layer_norm_joins_the_deferred_reductions():
    from dig_amd import ops
    g = gen(9)
    x, gy = randn(g, 300, 128), randn(g, 300, 128)
    w, b = (1 + 0.2 * randn(g, 128)).requires_grad_(), randn(g, 128).requires_grad_()
    now = torch.autograd.grad(ops.layer_norm(x, w, b), (w, b), gy)
    with ops.deferred_reductions() as red:
        later = torch.autograd.grad(ops.layer_norm(x, w, b), (w, b), gy)
    red.flush()
    q = norm64(x, w.detach(), b.detach(), 1e-5, gy)
    for a, c, ref, size in ((now[0], later[0], q['gw'], (q['gy'] * q['h']).abs().sum(0)), (now[1], later[1], q['gb'], q['gy'].abs().sum(0))):
        close(c, ref, (300 / 64 + 128 + 64) * U * size, 'deferred')
        assert (a - c).abs().max() <= 1e-4


# ------------------------------------------------------------------------------------------------ class losses
def head64(x, w, b, tau):
    z = x.double() @ w.double().t()
    return (z + b.double() if b is not None else z) / tau


def head_bounds(x, w, b, z, tau):
    """-> dz [N]: how far a logit / tau may be.  A product of D terms in float32: (D + 8) u sum |x w|.  float32 inputs enter as
    two 11-bit numbers each: 2^-22 of a factor lost, 2^-22 of the term dropped, 2^-39 of the tensor's largest value at small
    entries; three partial products of D terms."""
    D = x.size(1)
    s = (x.double().abs() @ w.double().abs().t()).amax(1)
    n = (3 * D if x.dtype == torch.float32 else D) + 8
    dz = n * U * s
    if x.dtype == torch.float32:
        dz = dz + 3 * 2.0 ** -22 * s + 2.0 ** -39 * D * (x.abs().max() * w.double().abs().max() * 2)
    zb = z.masked_fill(~torch.isfinite(z), 0).abs().amax(1)
    return dz / tau + 4 * U * zb + 4 * U * (b.double().abs().masked_fill(~torch.isfinite(b), 0).max() / tau if b is not None else 0.0)


def check_head(x, w, b, z, e, rows, loss_size, tau, got, scale, loss64):
    """z logits / tau, e = d loss_n / d z_n / tau as float64 [N, V] already times the row's incoming gradient (``scale`` [N]);
    rows: the losses [N].  e is off by |p| (2 dz + 8 u (1 + |z - lse|)) times the row's gradient, and half a step of the type it
    is kept in (float32: two halves, 2^-22); its products add that against |W| and |x|."""
    t = x.dtype
    V, (N, D) = w.size(0), x.shape
    dz = head_bounds(x, w, b, z, tau)
    zf = z.masked_fill(~torch.isfinite(z), 0)
    lse = torch.logsumexp(z, 1)
    # exp of a difference of size s: 3 u s in the exponent's product and difference; sums over V in a tree of tiles
    spread = (lse[:, None] - zf).abs()
    p = torch.exp(z - lse[:, None])
    dl = 2 * dz + 8 * U * (1 + (p * spread).sum(1)) + 40 * U
    tol_rows = loss_size * (dl + 4 * U * (zf.abs().amax(1) + lse.abs())) + 16 * U * rows.abs()
    if 'rows' in got:
        close(got['rows'], rows, tol_rows, 'rows')
    if 'out' in got:
        close(got['out'], loss64, (tol_rows.sum() + (N / 1024 + 64) * U * rows.abs().sum()) / got['div'], 'loss')
    a = scale.abs()[:, None]
    keep = {torch.float32: 2.0 ** -22, torch.bfloat16: half(torch.bfloat16), torch.float16: half(torch.float16)}[t]
    # entries far below the row's gradient are kept to 2^-24 / 2^15 of it in float16 (its smallest step over the scale)
    floor = {torch.float32: 2.0 ** -39, torch.bfloat16: 0.0, torch.float16: 2.0 ** -39}[t] * a.max()
    de = a * p * (2 * dz[:, None] + dl[:, None] + 8 * U * (1 + spread)) + (keep + 8 * U) * e.abs() + floor * (a != 0)
    wd, xd = w.double().abs(), x.double().abs().masked_fill(a == 0, 0.0)
    lost = 3 * 2.0 ** -22 if t == torch.float32 else 0.0
    tiny = 2.0 ** -39 * 2 if t == torch.float32 else 0.0
    ea = e.abs()
    n = 3 if t == torch.float32 else 1
    close(got['gx'], e @ w.double(), half(t) * (e @ w.double()).abs() * 1.01 + de @ wd + ((n * V + 64) * U + lost) * (ea @ wd) + tiny * wd.max() * ea.sum(1, keepdim=True) + torch.finfo(t).tiny, 'gx')
    xz = x.double().masked_fill(a == 0, 0.0)
    gw = e.t() @ xz
    close(got['gw'], gw, half(t) * gw.abs() * 1.01 + de.t() @ xd + ((n * N + 64) * U + lost) * (ea.t() @ xd) + tiny * xd.max() * ea.sum(0)[:, None] + torch.finfo(t).tiny, 'gw')
    if 'gb' in got:
        gb = e.sum(0)
        close(got['gb'], gb, half(t) * gb.abs() * 1.01 + de.sum(0) + (N + 64) * U * ea.sum(0) + torch.finfo(t).tiny, 'gb')


def run_classes(x, w, b, target, reduction, g, ignore=-100):
    from dig_amd import ops
    out = ops.linear_cross_entropy(x, w, target, b, ignore_index=ignore, reduction=reduction)
    leaves = [p for p in (x, w, b) if p is not None]
    gr = torch.autograd.grad(out, leaves, g)
    assert all(p.dtype == q.dtype and p.shape == q.shape for p, q in zip(leaves, gr)) and out.dtype == torch.float32
    got = dict(zip(('gx', 'gw', 'gb'), gr))
    got['rows' if reduction == 'none' else 'out'] = out.detach()
    return got


def ref_classes(x, w, b, target, reduction, g, ignore=-100):
    z = head64(x, w, b, 1.0)
    live = target != ignore
    at = torch.where(live, target, 0)
    lp = torch.log_softmax(z, 1)
    rows = torch.where(live, -lp.gather(1, at[:, None])[:, 0], 0.0)
    n = max(1, int(live.sum()))
    scale = (g.double() * live) if reduction == 'none' else g.double() * live / (n if reduction == 'mean' else 1)
    e = lp.exp()
    e.scatter_(1, at[:, None], torch.expm1(-rows)[:, None])
    e = torch.where(scale[:, None] != 0, e * scale[:, None], 0.0)
    loss = rows.sum() / (n if reduction == 'mean' else 1)
    return z, e, rows, loss, scale, n if reduction == 'mean' else 1


def classes_case(N, D, V, t, bias, seed, boost=6.0):
    g = gen(seed)
    w = randn(g, V, D) / math.sqrt(D)
    target = torch.randint(0, V, (N,), device=DEV, generator=g)
    x = randn(g, N, D) + boost * torch.rand(N, 1, device=DEV, generator=g) * w[target]
    b = (0.5 * randn(g, V)).to(t).requires_grad_() if bias else None
    return x.to(t).requires_grad_(), w.to(t).requires_grad_(), b, target, g


def one_classes(N, D, V, t, bias, reduction, ignored, seed=None):
    x, w, b, target, g = classes_case(N, D, V, t, bias, seed if seed is not None else N * 7 + D * 3 + V)
    target[torch.rand(N, device=DEV, generator=g) < ignored] = -100
    up = torch.rand(N, device=DEV, generator=g) + 0.5 if reduction == 'none' else torch.tensor(float(N) if t == torch.float16 else 1.7, device=DEV)
    got = run_classes(x, w, b, target, reduction, up)
    x, w, b = x.detach(), w.detach(), b.detach() if bias else None
    z, e, rows, loss, scale, div = ref_classes(x, w, b, target, reduction, up)
    got['div'] = div
    check_head(x, w, b, z, e, rows, 1.0, 1.0, got, scale, loss)


# one row, one class, sizes around the tiles (64, 128, 256) and the k step (64), more rows than classes and the reverse
HEAD = [(1, 1, 1), (1, 64, 1000), (3, 5, 2), (32, 128, 1195), (65, 64, 63), (64, 63, 65), (127, 130, 129), (300, 257, 511), (513, 192, 257),
        (1, 320, 9001), (2100, 40, 37), (700, 256, 5000)]


@pytest.mark.parametrize('t', list(TYPES))
@pytest.mark.parametrize('N,D,V', HEAD)
def test_linear_cross_entropy(N, D, V, t):
    one_classes(N, D, V, TYPES[t], bias=(N + V) % 2 == 1, reduction='mean', ignored=0.0)


@pytest.mark.parametrize('t', list(TYPES))
@pytest.mark.parametrize('reduction', ['none', 'sum', 'mean'])
@pytest.mark.parametrize('ignored', [0.0, 0.5, 1.0])
def test_linear_cross_entropy_reductions_and_ignored_rows(t, reduction, ignored):
    one_classes(150, 96, 700, TYPES[t], bias=True, reduction=reduction, ignored=ignored, seed=11)


@pytest.mark.parametrize('t', list(TYPES))
def test_linear_cross_entropy_many_tiles(t):
    """enough tiles for the large tile shape in all four products, and split products where one side is short"""
    one_classes(2048, 512, 8192 + 130, TYPES[t], bias=False, reduction='mean', ignored=0.1)


def test_linear_cross_entropy_in_pieces_of_the_vocabulary():
    """N x V beyond one piece of the gradient's workspace (512 MiB): the last piece is ragged, gx is added over the pieces"""
    one_classes(16384, 16, 33000, torch.bfloat16, bias=True, reduction='mean', ignored=0.3)


@pytest.mark.parametrize('t', list(TYPES))
@pytest.mark.parametrize('N,D,V', [(70, 80, 300), (600, 640, 900)])
def test_ignored_rows_may_hold_anything(N, D, V, t):
    """NaN, infinities and the type's lowest value in rows that are ignored change no bit of any result (float32: nor the scale
    of the two 16-bit parts that the others are kept in)"""
    from dig_amd import ops
    t = TYPES[t]
    x, w, b, target, g = classes_case(N, D, V, t, True, 3)
    target[::3] = -100
    one = torch.tensor(1.0, device=DEV)
    want = run_classes(x, w, b, target, 'mean', one)
    y = x.detach().clone()
    y[0], y[3], y[6], y[9] = float('nan'), float('inf'), torch.finfo(t).min, torch.finfo(t).max
    got = run_classes(y.requires_grad_(), w, b, target, 'mean', one)
    for k in want:
        assert torch.equal(got[k], want[k]), k
    # the same rows without a teacher
    index = torch.randint(0, V, (N, 4), device=DEV, generator=g)
    index[::3] = -1
    tl = randn(g, N, 4)
    res = []
    for rows in (x, y):
        out = ops.linear_distillation(rows, w, index, tl, b, temperature=2.0)
        res.append((out.detach(),) + torch.autograd.grad(out, (rows, w, b)))
    assert all(torch.equal(p, q) for p, q in zip(*res))


def test_every_row_ignored_is_zero():
    x, w, b, target, g = classes_case(9, 64, 100, torch.float32, True, 4)
    target.fill_(-100)
    got = run_classes(x, w, b, target, 'mean', torch.tensor(2.0, device=DEV))
    assert float(got['out']) == 0.0 and not got['gx'].any() and not got['gw'].any() and not got['gb'].any()


def test_another_ignore_index_and_a_target_that_is_no_class():
    x, w, b, target, g = classes_case(12, 64, 100, torch.float32, False, 5)
    target[3] = 7
    target[5] = 100
    got = run_classes(x, w, None, target, 'none', torch.ones(12, device=DEV), ignore=7)
    rows = got['rows']
    assert float(rows[3]) == 0.0 and not got['gx'][3].any()
    assert torch.isnan(rows[5]) and torch.isnan(got['gx'][5]).all()
    ok = [i for i in range(12) if i not in (5,) and int(target[i]) != 7]
    assert torch.isfinite(rows[ok]).all() and torch.isfinite(got['gx'][ok]).all()
    target[5] = -1
    got = run_classes(x, w, None, target, 'none', torch.ones(12, device=DEV), ignore=7)
    assert torch.isnan(got['rows'][5])


def test_masked_classes_and_a_bias_of_the_lowest_value():
    """a bias of -inf, or of the type's lowest value, takes classes out: probability 0, no gradient, and the rest as if alone"""
    for low in (float('-inf'), torch.finfo(torch.float32).min):
        x, w, b, target, g = classes_case(40, 64, 600, torch.float32, True, 6)
        bd = b.detach().clone()
        bd[300:] = low
        target = target % 300
        got = run_classes(x, w, bd.requires_grad_(), target, 'mean', torch.tensor(1.0, device=DEV))
        x, w, bd = x.detach(), w.detach(), bd.detach()
        z, e, rows, loss, scale, div = ref_classes(x, w[:300], bd[:300], target, 'mean', torch.tensor(1.0, device=DEV))
        assert not got['gw'][300:].any() and not got['gb'][300:].any()
        part = dict(out=got['out'], gx=got['gx'], gw=got['gw'][:300], gb=got['gb'][:300], div=div)
        check_head(x, w[:300], bd[:300], z, e, rows, 1.0, 1.0, part, scale, loss)


def test_a_certain_prediction_keeps_its_small_loss_and_gradient():
    """logit gaps up to 80: the loss and the target's gradient come from what the other classes hold, not from 1 - 1"""
    from dig_amd import ops
    N, V = 64, 32
    gap = torch.linspace(0, 80, N, device=DEV)
    x = torch.zeros(N, 64, device=DEV, dtype=torch.bfloat16)
    x[:, 0] = gap.to(torch.bfloat16)
    x.requires_grad_()
    w = torch.zeros(V, 64, device=DEV, dtype=torch.bfloat16)
    w[5, 0] = 1
    target = torch.full((N,), 5, device=DEV)
    rows = ops.linear_cross_entropy(x, w, target, reduction='none')
    want = torch.log1p(31 * torch.exp(-x.detach()[:, 0].double()))
    assert ((rows.double() - want).abs() <= 64 * U * want).all()             # sums of one sign: relative errors only
    (gx,) = torch.autograd.grad(rows.sum(), x)
    gw = torch.expm1(-want)
    assert ((gx[:, 0].double() - gw).abs() <= (2 * half(torch.bfloat16) + 80 * U) * gw.abs()).all()


def test_logits_of_every_size():
    """logits of +-1e4: nothing overflows, the statistics are those of the largest"""
    x, w, b, target, g = classes_case(33, 64, 500, torch.float32, False, 8)
    x = (x.detach() * 4000).requires_grad_()
    got = run_classes(x, w, None, target, 'mean', torch.tensor(1.0, device=DEV))
    x, w = x.detach(), w.detach()
    z, e, rows, loss, scale, div = ref_classes(x, w, None, target, 'mean', torch.tensor(1.0, device=DEV))
    got['div'] = div
    check_head(x, w, None, z, e, rows, 1.0, 1.0, got, scale, loss)


def test_strided_rows_and_weights_and_leading_dimensions():
    from dig_amd import ops
    for t in TYPES.values():
        x, w, b, target, g = classes_case(60, 64, 130, t, True, 9)
        x, w, b = x.detach(), w.detach(), b.detach()
        ref = ops.linear_cross_entropy(x, w, target, b, reduction='none')
        xw = torch.zeros(60, 75, device=DEV, dtype=t)
        xw[:, 3:67] = x
        ww = torch.zeros(130, 81, device=DEV, dtype=t)
        ww[:, 9:73] = w
        assert torch.equal(ops.linear_cross_entropy(xw[:, 3:67], ww[:, 9:73], target, b, reduction='none'), ref)
        assert torch.equal(ops.linear_cross_entropy(x, w.t().contiguous().t(), target, b, reduction='none'), ref)
        out = ops.linear_cross_entropy(x.reshape(4, 15, 64), w, target.reshape(4, 15), b, reduction='none')
        assert out.shape == (4, 15) and torch.equal(out.reshape(-1), ref)
        one = ops.linear_cross_entropy(x[7], w, target[7], b, reduction='none')
        # a row alone takes other tiles: the same value up to the order of the sums of 64 products and 130 classes
        assert one.shape == () and abs(float(one) - float(ref[7])) <= 400 * U * (1 + float(ref[7]) + 8 * 10)


def test_only_the_gradients_that_are_wanted():
    from dig_amd import ops
    x, w, b, target, g = classes_case(100, 64, 300, torch.float32, True, 10)
    full = run_classes(x, w, b, target, 'sum', torch.tensor(1.0, device=DEV))
    for k, name in ((0, 'gx'), (1, 'gw'), (2, 'gb')):
        ps = [p.detach().requires_grad_(i == k) for i, p in enumerate((x, w, b))]
        (gr,) = torch.autograd.grad(ops.linear_cross_entropy(ps[0], ps[1], target, ps[2], reduction='sum'), ps[k])
        assert torch.equal(gr, full[name])


def test_empty_batch():
    from dig_amd import ops
    x = torch.empty(0, 64, device=DEV, requires_grad=True)
    w = torch.randn(50, 64, device=DEV, requires_grad=True)
    t = torch.empty(0, dtype=torch.int64, device=DEV)
    for red in ('mean', 'sum', 'none'):
        out = ops.linear_cross_entropy(x, w, t, reduction=red)
        gx, gw = torch.autograd.grad(out.sum(), (x, w))
        assert float(out.detach().sum()) == 0.0 and gx.shape == (0, 64) and not gw.any()
    out = ops.linear_distillation(x, w, torch.empty(0, 3, dtype=torch.int64, device=DEV), torch.empty(0, 3, device=DEV))
    assert float(out.detach()) == 0.0


def test_gradient_against_differences():
    """(L(x + h d) - L(x - h d)) / 2h: the third derivative of the loss along a unit direction is below |w|^3, each loss is off by
    1e-6 at most at these sizes; h = 0.05 leaves 1e-6 / h + h^2 |w|^3 / 6"""
    from dig_amd import ops
    for which in range(3):
        x, w, b, target, g = classes_case(40, 64, 90, torch.float32, True, 12, boost=1.0)
        ps = [x, w, b]
        out = ops.linear_cross_entropy(*ps[:2], target, b, reduction='sum')
        gr = torch.autograd.grad(out, ps)[which]
        d = randn(g, *ps[which].shape)
        d /= d.norm()
        h = 0.05
        vals = []
        for s in (h, -h):
            q = [p.detach() for p in ps]
            q[which] = q[which] + s * d
            vals.append(ops.linear_cross_entropy(*q[:2], target, q[2], reduction='none').double().sum())
        diff = (vals[0] - vals[1]) / (2 * h)
        # sum of 40 rows: |third derivative| <= sum of (|d z|)^3 <= (|row or class direction| * |w| or |x|)^3
        reach = float(max(w.detach().norm(dim=1).max(), x.detach().norm(dim=1).max(), 1.0)) ** 3
        assert abs(float(diff) - float((gr.double() * d).sum())) <= 40 * 1e-6 / h + h * h * reach / 6


# ------------------------------------------------------------------------------------------------ distillation
def ref_teacher(x, w, b, index, teacher, tau, reduction, g):
    z = head64(x, w, b, tau)
    there = (index >= 0) & (teacher.double() != float('-inf'))
    live = there.any(1)
    a = torch.where(there, teacher.double() / tau, float('-inf'))
    a[~live] = 0.0
    q = torch.where(there, torch.softmax(a, 1), 0.0)
    lp = torch.log_softmax(z, 1)
    at = index.clamp(min=0)
    lk = lp.gather(1, at)
    rows = tau * tau * (torch.xlogy(q, q) - torch.where(q > 0, q * lk, 0.0)).sum(1)
    size = tau * tau * (1 + (q * torch.where(q > 0, a - a.amax(1, keepdim=True), 0.0).abs()).sum(1))
    n = max(1, int(live.sum()))
    scale = tau * (g.double() * live if reduction == 'none' else g.double() * live / (n if reduction == 'mean' else 1))
    e = lp.exp()
    e.scatter_add_(1, at, -q)
    return z, e * scale[:, None], rows, size, scale, n if reduction == 'mean' else 1


def teacher_case(N, D, V, K, t, bias, seed, ragged):
    g = gen(seed)
    w = randn(g, V, D) / math.sqrt(D)
    index = torch.rand(N, V, device=DEV, generator=g).topk(K, 1).indices
    teacher = 2 * randn(g, N, K)
    x = randn(g, N, D) + 2.0 * w[index[:, 0]]
    if ragged:
        gone = torch.arange(K, device=DEV) >= (torch.rand(N, 1, device=DEV, generator=g) * (K + 1)).long()
        index = index.masked_fill(gone, -1)
    b = (0.5 * randn(g, V)).to(t).requires_grad_() if bias else None
    return x.to(t).requires_grad_(), w.to(t).requires_grad_(), b, index, teacher.to(t), g


def one_teacher(N, D, V, K, t, bias, reduction, ragged, tau, seed=21, change=None):
    from dig_amd import ops
    x, w, b, index, teacher, g = teacher_case(N, D, V, K, t, bias, seed, ragged)
    if change:
        change(index, teacher)
    up = torch.rand(N, device=DEV, generator=g) + 0.5 if reduction == 'none' else torch.tensor(float(N) if t == torch.float16 else 1.3, device=DEV)
    out = ops.linear_distillation(x, w, index, teacher, b, temperature=tau, reduction=reduction)
    leaves = [p for p in (x, w, b) if p is not None]
    got = dict(zip(('gx', 'gw', 'gb'), torch.autograd.grad(out, leaves, up)))
    got['rows' if reduction == 'none' else 'out'] = out.detach()
    x, w, b = x.detach(), w.detach(), b.detach() if bias else None
    z, e, rows, size, scale, div = ref_teacher(x, w, b, index, teacher, tau, reduction, up)
    got['div'] = div
    # an entry of a listed class is p - q with q off by 16 u (1 + its exponent): inside the keep term's 8 u |e| + this
    e_ref = e
    check_teacher(x, w, b, z, e_ref, rows, size, tau, got, scale, rows.sum() / div, index, teacher)
    return got


def check_teacher(x, w, b, z, e, rows, size, tau, got, scale, loss, index, teacher):
    """as check_head, with the rounding of q beside that of p: q is off by 16 u (1 + its exponent's size) relative"""
    V = w.size(0)
    there = (index >= 0) & (teacher.double() != float('-inf'))
    a = torch.where(there, teacher.double() / tau, 0.0)
    dq = 16 * U * (2 + 2 * a.abs().amax())
    extra = dq * scale.abs()[:, None]                         # of an entry, |q| <= 1
    N, D = x.shape
    if 'gx' in got:
        wd, xd = w.double().abs(), x.double().abs()
        K = index.size(1)
        got = dict(got)
        slack = dict(gx=extra * wd.amax() * K, gw=(extra.amax() * xd.sum(0) * 1.0)[None].expand(V, D), gb=extra.amax() * N)
        ref = dict(gx=e @ w.double(), gw=e.t() @ x.double(), gb=e.sum(0))
        for k in ('gx', 'gw', 'gb'):
            if k in got:            # move the value towards the reference by the slack: what is left is check_head's own bound
                d = got[k].double() - ref[k]
                got[k] = ref[k] + d.sign() * (d.abs() - slack[k]).clamp(min=0)
    check_head(x, w, b, z, e, rows, size, tau, got, scale, loss)


TEACH = [(1, 64, 100, 1), (1, 5, 7, 7), (64, 128, 1195, 16), (65, 63, 130, 3), (300, 257, 511, 64), (130, 96, 3000, 130), (700, 520, 3000, 32),
         (3, 64, 3000, 2048)]


@pytest.mark.parametrize('t', list(TYPES))
@pytest.mark.parametrize('N,D,V,K', TEACH)
def test_linear_distillation(N, D, V, K, t):
    one_teacher(N, D, V, K, TYPES[t], bias=N % 2 == 0, reduction='mean', ragged=N > 600, tau=2.0)


@pytest.mark.parametrize('t', list(TYPES))
@pytest.mark.parametrize('reduction', ['none', 'sum', 'mean'])
@pytest.mark.parametrize('tau', [1.0, 4.0])
def test_linear_distillation_short_lists_and_reductions(t, reduction, tau):
    one_teacher(120, 64, 400, 9, TYPES[t], bias=True, reduction=reduction, ragged=True, tau=tau)


def test_linear_distillation_equal_indices_and_absent_entries_that_hold_anything():
    def change(index, teacher):
        index[0] = 17                              # one class, listed nine times
        index[1, 1] = index[1, 0]
        teacher[2, :] = float('-inf')              # a row without entries
        index[3, :] = -5
        teacher[3, 0] = float('nan')
        index[4, 2], teacher[4, 2] = -1, float('inf')
        teacher[5, 3] = float('-inf')
        teacher[6, 4] = torch.finfo(teacher.dtype).min
    for t in TYPES.values():
        got = one_teacher(30, 64, 200, 9, t, True, 'none', False, 2.0, change=change)
        assert float(got['rows'][2]) == 0.0 and float(got['rows'][3]) == 0.0
        assert not got['gx'][2].any() and not got['gx'][3].any()


def test_linear_distillation_index_beyond_the_classes_is_nan():
    from dig_amd import ops
    x, w, b, index, teacher, g = teacher_case(20, 64, 50, 4, torch.float32, False, 30, False)
    index[3, 2] = 50
    index[4, 1] = 1 << 40
    rows = ops.linear_distillation(x, w, index, teacher, reduction='none')
    assert torch.isnan(rows[3]) and torch.isnan(rows[4]) and torch.isfinite(rows[:3]).all() and torch.isfinite(rows[5:]).all()
    (gx,) = torch.autograd.grad(rows, x, torch.ones(20, device=DEV))
    assert torch.isnan(gx[3]).all() and torch.isfinite(gx[:3]).all() and torch.isfinite(gx[5:]).all()


def test_distillation_of_one_class_is_the_cross_entropy():
    """K = 1, tau = 1: q is one, the loss the label's.  Both are checked against float64 elsewhere; here the two against each
    other, within the sum of their bounds at this size (64 products and 200 classes of order 1 and 10)"""
    from dig_amd import ops
    x, w, b, target, g = classes_case(50, 64, 200, torch.float32, True, 31)
    a = ops.linear_cross_entropy(x, w, target, b, reduction='none')
    c = ops.linear_distillation(x, w, target[:, None], torch.zeros(50, 1, device=DEV), b, reduction='none')
    assert ((a - c).abs() <= 1000 * U * (1 + a.abs() + 10)).all()


# ------------------------------------------------------------------------------------------------ together, streams, graphs
class Head:
    """the operators as they are used: norm -> classes, and norm -> teacher, over one weight"""

    def __init__(self, t, seed=40, N=96, D=128, V=1195, K=8):
        g = gen(seed)
        self.h = (randn(g, N, D) * 1.3).to(t).requires_grad_()
        self.nw, self.nb = (1 + 0.1 * randn(g, D)).to(t).requires_grad_(), (0.1 * randn(g, D)).to(t).requires_grad_()
        self.w, self.b = (randn(g, V, D) / math.sqrt(D)).to(t).requires_grad_(), (0.1 * randn(g, V)).to(t).requires_grad_()
        self.target = torch.randint(0, V, (N,), device=DEV, generator=g)
        self.target[::5] = -100
        self.index = torch.rand(N, V, device=DEV, generator=g).topk(K, 1).indices
        self.index[1] = -1
        self.teacher = randn(g, N, K)

    leaves = property(lambda s: (s.h, s.nw, s.nb, s.w, s.b))

    def step(self):
        from dig_amd import ops
        x = ops.layer_norm(self.h, self.nw, self.nb)
        loss = 0.5 * ops.linear_cross_entropy(x, self.w, self.target, self.b)
        loss = loss + 0.5 * ops.linear_distillation(x, self.w, self.index, self.teacher, self.b, temperature=2.0)
        return (loss.detach(),) + torch.autograd.grad(loss, self.leaves)


def test_a_head_step_against_float64_autograd():
    s = Head(torch.float32)
    got = s.step()
    h, nw, nb, w, b = (p.detach().double().requires_grad_() for p in s.leaves)
    d = h - h.mean(1, keepdim=True)
    x = d / (d.square().mean(1, keepdim=True) + 1e-5).sqrt() * nw + nb
    z = x @ w.t() + b
    keep = s.target >= 0
    ce = -torch.log_softmax(z, 1)[keep].gather(1, s.target[keep][:, None]).mean()
    live = s.index[:, 0] >= 0
    q = torch.softmax(s.teacher[live].double() / 2, 1)
    lp = torch.log_softmax(z[live] / 2, 1).gather(1, s.index[live])
    loss = 0.5 * ce + 0.5 * 4 * (q * (q.log() - lp)).sum(1).mean()
    want = (loss.detach(),) + torch.autograd.grad(loss, (h, nw, nb, w, b))
    # 2-norms: D = 128 products of two 22-bit factors, 1195 classes, 96 rows: every sum is shorter than 3 * 1195 terms of either
    # sign, whose errors grow as the root: 60 u; ten operations in a row
    for a, r in zip(got, want):
        assert float((a.double() - r).norm() / r.norm()) <= 10 * 60 * U


@pytest.mark.parametrize('t', list(TYPES))
def test_the_same_bits_every_time_and_on_another_stream(t):
    s = Head(TYPES[t])
    first = s.step()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, s.step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = s.step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, other))


@pytest.mark.hipgraph
@pytest.mark.parametrize('t', ['f32', 'bf16'])
def test_a_captured_head_step_replays_the_eager_one(t):
    """two steps captured into two graphs of their own memory, replayed in turn with eager work between, on changing inputs"""
    t = TYPES[t]
    heads = [Head(t, seed=50, N=96), Head(t, seed=51, N=33, D=64, V=300)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in heads:
            s.step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in heads:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s.step())
        graphs.append(g)
    for k in range(4):
        for s, g, o in zip(heads, graphs, outs):
            with torch.no_grad():
                s.h.mul_(0.9).add_(0.01)
                s.target.copy_(torch.roll(s.target, 1))
            g.replay()
            want = s.step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(o, want)), (k, t)


def test_what_is_saved_may_be_packed_elsewhere():
    """saved tensors that come back from the host at other addresses, and a second backward of the same graph"""
    from dig_amd import ops
    s = Head(torch.float32, seed=62)
    want = s.step()
    with torch.autograd.graph.save_on_cpu():
        got = s.step()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    x = ops.layer_norm(s.h, s.nw, s.nb)
    loss = ops.linear_cross_entropy(x, s.w, s.target, s.b)
    a = torch.autograd.grad(loss, s.leaves, retain_graph=True)
    kept = [p.clone() for p in a]
    c = torch.autograd.grad(loss, s.leaves, grad_outputs=torch.tensor(2.0, device=DEV))
    assert all(torch.equal(p, q) for p, q in zip(a, kept)) and all(torch.equal(2 * p, q) for p, q in zip(a, c))


def test_two_steps_in_flight_on_two_streams():
    a, b = Head(torch.float32, seed=60), Head(torch.bfloat16, seed=61, N=200, D=192, V=2000)
    wa, wb = a.step(), b.step()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (sa, sb):
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(sa):
            ga = a.step()
        with torch.cuda.stream(sb):
            gb = b.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ga, wa)) and all(torch.equal(p, q) for p, q in zip(gb, wb))


def test_a_protein_class_head_trains_on_the_fused_loss():
    """ProNet's class head under the fused loss: the gradients that its last layer gets from the logits and a plain log-softmax"""
    from dig_amd import ops
    g = gen(70)
    y = randn(g, 32, 128).requires_grad_()
    lin_w, lin_b = (randn(g, 384, 128) / 11).requires_grad_(), torch.zeros(384, device=DEV, requires_grad=True)
    target = torch.randint(0, 384, (32,), device=DEV, generator=g)
    a = torch.autograd.grad(ops.linear_cross_entropy(y, lin_w, target, lin_b), (y, lin_w, lin_b))
    z = ops.linear(y, lin_w, lin_b)
    loss = -torch.log_softmax(z, 1).gather(1, target[:, None]).mean()
    c = torch.autograd.grad(loss, (y, lin_w, lin_b))
    for p, q in zip(a, c):                                   # two float32 routes of 384-term sums
        assert float((p - q).norm() / q.norm()) <= 2 * 384 * U


def test_refusals_on_the_device():
    from dig_amd import _hip, ops
    x, w = torch.randn(4, 64, device=DEV), torch.randn(10, 64, device=DEV)
    t = torch.zeros(4, dtype=torch.int64, device=DEV)
    idx, tl = torch.zeros(4, 2, dtype=torch.int64, device=DEV), torch.zeros(4, 2, device=DEV)
    bad = [lambda: ops.layer_norm(x.double()), lambda: ops.layer_norm(x, torch.ones(63, device=DEV)), lambda: ops.layer_norm(x, torch.ones(64)),
           lambda: ops.layer_norm(x, torch.ones(64, device=DEV, dtype=torch.bfloat16)),
           lambda: ops.layer_norm(x, torch.ones(64, device=DEV), torch.ones(64, device=DEV, dtype=torch.float16)),
           lambda: ops.layer_norm(x[:, :0]), lambda: ops.layer_norm(x[0, 0]),
           lambda: ops.linear_cross_entropy(x, w.half(), t), lambda: ops.linear_cross_entropy(x, w[:, :63], t),
           lambda: ops.linear_cross_entropy(x, w, t.int()), lambda: ops.linear_cross_entropy(x, w, t[:3]),
           lambda: ops.linear_cross_entropy(x, w, t, torch.zeros(9, device=DEV)), lambda: ops.linear_cross_entropy(x, w, t, reduction='avg'),
           lambda: ops.linear_cross_entropy(x, w[:0], t), lambda: ops.linear_cross_entropy(x, w, t.cpu()),
           lambda: ops.linear_distillation(x, w, idx, tl, temperature=0.0), lambda: ops.linear_distillation(x, w, idx, tl[:, :1]),
           lambda: ops.linear_distillation(x, w, idx[:, :0], tl[:, :0]), lambda: ops.linear_distillation(x, w, idx.repeat(1, 1025), tl.repeat(1, 1025)), lambda: ops.linear_distillation(x, w, idx.int(), tl),
           lambda: ops.linear_distillation(x, w, idx, tl, temperature=float('nan')), lambda: ops.linear_distillation(x, w, idx[0], tl[0])]
    for k, f in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError)):
            f()
            raise AssertionError(f'call {k} was taken')
    # once differentiable: a second derivative is refused, not wrong
    xr = x.clone().requires_grad_()
    (gx,) = torch.autograd.grad(ops.linear_cross_entropy(xr, w, t), xr, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gx.sum(), xr)
    assert issubclass(_hip.Dig3dError, RuntimeError)


# ------------------------------------------------------------------------------------------------ the ends of the ranges
@pytest.mark.parametrize('N,V', [(40, 300), (600, 900)])
def test_tensors_whose_product_is_below_the_types_range(N, V):
    """x and w of 1e-25: every logit is 0 in float32, the loss log V to the rounding of a sum and a logarithm; the gradients
    are those of softmax = 1 / V (e off by 8 u and its two halves, the operands by 2^-22 and 2^-39 of the largest)"""
    from dig_amd import ops
    g = gen(80)
    x, w = (randn(g, N, 64) * 1e-25).requires_grad_(), (randn(g, V, 64) * 1e-25).requires_grad_()
    target = torch.randint(0, V, (N,), device=DEV, generator=g)
    rows = ops.linear_cross_entropy(x, w, target, reduction='none')
    close(rows, torch.full((N,), math.log(V), dtype=torch.float64, device=DEV), 64 * U * math.log(V), 'rows')
    gx, gw = torch.autograd.grad(rows.sum(), (x, w))
    e = torch.full((N, V), 1.0 / V, dtype=torch.float64, device=DEV)
    e[torch.arange(N, device=DEV), target] -= 1.0
    xd, wd = x.detach().double(), w.detach().double()
    for got, want, size, n, top in ((gx, e @ wd, e.abs() @ wd.abs(), V, wd.abs().max()), (gw, e.t() @ xd, e.abs().t() @ xd.abs(), N, xd.abs().max())):
        close(got, want, ((3 * n + 80) * U + 6 * 2.0 ** -22) * size + 2.0 ** -38 * n * top, 'gradient')


@pytest.mark.parametrize('N,V', [(40, 300), (600, 900)])
@pytest.mark.parametrize('t', list(TYPES))
def test_no_class_left_and_infinite_logits_are_nan(N, V, t):
    from dig_amd import ops
    x, w, b, target, g = classes_case(N, 64, V, TYPES[t], True, 81)
    none = torch.full_like(b, float('-inf')).requires_grad_()
    rows = ops.linear_cross_entropy(x, w, target, none, reduction='none')
    assert torch.isnan(rows).all() and torch.isnan(torch.autograd.grad(rows.sum(), x)[0]).all()
    for v in (0, int(target[0])):                  # beside a row's target, and as one
        up = b.detach().clone()
        up[v] = float('inf')
        assert torch.isnan(ops.linear_cross_entropy(x, w, target, up, reduction='none')).all()


def test_listed_logits_of_the_lowest_value_stay_entries():
    """at tau = 1/2 the lowest value over tau is beyond the type; alone in a row such entries share it equally, beside others
    they hold nothing, also where the head itself gives their class nothing"""
    from dig_amd import ops
    x, w, b, index, teacher, g = teacher_case(20, 64, 50, 4, torch.float32, True, 82, False)
    index[0] = torch.tensor([3, 9, 11, 40], device=DEV)
    index[1] = index[0]
    low, even = teacher.clone(), teacher.clone()
    low[0], even[0] = torch.finfo(torch.float32).min, 0.0
    low[1, 3] = torch.finfo(torch.float32).min
    even[1, 3] = float('-inf')
    a = ops.linear_distillation(x, w, index, low, b, temperature=0.5, reduction='none')
    c = ops.linear_distillation(x, w, index, even, b, temperature=0.5, reduction='none')
    assert torch.equal(a, c) and torch.isfinite(a).all()
    bd = b.detach().clone()
    bd[40] = float('-inf')
    a = ops.linear_distillation(x[1:2], w, index[1:2], low[1:2], bd, temperature=0.5, reduction='none')
    q = torch.softmax(teacher[1, :3].double() / 0.5, 0)
    lp = torch.log_softmax(head64(x.detach()[1:2], w.detach(), bd, 0.5), 1)[0]
    want = 0.25 * (q * (q.log() - lp[index[1, :3]])).sum()
    assert abs(float(a.detach()[0]) - float(want)) <= 2000 * U * (1 + abs(float(want)) + 20)


@pytest.mark.parametrize('reduction', ['none', 'sum', 'mean'])
@pytest.mark.parametrize('t', ['f32', 'bf16'])
def test_more_rows_than_one_workgroup_adds(t, reduction):
    one_classes(20000, 24, 40, TYPES[t], True, reduction, 0.2)


@pytest.mark.parametrize('N,D,V', [(40, 64, 300), (600, 128, 2000)])
def test_a_backward_leaves_what_the_forward_kept(N, D, V):
    from dig_amd import ops
    x, w, b, target, g = classes_case(N, D, V, torch.float32, True, 83)
    rows = ops.linear_cross_entropy(x, w, target, b, reduction='none')
    keep = [p for p in rows.grad_fn.saved_tensors if p is not None]
    before = [p.clone().view(torch.uint8) for p in keep]
    a = torch.autograd.grad(rows, (x, w, b), torch.full((N,), 3.0, device=DEV), retain_graph=True)
    torch.autograd.grad(rows, (x, w, b), torch.full((N,), 1e-3, device=DEV), retain_graph=True)
    assert all(torch.equal(p, q.view(torch.uint8)) for p, q in zip(before, keep))
    c = torch.autograd.grad(rows, (x, w, b), torch.full((N,), 3.0, device=DEV))
    assert all(torch.equal(p, q) for p, q in zip(a, c))


def test_temperatures_out_of_range_are_refused():
    from dig_amd import ops
    x, w = torch.randn(4, 64, device=DEV), torch.randn(10, 64, device=DEV)
    idx, tl = torch.zeros(4, 2, dtype=torch.int64, device=DEV), torch.zeros(4, 2, device=DEV)
    for tau in (1e-7, 1e7, -1.0, float('inf')):
        with pytest.raises(ValueError):
            ops.linear_distillation(x, w, idx, tl, temperature=tau)


@pytest.mark.parametrize('N,D,V', [(1, 1024, 4096), (16, 515, 5001), (16, 515, 17001), (64, 96, 20000), (200, 100, 3000)])
def test_few_float32_rows_of_many_classes(N, D, V):
    """sizes around those that float32 takes in place and 16-bit rows do not"""
    one_classes(N, D, V, torch.float32, True, 'none', 0.2)
    one_teacher(N, D, V, 12, torch.float32, False, 'mean', True, 2.0)


def test_offsets_beyond_32_bits():
    """more than 2^31 elements of W, and of the rows of a layer norm: what lies behind them is what it is alone"""
    from dig_amd import ops
    g = gen(90)
    N, D, V = 4, 2048, 1_100_000
    w = torch.empty(V, D, device=DEV, dtype=torch.bfloat16)
    for i in range(0, V, 100_000):
        w[i:i + 100_000] = (randn(g, 100_000, D) / math.sqrt(D)).to(torch.bfloat16)
    x = randn(g, N, D).to(torch.bfloat16).requires_grad_()
    w.requires_grad_()
    target = torch.tensor([0, V - 1, V - 70_000, 1_048_577], device=DEV)
    rows = ops.linear_cross_entropy(x, w, target, reduction='none')
    gx, gw = torch.autograd.grad(rows.sum(), (x, w))
    xd, wd = x.detach().double(), w.detach()
    z = torch.cat([xd @ wd[i:i + 100_000].double().t() for i in range(0, V, 100_000)], 1)
    lse = torch.logsumexp(z, 1)
    want = lse - z.gather(1, target[:, None])[:, 0]
    # (D + 8) u of the terms in a logit, 8 u of every exponential, 40 levels of additions, twice (the sum and the target)
    size = (xd.abs() @ wd[target].double().abs().t()).amax()
    tol = 2 * ((D + 8) * U * float(size) + 100 * U)
    close(rows, want, tol * (1 + want.abs()), 'rows')
    e = torch.exp(z - lse[:, None])
    e[torch.arange(N, device=DEV), target] -= 1
    # two bf16 numbers of e: 2^-16 of an entry; the result's half step; V additions in ranges of at most 2^15 terms a chain
    ref, mag = torch.zeros(N, D, dtype=torch.float64, device=DEV), torch.zeros(N, D, dtype=torch.float64, device=DEV)
    for i in range(0, V, 100_000):
        ref += e[:, i:i + 100_000] @ wd[i:i + 100_000].double()
        mag += e[:, i:i + 100_000].abs() @ wd[i:i + 100_000].double().abs()
    close(gx, ref, half(torch.bfloat16) * ref.abs() * 1.01 + (2.0 ** -16 + 4 * tol + 2.0 ** 15 * U) * mag, 'gx')
    for i in (0, 1_048_570, V - 8):
        part = e[:, i:i + 8].t() @ xd
        close(gw[i:i + 8], part, half(torch.bfloat16) * part.abs() * 1.01 + (2.0 ** -16 + 4 * tol) * (e[:, i:i + 8].abs().t() @ xd.abs()) + 1e-30, 'gw')
    del w, gw, z, wd, e
    R, C = 2_200_000, 1000
    rows = torch.empty(R, C, device=DEV, dtype=torch.bfloat16)
    rows[:5], rows[-5:] = randn(g, 5, C).to(torch.bfloat16), randn(g, 5, C).to(torch.bfloat16)
    rows[5:-5] = 1.0
    y = ops.layer_norm(rows)
    assert torch.equal(y[-5:], ops.layer_norm(rows[-5:].clone())) and torch.equal(y[:5], ops.layer_norm(rows[:5].clone())) and not y[5:-5].any()


def test_an_ignore_index_beyond_the_type_is_refused():
    from dig_amd import ops
    with pytest.raises(ValueError):
        ops.linear_cross_entropy(torch.randn(4, 64, device=DEV), torch.randn(10, 64, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV),
                                 ignore_index=1 << 64)


@pytest.mark.parametrize('t', ['f32', 'bf16'])
def test_many_rows_of_a_teacher_with_few_classes(t):
    one_teacher(9000, 24, 40, 6, TYPES[t], True, 'mean', True, 2.0)


def test_many_ignored_rows_of_huge_values_leave_the_scale_alone():
    """float32, several rows a wave: the ignored ones hold the type's largest value and do not set the scale of the others"""
    x, w, b, target, g = classes_case(9000, 24, 40, torch.float32, True, 95)
    target[torch.rand(9000, device=DEV, generator=g) < 0.5] = -100
    clean = run_classes(x, w, b, target, 'mean', torch.tensor(1.0, device=DEV))
    y = x.detach().clone()
    y[target == -100] = torch.finfo(torch.float32).max
    got = run_classes(y.requires_grad_(), w, b, target, 'mean', torch.tensor(1.0, device=DEV))
    assert all(torch.equal(clean[k], got[k]) for k in clean)


@pytest.mark.parametrize('t', list(TYPES))
@pytest.mark.parametrize('R,C', [(600, 5000), (3, 12289), (5, 16384), (530, 8193)])
def test_layer_norm_of_long_rows(R, C, t):
    from dig_amd import ops
    g = gen(R + C)
    x = (randn(g, R, C) + 0.5).to(TYPES[t]).requires_grad_()
    w, b = (1 + 0.2 * randn(g, C)).to(TYPES[t]).requires_grad_(), (0.1 * randn(g, C)).to(TYPES[t]).requires_grad_()
    gy = randn(g, R, C).to(TYPES[t])
    y = ops.layer_norm(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), gy)
    check_norm(x.detach(), w.detach(), b.detach(), 1e-5, gy, y.detach(), gx, gw, gb)


@pytest.mark.parametrize('t', list(TYPES))
@pytest.mark.parametrize('N,D,V,K', [(5, 40, 30, 3), (2100, 72, 90, 33), (2050, 600, 70, 20), (2049, 64, 300, 64), (70, 128, 900, 300)])
def test_teacher_rows_of_one_wave_and_of_four(N, D, V, K, t):
    def change(index, teacher):
        index[0, -1] = index[0, 0]                 # a class listed twice, by the first and the last entry
        index[1, :] = -1
    one_teacher(N, D, V, K, TYPES[t], True, 'none', True, 2.0, change=change)

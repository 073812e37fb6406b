"""GPU: the class losses where their arithmetic comes to its ends — classes masked by the type's lowest value, rows with a single class
left, rows without a number beside others, and float32 operands whose sizes lie far apart — against float64 formulas.

Tolerances as in test_gpu_head.py: sums of the roundings that are made, derived before any run.  Each case runs at a size that the
kernels of head_small.h take in place and at one that the general path takes."""
import math

import pytest
import torch

from tests.test_gpu_head import DEV, TYPES, U, check_head, check_teacher, classes_case, close, gen, half, norm64, randn, ref_classes, ref_teacher

pytestmark = pytest.mark.gpu
SMALL, GENERAL = (40, 64, 600), (600, 64, 1100)          # rows, width, classes


def teacher_lists(g, N, V, K):
    return torch.rand(N, V, device=DEV, generator=g).topk(K, 1).indices, 2 * randn(g, N, K)


# ------------------------------------------------------------------------------------------------ masked classes
@pytest.mark.parametrize('t', list(TYPES))
@pytest.mark.parametrize('N,D,V', [SMALL, GENERAL])
def test_whole_tiles_of_classes_masked_by_the_lowest_value(N, D, V, t):
    """300 classes and behind them only masked ones: probability 0, no gradient, the others as if alone"""
    from dig_amd import ops
    x, w, b, target, g = classes_case(N, D, V, TYPES[t], True, 101)
    target = target % 300
    index, teacher = teacher_lists(g, N, 300, 5)
    one = torch.tensor(float(N) if t == 'f16' else 1.0, device=DEV)
    xd, wd, bd = x.detach(), w.detach()[:300], b.detach()[:300]
    for value in (torch.finfo(TYPES[t]).min, float('-inf')) + (() if t == 'f16' else (-1e10, -1e30)):
        low = b.detach().clone()
        low[300:] = value
        low.requires_grad_()
        out = ops.linear_cross_entropy(x, w, target, low)
        got = dict(zip(('gx', 'gw', 'gb'), torch.autograd.grad(out, (x, w, low), one)), out=out.detach())
        z, e, rows, loss, scale, div = ref_classes(xd, wd, bd, target, 'mean', one)
        assert not got['gw'][300:].any() and not got['gb'][300:].any(), value
        check_head(xd, wd, bd, z, e, rows, 1.0, 1.0, dict(got, gw=got['gw'][:300], gb=got['gb'][:300], div=div), scale, loss)
        for tau in (1.0, 0.5):             # at 1/2 logits of the lowest value are beyond the type's range
            out = ops.linear_distillation(x, w, index, teacher, low, temperature=tau)
            got = dict(zip(('gx', 'gw', 'gb'), torch.autograd.grad(out, (x, w, low), one)), out=out.detach())
            z, e, rows, size, scale, div = ref_teacher(xd, wd, bd, index, teacher, tau, 'mean', one)
            assert not got['gw'][300:].any() and not got['gb'][300:].any(), (value, tau)
            check_teacher(xd, wd, bd, z, e, rows, size, tau, dict(got, gw=got['gw'][:300], gb=got['gb'][:300], div=div), scale, rows.sum() / div,
                          index, teacher)


@pytest.mark.parametrize('t', ['f32', 'bf16'])
@pytest.mark.parametrize('N,D,V', [SMALL, GENERAL])
def test_every_class_at_the_lowest_value(N, D, V, t):
    """the bias swallows every product: all logits equal, the loss log V to the rounding of a sum and a logarithm, softmax = 1 / V.
    gx: V products of e, off by 16 u, and of w; in 16 bits e is rounded to half a step"""
    from dig_amd import ops
    x, w, b, target, g = classes_case(N, D, V, TYPES[t], True, 102)
    e = torch.full((N, V), 1.0 / V, dtype=torch.float64, device=DEV)
    e[torch.arange(N, device=DEV), target] -= 1.0
    wd = w.detach().double()
    keep = 2.0 ** -22 if t == 'f32' else half(TYPES[t])
    for value in (torch.finfo(TYPES[t]).min, -1e10):
        low = torch.full_like(b, value).requires_grad_()
        rows = ops.linear_cross_entropy(x, w, target, low, reduction='none')
        close(rows.detach(), torch.full((N,), math.log(V), dtype=torch.float64, device=DEV), 64 * U * math.log(V), 'rows')
        (gx,) = torch.autograd.grad(rows.sum(), x)
        close(gx, e @ wd, half(TYPES[t]) * (e @ wd).abs() * 1.01 + (keep + (6 * V + 200) * U) * (e.abs() @ wd.abs()), 'gx')


# ------------------------------------------------------------------------------------------------ one class left
@pytest.mark.parametrize('t', list(TYPES))
@pytest.mark.parametrize('N,D,V', [(40, 64, 1), (600, 64, 1), SMALL, GENERAL])
def test_the_target_is_the_only_class_left(N, D, V, t):
    """loss 0 and no gradient, whatever the size of its logit"""
    from dig_amd import ops
    t = TYPES[t]
    at = V // 2
    w = torch.zeros(V, D, device=DEV, dtype=t)
    w[at, 0] = 1
    w.requires_grad_()
    b = torch.full((V,), float('-inf'), device=DEV, dtype=t)
    b[at] = 0
    b.requires_grad_()
    target = torch.full((N,), at, device=DEV)
    for logit in (0.0, -80.0, -100.0, -1e4, 1e4):
        x = torch.zeros(N, D, device=DEV, dtype=t)
        x[:, 0] = logit
        x.requires_grad_()
        for red in ('mean', 'none'):
            out = ops.linear_cross_entropy(x, w, target, b, reduction=red)
            assert not out.detach().any(), (logit, red, out)
            for name, gr in zip('xwb', torch.autograd.grad(out.sum(), (x, w, b))):
                assert not gr.any(), (logit, red, name)


# ------------------------------------------------------------------------------------------------ a row without a number
@pytest.mark.parametrize('N,D,V', [(40, 64, 600), (600, 64, 900)])
@pytest.mark.parametrize('what', ['index', 'teacher', 'row', 'target'])
def test_a_row_without_a_number_counts_once(N, D, V, what):
    """the mean over 32 or 512 rows, one of them NaN: the loss and w's gradient are NaN, the other rows' gradients are those of the
    sum over the count of rows (a power of two: the same bits)"""
    from dig_amd import ops
    x, w, b, target, g = classes_case(N, D, V, torch.float32, True, 103)
    n = 32 if N < 512 else 512
    index, teacher = teacher_lists(g, N, V, 4)
    index[n:], target[n:] = -1, -100
    x = x.detach()
    if what == 'index':
        index[3, 1] = V
    elif what == 'teacher':
        teacher[3, 1] = float('nan')
    elif what == 'row':
        x[3, 5] = float('nan')
    else:
        target[3] = V
    x.requires_grad_()
    losses = []
    if what != 'target':
        losses.append(lambda red: ops.linear_distillation(x, w, index, teacher, b, temperature=2.0, reduction=red))
    if what in ('row', 'target'):
        losses.append(lambda red: ops.linear_cross_entropy(x, w, target, b, reduction=red))
    others = [i for i in range(N) if i != 3]
    for f in losses:
        mean = f('mean')
        gm, gw = torch.autograd.grad(mean, (x, w))
        (gs,) = torch.autograd.grad(f('sum'), x)
        assert torch.isnan(mean.detach()) and torch.isnan(gw).any() and torch.isnan(gm[3]).all()
        assert torch.isfinite(gs[others]).all() and gs[others].any()
        assert torch.equal(gm[others] * n, gs[others])


# ------------------------------------------------------------------------------------------------ rows without a loss
@pytest.mark.parametrize('t', list(TYPES))
@pytest.mark.parametrize('N,D,V', [SMALL, GENERAL])
def test_ignored_rows_beside_a_class_without_a_number(N, D, V, t):
    """a class whose bias is NaN or +inf makes every row's loss NaN; a row without a loss has none, and no gradient"""
    from dig_amd import ops
    x, w, b, target, g = classes_case(N, D, V, TYPES[t], True, 104)
    index, teacher = teacher_lists(g, N, V, 4)
    for value in (float('nan'), float('inf')):
        bad = b.detach().clone()
        bad[V - 2] = value
        bad.requires_grad_()
        for every in (False, True):
            tg, ix = target.clone(), index.clone()
            if every:
                tg[:], ix[:] = -100, -1
            else:
                tg[::3], ix[::3] = -100, -1
            for f in (lambda: ops.linear_cross_entropy(x, w, tg, bad), lambda: ops.linear_distillation(x, w, ix, teacher, bad)):
                out = f()
                gx, gw, gb = torch.autograd.grad(out, (x, w, bad))
                assert not gx[::3].any(), (value, every)
                if every:
                    assert float(out.detach()) == 0.0 and not gx.any() and not gw.any() and not gb.any()
                else:
                    assert torch.isnan(out.detach()) and torch.isnan(gx[1]).all()


@pytest.mark.parametrize('t', list(TYPES))
@pytest.mark.parametrize('N,D,V', [SMALL, GENERAL])
def test_what_reaches_an_ignored_row_is_not_used(N, D, V, t):
    """one loss per row: an incoming gradient of NaN or infinity at a row without a loss changes no bit"""
    from dig_amd import ops
    x, w, b, target, g = classes_case(N, D, V, TYPES[t], True, 105)
    index, teacher = teacher_lists(g, N, V, 4)
    target[::4], index[::4] = -100, -1
    up = torch.rand(N, device=DEV, generator=g) + 0.5
    for f in (lambda: ops.linear_cross_entropy(x, w, target, b, reduction='none'),
              lambda: ops.linear_distillation(x, w, index, teacher, b, reduction='none')):
        want = torch.autograd.grad(f(), (x, w, b), up)
        bad = up.clone()
        bad[0], bad[4], bad[8] = float('nan'), float('inf'), float('-inf')
        got = torch.autograd.grad(f(), (x, w, b), bad)
        assert all(torch.equal(p, q) for p, q in zip(got, want)) and all(torch.isfinite(p).all() for p in want)


@pytest.mark.parametrize('t', list(TYPES))
@pytest.mark.parametrize('N,D,V', [SMALL, GENERAL])
def test_a_gradient_without_a_number_reaches_the_rows_with_a_loss(N, D, V, t):
    """mean and sum under an incoming gradient of NaN or infinity: none of it in rows without a loss"""
    from dig_amd import ops
    x, w, b, target, g = classes_case(N, D, V, TYPES[t], True, 112)
    index, teacher = teacher_lists(g, N, V, 4)
    target[::4], index[::4] = -100, -1
    for red in ('mean', 'sum'):
        for f in (lambda: ops.linear_cross_entropy(x, w, target, b, reduction=red), lambda: ops.linear_distillation(x, w, index, teacher, b, reduction=red)):
            for value in (float('nan'), float('inf'), float('-inf')):
                gx, gw, gb = torch.autograd.grad(f(), (x, w, b), torch.tensor(value, device=DEV))
                assert not gx[::4].any(), (red, value)
                assert not torch.isfinite(gx[1]).any() and not torch.isfinite(gb[target[1]])


# ------------------------------------------------------------------------------------------------ float32 entry by entry
def check_entries(x, w, b, target, out, gx, gw, gb):
    """sum over rows, every entry against its own terms, no floor: x and w of 24 bits each (a product keeps 22 at least), sums of
    6 products a term in float32 of any order; p off by its logit's and its sum's errors; the target's p - 1 by its rest's."""
    N, D = x.shape
    V = w.size(0)
    xd, wd, bd = x.double(), w.double(), b.double()
    z, e, rows, loss, scale, _ = ref_classes(x, w, b, target, 'sum', torch.ones((), device=DEV))
    dz = ((6 * D + 64) * U + 2.0 ** -22) * (xd.abs() @ wd.abs().t()) + 4 * U * (z.abs() + bd.abs())
    lse = torch.logsumexp(z, 1, keepdim=True)
    p = torch.exp(z - lse)
    rel = dz + 8 * U * (1 + (z - lse).abs())
    de = p * (rel + (p * rel).sum(1, keepdim=True) + 40 * U)
    at = torch.where(scale != 0, target, 0)[:, None]
    rest = p.scatter(1, at, 0.0)
    have = rest.sum(1, keepdim=True).clamp(min=1e-300)
    own = rel.gather(1, at) + (rest * rel).sum(1, keepdim=True) / have + 64 * U
    de.scatter_(1, at, have * own)
    live = (scale != 0)[:, None]
    de, e = torch.where(live, de, 0.0), torch.where(live, e, 0.0)
    # a loss: of the rest's share, and of the difference of two logits where that is what it is
    tol = torch.where(live, have * own + dz.gather(1, at) + 8 * U * rows[:, None], 0.0).sum() + N * U * rows.sum()
    close(out, loss, tol, 'loss')
    for name, got, want, size, off, n in (('gx', gx, e @ wd, e.abs() @ wd.abs(), de @ wd.abs(), V), ('gw', gw, e.t() @ xd, e.abs().t() @ xd.abs(), de.t() @ xd.abs(), N),
                                          ('gb', gb, e.sum(0), e.abs().sum(0), de.sum(0), N)):
        close(got, want, off + (2.0 ** -22 + (6 * n + 64) * U) * size + 1e-36, name)


# the rows of gw of classes that no row gives more than 1e-8 .. 1e-30; predictions that are nearly certain; one row, class or column of x
# or w 1e8 times the others, or 1e-8; what the path of a size holds does not depend on the size
SPREADS = ['unlikely', 'certain', 'row', 'class', 'column of x', 'column of w', 'small column of w', 'everything']


@pytest.mark.parametrize('N,D,V', [SMALL, GENERAL, (300, 257, 2000)])
@pytest.mark.parametrize('spread', SPREADS)
def test_float32_entries_far_apart_in_size(N, D, V, spread):
    from dig_amd import ops
    x, w, b, target, g = classes_case(N, D, V, torch.float32, True, 106, boost=2.0)
    x, w, b = x.detach().clone(), w.detach().clone(), b.detach().clone()
    if spread in ('unlikely', 'everything'):
        b[V // 2:] -= torch.linspace(18, 69, V - V // 2, device=DEV)         # 1e-8 .. 1e-30
        target %= V // 2
    if spread == 'certain':
        b[7] += 25
        target[:] = 7
    if spread in ('row', 'everything'):
        x[3] *= 1e8
        target[3] = (x[3:4].double() @ w.double().t()).argmax()              # its own class: the others of its row hold nothing
    if spread == 'class':
        w[V - 3] *= 1e8
        w[V - 3] = -w[V - 3].abs() * x.sign().sum(0).sign()                  # rarely a row's largest
    if spread == 'column of x':
        x[:, 2] *= 1e8
        w[:, 2] *= 1e-8
    if spread == 'column of w':
        w[:, 2] *= 1e8
        x[:, 2] *= 1e-8
    if spread == 'small column of w':
        w[:, 2] *= 1e-8
        x[:, 3] *= 1e-8
    target[5] = -100
    leaves = [p.requires_grad_() for p in (x, w, b)]
    out = ops.linear_cross_entropy(x, w, target, b, reduction='sum')
    grads = torch.autograd.grad(out, leaves)
    check_entries(x.detach(), w.detach(), b.detach(), target, out.detach(), *grads)


@pytest.mark.parametrize('N,D,V', [SMALL, GENERAL])
def test_one_huge_row_leaves_the_others_alone(N, D, V):
    """a live row of 1e30, and one of the type's largest value: every other row's loss and gradient keep their bits"""
    from dig_amd import ops
    x, w, b, target, g = classes_case(N, D, V, torch.float32, True, 107)
    up = torch.ones(N, device=DEV)

    def rows_of(x):
        rows = ops.linear_cross_entropy(x, w, target, b, reduction='none')
        return rows.detach(), torch.autograd.grad(rows, x, up)[0]
    want, gx = rows_of(x)
    for value in (1e30, torch.finfo(torch.float32).max):
        y = x.detach().clone()
        y[9] = value
        got, gy = rows_of(y.requires_grad_())
        others = torch.arange(N, device=DEV) != 9
        assert torch.equal(got[others], want[others]) and torch.equal(gy[others], gx[others]), value


@pytest.mark.parametrize('N,D,V,K', [(40, 64, 600, 6), (600, 64, 1100, 6)])
def test_distillation_of_unlikely_classes(N, D, V, K):
    """rows of gw of classes outside the lists that hold 1e-8 .. 1e-30: entry by entry"""
    from dig_amd import ops
    x, w, b, target, g = classes_case(N, D, V, torch.float32, True, 108, boost=2.0)
    x, w, b = x.detach(), w.detach(), b.detach().clone()
    H = V // 2
    b[H:] -= torch.linspace(18, 69, V - H, device=DEV)
    index, teacher = teacher_lists(g, N, H, K)
    wg = w.clone().requires_grad_()
    (gw,) = torch.autograd.grad(ops.linear_distillation(x, wg, index, teacher, b, temperature=1.0, reduction='sum'), wg)
    z, e, rows, size, scale, div = ref_teacher(x, w, b, index, teacher, 1.0, 'sum', torch.ones((), device=DEV))
    xd = x.double()
    dz = ((6 * D + 64) * U + 2.0 ** -22) * (xd.abs() @ w.double().abs().t()) + 4 * U * (z.abs() + b.double().abs())
    lse = torch.logsumexp(z, 1, keepdim=True)
    p = torch.exp(z - lse)
    rel = dz + 8 * U * (1 + (z - lse).abs())
    de = p * (rel + (p * rel).sum(1, keepdim=True) + 40 * U)
    want = e[:, H:].t() @ xd
    close(gw[H:], want, de[:, H:].t() @ xd.abs() + (2.0 ** -22 + (6 * N + 64) * U) * (e[:, H:].t() @ xd.abs()) + 1e-36, 'gw')


# what a sum of D products in the small tiles' order is off by at most, in u of the sum of their sizes: the products of a matrix
# instruction in any order, the additions of a block of them, the blocks, and 8 for what follows
CHAINS = {'in place': lambda D: 4 + 8 + D / 32 + 8, '16 bits': lambda D: 32 + 16 + D / 512 + 8, 'three numbers': lambda D: 32 + 24 + D / 128 + 8 + 4}


@pytest.mark.parametrize('t,D,V,kind', [('bf16', 65536, 2, '16 bits'), ('f16', 65536, 2, '16 bits'), ('f32', 65536, 2, 'three numbers'),
                                        ('f32', 4096, 16384, 'in place')])
def test_long_sums_of_few_rows(t, D, V, kind):
    """64 rows whose D products are all equal, so that a chain's roundings all go one way; every other class has the logit 0"""
    from dig_amd import ops
    g = gen(113)
    N, at = 64, V - 1
    a = (1 + torch.rand(N, 1, device=DEV, generator=g)).to(TYPES[t])
    w = torch.zeros(V, D, device=DEV, dtype=TYPES[t])
    w[at] = -40 / (1.5 * D)
    rows = ops.linear_cross_entropy(a.expand(N, D).contiguous(), w, torch.full((N,), at, device=DEV), reduction='none')
    z = a[:, 0].double() * w[at, 0].double() * D
    want = torch.log((V - 1) + torch.exp(z)) - z
    close(rows, want, CHAINS[kind](D) * U * z.abs() + 16 * U * want, 'rows')


# ------------------------------------------------------------------------------------------------ saved tensors elsewhere
class _Moved(torch.autograd.graph.saved_tensors_hooks):
    """what is saved comes back elsewhere: 'offset' rows at another alignment and pitch; 'gaps' everything with a gap behind
    each element; 'turned' matrices whose columns are contiguous"""

    def __init__(self, how):
        def unpack(t):
            if how == 'gaps' and t.dim():
                return torch.stack((t, t.flip(0)), -1)[..., 0]
            if t.dim() != 2 or how == 'gaps':
                return t
            if how == 'turned':
                return t.t().contiguous().t()
            wide = torch.zeros(t.size(0), t.size(1) + 3, dtype=t.dtype, device=t.device)
            wide[:, 1:1 + t.size(1)] = t
            return wide[:, 1:1 + t.size(1)]
        super().__init__(lambda t: t.detach().clone(), unpack)


HOW = ['offset', 'gaps', 'turned']


@pytest.mark.parametrize('how', HOW)
def test_saved_norms_that_come_back_elsewhere(how):
    from dig_amd import ops
    g = gen(110)
    x, gy = randn(g, 70, 130).requires_grad_(), randn(g, 70, 130)
    w, b = (1 + 0.2 * randn(g, 130)).requires_grad_(), randn(g, 130).requires_grad_()
    want = torch.autograd.grad(ops.layer_norm(x, w, b), (x, w, b), gy)
    with _Moved(how):
        y = ops.layer_norm(x, w, b)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, (x, w, b), gy), want))


@pytest.mark.parametrize('how', HOW)
@pytest.mark.parametrize('t', list(TYPES))
@pytest.mark.parametrize('N,D,V', [(32, 128, 8192), (100, 64, 4000), (40, 64, 600), (600, 128, 900)])
def test_saved_rows_that_come_back_elsewhere(N, D, V, t, how):
    """the backward may then copy what the forward read in place, or take other kernels than it: the same bounds"""
    from dig_amd import ops
    x, w, b, target, g = classes_case(N, D, V, TYPES[t], True, 109)
    index, teacher = teacher_lists(g, N, V, 4)
    teacher = teacher.to(TYPES[t])
    one = torch.tensor(float(N) if t == 'f16' else 1.0, device=DEV)
    xd, wd, bd = x.detach(), w.detach(), b.detach()
    with _Moved(how):
        out = ops.linear_cross_entropy(x, w, target, b)
        got = dict(zip(('gx', 'gw', 'gb'), torch.autograd.grad(out, (x, w, b), one)), out=out.detach())
    z, e, rows, loss, scale, div = ref_classes(xd, wd, bd, target, 'mean', one)
    check_head(xd, wd, bd, z, e, rows, 1.0, 1.0, dict(got, div=div), scale, loss)
    with _Moved(how):
        out = ops.linear_distillation(x, w, index, teacher, b, temperature=2.0)
        got = dict(zip(('gx', 'gw', 'gb'), torch.autograd.grad(out, (x, w, b), one)), out=out.detach())
    z, e, rows, size, scale, div = ref_teacher(xd, wd, bd, index, teacher, 2.0, 'mean', one)
    check_teacher(xd, wd, bd, z, e, rows, size, 2.0, dict(got, div=div), scale, rows.sum() / div, index, teacher)


# ------------------------------------------------------------------------------------------------ deferred reductions
def test_a_norm_used_twice_joins_the_deferred_reductions():
    """one weight under two biases, one bias under two weights, one tensor as both: every use reaches the gradient.  Each use adds
    300 rows in chains of at most 300 / 64 + 128 and joins the others' in at most 64 steps; h is off as in check_norm"""
    from dig_amd import ops
    g = gen(111)
    x, z = randn(g, 300, 128), randn(g, 300, 128) * 1.5 + 0.3
    w, v, b, c, p = ((1 + 0.2 * randn(g, 128)).requires_grad_() for _ in range(5))
    none = torch.empty(0, 128, device=DEV)
    uses = [(none, w, b), (x, w, b), (z, w, c), (x, v, b), (z, p, p), (z, v, None), (none, None, c)]
    gys = [randn(g, u[0].size(0), 128) for u in uses]
    ops.backward(sum((ops.layer_norm(*u) * gy).sum() for u, gy in zip(uses, gys)), [w, v, b, c, p])
    want = {id(t): [0.0, 0.0] for t in (w, v, b, c, p)}
    for (rows, weight, bias), gy in zip(uses, gys):
        if not rows.size(0):
            continue
        q = norm64(rows, weight.detach(), None, 1e-5, gy)
        reach = 64 * U * (q['x'].abs().amax(1, keepdim=True) * q['r'] + q['h'].abs())
        n = (300 / 64 + 128 + 64) * U
        parts = [(weight, q['gw'], n * (q['gy'] * q['h']).abs().sum(0) + (q['gy'].abs() * reach).sum(0)), (bias, q['gb'], n * q['gy'].abs().sum(0))]
        for leaf, value, tol in parts:
            if leaf is not None:
                want[id(leaf)][0] = want[id(leaf)][0] + value
                want[id(leaf)][1] = want[id(leaf)][1] + tol
    for name, leaf in zip('wvbcp', (w, v, b, c, p)):
        close(leaf.grad, *want[id(leaf)], name)


# ------------------------------------------------------------------------------------------------ a model's own head
@pytest.mark.parametrize('level', ['aminoacid', 'allatom'])
def test_a_protein_model_trains_its_class_head_without_logits(level):
    """ProNet with its last layer taken out gives the rows that layer would have got; the fused loss over that layer's weight gives
    them, the weight and the bias the gradients of the formula, and the model's own backward goes on from there"""
    from dig_amd import ops
    from dig_amd.synthetic import make_protein_batch
    import dig_amd.threedgraph.method as M
    torch.manual_seed(0)
    model = M.ProNet(level=level, num_blocks=2, hidden_channels=64, mid_emb=32, out_channels=384).to(DEV)
    batch = make_protein_batch(6, 20, 40, 33, device=DEV)
    target = torch.arange(6, device=DEV) * 61
    logits = model(batch)
    head, model.lin_out = model.lin_out, torch.nn.Identity()
    h = model(batch)
    assert h.shape == (6, 64) and torch.equal(head(h), logits)
    rows = h.detach().requires_grad_()
    leaves = (rows, head.weight, head.bias)
    out = ops.linear_cross_entropy(rows, head.weight, target, head.bias)
    got = dict(zip(('gx', 'gw', 'gb'), torch.autograd.grad(out, leaves)), out=out.detach())
    x, w, b = (p.detach() for p in leaves)
    one = torch.ones((), device=DEV)
    z, e, lr, loss, scale, div = ref_classes(x, w, b, target, 'mean', one)
    check_head(x, w, b, z, e, lr, 1.0, 1.0, dict(got, div=div), scale, loss)
    params = [p for p in model.parameters()]
    end = torch.autograd.grad(ops.linear_cross_entropy(h, head.weight, target, head.bias), params, retain_graph=True)
    step = torch.autograd.grad(h, params, got['gx'])
    assert all(torch.equal(p, q) for p, q in zip(end, step)) and any(p.any() for p in end)

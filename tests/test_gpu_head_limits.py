"""GPU: the class losses where their arithmetic comes to its ends — classes masked by the type's lowest value, rows with a single class
left, rows without a number beside others, and float32 operands whose sizes lie far apart — against float64 formulas.

Tolerances as in test_gpu_head.py: sums of the roundings that are made, derived before any run.  Each case runs at a size that the
kernels of head_small.h take in place and at one that the general path takes."""
import math

import pytest
import torch

from tests.test_gpu_head import DEV, TYPES, U, check_head, check_teacher, classes_case, close, gen, half, head64, randn, ref_classes, ref_teacher

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

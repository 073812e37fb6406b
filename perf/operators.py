"""What the operators of a trained output head cost: the last normalisation of the hidden rows, the loss over the classes of
the head's product, and the same loss against a teacher's largest logits.  Each case is one pass as a training step (value and
gradients) or an evaluation makes it; the plain forms are elementary torch operations in 32 bits."""
import math

import torch

own = False

TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    ln = dict(op='norm', eps=1e-5, affine=True, grad=True, strided=False)
    ce = dict(op='classes', bias=False, ignored=0.0, reduction='mean', grad=True)
    kd = dict(op='teacher', bias=False, reduction='mean', temperature=2.0, ragged=False, grad=True)
    return [
        # atoms of 32 small molecules, the hidden width of the energy models: a launch-bound call
        dict(ln, name='norm 608x128 f32', rows=608, width=128, type='f32'),
        # 128 molecules of 128 atoms at 256 channels
        dict(ln, name='norm 16384x256 f32', rows=16384, width=256, type='f32'),
        # an odd width inside a wider buffer: rows that start anywhere
        dict(ln, name='norm 8191x1021 bf16', rows=8191, width=1021, type='bf16', strided=True),
        # a long batch of sequence positions
        dict(ln, name='norm 131072x1024 bf16', rows=131072, width=1024, type='bf16'),
        # one position in serving
        dict(ln, name='norm 1x8192 f16', rows=1, width=8192, type='f16', grad=False),
        # the class head of a protein model: 32 graphs, about a thousand classes
        dict(ce, name='classes 32x128x1195 f32', rows=32, width=128, classes=1195, type='f32', bias=True),
        # node classification over a large vocabulary at the models' own width and type
        dict(ce, name='classes 2048x256x32768 f32', rows=2048, width=256, classes=32768, type='f32'),
        # nothing a multiple of anything, one loss per row, a mask of half of the rows
        dict(ce, name='classes 1009x321x10007 f16', rows=1009, width=321, classes=10007, type='f16', bias=True, ignored=0.5,
             reduction='none'),
        # a batch of sequences over a large vocabulary, padding ignored
        dict(ce, name='classes 4096x2048x131072 bf16', rows=4096, width=2048, classes=131072, type='bf16', ignored=0.1),
        # the score of one position in evaluation: the weight is read once
        dict(ce, name='classes 1x1024x32768 bf16', rows=1, width=1024, classes=32768, type='bf16', grad=False),
        # a class head taught by a larger model's sixteen best classes
        dict(kd, name='teacher 64x128x1195 f32', rows=64, width=128, classes=1195, top=16, type='f32', bias=True),
        # positions taught by 64 logits each, some rows short or empty
        dict(kd, name='teacher 4096x1024x32000 bf16', rows=4096, width=1024, classes=32000, top=64, type='bf16', ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['norm', 'classes', 'teacher'])
    c = dict(op=op, type=rng.choice(['f32', 'bf16', 'f16']), grad=rng.random() < 0.8)
    if op == 'norm':
        c['width'] = _log(rng, 8, 8192)
        c['rows'] = _log(rng, 1, min(131072, (1 << 27) // c['width']))
        c.update(eps=rng.choice([1e-5, 1e-6]), affine=rng.random() < 0.8, strided=rng.random() < 0.3)
        return c
    c['width'] = _log(rng, 16, 2048)
    c['classes'] = _log(rng, 2 if op == 'classes' else 100, 131072)
    # at most a quarter of the largest listed product, whatever the type
    c['rows'] = _log(rng, 1, max(2, min(8192, (1 << 38) // (c['width'] * c['classes']))))
    c.update(bias=rng.random() < 0.5, reduction=rng.choice(['mean', 'sum', 'none']))
    if op == 'classes':
        c['ignored'] = rng.choice([0.0, 0.1, 0.5])
    else:
        c.update(top=min(c['classes'], _log(rng, 2, 128)), temperature=rng.choice([1.0, 2.0, 4.0]), ragged=rng.random() < 0.5)
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _normal(gen, *shape):
    return torch.randn(*shape, device='cuda', generator=gen)


def _uniform(gen, *shape):
    return torch.rand(*shape, device='cuda', generator=gen)


def prepare(case, seed):
    t = TYPES[case['type']]
    gen = torch.Generator(device='cuda').manual_seed(seed)
    R, D = case['rows'], case['width']
    s = dict(case=case)
    if case['op'] == 'norm':
        wide = D + 11 if case['strided'] else D
        x = (_normal(gen, R, wide) * (0.5 + _uniform(gen, R, 1)) + 0.3 * _normal(gen, R, 1)).to(t)
        s['x'] = x[:, 5:5 + D] if case['strided'] else x
        s['w'] = (1.0 + 0.2 * _normal(gen, D)).to(t) if case['affine'] else None
        s['b'] = (0.1 * _normal(gen, D)).to(t) if case['affine'] else None
        if case['grad']:
            s['g'] = _normal(gen, R, D).to(t)
    else:
        V = case['classes']
        w = _normal(gen, V, D) / math.sqrt(D)
        x = _normal(gen, R, D)
        if case['op'] == 'classes':
            target = torch.randint(0, V, (R,), device='cuda', generator=gen)
            # a head that has learnt something: the right class stands out by 0 to 10
            x += 10.0 * _uniform(gen, R, 1) * w[target]
            target[_uniform(gen, R) < case['ignored']] = -100
            s['target'] = target
        else:
            K = case['top']
            start = torch.randint(0, V, (R, 1), device='cuda', generator=gen)
            step = (_uniform(gen, R, 1) * (V // K)).long().clamp_(min=1)
            index = (start + step * torch.arange(K, device='cuda')) % V
            teacher = (2.0 * _normal(gen, R, K)).sort(1, descending=True).values
            x += 3.0 * _uniform(gen, R, 1) * w[index[:, 0]]
            if case['ragged']:
                # the teacher's list ends early, and for some rows at once
                n = (_uniform(gen, R, 1) * (K + 1)).long()
                gone = torch.arange(K, device='cuda') >= n
                index = index.masked_fill(gone, -1)
                teacher = teacher.masked_fill(gone, float('-inf'))
            s['index'], s['teacher'] = index, teacher.to(t)
        s['x'], s['w'] = x.to(t), w.to(t)
        s['b'] = (0.5 * _normal(gen, V)).to(t) if case['bias'] else None
        if case['grad']:
            # 16-bit floats come with the loss scale that keeps their gradients in range
            up = float(R) if case['type'] == 'f16' and case['reduction'] == 'mean' else 1.0
            s['g'] = up * (0.5 + _uniform(gen, R)) if case['reduction'] == 'none' else up * (0.5 + _uniform(gen, 1)[0])
    if case['grad']:
        for k in ('x', 'w', 'b'):
            if s[k] is not None:
                s[k] = s[k].detach().requires_grad_()
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    c = s['case']
    if own:
        from dig_amd import ops
        if c['op'] == 'norm':
            out = ops.layer_norm(s['x'], s['w'], s['b'], eps=c['eps'])
        elif c['op'] == 'classes':
            out = ops.linear_cross_entropy(s['x'], s['w'], s['target'], s['b'], reduction=c['reduction'])
        else:
            out = ops.linear_distillation(s['x'], s['w'], s['index'], s['teacher'], s['b'], temperature=c['temperature'],
                                          reduction=c['reduction'])
        res = {'out': out.detach()}
        if c['grad']:
            leaves = [k for k in ('x', 'w', 'b') if s[k] is not None]
            res.update(zip(['g' + k for k in leaves], torch.autograd.grad(out, [s[k] for k in leaves], s['g'])))
        return res
    with torch.no_grad():
        return {'norm': _plain_norm, 'classes': _plain_classes, 'teacher': _plain_teacher}[c['op']](s, c)


def _plain_norm(s, c):
    x, t = s['x'].float(), s['x'].dtype
    d = x - x.mean(1, keepdim=True)
    r = torch.rsqrt((d * d).mean(1, keepdim=True) + c['eps'])
    h = d * r
    y = h * s['w'].float() + s['b'].float() if c['affine'] else h
    res = {'out': y.to(t)}
    if c['grad']:
        g = s['g'].float()
        gh = g * s['w'].float() if c['affine'] else g
        gx = r * (gh - gh.mean(1, keepdim=True) - h * (gh * h).mean(1, keepdim=True))
        res['gx'] = gx.to(t)
        if c['affine']:
            res['gw'], res['gb'] = (g * h).sum(0).to(t), g.sum(0).to(t)
    return res


def _plain_logits(s):
    z = s['x'].float() @ s['w'].float().t()
    return z if s['b'] is None else z.add_(s['b'].float())


def _plain_finish(s, c, loss, live, e, scale):
    """The reduction of the rows' losses, and the gradients of x, w and b from e = d loss_n / d logits_n / scale."""
    t, n = s['x'].dtype, live.sum().clamp(min=1).float()
    res = {'out': loss if c['reduction'] == 'none' else loss.sum() / n if c['reduction'] == 'mean' else loss.sum()}
    if c['grad']:
        g = s['g'].float() * live.float() * scale
        e *= (g / n if c['reduction'] == 'mean' else g).unsqueeze(1)
        res['gx'] = (e @ s['w'].float()).to(t)
        res['gw'] = (e.t() @ s['x'].float()).to(t)
        if s['b'] is not None:
            res['gb'] = e.sum(0).to(t)
    return res


def _plain_classes(s, c):
    z = _plain_logits(s)
    live = s['target'] != -100
    at = s['target'].clamp(min=0).unsqueeze(1)
    m = z.amax(1, keepdim=True)
    zt = z.gather(1, at) - m
    e = z.sub_(m).exp_()
    # the other classes apart: where the right one has nearly all, its loss and its gradient are what the others have
    e.scatter_(1, at, 0.0)
    others = e.sum(1, keepdim=True)
    loss = torch.where(zt < 0, (others + zt.exp()).log() - zt, torch.log1p(others)).squeeze(1) * live
    if c['grad']:
        total = others + zt.exp()
        e /= total
        e.scatter_(1, at, -others / total)
    return _plain_finish(s, c, loss, live, e, 1.0)


def _plain_teacher(s, c):
    tau = c['temperature']
    z = _plain_logits(s) / tau
    there = (s['index'] >= 0) & (s['teacher'] != float('-inf'))
    live = there.any(1)
    at = s['index'].clamp(min=0)
    a = (s['teacher'].float() / tau).masked_fill(~there, float('-inf'))
    top = a.amax(1, keepdim=True).masked_fill(~live.unsqueeze(1), 0.0)
    q = (a - top).exp()
    sum_q = q.sum(1, keepdim=True).masked_fill(~live.unsqueeze(1), 1.0)
    q /= sum_q
    log_q = (a - top - sum_q.log()).masked_fill(~there, 0.0)
    m = z.amax(1, keepdim=True)
    zt = z.gather(1, at)
    e = z.sub_(m).exp_()
    total = e.sum(1, keepdim=True)
    log_p = zt - m - total.log()
    loss = tau * tau * (q * (log_q - log_p)).sum(1)
    if c['grad']:
        e /= total
        e.scatter_add_(1, at, -q)
    return _plain_finish(s, c, loss, live, e, tau)


# ------------------------------------------------------------------------------------------------ what it cannot do without
def work(case):
    R, D, size = case['rows'], case['width'], 4 if case['type'] == 'f32' else 2
    if case['op'] == 'norm':
        par = 2 * D if case['affine'] else 0
        n = (4 * R * D + 2 * par if case['grad'] else 2 * R * D + par) * size
        return {'bytes': n, 'flops': (18 if case['grad'] else 8) * R * D}
    V = case['classes']
    read = (R * D + V * D + (V if case['bias'] else 0)) * size
    n = 2 * read if case['grad'] else read
    n += R * 8 if case['op'] == 'classes' else R * case['top'] * (8 + size)
    n += 4 * R if case['reduction'] == 'none' else 4
    return {'bytes': n, 'flops': (6 if case['grad'] else 2) * R * V * D}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    p = {k: s[k].detach().double().requires_grad_(case['grad']) for k in ('x', 'w', 'b') if s[k] is not None}
    if case['op'] == 'norm':
        x = p['x']
        mean = x.sum(1, keepdim=True) / case['width']
        var = (x * x).sum(1, keepdim=True) / case['width'] - mean ** 2
        out = (x - mean) / torch.sqrt(var + case['eps'])
        if case['affine']:
            out = torch.addcmul(p['b'], out, p['w'])
    else:
        z = torch.matmul(p['x'], p['w'].t())
        if 'b' in p:
            z = z + p['b']
        if case['op'] == 'classes':
            keep = (s['target'] >= 0).nonzero().squeeze(1)
            rows = torch.logsumexp(z[keep], 1) - z[keep, s['target'][keep]]
        else:
            tau = case['temperature']
            keep = ((s['index'] >= 0) & (s['teacher'].double() > float('-inf'))).any(1).nonzero().squeeze(1)
            index, teacher = s['index'][keep], s['teacher'][keep].double()
            q = torch.softmax(torch.where(index < 0, float('-inf'), teacher / tau), 1)
            log_p = torch.log_softmax(z[keep] / tau, 1).gather(1, index.clamp(min=0))
            rows = tau ** 2 * (torch.special.xlogy(q, q) - q * log_p).sum(1)
        out = torch.zeros(case['rows'], dtype=torch.float64, device='cuda').index_add(0, keep, rows)
        if case['reduction'] != 'none':
            out = out.sum() / (max(1, keep.numel()) if case['reduction'] == 'mean' else 1)
    res = {'out': out.detach()}
    if case['grad']:
        res.update(zip(['g' + k for k in p], torch.autograd.grad(out, list(p.values()), s['g'].double())))
    return res

"""Losses over the classes of a linear output head, the logits never kept (csrc/head.hip): cross entropy against labels and
distillation from a teacher's largest logits.  Reached as ``dig_amd.ops.linear_cross_entropy`` / ``linear_distillation``; the heads
they train are ``nn.Linear``-shaped (``ProNet.lin_out``, method/pronet/pronet.py:349-352)."""
import torch
from torch.autograd import Function

from . import _hip, ops
from ._hip import call, ptr
from .graph import _stream

_REDUCTIONS = ('none', 'mean', 'sum')


def _pitch(t):
    return t.stride(0) if t.size(0) > 1 else t.size(1)


def _workspace(x, w, V, backward, needs):
    N, D = x.shape
    kib = _hip.query('dig3d_head_ws_kib', ops._DTYPES[x.dtype], _pitch(x), ptr(x), _pitch(w), ptr(w), N, D, V, backward, needs)
    if kib < 0:
        raise _hip.Dig3dError(f'class head of {N} rows x {D} x {V} classes is beyond the supported sizes')
    return torch.empty(max(kib, 1) * 1024, dtype=torch.uint8, device=x.device), kib


class _HeadLoss(Function):
    """loss of the classes of x w^T + bias; ``teacher``: (index, logits) instead of targets."""

    @staticmethod
    def forward(ctx, x, w, bias, target, index, teacher, tau, ignore_index, reduction):
        (N, D), V, dev = x.shape, w.size(0), x.device
        ctx.meta = (tau, ignore_index, reduction)
        f32 = dict(dtype=torch.float32, device=dev)
        dt = ops._DTYPES[x.dtype]
        if N == 0:
            ctx.save_for_backward(x, w, bias)
            return torch.zeros(N, **f32) if reduction == 'none' else torch.zeros((), **f32)
        scal = torch.empty(516, **f32)
        rows = torch.empty(3, N, **f32)                     # lse, loss, live
        lse, loss, live = rows[0], rows[1], rows[2]
        with torch.cuda.device(dev):
            st = _stream()
            ws, kib = _workspace(x, w, V, 0, 0)
            call('dig3d_head_lse', dt, ptr(x), _pitch(x), ptr(w), _pitch(w), ptr(bias), ptr(target), ignore_index, tau, N, D, V,
                 ptr(scal), ptr(lse), ptr(loss) if target is not None else None, ptr(ws), kib, st)
            q = None
            if index is not None:
                K = index.size(1)
                q = torch.empty(2, N, K, **f32)
                call('dig3d_head_teacher', dt, ptr(x), _pitch(x), ptr(w), _pitch(w), ptr(bias), ptr(index), ptr(teacher),
                     ops._DTYPES[teacher.dtype], K, tau, N, D, V, ptr(lse), ptr(q), q.data_ptr() + 4 * N * K, ptr(loss), ptr(live), st)
            count = out = None
            if reduction != 'none':
                out, count = torch.empty((), **f32), torch.empty((), **f32)
                call('dig3d_head_total', ptr(loss), ptr(target), ignore_index, ptr(live) if index is not None else None, N,
                     int(reduction == 'mean'), ptr(out), ptr(count), st)
        ctx.save_for_backward(x, w, bias, target, index, q, scal, rows, count)
        return loss.clone() if reduction == 'none' else out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        tau, ignore_index, reduction = ctx.meta
        none = (None,) * 6
        needs = ctx.needs_input_grad[:3]
        if len(ctx.saved_tensors) == 3:
            return tuple(torch.zeros_like(t) if n else None for t, n in zip(ctx.saved_tensors, needs)) + none
        x, w, bias, target, index, q, scal, rows, count = ctx.saved_tensors
        (N, D), V = x.shape, w.size(0)
        new = lambda n, *shape: torch.empty(*shape, dtype=x.dtype, device=x.device) if n else None
        gx, gw, gb = new(needs[0], N, D), new(needs[1], V, D), new(needs[2], V)
        g = g.to(torch.float32).contiguous()
        K = index.size(1) if index is not None else 0
        with torch.cuda.device(x.device):
            ws, kib = _workspace(x, w, V, 1, needs[0] + 2 * needs[1] + 4 * needs[2])
            call('dig3d_head_bwd', ops._DTYPES[x.dtype], ptr(x), _pitch(x), ptr(w), _pitch(w), ptr(bias), ptr(target), ignore_index, ptr(index),
                 ptr(q), q.data_ptr() + 4 * N * K if K else None, rows.data_ptr() + 8 * N if K else None, K, tau, N, D, V, ptr(g),
                 int(reduction == 'none'), ptr(count) if reduction == 'mean' else None, ptr(scal), ptr(rows), rows.data_ptr() + 4 * N,
                 ptr(gx), ptr(gw), ptr(gb), ptr(ws), kib, _stream())
        return (gx, gw, gb) + none


def _check_head(name, x, weight, bias, reduction):
    if reduction not in _REDUCTIONS:
        raise ValueError(f"{name}: reduction is one of {_REDUCTIONS}, got {reduction!r}")
    x2, _ = ops._check_rows(name, x)
    if not weight.is_cuda or weight.device != x2.device:
        raise _hip.Dig3dError(f'{name}: weight is on {weight.device}, the rows on {x2.device}')
    if weight.dim() != 2 or weight.size(1) != x2.size(1) or weight.size(0) < 1 or weight.dtype != x2.dtype:
        raise RuntimeError(f'{name}: expected weight [V, {x2.size(1)}] of {x2.dtype} with V >= 1, got {tuple(weight.shape)} {weight.dtype}')
    weight, _ = ops._check_rows(name, weight)
    if bias is not None:
        bias = ops._check_vector(name, 'bias', bias, weight.size(0), x2, (x2.dtype,))
    return x2, weight, bias


def _check_index(name, what, t, shape, x):
    if not t.is_cuda or t.device != x.device:
        raise _hip.Dig3dError(f'{name}: {what} is on {t.device}, the rows on {x.device}')
    if t.dtype != torch.int64 or tuple(t.shape) != tuple(shape):
        raise RuntimeError(f'{name}: expected {what} {list(shape)} of torch.int64, got {tuple(t.shape)} {t.dtype}')


def linear_cross_entropy(x, weight, target, bias=None, ignore_index=-100, reduction='mean'):
    """Softmax cross entropy of the classes ``x @ weight.T + bias`` (x [..., D], weight [V, D], bias [V] or None, all float32,
    bfloat16 or float16) against ``target`` [...] (int64), without keeping the logits: the forward reduces them tile by tile, the
    backward forms them again in pieces of the vocabulary.

    -> float32: the mean over the rows whose target is not ``ignore_index`` (0 if there are none), their sum, or with
    ``reduction='none'`` one loss per row (0 for an ignored one).  Ignored rows take no part in any gradient, whatever they
    hold.  A target outside [0, V) gives NaN, in the loss and the gradients.  Differentiable once, in x, weight and bias; the
    gradients have the type of their inputs and the same bits every time."""
    x2, weight, bias = _check_head('linear_cross_entropy', x, weight, bias, reduction)
    _check_index('linear_cross_entropy', 'target', target, x.shape[:-1], x2)
    loss = _HeadLoss.apply(x2, weight, bias, target.reshape(-1).contiguous(), None, None, 1.0, int(ignore_index), reduction)
    return loss.reshape(target.shape) if reduction == 'none' else loss


def linear_distillation(x, weight, teacher_index, teacher_logits, bias=None, temperature=1.0, reduction='mean'):
    """Distillation of the head ``x @ weight.T + bias`` from a teacher's K largest logits: per row
    ``temperature**2 * KL(q || p)`` with q the softmax of ``teacher_logits`` [..., K] / temperature over the listed classes
    ``teacher_index`` [..., K] (int64) and p the head's softmax over ALL classes at the same temperature, the head's logits never
    kept.

    An entry with a negative index or the logit -inf is absent, whatever else it holds; a row without entries has the loss 0, no
    gradient, and is not counted by the mean.  Equal indices of a row add up.  An index >= V gives NaN.  The teacher takes no
    gradient.  Types, reductions and gradients as ``linear_cross_entropy``; teacher_logits float32, bfloat16 or float16."""
    name = 'linear_distillation'
    x2, weight, bias = _check_head(name, x, weight, bias, reduction)
    if not (isinstance(temperature, (int, float)) and 0.0 < float(temperature) < float('inf')):
        raise ValueError(f'{name}: temperature is a positive number, got {temperature!r}')
    if teacher_index.dim() != x.dim() or teacher_index.size(-1) < 1:
        raise RuntimeError(f'{name}: expected teacher_index [..., K] with K >= 1 for rows {tuple(x.shape)}, got {tuple(teacher_index.shape)}')
    K = teacher_index.size(-1)
    _check_index(name, 'teacher_index', teacher_index, tuple(x.shape[:-1]) + (K,), x2)
    if teacher_logits.shape != teacher_index.shape or teacher_logits.dtype not in ops._DTYPES or teacher_logits.device != x2.device:
        raise RuntimeError(f'{name}: expected teacher_logits {list(teacher_index.shape)} of float32, bfloat16 or float16 on {x2.device}, got '
                           f'{tuple(teacher_logits.shape)} {teacher_logits.dtype} on {teacher_logits.device}')
    index = teacher_index.reshape(-1, K).contiguous()
    teacher = teacher_logits.detach().reshape(-1, K).contiguous()
    loss = _HeadLoss.apply(x2, weight, bias, None, index, teacher, float(temperature), 0, reduction)
    return loss.reshape(x.shape[:-1]) if reduction == 'none' else loss

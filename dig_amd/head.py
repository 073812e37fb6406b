"""Losses over the classes of a linear output head, the logits never kept (csrc/head.hip): cross entropy against labels and
distillation from a teacher's largest logits.  Reached as ``dig_amd.ops.linear_cross_entropy`` / ``linear_distillation``; the heads
they train are ``nn.Linear``-shaped (``ProNet.lin_out``, method/pronet/pronet.py:349-352)."""
import torch
from torch.autograd import Function

from . import _hip, ops
from ._hip import ptr

_REDUCTIONS = {'none': 0, 'mean': 1, 'sum': 2}
_TOP_MAX = 2048                                    # entries of a teacher's row (csrc/head.hip: TC_MAX)


def _call(name, dev, backward, needs, x, w, bias, target, index, teacher, keep, tau, ignore_index, reduction, *last):
    """one C entry on these operands and a fresh workspace; ``last``: its arguments between ``keep`` and the workspace"""
    (N, D), V, dt = x.shape, w.size(0), ops._DTYPES[x.dtype]
    operands = (dt, x.data_ptr(), ops._pitch(x), w.data_ptr(), ops._pitch(w))
    kib = _hip.query('dig3d_head_ws_kib', *operands, N, D, V, backward, needs)
    if kib < 0:
        raise _hip.Dig3dError(f'class head of {N} rows x {D} x {V} classes is beyond the supported sizes (2^24 rows, 2^20 channels, 2^28 classes)')
    ws = torch.empty(max(kib, 1) * 1024, dtype=torch.uint8, device=x.device)
    K, tdt = (0, 0) if index is None else (index.size(1), ops._DTYPES[teacher.dtype])
    ops._on_device(dev, name, *operands, ptr(bias), ptr(target), ignore_index, ptr(index), ptr(teacher), tdt, K, tau, N, D, V, reduction,
                   keep.data_ptr(), *last, ws.data_ptr(), kib)


class _HeadLoss(Function):
    """The loss of the classes of x w^T + bias against targets, or against a teacher's entries (index, teacher)."""

    @staticmethod
    def forward(ctx, x, w, bias, target, index, teacher, tau, ignore_index, reduction):
        N, D = x.shape
        f32 = dict(dtype=torch.float32, device=x.device)
        out = torch.empty(N, **f32) if reduction == 0 else torch.empty((), **f32)
        if N == 0:
            ctx.meta = None
            ctx.save_for_backward(x, w, bias)
            return out.zero_()
        keep = torch.empty(8 + N * (4 + 2 * (0 if index is None else index.size(1))), **f32)
        _call('dig3d_head_fwd', x.get_device(), 0, 0, x, w, bias, target, index, teacher, keep, tau, ignore_index, reduction, out.data_ptr())
        ctx.meta = (tau, ignore_index, reduction)
        ctx.save_for_backward(x, w, bias, target, index, teacher, keep)
        return out

    @staticmethod
    @ops._once
    def backward(ctx, g):
        needs = ctx.needs_input_grad[:3]
        saved = ctx.saved_tensors
        x, w, bias = saved[:3]
        if ctx.meta is None:
            return tuple(torch.zeros_like(t) if n else None for t, n in zip((x, w, bias), needs)) + (None,) * 6
        saved = [ops._same_rows(x), ops._same_rows(w)] + [t if t is None else t.contiguous() for t in saved[2:]]
        gx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if needs[0] else None
        gw = torch.empty(w.shape, dtype=x.dtype, device=x.device) if needs[1] else None
        gb = torch.empty(bias.shape, dtype=x.dtype, device=x.device) if needs[2] else None
        if g.dtype != torch.float32 or not g.is_contiguous():
            g = g.to(torch.float32).contiguous()
        _call('dig3d_head_bwd', x.get_device(), 1, needs[0] + 2 * needs[1] + 4 * needs[2], *saved, *ctx.meta, g.data_ptr(), ptr(gx), ptr(gw),
              ptr(gb))
        return gx, gw, gb, None, None, None, None, None, None


def _check_head(name, x, weight, bias, reduction):
    if reduction not in _REDUCTIONS:
        raise ValueError(f'{name}: reduction is one of {tuple(_REDUCTIONS)}, got {reduction!r}')
    x2 = ops._check_rows(name, x)
    if weight.get_device() != x2.get_device():
        raise _hip.Dig3dError(f'{name}: weight is on {weight.device}, the rows on {x2.device}')
    if weight.dim() != 2 or weight.size(1) != x2.size(1) or weight.size(0) < 1 or weight.dtype != x2.dtype:
        raise RuntimeError(f'{name}: expected weight [V, {x2.size(1)}] of {x2.dtype} with V >= 1, got {tuple(weight.shape)} {weight.dtype}')
    weight = ops._check_rows(name, weight)
    if bias is not None:
        bias = ops._check_vector(name, 'bias', bias, weight.size(0), x2, (x2.dtype,))
    return x2, weight, bias


def _check_index(name, what, t, shape, x):
    if t.get_device() != x.get_device():
        raise _hip.Dig3dError(f'{name}: {what} is on {t.device}, the rows on {x.device}')
    if t.dtype != torch.int64 or tuple(t.shape) != tuple(shape):
        raise RuntimeError(f'{name}: expected {what} {list(shape)} of torch.int64, got {tuple(t.shape)} {t.dtype}')


def linear_cross_entropy(x, weight, target, bias=None, ignore_index=-100, reduction='mean'):
    """Softmax cross entropy of the classes ``x @ weight.T + bias`` (x [..., D], weight [V, D], bias [V] or None, all float32,
    bfloat16 or float16) against ``target`` [...] (int64), without keeping the logits: the forward reduces them tile by tile, the
    backward forms them again in pieces of the vocabulary.

    -> float32: the mean over the rows whose target is not ``ignore_index`` (0 if there are none), their sum, or with
    ``reduction='none'`` one loss per row (0 for an ignored one).  Ignored rows take no part in any gradient, whatever they
    hold.  A target outside [0, V) gives NaN, in the loss and the gradients, and so does a row without a finite logit or with an
    infinite one; such a row counts once in the mean.  A bias of -inf or of the type's lowest value takes its class out.
    Differentiable once, in x, weight and bias; the gradients have the type of their inputs and the same bits every time.

    Precision: sums, statistics and losses in float32.  float32 rows and weights enter with all 24 bits (products to 2^-23 of a
    term) at every size.  In 16 bits the gradient of the logits is float32 or two numbers of the type where the products are
    small (up to 128 rows, or N D V up to 2^31), and beyond is rounded once to the type, half a step of each entry (the
    gradients are then off by 1.1 to 1.4 times what their own rounding costs); in float16 an entry below 2^-29 of the
    largest incoming gradient of a row keeps fewer bits."""
    x2, weight, bias = _check_head('linear_cross_entropy', x, weight, bias, reduction)
    _check_index('linear_cross_entropy', 'target', target, x.shape[:-1], x2)
    if not -1 << 63 <= int(ignore_index) < 1 << 63:
        raise ValueError(f'linear_cross_entropy: ignore_index is an int64, got {ignore_index}')
    loss = _HeadLoss.apply(x2, weight, bias, target.reshape(-1).contiguous(), None, None, 1.0, int(ignore_index), _REDUCTIONS[reduction])
    return loss if reduction != 'none' or x.dim() == 2 else loss.reshape(target.shape)


def linear_distillation(x, weight, teacher_index, teacher_logits, bias=None, temperature=1.0, reduction='mean'):
    """Distillation of the head ``x @ weight.T + bias`` from a teacher's K largest logits: per row
    ``temperature**2 * KL(q || p)`` (temperature from 1e-6 to 1e6) with q the softmax of ``teacher_logits`` [..., K] /
    temperature over the listed classes ``teacher_index`` [..., K] (int64) and p the head's softmax over ALL classes at the same
    temperature, the head's logits never kept.

    An entry with a negative index or the logit -inf is absent, whatever else it holds; a row without entries has the loss 0, no
    gradient, and is not counted by the mean.  Equal indices of a row add up.  An index >= V or a NaN among the listed logits gives
    NaN; such a row counts once in the mean.  The teacher takes no gradient.  K is at most 2048.  Types, reductions, gradients
    and precision as ``linear_cross_entropy``; teacher_logits float32, bfloat16 or float16."""
    name = 'linear_distillation'
    x2, weight, bias = _check_head(name, x, weight, bias, reduction)
    if not (isinstance(temperature, (int, float)) and 1e-6 <= float(temperature) <= 1e6):
        raise ValueError(f'{name}: temperature is a number from 1e-6 to 1e6, got {temperature!r}')
    if teacher_index.dim() != x.dim() or not 1 <= teacher_index.size(-1) <= _TOP_MAX:
        raise RuntimeError(f'{name}: expected teacher_index [..., K] with 1 <= K <= {_TOP_MAX} for rows {tuple(x.shape)}, got {tuple(teacher_index.shape)}')
    K = teacher_index.size(-1)
    if x2.size(0) * K > 1 << 31:
        raise RuntimeError(f'{name}: {x2.size(0)} rows of {K} entries are beyond 2^31 entries in one call')
    _check_index(name, 'teacher_index', teacher_index, tuple(x.shape[:-1]) + (K,), x2)
    if teacher_logits.shape != teacher_index.shape or teacher_logits.dtype not in ops._DTYPES or teacher_logits.get_device() != x2.get_device():
        raise RuntimeError(f'{name}: expected teacher_logits {list(teacher_index.shape)} of float32, bfloat16 or float16 on {x2.device}, got '
                           f'{tuple(teacher_logits.shape)} {teacher_logits.dtype} on {teacher_logits.device}')
    index = teacher_index.reshape(-1, K).contiguous()
    teacher = teacher_logits.detach().reshape(-1, K).contiguous()
    loss = _HeadLoss.apply(x2, weight, bias, None, index, teacher, float(temperature), 0, _REDUCTIONS[reduction])
    return loss if reduction != 'none' or x.dim() == 2 else loss.reshape(x.shape[:-1])

"""Dense-head operators on MI355X: the layer that makes logits, what the logits say, and learning from a teacher's.

The heads of the scene-graph model are Linear (+ ReLU) stacks that end in a log-softmax
(SGH/model/pointnets/network_PointNet.py:188-271) on torch's library products; these three operators are the general form of
such a head on hand-written kernels (csrc/linear_act.hip, csrc/label_probs.hip), for fp32, bf16 and fp16:

* ``linear_act``      act(x W^T + b) + residual in one kernel, with gradients for x, W, b and the residual;
* ``label_log_probs`` log probability of given labels, entropy of every row and its best alternatives, with gradients;
* ``distill_top_k``   divergence of a teacher's top logits (``label_log_probs(..., top=k)`` makes them) from the student's
                      softmax, with its gradient.

Leading axes are free; tensors must be on the GPU (RuntimeError otherwise), work runs on the current stream of their device, and
nothing is synchronised or kept between calls.  Each operator is differentiable once.
"""
import collections

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from pointnet2_ops import _ext

ACTIVATIONS = tuple(_ext.ACTIVATIONS)

LabelLogProbs = collections.namedtuple("LabelLogProbs", "log_prob entropy top_log_prob top_index")


def _once(backward):
    """once_differentiable, without its price where no graph of the backward pass is being built."""
    guarded = once_differentiable(backward)

    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


def _matrix(t, name):
    """(..., C) -> (rows, C) with a contiguous last axis; a copy only where the strides allow no view."""
    if not isinstance(t, torch.Tensor) or t.dim() < 1:
        _ext._fail(f"{name} must be a tensor with at least one axis")
    if t.dim() != 2:
        t = t.reshape(-1, t.size(-1)) if t.size(-1) else t.reshape(t.shape[:-1].numel(), 0)
    return t if t.size(1) == 1 or t.stride(1) == 1 else t.contiguous()


class _LinearAct(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        need_dx, need_dw, need_db = ctx.needs_input_grad[:3]
        y, slope = _ext.linear_act(x, weight, bias, activation, residual, want_slope=need_dx or need_dw or need_db)
        ctx.save_for_backward(x if need_dw else None, weight if need_dx else None, slope)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        need_dx, need_dw, need_db, need_dr, _ = ctx.needs_input_grad
        dx = dw = db = None
        if need_dx or need_dw or need_db:
            x, weight, slope = ctx.saved_tensors
            dx, dw, db = _ext.linear_act_grad(_matrix(dy, "dy"), slope, x, weight, need_dx, need_dw,
                                              ctx.bias_dtype if need_db else None)
        return dx, dw, db, dy if need_dr else None, None


def linear_act(x, weight, bias=None, activation="none", residual=None):
    """act(x weight^T + bias) + residual.

    x (..., K); weight (N, K) of x's type; bias (N) of x's type or fp32; residual of x's type, broadcast to (..., N);
    activation one of ``ACTIVATIONS``: none, relu, gelu (erf), gelu_tanh, silu.  -> (..., N) of x's type.
    Products accumulate in fp32; bias, activation and residual are applied to the accumulator and the result is rounded once.
    The backward pass keeps the activation's slope (one tensor like y); all its sums run in a fixed order."""
    xm, wm = _matrix(x, "x"), _matrix(weight, "weight")
    if weight.dim() != 2:
        _ext._fail("weight must have shape (N, K)")
    shape = x.shape[:-1] + weight.shape[:1]
    rm = None
    if residual is not None:
        try:
            rm = _matrix(residual.expand(shape), "residual")
        except RuntimeError:
            _ext._fail(f"residual must broadcast to {tuple(shape)}")
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad) or
                                    (residual is not None and residual.requires_grad)):
        y = _LinearAct.apply(xm, wm, bias, rm, activation)
    else:
        y, _ = _ext.linear_act(xm, wm, bias, activation, rm)
    return y if x.dim() == 2 else y.view(shape)


class _LabelLogProbs(Function):
    @staticmethod
    def forward(ctx, logits, labels, top, ignore_index):
        lp, ent, tlp, tix, stats = _ext.label_logprobs(logits, labels, top, ignore_index, want_stats=True)
        ctx.save_for_backward(logits, labels, stats, ent)
        ctx.ignore_index = ignore_index
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(tlp, tix)
        return lp, ent, tlp, tix

    @staticmethod
    @_once
    def backward(ctx, g_lp, g_ent, _tlp, _tix):
        if g_lp is None and g_ent is None:
            return None, None, None, None
        logits, labels, stats, ent = ctx.saved_tensors
        g_lp, g_ent = (None if g is None else g.contiguous() for g in (g_lp, g_ent))
        return _ext.label_logprobs_grad(logits, labels, stats, ent, g_lp, g_ent, ctx.ignore_index), None, None, None


def label_log_probs(logits, labels, top=0, ignore_index=-100):
    """Log probability of the given labels, entropy and best alternatives of rows of logits (or of log probabilities).

    logits (..., V); labels (...) int64.  -> LabelLogProbs, everything fp32 but the indices:
      log_prob (...): log softmax(logits)[label]; 0 where label == ignore_index, NaN where the label lies outside [0, V);
      entropy (...): of the row's softmax, in nats;
      top_log_prob, top_index (..., top): the `top` <= min(V, 64) best entries, best first, equal logits by ascending index
      (None, None for top = 0).  A masked entry (-inf) has probability 0 and is no alternative: unused slots hold -inf and -1.
    A row of nothing but -inf has log_prob -inf, entropy 0, no alternatives and gradient 0; a row with NaN or +inf is NaN.
    log_prob and entropy are differentiable in the logits, the alternatives are not."""
    lm = _matrix(logits, "logits")
    shape = logits.shape[:-1]
    if not isinstance(labels, torch.Tensor) or labels.shape != shape:
        _ext._fail(f"labels must be a tensor of shape {tuple(shape)}")
    ym = labels.reshape(-1)
    if not ym.is_contiguous():
        ym = ym.contiguous()
    if logits.requires_grad and torch.is_grad_enabled():
        lp, ent, tlp, tix = _LabelLogProbs.apply(lm, ym, int(top), int(ignore_index))
    else:
        lp, ent, tlp, tix, _ = _ext.label_logprobs(lm, ym, top, ignore_index)
    if logits.dim() != 2:
        lp, ent = lp.view(shape), ent.view(shape)
        if tlp is not None:
            tlp, tix = tlp.view(shape + (-1,)), tix.view(shape + (-1,))
    return LabelLogProbs(lp, ent, tlp, tix)


class _DistillTopK(Function):
    @staticmethod
    def forward(ctx, logits, index, values, temperature):
        loss, stats = _ext.distill_topk(logits, index, values, temperature, want_stats=True)
        ctx.save_for_backward(logits, index, values, stats)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @_once
    def backward(ctx, g):
        logits, index, values, stats = ctx.saved_tensors
        return _ext.distill_topk_grad(logits, index, values, ctx.temperature, stats, g.contiguous()), None, None, None


def distill_top_k(logits, teacher_index, teacher_logits, temperature=1.0):
    """Row losses temperature^2 KL(q || p) of a student against the k best logits of a teacher.

    logits (..., V) of the student; teacher_index (..., k) int64, teacher_logits (..., k) (logits or log probabilities: only their
    differences count).  q = softmax(teacher_logits / temperature) over the row's k entries, p = softmax(logits / temperature) over
    all V.  -> (...) fp32, differentiable in the logits; the teacher is a constant (RuntimeError if it requires a gradient).
    A slot with a negative index or the value -inf is unused; a row without a used slot has loss 0 and gradient 0 (so padded rows
    take teacher_index = -1).  An index >= V makes its row NaN; an index may occur more than once."""
    lm = _matrix(logits, "logits")
    shape = logits.shape[:-1]
    for t, name in ((teacher_index, "teacher_index"), (teacher_logits, "teacher_logits")):
        if not isinstance(t, torch.Tensor) or t.dim() != logits.dim() or t.shape[:-1] != shape:
            _ext._fail(f"{name} must be a tensor of shape {tuple(shape) + ('k',)}")
    if teacher_logits.requires_grad:
        _ext._fail("teacher_logits must not require a gradient (detach the teacher)")
    im, vm = (t.reshape(-1, t.size(-1)) if t.dim() != 2 and t.size(-1) else t for t in (teacher_index, teacher_logits))
    im, vm = im.contiguous(), vm.contiguous()
    if logits.requires_grad and torch.is_grad_enabled():
        loss = _DistillTopK.apply(lm, im, vm, float(temperature))
    else:
        loss, _ = _ext.distill_topk(lm, im, vm, temperature)
    return loss if logits.dim() == 2 else loss.view(shape)

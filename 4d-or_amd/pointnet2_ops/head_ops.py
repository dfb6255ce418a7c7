"""Dense-head operators on MI355X: the layer that makes logits, what the logits say, and learning from a teacher's.

The heads of the scene-graph model are Linear (+ ReLU) stacks that end in a log-softmax
(SGH/model/pointnets/network_PointNet.py:188-271) on torch's library products; these three operators are the general form of
such a head on hand-written kernels (csrc/linear_act.hip, csrc/label_probs.hip), for fp32, bf16 and fp16:

* ``linear_act``      act(x W^T + b) + residual in one kernel, with gradients for x, W, b and the residual;
* ``label_log_probs`` log probability of given labels, entropy of every row and its best alternatives, with gradients;
* ``distill_top_k``   divergence of a teacher's top logits (``label_log_probs(..., top=k)`` makes them) from the student's
                      softmax, with its gradient.

Leading axes are free; tensors must be on the GPU (RuntimeError otherwise), work runs on the current stream of their device, and
nothing is synchronised or kept between calls.  Each operator is differentiable once, in reverse mode.  The kernels run outside
torch's dispatcher: dual tensors of forward mode, recording by ``torch.jit.trace`` / ``make_fx`` / export, subclasses with
``__torch_dispatch__`` and tensors without memory of their own are refused (RuntimeError).  So is a backward pass that is captured into
a graph while an eager graph of the same leaves lives on another stream (torch would break the capture): drop that graph first, or
capture with leaves of its own.
"""
import collections
import os

import torch

from pointnet2_ops import _ext

try:
    from pointnet2_ops import _heads
except ImportError as e:
    raise ImportError(f"pointnet2_ops._heads: {e}. Build it with `make -C {os.path.join(_ext._PKG_DIR, 'csrc')}` (or "
                      "__graft_entry__.build()); there is no CPU/PyTorch fallback.") from e

ACTIVATIONS = tuple(_ext.ACTIVATIONS)

LabelLogProbs = collections.namedtuple("LabelLogProbs", "log_prob entropy top_log_prob top_index")

# arguments, allocation and autograd nodes: csrc/head_binding.cpp, around the entry points of the library that _ext has loaded
_heads.bind(_ext.address, _ext._call)


def _timed():
    return _ext.TIMER is not None and _ext.TIMER.enabled


def _tensors(**named):
    """The reason of a refused call whose arguments are no tensors."""
    for name, t in named.items():
        if not isinstance(t, torch.Tensor):
            _ext._fail(f"{name} must be a torch.Tensor")


def linear_act(x, weight, bias=None, activation="none", residual=None):
    """act(x weight^T + bias) + residual.

    x (..., K); weight (N, K) of x's type; bias (N) of x's type or fp32; residual of x's type, broadcast to (..., N);
    activation one of ``ACTIVATIONS``: none, relu, gelu (erf), gelu_tanh, silu.  -> (..., N) of x's type.
    Products accumulate in fp32; bias, activation and residual are applied to the accumulator and the result is rounded once.
    The backward pass keeps the activation's slope (one tensor like y); all its sums run in a fixed order."""
    act = _ext.ACTIVATIONS.get(activation) if isinstance(activation, str) else None
    if act is None:
        _ext._fail(f"activation must be one of {', '.join(ACTIVATIONS)}")
    try:
        return _heads.linear_act(x, weight, bias, act, residual, _timed())
    except TypeError:
        _tensors(x=x, weight=weight, **{n: t for n, t in (("bias", bias), ("residual", residual)) if t is not None})
        raise


def label_log_probs(logits, labels, top=0, ignore_index=-100):
    """Log probability of the given labels, entropy and best alternatives of rows of logits (or of log probabilities).

    logits (..., V); labels (...) int64.  -> LabelLogProbs, everything fp32 but the indices:
      log_prob (...): log softmax(logits)[label]; 0 where label == ignore_index, NaN where the label lies outside [0, V);
      entropy (...): of the row's softmax, in nats;
      top_log_prob, top_index (..., top): the `top` <= min(V, 64) best entries, best first, equal logits by ascending index
      (None, None for top = 0).  A masked entry (-inf) has probability 0 and is no alternative: unused slots hold -inf and -1.
    A row of nothing but -inf has log_prob -inf, entropy 0, no alternatives and gradient 0; a row with NaN or +inf is NaN.
    log_prob and entropy are differentiable in the logits, the alternatives are not."""
    top, ignore_index = int(top), int(ignore_index)
    try:
        return LabelLogProbs(*_heads.label_log_probs(logits, labels, top, ignore_index, _timed()))
    except TypeError:
        _tensors(logits=logits, labels=labels)
        raise


def distill_top_k(logits, teacher_index, teacher_logits, temperature=1.0):
    """Row losses temperature^2 KL(q || p) of a student against the k best logits of a teacher.

    logits (..., V) of the student; teacher_index (..., k) int64, teacher_logits (..., k) (logits or log probabilities: only their
    differences count).  q = softmax(teacher_logits / temperature) over the row's k entries, p = softmax(logits / temperature) over
    all V.  -> (...) fp32, differentiable in the logits; the teacher is a constant (RuntimeError if it requires a gradient).
    A slot with a negative index or the value -inf is unused; a row without a used slot has loss 0 and gradient 0 (so padded rows
    take teacher_index = -1).  An index >= V of a used slot makes its row NaN; an index may occur more than once.  Where the teacher has
    an entry that is masked (-inf) for the student the loss is +inf; a student's row of nothing but -inf has gradient 0."""
    try:
        return _heads.distill_top_k(logits, teacher_index, teacher_logits, float(temperature), _timed())
    except TypeError:
        _tensors(logits=logits, teacher_index=teacher_index, teacher_logits=teacher_logits)
        raise

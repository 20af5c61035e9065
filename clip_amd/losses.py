"""Losses of the vocabulary decoder with their gradients, and a teacher's top scores, on the HIP kernels.

    loss = linear_cross_entropy(hidden, decoder_weight, decoder_bias, labels)     # == F.cross_entropy(hidden @ W.T + b, labels)
    loss.backward()                                                               # gradients of hidden, W and b

    values, index = topk_logits(teacher_scores, 64)                               # once, from the teacher
    loss = linear_distillation(hidden, decoder_weight, decoder_bias, values, index, temperature=2.0)

What sentclf/bert_model.py:165,175-179 computes as decoder scores + CrossEntropyLoss, here in one pass that keeps no
[n, vocab] scores, forward or backward.  hidden and weight are bf16 or fp16 (their gradients too), the bias and all losses
fp32.  Rows that take no part (labels equal to ignore_index, teacher rows without an entry) cost nothing in the products.
Everything is queued on the current stream of the tensors' device; there is no host wait and no CPU execution path."""
import ctypes as C

import torch

from . import _lib

_OPERANDS = {torch.bfloat16: _lib.PRECISION_BF16, torch.float16: _lib.PRECISION_F16}
_SCORES = {**_OPERANDS, torch.float32: _lib.PRECISION_FP32}
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _linear(hidden, weight, bias):
    if not isinstance(hidden, torch.Tensor) or not isinstance(weight, torch.Tensor):
        raise TypeError("hidden and weight must be tensors")
    if hidden.device.type != "cuda":
        raise RuntimeError("hidden must be on an MI355X (cuda); clip_amd has no CPU execution path")
    if hidden.dtype not in _OPERANDS or weight.dtype != hidden.dtype:
        raise TypeError(f"hidden and weight must both be bfloat16 or float16, not {hidden.dtype} and {weight.dtype}")
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"hidden {tuple(hidden.shape)} does not fit a [vocab, hidden] weight of {tuple(weight.shape)}")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != weight.shape[:1]):
        raise TypeError(f"bias must be float32 [{weight.shape[0]}], not {bias.dtype} {tuple(bias.shape)}")
    for t in (weight, bias):
        if t is not None and t.device != hidden.device:
            raise RuntimeError(f"tensors on {hidden.device} and {t.device}")


def _rows(t):
    """[n, H] with unit stride along a row (any row stride)"""
    t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 and (t.shape[0] < 2 or t.stride(0) >= t.shape[1]) else t.contiguous()


def _decoder(w):
    """[V, H] as the kernels read it: 16-byte aligned rows (a parameter is; anything else is copied)"""
    ok = w.stride(1) == 1 and w.stride(0) % 8 == 0 and w.shape[1] <= w.stride(0) <= 1 << 22 and w.data_ptr() % 16 == 0
    return w if ok else w.contiguous()


def _describe(hidden, weight, bias):
    return _lib.ClipLinear(_OPERANDS[hidden.dtype], hidden.shape[0], hidden.shape[1], weight.shape[0], hidden.data_ptr(),
                           hidden.stride(0), weight.data_ptr(), weight.stride(0), None if bias is None else bias.data_ptr())


def _workspace(lib, d, k, grad, device):
    need = C.c_int64()
    _lib.check(lib.clip_linear_loss_workspace(C.byref(d), k, grad, C.byref(need)))
    return torch.empty(need.value, dtype=torch.uint8, device=device)


class _LinearLoss(torch.autograd.Function):
    """hidden, weight, bias and the targets (labels, or a teacher's values and index) -> loss"""

    @staticmethod
    def forward(ctx, hidden, weight, bias, labels, values, index, ignore_index, temperature, reduction):
        rows, w = _rows(hidden), _decoder(weight)
        b = None if bias is None else bias.contiguous()
        lib, n, dev = _lib.load(), rows.shape[0], hidden.device
        k = 0 if labels is not None else values.shape[1]
        with torch.cuda.device(dev):
            d = _describe(rows, w, b)
            # the loss has storage of its own: a caller may change it in place before the backward pass reads what is kept
            kept = torch.empty((2 + max(k, 1)) * n, dtype=torch.float32, device=dev)
            row_loss, lse, target = kept[:n], kept[n:2 * n], kept[2 * n:]
            loss = torch.empty(n if reduction == 0 else (), dtype=torch.float32, device=dev)
            if reduction == 0:
                row_loss = loss
            work = _workspace(lib, d, k, 0, dev)
            tail = (reduction, _lib.ptr(row_loss), _lib.ptr(lse), _lib.ptr(target), _lib.ptr(loss), _lib.ptr(work), work.numel(),
                    _lib.stream_ptr())
            if labels is not None:
                _lib.check(lib.clip_linear_ce(C.byref(d), _lib.ptr(labels), ignore_index, *tail))
            else:
                _lib.check(lib.clip_linear_distill(C.byref(d), _lib.ptr(values), _lib.ptr(index), k, temperature, *tail))
        ctx.save_for_backward(hidden, weight, bias, labels, values, index, lse, target)
        ctx.args = ignore_index, temperature, reduction
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        hidden, weight, bias, labels, values, index, lse, target = ctx.saved_tensors
        ignore_index, temperature, reduction = ctx.args
        rows, w = _rows(hidden), _decoder(weight)
        b = None if bias is None else bias.contiguous()
        lib, dev = _lib.load(), hidden.device
        k = 0 if labels is not None else values.shape[1]
        grad = grad.to(torch.float32).contiguous()
        with torch.cuda.device(dev):
            d = _describe(rows, w, b)
            dh = torch.empty(rows.shape, dtype=rows.dtype, device=dev) if ctx.needs_input_grad[0] else None
            dw = torch.empty(w.shape, dtype=w.dtype, device=dev) if ctx.needs_input_grad[1] else None
            db = torch.empty(w.shape[0], dtype=torch.float32, device=dev) if bias is not None and ctx.needs_input_grad[2] else None
            work = _workspace(lib, d, k, 1, dev)
            tail = (reduction, _lib.ptr(lse), _lib.ptr(target), _lib.ptr(grad), _lib.ptr(dh), rows.shape[1], _lib.ptr(dw), rows.shape[1],
                    _lib.ptr(db), _lib.ptr(work), work.numel(), _lib.stream_ptr())
            if labels is not None:
                _lib.check(lib.clip_linear_ce_grad(C.byref(d), _lib.ptr(labels), ignore_index, *tail))
            else:
                _lib.check(lib.clip_linear_distill_grad(C.byref(d), _lib.ptr(values), _lib.ptr(index), k, temperature, *tail))
        return (None if dh is None else dh.view(hidden.shape), dw, db) + (None,) * 6


def _reduction(reduction):
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'none', 'mean' or 'sum', not {reduction!r}")
    return _REDUCTIONS[reduction]


def linear_cross_entropy(hidden, weight, bias, labels, *, ignore_index=-100, reduction="mean"):
    """F.cross_entropy(hidden @ weight.T + bias, labels, ignore_index=..., reduction=...) without the scores, differentiable in
    hidden [..., H] and weight [V, H] (bf16 or fp16; H a multiple of 64) and in bias (fp32 [V], or None).  labels: integers of
    hidden's leading shape.  The mean is over the rows that are not ignored (NaN if there is none, with zero gradients); a
    label outside [0, V) that is not ignore_index makes the loss and the gradients NaN."""
    code = _reduction(reduction)
    _linear(hidden, weight, bias)
    if labels.dtype not in (torch.int64, torch.int32) or labels.shape != hidden.shape[:-1]:
        raise ValueError(f"labels must be integers of shape {tuple(hidden.shape[:-1])}, not {labels.dtype} {tuple(labels.shape)}")
    if labels.device != hidden.device:
        raise RuntimeError(f"tensors on {hidden.device} and {labels.device}")
    flat = labels.reshape(-1).to(torch.int64).contiguous()
    loss = _LinearLoss.apply(hidden, weight, bias, flat, None, None, int(ignore_index), 1.0, code)
    return loss.view(labels.shape) if code == 0 else loss


def linear_distillation(hidden, weight, bias, teacher_values, teacher_index, *, temperature=1.0, reduction="mean"):
    """temperature^2 KL(p || q) per row, p the softmax of the teacher's listed scores teacher_values [..., k] / temperature, q the
    student's softmax over the whole vocabulary of (hidden @ weight.T + bias) / temperature; teacher_index [..., k] holds the
    scores' vocabulary ids (topk_logits gives both).  An entry with a negative id or the value -inf is left out, a row without
    entries contributes nothing.  Differentiable in hidden, weight and bias (not in the teacher).  k <= 1024."""
    code = _reduction(reduction)
    _linear(hidden, weight, bias)
    lead = tuple(hidden.shape[:-1])
    if teacher_index.dtype != torch.int64 or teacher_index.dim() != hidden.dim() or tuple(teacher_index.shape[:-1]) != lead or \
            teacher_values.shape != teacher_index.shape or not teacher_values.is_floating_point():
        raise ValueError(f"teacher values / index must be floating point / int64 of shape {lead + ('k',)}, not {teacher_values.dtype} "
                         f"{tuple(teacher_values.shape)} / {teacher_index.dtype} {tuple(teacher_index.shape)}")
    k = teacher_index.shape[-1]
    if not 1 <= k <= 1024:
        raise ValueError(f"{k} teacher entries per row (1 .. 1024)")
    if not (0.0 < float(temperature) < float("inf")):
        raise ValueError(f"temperature must be positive, not {temperature}")
    for t in (teacher_values, teacher_index):
        if t.device != hidden.device:
            raise RuntimeError(f"tensors on {hidden.device} and {t.device}")
    values = teacher_values.detach().to(torch.float32).reshape(-1, k).contiguous()
    index = teacher_index.reshape(-1, k).contiguous()
    loss = _LinearLoss.apply(hidden, weight, bias, None, values, index, 0, float(temperature), code)
    return loss.view(lead) if code == 0 else loss


def topk_logits(logits, k):
    """The k largest scores of every row of logits [..., V] (fp32, bf16 or fp16) -> (values [..., k], index int64 [..., k]), largest
    first, ties to the lowest index, NaN above everything.  1 <= k <= min(V, 1024).  Not differentiable."""
    if logits.device.type != "cuda":
        raise RuntimeError("logits must be on an MI355X (cuda); clip_amd has no CPU execution path")
    if logits.dtype not in _SCORES or logits.dim() < 1:
        raise TypeError(f"logits must be float32, bfloat16 or float16 with at least one dimension, not {logits.dtype}")
    k, vocab = int(k), logits.shape[-1]
    if not 1 <= k <= min(vocab, 1024):
        raise ValueError(f"k = {k} of {vocab} scores (1 .. min(vocab, 1024))")
    rows = _rows(logits.detach())
    n = rows.shape[0]
    with torch.cuda.device(logits.device):
        values = torch.empty((n, k), dtype=rows.dtype, device=rows.device)
        index = torch.empty((n, k), dtype=torch.int64, device=rows.device)
        _lib.check(_lib.load().clip_topk_scores(_SCORES[rows.dtype], _lib.ptr(rows), rows.stride(0), n, vocab, k, _lib.ptr(values),
                                                _lib.ptr(index), _lib.stream_ptr()))
    lead = logits.shape[:-1]
    return values.view(*lead, k), index.view(*lead, k)

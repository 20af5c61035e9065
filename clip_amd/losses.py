"""Losses of the vocabulary decoder with their gradients, and a teacher's top scores, on the HIP kernels.

    loss = linear_cross_entropy(hidden, decoder_weight, decoder_bias, labels)     # == F.cross_entropy(hidden @ W.T + b, labels)
    loss.backward()                                                               # gradients of hidden, W and b

    values, index = topk_logits(teacher_scores, 64)                               # once, from the teacher
    loss = linear_distillation(hidden, decoder_weight, decoder_bias, values, index, temperature=2.0)

What sentclf/bert_model.py:165,175-179 computes as decoder scores + CrossEntropyLoss, here in one pass that keeps no
[n, vocab] scores, forward or backward.  hidden and weight are bf16 or fp16 (their gradients too), the bias and all losses
fp32.  Rows that take no part (labels equal to ignore_index, teacher rows without an entry) cost nothing in the products.
Everything is queued on the current stream of the tensors' device; there is no host wait and no CPU execution path.
Refused: second and forward-mode derivatives, and tracing (a trace would hold the outputs' allocation and not what fills them;
torch.compile runs these calls outside its graphs).
The tensor handling is in csrc/torch_losses.cpp (lib/_clip_torch.so), over the C ABI (clip_linear_ce and its neighbours).

In a HIP graph: make one eager call of the same sizes first, and let go of eager losses of the same leaves before the capture (torch
ties a leaf's gradient accumulation to the stream of the graph that is alive)."""
import ctypes as C
import importlib.util
import os

import torch  # noqa: F401  (the binding links against it)

from . import _lib

EXT_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "_clip_torch.so")
_ext = None


def load():
    """The torch binding, bound to the library that _lib loads.  There is no fallback: a missing file raises."""
    global _ext
    if _ext is None:
        if not os.path.isfile(EXT_PATH):
            raise ImportError(f"{EXT_PATH} not found: build it with `python -c 'import __graft_entry__ as g; g.build()'`")
        lib = _lib.load()
        spec = importlib.util.spec_from_file_location("_clip_torch", EXT_PATH)
        ext = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(ext)
        ext.bind([C.cast(getattr(lib, "clip_" + name), C.c_void_p).value for name in
                  ("linear_loss_workspace", "linear_ce", "linear_ce_grad", "linear_distill", "linear_distill_grad", "topk_scores",
                   "last_error")])
        _ext = ext
    return _ext


def linear_cross_entropy(hidden, weight, bias, labels, *, ignore_index=-100, reduction="mean"):
    """F.cross_entropy(hidden @ weight.T + bias, labels, ignore_index=..., reduction=...) without the scores, differentiable in
    hidden [..., H] and weight [V, H] (bf16 or fp16; H a multiple of 64, at most 8192) and in bias (fp32 [V], or None).  labels:
    int64 or int32 of hidden's leading shape.  The mean is over the rows that are not ignored (NaN if there is none, with zero
    gradients); a label outside [0, V) that is not ignore_index makes the loss and the gradients NaN.  fp16 with reduction="none":
    the score gradients are held to 2^-40 of the largest upstream gradient, so rows weighted below 2^-20 of it lose bits of theirs."""
    return (_ext or load()).linear_cross_entropy(hidden, weight, bias, labels, ignore_index, reduction)


def linear_distillation(hidden, weight, bias, teacher_values, teacher_index, *, temperature=1.0, reduction="mean"):
    """temperature^2 KL(p || q) per row, p the softmax of the teacher's listed scores teacher_values [..., k] / temperature, q the
    student's softmax over the whole vocabulary of (hidden @ weight.T + bias) / temperature; teacher_index [..., k] (int64) holds
    the scores' vocabulary ids (topk_logits gives both).  An entry with a negative id or the value -inf is left out, a row
    without entries contributes nothing.  Differentiable in hidden, weight and bias (not in the teacher).  k <= 1024,
    1e-6 <= temperature <= 1e6, scores / temperature up to 2^30."""
    return (_ext or load()).linear_distillation(hidden, weight, bias, teacher_values, teacher_index, temperature, reduction)


def topk_logits(logits, k):
    """The k largest scores of every row of logits [..., V] (fp32, bf16 or fp16) -> (values [..., k], index int64 [..., k]), largest
    first, ties to the lowest index, NaN above everything.  1 <= k <= min(V, 1024).  Not differentiable."""
    return (_ext or load()).topk_logits(logits, k)

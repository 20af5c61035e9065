"""clip_amd.losses without a GPU: what is refused before any device work, and the workspace sizes."""
import ctypes as C

import pytest
import torch

from clip_amd import _lib, losses


def _desc(**kw):
    d = dict(operand=_lib.PRECISION_BF16, n=8, hidden_size=128, vocab=1000, dev_hidden=4096, ld_hidden=128, dev_weight=4096,
             ld_weight=128, dev_bias=None)
    d.update(kw)
    return _lib.ClipLinear(**d)


def _need(k=0, grad=0, **kw):
    out = C.c_int64(-1)
    rc = _lib.load().clip_linear_loss_workspace(C.byref(_desc(**kw)), k, grad, C.byref(out))
    return rc, out.value


@pytest.mark.parametrize("kw", [dict(operand=_lib.PRECISION_FP32), dict(operand=7), dict(n=-1), dict(n=1 << 21), dict(n=1 << 18, hidden_size=8192, ld_hidden=8192, ld_weight=8192), dict(n=1 << 20, vocab=1 << 30), dict(hidden_size=0),
                                dict(hidden_size=96), dict(hidden_size=8256, ld_weight=8256, ld_hidden=8256), dict(vocab=0),
                                dict(vocab=(1 << 30) + 1), dict(ld_weight=120), dict(ld_weight=132), dict(ld_weight=(1 << 22) + 8),
                                dict(ld_hidden=64)])
def test_sizes_refused(kw):
    assert _need(**kw)[0] == _lib.CLIP_ERR_ARG
    assert _lib.load().clip_last_error()


def test_workspace_is_bounded():
    assert _need()[0] == 0 and _need(n=0)[0] == 0 and _need(n=0, grad=1)[0] == 0
    assert _need(n=1, ld_hidden=0)[0] == 0              # one row needs no stride
    for grad in (0, 1):
        sizes = [_need(n=n, vocab=30522, hidden_size=768, ld_hidden=768, ld_weight=768, grad=grad)[1] for n in (1, 300, 4096, 16384, 65536)]
        assert sizes == sorted(sizes)
    # the gradients' workspace: one 512-MiB piece of 16-bit score gradients at most, rows, and fp32 partials of the hidden
    # rows' gradient; the fp32 scores alone would be 65536 x 262144 x 4 = 64 GiB
    rc, need = _need(n=65536, vocab=262144, hidden_size=768, ld_hidden=768, ld_weight=768, grad=1)
    assert rc == 0 and need < 20 << 30
    assert _need(k=1025)[0] == _lib.CLIP_ERR_ARG and _need(k=-1)[0] == _lib.CLIP_ERR_ARG
    assert _need(k=64)[1] > _need()[1]


BOUND = 1 << 30                  # bytes of a piece's score gradients, and of its (max, sum) pairs
SHAPES = [(1, 30522, 768, 0), (64, 1 << 24, 64, 0), (64, 1 << 30, 64, 0), (300, 30522, 768, 8), (4096, 30522, 768, 1024), (16384, 30522, 768, 0), (16384, 1 << 22, 128, 3),
          (1 << 17, 262221, 64, 0), (1 << 20, 262221, 64, 0), (1 << 20, 262221, 64, 64), ((1 << 21) - 256, 30522, 768, 0), ((1 << 21) - 257, 1 << 23, 128, 16)]


@pytest.mark.parametrize("n,vocab,hidden,k", SHAPES)
def test_workspace_of_a_loss(n, vocab, hidden, k):
    """the copied rows, a list's log p, and (max, sum) pairs: of the whole vocabulary (8 bytes per row and 64 columns) or of a
    bounded piece, with one joined pair per row"""
    rc, need = _need(k=k, n=n, vocab=vocab, hidden_size=hidden, ld_hidden=hidden, ld_weight=hidden)
    assert rc == 0
    rows, pair_rows = -(-n // 256) * 256, 64 if n <= 64 else -(-n // 256) * 256
    pairs = pair_rows * -(-vocab // 256) * 32
    assert need <= rows * (2 * hidden + 8) + 4 * n * k + (pairs if pairs <= BOUND else BOUND + 8 * rows) + 8 * 256


def test_calls_refused_without_a_device():
    lib, d = _lib.load(), _desc()
    p = C.c_void_p(4096)
    big = 1 << 40
    ok = [p, -100, 1, p, p, p, p, p, big, None]

    def ce(**at):
        args = list(ok)
        for i, v in at.items():
            args[int(i[1:])] = v
        return lib.clip_linear_ce(C.byref(at.pop("desc", d)) if "desc" in at else C.byref(d), *args)
    assert ce(_0=None) == _lib.CLIP_ERR_ARG                  # labels
    assert ce(_2=3) == ce(_2=-1) == _lib.CLIP_ERR_ARG        # reduction
    for out in ("_3", "_4", "_5", "_6"):
        assert ce(**{out: None}) == _lib.CLIP_ERR_ARG
    assert ce(_7=None) == _lib.CLIP_ERR_ARG and ce(_7=C.c_void_p(4104)) == _lib.CLIP_ERR_ARG
    assert ce(_8=100) == _lib.CLIP_ERR_CAPACITY and b"clip_linear_loss_workspace" in lib.clip_last_error()
    assert lib.clip_linear_ce(None, *ok) == _lib.CLIP_ERR_ARG
    for bad in (_desc(dev_weight=None), _desc(dev_weight=4100), _desc(dev_hidden=None), _desc(hidden_size=100)):
        assert lib.clip_linear_ce(C.byref(bad), *ok) == _lib.CLIP_ERR_ARG
    for k, t in ((0, 1.0), (1025, 1.0), (4, 0.0), (4, -1.0), (4, float("inf")), (4, float("nan"))):
        assert lib.clip_linear_distill(C.byref(d), p, p, k, t, 1, p, p, p, p, p, big, None) == _lib.CLIP_ERR_ARG
        assert lib.clip_linear_distill_grad(C.byref(d), p, k, t, 1, p, p, p, p, 128, p, 128, p, p, big, None) == _lib.CLIP_ERR_ARG
    grad = [p, -100, 1, p, p, p, p, 128, p, 128, p, p, big, None]
    for i, v in ((0, None), (3, None), (4, None), (5, None), (7, 64), (8, C.c_void_p(4100)), (9, 64), (9, 130), (11, None)):
        args = list(grad)
        args[i] = v
        assert lib.clip_linear_ce_grad(C.byref(d), *args) == _lib.CLIP_ERR_ARG, i
    args = list(grad)
    args[12] = 1000
    assert lib.clip_linear_ce_grad(C.byref(d), *args) == _lib.CLIP_ERR_CAPACITY
    for args in ((3, p, 10, 1, 10, 1, p, p, None), (1, p, 10, 1, 10, 11, p, p, None), (1, p, 10, 1, 10, 0, p, p, None),
                 (1, p, 2000, 1, 2000, 1025, p, p, None), (1, None, 10, 1, 10, 1, p, p, None), (1, p, 9, 2, 10, 1, p, p, None),
                 (1, C.c_void_p(4098), 10, 1, 10, 1, p, p, None), (0, C.c_void_p(4097), 10, 1, 10, 1, p, p, None),
                 (1, p, 10, -1, 10, 1, p, p, None)):
        assert lib.clip_topk_scores(*args) == _lib.CLIP_ERR_ARG


def test_python_refuses_cpu_tensors():
    h, w, y = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(5, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU"):
        losses.linear_cross_entropy(h, w, None, y)
    with pytest.raises(RuntimeError, match="no CPU"):
        losses.linear_distillation(h, w, None, torch.zeros(2, 1), y[:, None])
    with pytest.raises(RuntimeError, match="no CPU"):
        losses.topk_logits(torch.zeros(2, 5), 1)
    with pytest.raises(TypeError):
        losses.linear_cross_entropy([1.0], w, None, y)
    with pytest.raises(ValueError, match="reduction"):
        losses.linear_cross_entropy(h, w, None, y, reduction="max")


def test_missing_binding_raises(monkeypatch):
    monkeypatch.setattr(losses, "_ext", None)
    monkeypatch.setattr(losses, "EXT_PATH", losses.EXT_PATH + ".missing")
    with pytest.raises(ImportError, match="build"):
        losses.topk_logits(torch.zeros(2, 5), 1)


def test_forward_mode_derivatives_are_refused():
    """a dual number's tangent would be lost without a word: the kernels read values only"""
    import torch.autograd.forward_ad as fw
    h, w, b = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(5, 64, dtype=torch.bfloat16), torch.zeros(5)
    y = torch.zeros(2, dtype=torch.int64)
    with fw.dual_level():
        for i in range(3):
            for grad in (False, True):
                args = [fw.make_dual(t, torch.ones_like(t)) if i == j else t.clone().requires_grad_(grad) for j, t in enumerate((h, w, b))]
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    losses.linear_cross_entropy(*args, y)
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    losses.linear_distillation(*args, torch.zeros(2, 1), y[:, None])
        with pytest.raises(RuntimeError, match="no CPU"):       # plain tensors pass that check
            losses.linear_cross_entropy(h, w, b, y)


def test_tracing_is_refused():
    """a trace would hold the outputs' allocation and nothing that fills them"""
    from torch.fx.experimental.proxy_tensor import make_fx
    h, w = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(5, 64, dtype=torch.bfloat16)
    y = torch.zeros(2, dtype=torch.int64)
    for call in (lambda h: losses.linear_cross_entropy(h, w, None, y), lambda h: losses.linear_distillation(h, w, None, torch.zeros(2, 1), y[:, None]),
                 lambda h: losses.topk_logits(h, 3)[0]):
        with pytest.raises(NotImplementedError, match="traced"):
            torch.jit.trace(call, (h,), check_trace=False)
        with pytest.raises(NotImplementedError, match="traced"):
            make_fx(call)(h)
        with pytest.raises(RuntimeError, match="no CPU"):
            call(h)


@pytest.mark.parametrize("n,vocab,hidden,k", SHAPES)
def test_workspace_of_the_gradients(n, vocab, hidden, k):
    """rows, what is known of each, fp32 partials of their gradient, a distillation's table of target sums, and one piece of 16-bit
    score gradients with its column sums"""
    rc, need = _need(k=k, grad=1, n=n, vocab=vocab, hidden_size=hidden, ld_hidden=hidden, ld_weight=hidden)
    assert rc == 0
    rows = -(-n // 256) * 256
    piece = min(2 * rows * (-(-vocab // 256) * 256), BOUND)
    table = rows * (16 + 64) + 64 * vocab if k else 0
    assert need <= rows * (2 * hidden + 24) + table + piece * 33 // 32 + max(8 * rows * (hidden + 255), 2 * 128 << 20) + 12 * 256

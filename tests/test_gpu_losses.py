"""clip_amd.losses on the GPU: the decoder losses and their gradients against 64-bit forms, over the sizes, masks,
strides and layouts where tiles end; a teacher's top scores bit for bit; refusals; streams and graphs."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "helpers"))
import loss_case as R  # noqa: E402
from clip_amd import losses  # noqa: E402

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
INF, NAN = float("inf"), float("nan")


def _labels(n, vocab, seed, ignored=0.0, ignore=-100):
    g = torch.Generator().manual_seed(seed + 1)
    y = torch.randint(0, vocab, (n,), generator=g)
    y[torch.rand(n, generator=g) < ignored] = ignore
    return y.cuda()


def _teacher(n, vocab, k, seed, dropped=0.0):
    g = torch.Generator().manual_seed(seed + 2)
    values = 3 * torch.randn(n, k, generator=g)
    index = torch.stack([torch.randperm(vocab, generator=g)[:k] for _ in range(n)]) if n else torch.zeros(0, k, dtype=torch.int64)
    index[torch.rand(n, k, generator=g) < dropped] = -1
    return values.cuda(), index.cuda()


def _check(h, w, b, run, p, live, temperature, reduction, seed, entropy=None):
    """run(h, w, b) -> loss; compares loss and gradients"""
    leaves = [t.detach().clone().requires_grad_() if t is not None else None for t in (h, w, b)]
    n = h.shape[0]
    loss = run(*leaves)
    count = int(live.sum())
    if reduction == "none":
        up = torch.randn(n, generator=torch.Generator().manual_seed(seed)).cuda()
        row_grad = up
    else:
        up = torch.tensor(0.7, device="cuda")
        row_grad = (up / (max(count, 1) if reduction == "mean" else 1)).expand(n)
    inputs = [t for t in leaves if t is not None]
    grads = torch.autograd.grad(loss, inputs, up)
    (ref, dh, dw, db), (e_loss, e_h, e_w, e_b) = R.reference(h, w, b, p, live, temperature, row_grad, entropy)
    if reduction == "none":
        R.assert_within("loss", loss.detach(), ref, e_loss)
    else:
        total, err = ref.sum(), e_loss.sum() + n * 2.0 ** -24 * ref.abs().sum()
        if reduction == "mean":
            total, err = total / count if count else ref.new_tensor(NAN), err / max(count, 1)
        R.assert_within("loss", loss.detach(), total, err)
    R.assert_within("dh", grads[0], dh, e_h)
    R.assert_within("dw", grads[1], dw, e_w)
    if b is not None:
        R.assert_within("db", grads[2], db, e_b)
    assert grads[0].dtype == h.dtype and grads[1].dtype == w.dtype
    return loss.detach(), grads


SIZES = [(1, 1, 64), (1, 2, 64), (2, 63, 64), (3, 65, 128), (37, 2000, 128), (64, 128, 64), (65, 129, 192), (130, 777, 320),
         (257, 1000, 768), (300, 4099, 256), (1000, 300, 512), (513, 30522, 128), (20, 30522, 768), (2600, 1300, 128), (1500, 2500, 384),
         (1030, 5, 1024), (70, 500, 2048), (300, 600, 1152), (130, 300, 8192),
         # large tiles for the loss (192 of them), and below for gradients (500 blocks of 256^3)
         (257, 30700, 128), (129, 10300, 1408), (300, 9001, 1152), (1030, 4099, 1024), (2600, 8003, 128), (1500, 10001, 384), (20500, 700, 256), (4100, 65, 256),
         (257, 128100, 128), (129, 24001, 1408), (300, 14501, 1152), (1030, 6500, 1024), (2600, 24003, 128), (1500, 15001, 384)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,vocab,hidden", SIZES)
def test_cross_entropy_sizes(n, vocab, hidden, dtype):
    h, w, b = R.make(n, vocab, hidden, dtype, n + vocab)
    y = _labels(n, vocab, n)
    p, live = R.targets_ce(y, vocab, -100)
    _check(h, w, b, lambda h, w, b: losses.linear_cross_entropy(h, w, b, y), p, live, 1.0, "mean", 5)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("ignored", [0.0, 0.6, 0.97, 1.1])
@pytest.mark.parametrize("vocab", [523, 30523, 128100])
def test_cross_entropy_reductions_and_ignored_rows(vocab, dtype, reduction, ignored):
    n, hidden = 401, 128
    h, w, b = R.make(n, vocab, hidden, dtype, 3)
    y = _labels(n, vocab, 4, ignored, ignore=-7)
    p, live = R.targets_ce(y, vocab, -7)
    if ignored:                       # whatever an ignored row holds stays there
        h[~live] = NAN
        h[~live, 0] = INF
    _, grads = _check(h, w, b, lambda h, w, b: losses.linear_cross_entropy(h, w, b, y, ignore_index=-7, reduction=reduction), p, live,
                      1.0, reduction, 6)
    assert not grads[0][~live].any()
    if ignored > 1:
        assert not any(g.any() for g in grads)


@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("distill", [False, True])
@pytest.mark.parametrize("n", [1500, 4097, 9001, 70001])
def test_ignored_rows_among_many(n, distill, reduction):
    # live rows counted by the copying workgroups, small and large, or beforehand
    vocab, hidden = 200, 128
    h, w, b = R.make(n, vocab, hidden, BF16, n)
    if distill:
        values, index = _teacher(n, vocab, 3, n, 0.8)
        p, live, entropy = R.targets_distill(values, index, vocab, 2.0)
    else:
        y = _labels(n, vocab, n, 0.6)
        (p, live), entropy = R.targets_ce(y, vocab, -100), None
    h[~live] = NAN
    _, grads = _check(h, w, b, lambda h, w, b: losses.linear_distillation(h, w, b, values, index, temperature=2.0, reduction=reduction) if distill
                      else losses.linear_cross_entropy(h, w, b, y, reduction=reduction), p, live, 2.0 if distill else 1.0, reduction, 6, entropy)
    assert not grads[0][~live].any()


def test_mean_over_no_rows():
    h, w, b = R.make(5, 70, 64, BF16, 1)
    y = torch.full((5,), -100).cuda()
    assert losses.linear_cross_entropy(h, w, b, y).isnan()
    assert losses.linear_cross_entropy(h, w, b, y, reduction="sum") == 0
    h, w, b = (t.requires_grad_() for t in (h[:0].clone(), w, b))
    for red in ("mean", "sum", "none"):
        loss = losses.linear_cross_entropy(h, w, b, y[:0], reduction=red)
        assert loss.isnan() if red == "mean" else not loss.any()
        grads = torch.autograd.grad(loss.sum(), (h, w, b))
        assert grads[0].shape == (0, 64) and not grads[1].any() and not grads[2].any()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_without_bias_and_with_entries_left_out(dtype):
    n, vocab, hidden = 90, 700, 64
    h, w, b = R.make(n, vocab, hidden, dtype, 8)
    y = _labels(n, vocab, 9)
    p, live = R.targets_ce(y, vocab, -100)
    _check(h, w, None, lambda h, w, b: losses.linear_cross_entropy(h, w, b, y), p, live, 1.0, "mean", 5)
    # a whole column tile and single entries at -inf, one at the type's lowest value
    b[128:256] = -INF
    b[[3, 699]] = -INF
    b[400] = torch.finfo(F32).min
    ok = torch.tensor([v for v in range(vocab) if b[v] > -1e30]).cuda()
    y = ok[torch.randint(0, len(ok), (n,), generator=torch.Generator().manual_seed(1)).cuda()]
    p, live = R.targets_ce(y, vocab, -100)
    b2 = torch.where(b == torch.finfo(F32).min, -INF, b)      # the same softmax; the bounds are made from finite scores
    leaves = [t.clone().requires_grad_() for t in (h, w, b)]
    loss = losses.linear_cross_entropy(*leaves, y, reduction="none")
    grads = torch.autograd.grad(loss.sum(), leaves)
    want, err = R.reference(h, w, b2, p, live, 1.0, torch.ones(n).cuda())
    for name, got, a, e in zip(("loss", "dh", "dw", "db"), (loss.detach(), *grads), want, err):
        R.assert_within(name, got, a, e)
    assert not grads[1][128:256].any() and not grads[2][128:256].any() and grads[2][400] == 0
    # a label whose entry is left out: an infinite loss, and -1 in its gradient
    y[0] = 3
    loss = losses.linear_cross_entropy(*leaves, y, reduction="none")
    assert loss[0] == INF and loss[1:].isfinite().all()
    assert torch.autograd.grad(loss[1:].sum() + loss[0], leaves)[2][3] == -1
    # nothing left at all
    assert losses.linear_cross_entropy(h, w, torch.full_like(b, -INF), y, reduction="none").isnan().all()


@pytest.mark.parametrize("n,vocab,hidden", [(140, 300, 64), (300, 30800, 128), (300, 128100, 128), (50, 300, 64)])
def test_non_finite_rows_stay_in_their_rows(n, vocab, hidden):
    h, w, b = R.make(n, vocab, hidden, BF16, 12)
    h[5], h[37, 3] = NAN, INF
    y = _labels(n, vocab, 13)
    y[9] = vocab                      # no such entry
    y[11] = -1
    bad = torch.zeros(n, dtype=torch.bool).cuda()
    bad[[5, 37, 9, 11]] = True
    leaves = [t.requires_grad_() for t in (h, w, b)]
    loss = losses.linear_cross_entropy(*leaves, y, reduction="none")
    assert torch.equal(loss.isnan(), bad)
    dh, dw, db = torch.autograd.grad(loss.sum(), leaves)
    assert torch.equal(dh.isnan().any(1), bad)
    assert dw.isnan().all() and db.isnan().all()
    assert losses.linear_cross_entropy(*leaves, y).isnan()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_strides_and_shapes(dtype):
    n, vocab, hidden = 66, 333, 128
    big_h = torch.randn(n, 3 * hidden + 5, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    big_w = (0.1 * torch.randn(vocab, hidden + 24, generator=torch.Generator().manual_seed(2))).to(dtype).cuda()
    b = torch.randn(2 * vocab, generator=torch.Generator().manual_seed(3)).cuda()[::2]
    y = _labels(n, vocab, 3, 0.2)
    p, live = R.targets_ce(y, vocab, -100)

    def loss(h, w, b):
        return losses.linear_cross_entropy(h, w, b, y)
    base = loss(big_h[:, 7:7 + hidden].contiguous(), big_w[:, 8:8 + hidden].contiguous(), b.contiguous())
    views_h = {"odd start": big_h[:, 7:7 + hidden], "transposed": big_h[:, 7:7 + hidden].t().contiguous().t()}
    views_w = {"strided": big_w[:, 8:8 + hidden], "unaligned": big_w.reshape(-1)[8:].as_strided((vocab, hidden), (hidden + 24, 1)),
               "transposed": big_w[:, 8:8 + hidden].t().contiguous().t()}
    for hv in views_h.values():
        for wv in views_w.values():
            assert torch.equal(loss(hv, wv, b), base)
    wide = big_h.detach().clone().requires_grad_()
    wfull = big_w.detach().clone().requires_grad_()
    got = torch.autograd.grad(loss(wide[:, 7:7 + hidden], wfull[:, 8:8 + hidden], b), (wide, wfull))
    _, want = _check(big_h[:, 7:7 + hidden], big_w[:, 8:8 + hidden], b, loss, p, live, 1.0, "mean", 2)
    assert not got[0][:, :7].any() and not got[1][:, :8].any()
    # [batch, width, H] with [batch, width] labels, int32 labels, one broadcast row
    h = big_h[:, 7:7 + hidden].contiguous()
    assert torch.equal(losses.linear_cross_entropy(h.view(6, 11, hidden), big_w[:, 8:8 + hidden], b, y.view(6, 11).int()), base)
    rows = losses.linear_cross_entropy(h[:1].expand(4, hidden), big_w[:, 8:8 + hidden], b, y[live][:1].expand(4), reduction="none")
    assert (rows == rows[0]).all()
    row3 = losses.linear_cross_entropy(h.view(6, 11, hidden), big_w[:, 8:8 + hidden], b, y.view(6, 11), reduction="none")
    assert row3.shape == (6, 11)
    # one row's loss has the same bits wherever it stands
    alone = losses.linear_cross_entropy(h[live][20:21], big_w[:, 8:8 + hidden], b, y[live][20:21], reduction="none")
    assert torch.equal(alone[0], row3.view(-1)[live][20])
    # one hidden vector, one label
    one = losses.linear_cross_entropy(h[live][0], big_w[:, 8:8 + hidden], b, y[live][0])
    assert one.shape == () and torch.equal(one, row3.view(-1)[live][0])


@pytest.mark.parametrize("n,vocab", [(40, 333), (130, 333), (300, 30801), (300, 128101)])
def test_weight_anywhere_in_a_flat_buffer(n, vocab):
    """a contiguous weight whose first row starts on 2 or 8 bytes, as a view into flat parameters may: loss and gradients"""
    hidden = 128
    h, w, b = R.make(n, vocab, hidden, BF16, 15)
    y = _labels(n, vocab, 16, 0.1)
    leaves = [t.clone().requires_grad_() for t in (h, w, b)]
    loss = losses.linear_cross_entropy(*leaves, y)
    want = (loss.detach(), *torch.autograd.grad(loss, leaves))
    for at in (1, 4):
        flat = torch.full((vocab * hidden + 8,), NAN, dtype=BF16, device="cuda")
        flat[at:at + vocab * hidden] = w.view(-1)
        flat.requires_grad_()
        view = flat[at:at + vocab * hidden].view(vocab, hidden)
        assert view.is_contiguous() and view.data_ptr() % 16 != 0
        loss = losses.linear_cross_entropy(leaves[0], view, leaves[2], y)
        dh, dflat, db = torch.autograd.grad(loss, (leaves[0], flat, leaves[2]))
        got = (loss.detach(), dh, dflat[at:at + vocab * hidden].view(vocab, hidden), db)
        assert all(torch.equal(g, r) for g, r in zip(got, want))
        assert not dflat[:at].any() and not dflat[at + vocab * hidden:].any()


def test_one_decoder_row_of_any_stride():
    # (torch calls a single row contiguous whatever its stride is)
    h, _, _ = R.make(9, 1, 64, BF16, 3)
    y = torch.zeros(9, dtype=torch.int64).cuda()
    wide = torch.randn(2, 131, generator=torch.Generator().manual_seed(4)).to(BF16).cuda()
    one = wide[:1, :64]
    assert one.is_contiguous() and one.stride(0) == 131
    leaves = [h.clone().requires_grad_(), one.detach().requires_grad_()]
    loss = losses.linear_cross_entropy(*leaves, None, y, reduction="none")
    p, live = R.targets_ce(y, 1, -100)
    want, err = R.reference(h, one, None, p, live, 1.0, torch.ones(9).cuda())
    for name, got, a, e in zip(("loss", "dh", "dw"), (loss.detach(), *torch.autograd.grad(loss.sum(), leaves)), want, err):
        R.assert_within(name, got, a, e)


@pytest.mark.parametrize("n,vocab", [(1, 500), (30, 500), (64, 500), (100, 500), (300, 500), (300, 31000), (1300, 31000), (300, 128100), (1300, 43000)])
def test_row_strides_by_size(n, vocab):
    """rows read in place (few), copied by aligned and by unaligned loads: the same bits from every layout"""
    hidden = 128
    big = torch.randn(n, 3 * hidden, generator=torch.Generator().manual_seed(n)).to(BF16).cuda()
    _, w, b = R.make(1, vocab, hidden, BF16, 2)
    y = _labels(n, vocab, 3, 0.3)
    values, index = _teacher(n, vocab, 5, 4, 0.2)
    y[0] = 7
    seen = []
    for at in (0, 8, 3, 2 * hidden):
        big2 = torch.zeros_like(big)
        big2[:, at:at + hidden] = big[:, :hidden]
        for h in (big2[:, at:at + hidden], big2[:, at:at + hidden].contiguous()):
            leaves = [t.detach().requires_grad_() for t in (h, w, b)]
            for loss in (losses.linear_cross_entropy(*leaves, y), losses.linear_distillation(*leaves, values, index)):
                seen.append((loss.detach(), *torch.autograd.grad(loss, leaves)))
    for i, got in enumerate(seen):
        assert all(torch.equal(a, b) for a, b in zip(got, seen[i % 2])), i


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("distill", [0, 2, 70])
@pytest.mark.parametrize("n,vocab", [(1, 600), (40, 600), (64, 600), (100, 600), (700, 600), (700, 21000), (700, 85500)])
def test_what_the_rounded_score_gradients_leave_is_put_back(n, vocab, distill, dtype):
    """The large entries of a row reach dhidden unrounded; dweight of at most 64 rows is made of high and low parts, whose
    product is off by the square of a half step."""
    hidden = 128
    h, w, b = R.make(n, vocab, hidden, dtype, n)
    w[2:] = 0                                     # the targets, each in columns of its own
    w[0, 64:] = 0
    w[1, :64] = 0
    up = torch.randn(n, generator=torch.Generator().manual_seed(n)).cuda()
    if distill:
        values, index = torch.full((n, distill), -INF).cuda(), torch.full((n, distill), -1).cuda()
        values[:, 0], values[:, -1], index[:, 0], index[:, -1] = 1.0, 0.5, 0, 1
        p, live, entropy = R.targets_distill(values, index, vocab, 1.0)
    else:
        y = torch.arange(n).cuda() % 2
        (p, live), entropy = R.targets_ce(y, vocab, -100), None
    leaves = [t.clone().requires_grad_() for t in (h, w, b)]
    loss = (losses.linear_distillation(*leaves, values, index, reduction="none") if distill else
            losses.linear_cross_entropy(*leaves, y, reduction="none"))
    dh, dw, _ = torch.autograd.grad(loss, leaves, up)
    q = torch.softmax(h.double() @ w.double().t() + b.double(), 1)
    large = (q - p).abs() >= 0.07 if distill else p > 0          # (a sixteenth, and away from it)
    u = R.half_step(dtype)
    (_, want_h, want_w, _), (_, e_h, e_w, _) = R.reference(h, w, b, p, live, 1.0, up, entropy, rounded_h=~large * 1.0,
                                                          rounded_w=u if n <= 64 else 1.0)
    R.assert_within("dh", dh, want_h, e_h)
    R.assert_within("dw", dw, want_w, e_w)


def test_gradients_of_some_inputs_only():
    h, w, b = R.make(70, 200, 64, BF16, 4)
    y = _labels(70, 200, 4)
    full = [t.clone().requires_grad_() for t in (h, w, b)]
    want = torch.autograd.grad(losses.linear_cross_entropy(*full, y), full)
    for i in range(3):
        args = [t.clone().requires_grad_(j == i) for j, t in enumerate((h, w, b))]
        got, = torch.autograd.grad(losses.linear_cross_entropy(*args, y), args[i])
        assert torch.equal(got, want[i])
    # an in-place change of the loss before the backward pass
    loss = losses.linear_cross_entropy(*full, y)
    loss *= 2.0
    assert torch.equal(torch.autograd.grad(loss, full)[2], 2 * want[2])
    again = torch.autograd.grad(losses.linear_cross_entropy(*full, y), full)
    assert all(torch.equal(a, b) for a, b in zip(again, want))          # the same bits every time


def test_large_scores_and_common_shift():
    # scores of some hundred: the softmax is taken relative to the row's maximum; bounds grow with the scores
    for dtype in (BF16, F16):
        h, w, b = R.make(50, 400, 128, dtype, 21, spread=2.0)
        b = b + 300.0
        y = _labels(50, 400, 2)
        p, live = R.targets_ce(y, 400, -100)
        _check(h, w, b, lambda h, w, b: losses.linear_cross_entropy(h, w, b, y, reduction="none"), p, live, 1.0, "none", 3)


def _saturated(n, vocab, dtype, spread, seed, least):
    """rows whose largest score is ahead of the next by `least` and more: their softmax is one-hot to fp32's last bit; scores big
    enough that two orders of the same fp32 sum differ by a part of it that shows"""
    h, w, b = R.make(16 * n, vocab, 128, dtype, seed, spread=spread)
    top = (h.double() @ w.double().t() + b.double()).topk(2, 1)
    keep = (top.values[:, 0] - top.values[:, 1] >= least).nonzero()[:n, 0]
    assert len(keep) == n
    return h[keep].contiguous(), w, b, top.indices[keep, 0]


def _check_one_hot(h, w, b, top, p, scale, up, grads):
    """dz = up scale (onehot(top) - p), the one rounding of the operand type on its way into dh and dw (and of the results), fp32 sums:
    no error of a score is let in"""
    n, vocab = p.shape
    u = R.half_step(h.dtype)
    q = torch.zeros_like(p)
    q[torch.arange(n), top] = 1.0
    dz = up * scale * (q - p)
    # exp2, reciprocals and products of c, q and p; p of values / T up to 13.5, off by three half steps (T, its reciprocal, the product)
    near = up * scale * 64 * R.F32 * (q + p)
    hd, wd = h.double(), w.double()
    for name, got, want, size in zip(("dh", "dw", "db"), grads, (dz @ wd, dz.t() @ hd, dz.sum(0)),
                                     ((u * dz.abs() + near) @ wd.abs(), (u * dz.abs() + near).t() @ hd.abs(), near.sum(0))):
        own = u if name != "db" else 0
        sums = (n if name != "dh" else 4) * R.F32 * {"dh": (dz.abs() + near) @ wd.abs(), "dw": dz.abs().t() @ hd.abs(), "db": (q + p).sum(0) * up * scale}[name]
        R.assert_within(name, got, want, size + sums + 1.01 * own * want.abs() + (R.TINY[h.dtype] if own else n * 2.0 ** -38 * up * scale))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,vocab", [(40, 700), (100, 700), (300, 128100)])
def test_large_scores_of_rows_that_are_sure(n, vocab, dtype):
    # scores of some 10 000: a label that is the row's largest score has no gradient, another one that of a one-hot softmax
    h, w, b, top = _saturated(n, vocab, dtype, 20.0, 61, 120.0)
    y = torch.where(torch.arange(n).cuda() % 2 == 0, top, (top + 1) % vocab)
    p = torch.zeros(n, vocab, dtype=torch.float64, device="cuda")
    p[torch.arange(n), y] = 1.0
    leaves = [t.clone().requires_grad_() for t in (h, w, b)]
    loss = losses.linear_cross_entropy(*leaves, y, reduction="sum")
    _check_one_hot(h, w, b, top, p, 1.0, 0.5, torch.autograd.grad(loss, leaves, torch.tensor(0.5).cuda()))
    # and no loss: exp2, log2 and a product next to the exact difference from the largest score
    rows = losses.linear_cross_entropy(h, w, b, y, reduction="none")
    assert rows[::2].abs().max() <= 16 * R.F32 and (rows[1::2] > 100).all()


@pytest.mark.parametrize("spread", [0.5, 1.0, 3.0, 20.0])
@pytest.mark.parametrize("n,vocab", [(60, 2000), (4000, 2000), (4000, 30001)])
def test_no_negative_losses(n, vocab, spread):
    # labels that are their rows' largest scores: losses down to fp32's last bits
    h, w, b = R.make(n, vocab, 128, BF16, 64, spread=spread)
    y = (h.double() @ w.double().t() + b.double()).argmax(1)
    rows = losses.linear_cross_entropy(h, w, b, y, reduction="none")
    assert (rows >= 0).all() and rows.isfinite().all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("temperature", [1e-3, 1e-5, 1e-6])
@pytest.mark.parametrize("n,vocab,k", [(40, 700, 5), (100, 700, 5), (100, 700, 90), (300, 128100, 5), (300, 128100, 90), (4500, 500, 5)])
def test_small_temperatures(n, vocab, k, temperature, dtype):
    # scores over T of some thousand to some million: q is one-hot, and the teacher's list names its entry in every other row
    h, w, b, top = _saturated(n, vocab, dtype, 0.5, 62, 100 * temperature)
    values, index = _teacher(n, vocab, k, 63)
    values *= temperature
    index[::2, 1] = top[::2]
    p, live, _ = R.targets_distill(values, index, vocab, temperature)
    leaves = [t.clone().requires_grad_() for t in (h, w, b)]
    loss = losses.linear_distillation(*leaves, values, index, temperature=temperature, reduction="sum")
    up = 0.5 / temperature
    _check_one_hot(h, w, b, top, p, temperature, up, torch.autograd.grad(loss, leaves, torch.tensor(up).cuda()))


def test_loss_differences():
    # central differences of the loss itself along +-1 directions; hidden values on a grid of 2^-5 that bf16 holds with the
    # step added.  Third derivative of logsumexp along d: a third cumulant of d.w_v, at most 8 M^3, M = max |d.w_v|.
    n, vocab, hidden = 40, 150, 64
    h, w, b = R.make(n, vocab, hidden, BF16, 31, spread=0.02)
    h = (h.float().clamp(-3, 3) * 32).round() / 32
    h = h.to(BF16)
    y = _labels(n, vocab, 3)
    sign = torch.Generator().manual_seed(5)
    dh_dir = (torch.randint(0, 2, h.shape, generator=sign) * 2 - 1).cuda().double()
    db_dir = (torch.randint(0, 2, b.shape, generator=sign) * 2 - 1).cuda().double()
    leaves = [t.clone().requires_grad_() for t in (h, w, b)]
    loss = losses.linear_cross_entropy(*leaves, y, reduction="sum")
    gh, _, gb = torch.autograd.grad(loss, leaves)

    def f(h, b):
        return losses.linear_cross_entropy(h.to(BF16), w, b.float(), y, reduction="none").double().sum()
    step = 2.0 ** -5
    hp, hm = h.double() + step * dh_dir, h.double() - step * dh_dir
    assert torch.equal(hp.to(BF16).double(), hp) and torch.equal(hm.to(BF16).double(), hm)
    p, live = R.targets_ce(y, vocab, -100)
    _, (e_loss, e_h, _, e_b) = R.reference(h, w, b, p, live, 1.0, torch.ones(n).cuda())
    m = (dh_dir @ w.double().t()).abs().amax(1)
    slope = (f(hp, b.double()) - f(hm, b.double())) / (2 * step)
    assert abs(slope - (gh.double() * dh_dir).sum()) <= (step ** 2 / 6 * 8 * m ** 3).sum() + e_loss.sum() / step + e_h.sum()
    step = 2.0 ** -4
    slope = (f(h, b.double() + step * db_dir) - f(h, b.double() - step * db_dir)) / (2 * step)
    assert abs(slope - (gb.double() * db_dir).sum()) <= n * step ** 2 / 6 * 8 + e_loss.sum() / step + e_b.sum()


@pytest.mark.parametrize("n,vocab,hidden", [(4500, 65537, 64), (4500, 120001, 128)])
def test_vocabulary_in_several_pieces(n, vocab, hidden):
    # 16-bit score gradients of 4500 x 65 536 are beyond one piece's bound: the products run piece by piece
    h, w, b = R.make(n, vocab, hidden, BF16, 77)
    y = _labels(n, vocab, 78, 0.01)
    y[0], y[1] = vocab - 1, 0
    p, live = R.targets_ce(y, vocab, -100)
    _check(h, w, b, lambda h, w, b: losses.linear_cross_entropy(h, w, b, y), p, live, 1.0, "mean", 5)


@pytest.mark.parametrize("distill", [False, True])
@pytest.mark.parametrize("n", [20, 100, 300])
def test_few_rows_in_several_pieces(n, distill):
    # rows of the weight so far apart that 32-bit byte offsets reach 256 of them
    vocab, hidden, ld = 600, 128, 1 << 22
    h, w, b = R.make(n, vocab, hidden, BF16, 79)
    far = torch.empty(vocab, ld, dtype=BF16, device="cuda")[:, :hidden]
    far.copy_(w)
    if distill:
        values, index = _teacher(n, vocab, 10, 80, 0.1)
        p, live, entropy = R.targets_distill(values, index, vocab, 1.5)
    else:
        y = _labels(n, vocab, 80, 0.2)
        (p, live), entropy = R.targets_ce(y, vocab, -100), None
    leaves = [h.clone().requires_grad_(), far.requires_grad_(), b.clone().requires_grad_()]
    loss = (losses.linear_distillation(*leaves, values, index, temperature=1.5, reduction="none") if distill else
            losses.linear_cross_entropy(*leaves, y, reduction="none"))
    grads = torch.autograd.grad(loss.sum(), leaves)
    want, err = R.reference(h, w, b, p, live, 1.5 if distill else 1.0, torch.ones(n).cuda(), entropy)
    for name, got, a, e in zip(("loss", "dh", "dw", "db"), (loss.detach(), *grads), want, err):
        R.assert_within(name, got, a, e)


@pytest.mark.parametrize("distill", [0, 3, 20])
def test_loss_of_pairs_beyond_one_piece(distill):
    # 2^17 rows x 70 001 entries: the (max, sum) pairs of the whole vocabulary are beyond one piece's bound
    n, vocab, hidden, step = 1 << 17, 70001, 128, 4096
    h, w, b = R.make(n, vocab, hidden, BF16, 83)
    if distill:
        values, index = _teacher(step, vocab, distill, 84, 0.2)
        values, index = values.repeat(n // step, 1), index.repeat(n // step, 1)
        index[:, 0] = torch.arange(n).cuda() % vocab
        index[::7] = -1
        loss = losses.linear_distillation(h, w, b, values, index, temperature=2.0, reduction="none")
    else:
        y = _labels(n, vocab, 85, 0.3)
        y[-1], y[-2] = vocab - 1, 0
        loss = losses.linear_cross_entropy(h, w, b, y, reduction="none")
    for i in (0, step * 13, n - step):
        at = slice(i, i + step)
        if distill:
            p, live, entropy = R.targets_distill(values[at], index[at], vocab, 2.0)
        else:
            (p, live), entropy = R.targets_ce(y[at], vocab, -100), None
        (want, *_), (err, *_) = R.reference(h[at], w, b, p, live, 2.0 if distill else 1.0, torch.ones(step).cuda(), entropy)
        R.assert_within("loss", loss[at], want, err)
        del p, want, err
    if distill:
        return
    for i in range(0, n, step):      # every row, by R.reference's bound of the loss
        hd, yi = h[i:i + step].double(), y[i:i + step]
        z = hd @ w.double().t() + b.double()
        lse = torch.logsumexp(z, 1)
        mag = z.abs().amax(1) + lse.abs()
        z_err = ((hidden + 2) * R.F32 * (hd.abs() @ w.double().abs().t() + b.abs())).amax(1) + 8 * R.F32 * mag
        off = (loss[i:i + step] - (lse - z.gather(1, yi.clamp(min=0)[:, None])[:, 0])).abs()
        assert (off <= 2 * z_err + (16 + vocab / 64) * R.F32 * (1 + mag))[yi >= 0].all()
        assert not loss[i:i + step][yi < 0].any()


def test_few_rows_of_pairs_beyond_one_piece():
    # 2^27 entries and more: a vocabulary of which 64 rows' pairs are beyond the bound (17 GB of weight)
    vocab, hidden, n = (1 << 27) + 77, 64, 64
    h, w, _ = R.make(n, 1 << 20, hidden, BF16, 86)
    w = w.repeat(129, 1)[:vocab]
    b = (torch.arange(vocab, device="cuda") % 1009).float() / 1009
    b[-1] = 18.0        # weighs as much as all others: it is in the second piece
    y = torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(87)).cuda()
    y[0], y[1], y[2] = vocab - 1, -100, 5
    loss = losses.linear_cross_entropy(h, w, b, y, reduction="none")
    hd, parts = h.double(), []
    for v in range(0, vocab, 1 << 20):
        parts.append(torch.logsumexp(hd @ w[v:v + (1 << 20)].double().t() + b[v:v + (1 << 20)].double(), 1))
    lse = torch.logsumexp(torch.stack(parts), 0)
    z = (hd * w[y.clamp(min=0)].double()).sum(1) + b[y.clamp(min=0)].double()
    assert loss[1] == 0
    # a score: 66 fp32 steps of its magnitudes' sum; the exponentials' sum: 64 columns in a tree, then 2^21 / 64 pairs one after the
    # other in a lane, rescaled once per eight
    z_err = 66 * R.F32 * (hd.abs().sum(1) * w[:1 << 20].abs().amax().double() + 18)
    err = 2 * z_err + (64 + (1 << 15) * 9 / 8) * R.F32 + 16 * R.F32 * (1 + lse.abs())
    off = (loss.double() - (lse - z))[y >= 0].abs()
    assert (off <= err[y >= 0]).all(), (off.max(), err.min())


# ---------------------------------------------------------------- distillation
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,vocab,hidden,k,temperature", [
    (1, 1, 64, 1, 1.0), (1, 30, 64, 30, 2.0), (3, 65, 128, 7, 0.5), (70, 1000, 128, 64, 2.0), (130, 777, 320, 65, 4.0),
    (33, 2000, 64, 200, 1.0), (300, 3001, 256, 16, 1.5), (9, 1500, 64, 1024, 3.0), (19, 30522, 768, 8, 1.0),
    (300, 30801, 128, 16, 1.5), (1100, 12345, 256, 100, 2.0), (300, 128100, 128, 16, 1.5), (1100, 25701, 256, 100, 2.0)])
def test_distillation_sizes(n, vocab, hidden, k, temperature, dtype):
    h, w, b = R.make(n, vocab, hidden, dtype, n + k)
    values, index = _teacher(n, vocab, k, n)
    p, live, entropy = R.targets_distill(values, index, vocab, temperature)
    _check(h, w, b, lambda h, w, b: losses.linear_distillation(h, w, b, values, index, temperature=temperature), p, live, temperature,
           "mean", 5, entropy)


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,vocab,k", [(150, 400, 12), (300, 30800, 12), (60, 400, 12), (150, 400, 65), (60, 400, 300), (300, 30800, 300),
                                       (300, 128100, 12), (300, 128100, 300)])
def test_distillation_ragged_empty_and_repeated_entries(n, vocab, k, dtype, reduction):
    hidden = 128
    h, w, b = R.make(n, vocab, hidden, dtype, 5)
    values, index = _teacher(n, vocab, k, 6, dropped=0.4)
    index[[0, 17, n - 1]] = -1            # nothing listed
    index[40] = -5
    values[41] = -INF
    values[42, 3:] = -INF
    values[43] = torch.finfo(F32).min     # the lowest finite value everywhere: a uniform teacher
    index[44, :5] = index[44, 5].clamp(min=0)   # one id several times
    index[46, k // 2:] = index[46, :k - k // 2].clone()  # the list twice
    index[47] = 7
    index[45] = vocab - 1
    p, live, entropy = R.targets_distill(values, index, vocab, 2.0)
    assert not live[[0, 17, n - 1, 40, 41]].any()
    h[~live] = NAN
    _, grads = _check(h, w, b, lambda h, w, b: losses.linear_distillation(h, w, b, values, index, temperature=2.0, reduction=reduction),
                      p, live, 2.0, reduction, 9, entropy)
    assert not grads[0][~live].any()


@pytest.mark.parametrize("n,vocab,k", [(30, 100, 4), (100, 100, 4), (300, 30800, 4), (300, 128100, 4), (30, 100, 90)])
def test_distillation_of_bad_entries_is_nan(n, vocab, k):
    h, w, b = R.make(n, vocab, 128, BF16, 5)
    values, index = _teacher(n, vocab, k, 6)
    index[3, 1] = vocab
    values[4, 2] = NAN
    values[5, 0] = INF
    bad = torch.zeros(n, dtype=torch.bool).cuda()
    bad[3:6] = True
    leaves = [t.requires_grad_() for t in (h, w, b)]
    loss = losses.linear_distillation(*leaves, values, index, reduction="none")
    assert torch.equal(loss.isnan(), bad)
    dh, dw, db = torch.autograd.grad(loss.sum(), leaves)
    assert torch.equal(dh.isnan().any(1), bad) and dw.isnan().all() and db.isnan().all()


@pytest.mark.parametrize("k", [1, 100])
def test_distillation_of_no_rows(k):
    h, w, b = (t.requires_grad_() for t in R.make(3, 200, 128, BF16, 5))
    values, index = _teacher(3, 200, k, 6)
    for rows in (0, 3):                       # none at all; none with an entry
        ix = index[:rows].clone().fill_(-1)
        for red in ("mean", "sum", "none"):
            loss = losses.linear_distillation(h[:rows], w, b, values[:rows], ix, reduction=red)
            assert loss.isnan() if red == "mean" else not loss.any()
            grads = torch.autograd.grad(loss.sum(), (h, w, b))
            assert not any(g.any() for g in grads)


def test_distillation_of_itself_is_zero():
    # the teacher lists the whole vocabulary with the student's own scores: loss and gradient vanish up to rounding
    n, vocab, hidden = 40, 60, 64
    h, w, b = R.make(n, vocab, hidden, BF16, 14)
    scores = h.float() @ w.float().t() + b
    values, index = losses.topk_logits(scores, vocab)
    p, live, entropy = R.targets_distill(values, index, vocab, 1.0)
    loss, grads = _check(h, w, b, lambda h, w, b: losses.linear_distillation(h, w, b, values, index, reduction="none"), p, live, 1.0,
                         "none", 3, entropy)
    assert loss.abs().max() < 1e-5 and grads[0].abs().max() < 1e-5


# ---------------------------------------------------------------- a teacher's top scores
def _topk_plain(x, k):
    """by a stable sort of 64-bit values, NaN first"""
    y = x.double()
    y = torch.where(y.isnan(), torch.inf, y)
    order = torch.argsort(torch.where(x.isnan(), 1, 0), dim=-1, descending=True, stable=True)
    first = torch.gather(y, -1, order).argsort(dim=-1, descending=True, stable=True)
    index = torch.gather(order, -1, first)[..., :k]
    return torch.gather(x, -1, index), index


def _same_topk(x, k):
    values, index = losses.topk_logits(x, k)
    want_v, want_i = _topk_plain(x, k)
    assert torch.equal(index, want_i)
    as_int = {F32: torch.int32}.get(x.dtype, torch.int16)
    assert torch.equal(values.contiguous().view(as_int), want_v.contiguous().view(as_int)), "values are the scores' own bits"


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,vocab,k", [(1, 1, 1), (2, 3, 3), (5, 17, 5), (7, 1000, 1000), (3, 255, 256 - 1), (4, 4097, 64), (9, 30522, 10),
                                       (2, 30522, 257), (3, 50001, 1024), (1, 200003, 128), (70, 8192, 1), (5, 300, 100), (5, 301, 128),
                                       (4, 1000, 128), (4, 1030, 64), (6, 1003, 200), (3, 2051, 256), (3, 3000, 1024), (2, 4099, 1024),
                                       (2, 9001, 1024), (2, 16500, 1024), (2, 5000, 700), (2, 17001, 129)])
def test_topk_sizes(n, vocab, k, dtype):
    g = torch.Generator().manual_seed(vocab)
    _same_topk((2.5 * torch.randn(n, vocab, generator=g)).to(dtype).cuda(), k)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("vocab,k", [(20000, 1), (20000, 64), (20000, 300), (20000, 1000), (600, 64), (600, 128), (600, 500), (5000, 700)])
def test_topk_orders_that_fill_the_list(dtype, vocab, k):
    up = torch.linspace(-50, 50, vocab)
    rows = [up, up.flip(0), torch.zeros(vocab), torch.full((vocab,), -INF), torch.full((vocab,), NAN), (torch.arange(vocab) % 7).float(),
            torch.where(torch.arange(vocab) % 2 == 0, 0.0, -0.0), torch.where(torch.arange(vocab) < 100, INF, -INF),
            torch.where(torch.arange(vocab) % 97 == 5, NAN, torch.finfo(F16).min), torch.full((vocab,), torch.finfo(dtype).min)]
    _same_topk(torch.stack(rows).to(dtype).cuda(), k)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_topk_strides_and_shapes(dtype):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(6, 5003, generator=g).to(dtype).cuda()
    for lo in range(9):
        _same_topk(x[:, lo:lo + 4990], 33)
    _same_topk(x.t().contiguous().t(), 5)
    _same_topk(x[::2, ::3], 5)
    v, i = losses.topk_logits(x.view(2, 3, 5003), 4)
    assert v.shape == i.shape == (2, 3, 4) and torch.equal(i.view(6, 4), _topk_plain(x, 4)[1])
    v, i = losses.topk_logits(x[0], 4)
    assert v.shape == (4,)
    v, i = losses.topk_logits(x[:0], 4)
    assert v.shape == i.shape == (0, 4)


@pytest.mark.parametrize("k", [5, 200])
def test_topk_of_the_longest_row(k):
    # 2^31 - 1 scores: ids up to the last of 32 bits
    vocab = (1 << 31) - 1
    x = torch.empty(1, vocab, dtype=F16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(5))
    x[0, [vocab - 1, 0, vocab - 2]] = torch.tensor([9.0, 9.0, 8.0], dtype=F16, device="cuda")
    values, index = losses.topk_logits(x, k)
    parts = [_topk_plain(x[:, i:i + (1 << 24)], k) for i in range(0, vocab, 1 << 24)]
    v = torch.cat([p[0] for p in parts], 1)
    i = torch.cat([p[1] + (at << 24) for at, p in enumerate(parts)], 1)
    want, at = _topk_plain(v, k)          # (parts and their ties are in the order of the ids)
    assert torch.equal(values, want) and torch.equal(index, torch.gather(i, 1, at))
    assert index[0, 0] == 0 and index[0, 1] == vocab - 1


def test_topk_of_more_rows_than_one_grid():
    n = (1 << 24) + 70001
    x = torch.randint(-3, 3, (n, 3), generator=torch.Generator().manual_seed(5), dtype=torch.int8).cuda().to(BF16)
    values, index = losses.topk_logits(x, 1)
    want = x.max(1).values
    first = torch.where(x[:, 0] == want, 0, torch.where(x[:, 1] == want, 1, 2))
    assert torch.equal(values[:, 0], want) and torch.equal(index[:, 0], first)


def test_losses_of_more_tiles_than_one_grid():
    # 2^20 rows of 64 columns over 2^18 + 77 entries: 2^24 tiles and more
    n, vocab, hidden = 1 << 20, (1 << 18) + 77, 64
    h, w, b = R.make(4096, vocab, hidden, BF16, 99)
    y = torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(6)).cuda()
    y[-1] = vocab - 1
    loss = losses.linear_cross_entropy(h.repeat(n // 4096, 1), w, b, y, reduction="none")
    for at in (slice(0, 128), slice(n - 128, n)):
        rows = h[at.start % 4096:at.start % 4096 + 128]
        p, live = R.targets_ce(y[at], vocab, -100)
        (want, *_), (err, *_) = R.reference(rows, w, b, p, live, 1.0, torch.ones(128).cuda())
        R.assert_within("loss", loss[at], want, err)
    # equal hidden rows have equal logsumexps: loss + score is off by the score's 64 fp32 sums (|h| |w| < 16) and the loss's rounding
    z = torch.cat([(h.double() * w.double()[y[i:i + 4096]]).sum(1) + b.double()[y[i:i + 4096]] for i in range(0, n, 4096)])
    lse = (loss.double() + z).view(-1, 4096)
    assert ((lse - lse[0]).abs() <= 2 * (66 * 16 + 32) * R.F32).all()


# ---------------------------------------------------------------- used together, streams, graphs
def test_teacher_to_student_step():
    """a teacher's scores -> its top entries -> the student's distillation and cross entropy on the same rows"""
    n, vocab = 120, 3000
    th, tw, tb = R.make(n, vocab, 256, BF16, 50)
    h, w, b = R.make(n, vocab, 128, BF16, 51)
    y = _labels(n, vocab, 52, 0.3)
    values, index = losses.topk_logits(th.float() @ tw.float().t() + tb, 20)
    leaves = [t.requires_grad_() for t in (h, w, b)]
    total = losses.linear_distillation(*leaves, values, index, temperature=2.0) + 0.5 * losses.linear_cross_entropy(*leaves, y)
    grads = torch.autograd.grad(total, leaves)
    p1, l1, ent = R.targets_distill(values, index, vocab, 2.0)
    p2, l2 = R.targets_ce(y, vocab, -100)
    a, ea = R.reference(h.detach(), w.detach(), b.detach(), p1, l1, 2.0, torch.full((n,), 1 / n).cuda(), ent)
    c, ec = R.reference(h.detach(), w.detach(), b.detach(), p2, l2, 1.0, torch.full((n,), 0.5 / int(l2.sum())).cuda())
    u = R.half_step(BF16)
    for name, got, x, y_, e, f in zip(("dh", "dw", "db"), grads, a[1:], c[1:], ea[1:], ec[1:]):
        R.assert_within(name, got, x + y_, e + f + (u if name != "db" else R.F32) * 1.01 * (x + y_).abs())


@pytest.mark.parametrize("held", [F32, BF16])
def test_decoder_as_a_linear_layer_holds_it(held):
    """the documented use: weight and bias of one type, the other one cast, gradients back in the layer's own type"""
    batch, width, hidden_size, vocab = 3, 20, 128, 900
    torch.manual_seed(7)
    decoder = torch.nn.Linear(hidden_size, vocab).to("cuda", held)
    hidden = torch.randn(batch, width, hidden_size, device="cuda", requires_grad=True)
    mlm_labels = _labels(batch * width, vocab, 8, 0.5).view(batch, width)
    teacher_scores = 2 * torch.randn(batch, width, vocab, device="cuda")
    weight, bias = decoder.weight.to(BF16), decoder.bias.float()
    loss = losses.linear_cross_entropy(hidden.to(BF16), weight, bias, mlm_labels)
    values, index = losses.topk_logits(teacher_scores, 64)
    loss = loss + losses.linear_distillation(hidden.to(BF16), weight, bias, values, index, temperature=2.0)
    loss.backward()
    h, w, b = hidden.detach().to(BF16).view(-1, hidden_size), decoder.weight.detach().to(BF16), decoder.bias.detach().float()
    n, y = batch * width, mlm_labels.view(-1)
    p1, l1 = R.targets_ce(y, vocab, -100)
    p2, l2, ent = R.targets_distill(values.view(n, 64), index.view(n, 64), vocab, 2.0)
    a, ea = R.reference(h, w, b, p1, l1, 1.0, torch.full((n,), 1 / int(l1.sum())).cuda())
    c, ec = R.reference(h, w, b, p2, l2, 2.0, torch.full((n,), 1 / n).cuda(), ent)
    for name, got, x, y_, e, f, u in (("dh", hidden.grad.view(n, -1), a[1], c[1], ea[1], ec[1], R.half_step(BF16)),
                                      ("dw", decoder.weight.grad, a[2], c[2], ea[2], ec[2], R.half_step(BF16)),
                                      ("db", decoder.bias.grad, a[3], c[3], ea[3], ec[3], R.half_step(held))):
        # (the two gradients, each rounded within its own bound, are added in bf16, and kept in the layer's type)
        R.assert_within(name, got, x + y_, e + f + 2.02 * u * (x + y_).abs() + 1.01 * u * (e + f))
    assert hidden.grad.dtype == F32 and decoder.weight.grad.dtype == decoder.bias.grad.dtype == held


@pytest.mark.parametrize("n,vocab", [(500, 3000), (500, 31000), (500, 128100), (50, 3000)])
def test_other_stream(n, vocab):
    h, w, b = R.make(n, vocab, 128, BF16, 60)
    y = _labels(n, vocab, 61)
    leaves = [t.requires_grad_() for t in (h, w, b)]
    want = torch.autograd.grad(losses.linear_cross_entropy(*leaves, y), leaves)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for s in (s1, s2, s1, s2):      # calls side by side: each has its own workspace
        with torch.cuda.stream(s):
            got.append(torch.autograd.grad(losses.linear_cross_entropy(*leaves, y), leaves))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_calls_from_several_threads():
    from concurrent.futures import ThreadPoolExecutor
    cases = []
    for n, vocab in ((40, 3000), (300, 2000), (1, 500), (600, 31000)):
        h, w, b = R.make(n, vocab, 128, BF16, n)
        y, (values, index) = _labels(n, vocab, n, 0.2), _teacher(n, vocab, 9, n)
        y[0] = 5
        cases.append((h, w, b, y, values, index))

    def step(case):
        h, w, b, y, values, index = case
        with torch.cuda.stream(torch.cuda.Stream()):
            leaves = [t.detach().requires_grad_() for t in (h, w, b)]
            ce = losses.linear_cross_entropy(*leaves, y)
            kd = losses.linear_distillation(*leaves, values, index, reduction="sum")
            out = (ce.detach(), kd.detach(), *torch.autograd.grad(ce, leaves), *torch.autograd.grad(kd, leaves), *losses.topk_logits(w, 5))
            torch.cuda.current_stream().synchronize()
        return out
    torch.cuda.synchronize()
    want = [step(c) for c in cases]
    with ThreadPoolExecutor(4) as pool:
        for _ in range(3):
            for got, ref in zip(pool.map(step, cases), want):
                assert all(torch.equal(x, r) for x, r in zip(got, ref))


def test_empty_shapes_and_inference_mode():
    h, w, b = R.make(6, 300, 128, BF16, 5)
    y = _labels(6, 300, 6)
    with torch.inference_mode():
        assert torch.equal(losses.linear_cross_entropy(h, w, b, y, reduction="none"),
                           losses.linear_cross_entropy(h.clone(), w.clone(), b.clone(), y.clone(), reduction="none"))
    empty = h[:0].view(2, 0, 128)
    assert losses.linear_cross_entropy(empty, w, b, y[:0].view(2, 0), reduction="none").shape == (2, 0)
    values, index = _teacher(0, 300, 4, 1)
    assert losses.linear_distillation(empty, w, b, values.view(2, 0, 4), index.view(2, 0, 4), reduction="none").shape == (2, 0)
    v, i = losses.topk_logits(w.view(3, 100, 128)[:, :0], 2)
    assert v.shape == i.shape == (3, 0, 2)


@pytest.mark.parametrize("n,vocab", [(90, 1111), (50, 1111), (400, 31111), (400, 128111), (4200, 4000)])
def test_captured_step_replays(n, vocab):
    hidden = 128
    h, w, b = R.make(n, vocab, hidden, BF16, 70)
    y = _labels(n, vocab, 71, 0.3)
    values, index = _teacher(n, vocab, 9, 72)
    leaves = [t.requires_grad_() for t in (h, w, b)]

    def step():
        loss = losses.linear_cross_entropy(*leaves, y)
        kd = losses.linear_distillation(*leaves, values, index, temperature=2.0)
        top = losses.topk_logits(b.detach().view(1, -1), 5)
        return (loss.detach(), kd.detach(), *torch.autograd.grad(loss, leaves), *torch.autograd.grad(kd, leaves), *top)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (80, 81, 82, 83):
        h2, w2, b2 = R.make(n, vocab, hidden, BF16, seed)
        with torch.no_grad():
            h.copy_(h2), w.copy_(w2), b.copy_(b2)
            y.copy_(_labels(n, vocab, seed, 0.5 if seed % 2 else 1.1))
            index.copy_(_teacher(n, vocab, 9, seed, 0.3)[1])
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        for got, want in zip(kept, step()):
            assert torch.equal(got, want) or (got.isnan().all() and want.isnan().all())


def test_capture_beside_a_living_eager_loss_is_refused():
    h, w, b = R.make(40, 300, 64, BF16, 70)
    y = _labels(40, 300, 71)
    h.requires_grad_()
    alive = losses.linear_cross_entropy(h, w, b, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="let go of eager losses"):
        with torch.cuda.graph(graph, stream=side):
            losses.linear_cross_entropy(h, w, b, y)
    want, = torch.autograd.grad(alive, h)
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got, = torch.autograd.grad(losses.linear_cross_entropy(h, w, b, y), h)
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_compiled_caller():
    # torch.compile leaves the calls outside its graphs: the same bits
    h, w, b = R.make(66, 333, 128, BF16, 1)
    y = _labels(66, 333, 2)

    def step(h, w, b):
        return 3 * losses.linear_cross_entropy((2 * h).relu(), w, b, y)
    leaves = [t.requires_grad_() for t in (h, w, b)]
    want = step(*leaves)
    got = torch.compile(step, backend="eager")(*leaves)
    assert torch.equal(got, want)
    assert all(torch.equal(x, r) for x, r in zip(torch.autograd.grad(got, leaves), torch.autograd.grad(want, leaves)))


def test_backward_accumulates_and_repeats():
    """.backward() into .grad, twice over one graph, and a weight shared by two losses"""
    h, w, b = R.make(60, 500, 128, BF16, 90)
    y = _labels(60, 500, 91, 0.2)
    h, w, b = (t.requires_grad_() for t in (h, w, b))
    loss = losses.linear_cross_entropy(h, w, b, y)
    loss.backward(retain_graph=True)
    first = [t.grad.clone() for t in (h, w, b)]
    loss.backward()
    assert all(torch.equal(t.grad, 2 * g) for t, g in zip((h, w, b), first))
    two = losses.linear_cross_entropy(h, w, b, y) + losses.linear_cross_entropy(h[:30], w, b, y[:30], reduction="sum")
    sep = torch.autograd.grad(losses.linear_cross_entropy(h[:30], w, b, y[:30], reduction="sum"), w)[0]
    assert torch.equal(torch.autograd.grad(two, w)[0], (first[1] + sep))


@pytest.mark.parametrize("up", [0.0, -2.0, 65536.0, 1e-30])
@pytest.mark.parametrize("n,vocab", [(90, 700), (40, 700), (300, 30800), (300, 128100)])
def test_upstream_gradients(n, vocab, up):
    h, w, b = R.make(n, vocab, 128, BF16, 40)
    y = _labels(n, vocab, 41)
    p, live = R.targets_ce(y, vocab, -100)
    leaves = [t.clone().requires_grad_() for t in (h, w, b)]
    for red in ("sum", "none"):
        loss = losses.linear_cross_entropy(*leaves, y, reduction=red)
        g = torch.full_like(loss, up)
        if red == "none":
            g[::3] *= -1
            g[7] = 0
        rows = g if red == "none" else g.expand(n)
        want, err = R.reference(h, w, b, p, live, 1.0, rows)
        for name, got, a, e in zip(("dh", "dw", "db"), torch.autograd.grad(loss, leaves, g), want[1:], err[1:]):
            R.assert_within(name, got, a, e)
    # an infinite or NaN gradient shows
    for bad in (INF, NAN):
        loss = losses.linear_cross_entropy(*leaves, y)
        assert not any(t.isfinite().all() for t in torch.autograd.grad(loss, leaves, torch.tensor(bad).cuda()))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,vocab", [(40, 700), (90, 700), (300, 128100)])
def test_rows_weighted_over_a_wide_range(n, vocab, dtype):
    """upstream gradients from 2^14 down to 2^-16 (whose dh both types still hold as normal numbers): fp16 score gradients are no
    finer than 2^-40 of the largest, as R.reference has it; rows of 2^-20 of it and more are as exact as the largest"""
    h, w, b = R.make(n, vocab, 128, dtype, 47)
    y = _labels(n, vocab, 48)
    p, live = R.targets_ce(y, vocab, -100)
    up = 2.0 ** (14 - torch.tensor([0, 10, 20, 24, 30]).repeat(n // 5)).cuda()
    leaves = [t.clone().requires_grad_() for t in (h, w, b)]
    got = torch.autograd.grad(losses.linear_cross_entropy(*leaves, y, reduction="none"), leaves, up)
    want, err = R.reference(h, w, b, p, live, 1.0, up)
    for name, g, a, e in zip(("dh", "dw", "db"), got, want[1:], err[1:]):
        if g.dtype == F16:      # 2^14 |h| of a label's row beyond 4: more than the type's 65 504 is infinite
            a = torch.where(a.abs() < 65520, a, a.sign() * INF)
        R.assert_within(name, g, a, e)
    # rows 2^0, 2^-10 and 2^-20: dh's own rounding (half a step of each value), what 2^-40 an entry comes to where all of a
    # row's entries are off by it, and the relative rounding of the entries
    u = R.half_step(dtype)
    wide = (torch.arange(n) % 5 < 3).cuda()
    q = torch.softmax(h.double() @ w.double().t() + b.double(), 1)
    dz = (up.double()[:, None] * (q - p)).abs()
    each = (2 * u * dz) @ w.double().abs() + (2.0 ** -40 * 2.0 ** 14 if dtype == F16 else 0.0) * w.double().abs().sum(0)
    assert ((got[0].double() - want[1]).abs() <= each + 2 * u * want[1].abs() + R.TINY[dtype])[wide].all()


@pytest.mark.parametrize("n,vocab,hidden", [(40, 701, 128), (130, 701, 128), (300, 30803, 128), (300, 128101, 128), (1300, 15003, 384)])
def test_bias_on_four_bytes(n, vocab, hidden):
    # (the 256-row tiles fetch it 16 bytes at a time)
    h, w, b = R.make(n, vocab, hidden, BF16, 49)
    y = _labels(n, vocab, 50, 0.1)
    leaves = [t.clone().requires_grad_() for t in (h, w, b)]
    loss = losses.linear_cross_entropy(*leaves, y)
    want = (loss.detach(), *torch.autograd.grad(loss, leaves))
    for at in (1, 2, 3):
        flat = torch.full((vocab + 8,), NAN, device="cuda")
        flat[at:at + vocab] = b
        bias = flat[at:at + vocab].requires_grad_()
        assert bias.data_ptr() % 16 == 4 * at
        loss = losses.linear_cross_entropy(leaves[0], leaves[1], bias, y)
        got = (loss.detach(), *torch.autograd.grad(loss, (leaves[0], leaves[1], bias)))
        assert all(torch.equal(g, r) for g, r in zip(got, want))


@pytest.mark.parametrize("n,vocab,hidden,dtype", [(300, 2301, 8192, BF16), (600, 5003, 4096, F16), (1100, 900, 2176, BF16)])
def test_wide_hidden_on_the_large_tiles(n, vocab, hidden, dtype):
    h, w, b = R.make(n, vocab, hidden, dtype, 51, spread=0.02)
    y = _labels(n, vocab, 52, 0.1)
    p, live = R.targets_ce(y, vocab, -100)
    _check(h, w, b, lambda h, w, b: losses.linear_cross_entropy(h, w, b, y), p, live, 1.0, "mean", 5)


@pytest.mark.parametrize("k", [0, 6])
def test_large_tiles_of_rows_far_apart(k):
    # a weight whose rows lie 90 000 elements apart (4.3 GB in all): pieces as 32-bit byte offsets allow, on the 256-row tiles
    n, vocab, hidden, ld, T = 2600, 24001, 128, 90000, 1.5 if k else 1.0
    h, w, b = R.make(n, vocab, hidden, BF16, 53)
    far = torch.empty(vocab, ld, dtype=BF16, device="cuda")[:, :hidden]
    far.copy_(w)
    if k:
        values, index = _teacher(n, vocab, k, 54, 0.1)
        p, live, entropy = R.targets_distill(values, index, vocab, T)
    else:
        y = _labels(n, vocab, 55, 0.2)
        (p, live), entropy = R.targets_ce(y, vocab, -100), None
    leaves = [h.clone().requires_grad_(), far.requires_grad_(), b.clone().requires_grad_()]
    loss = (losses.linear_distillation(*leaves, values, index, temperature=T, reduction="none") if k else
            losses.linear_cross_entropy(*leaves, y, reduction="none"))
    grads = torch.autograd.grad(loss.sum(), leaves)
    want, err = R.reference(h, w, b, p, live, T, torch.ones(n).cuda(), entropy)
    for name, got, a, e in zip(("loss", "dh", "dw", "db"), (loss.detach(), *grads), want, err):
        R.assert_within(name, got, a, e)


@pytest.mark.parametrize("n,vocab,hidden,k", [((1 << 21) - 1, 300, 64, 0), ((1 << 21) - 1, 300, 64, 3), (200001, 300, 8192, 0), (261887, 129, 8192, 0)])
def test_as_many_rows_as_are_allowed(n, vocab, hidden, k):
    """fewer than 2^21 rows and (n + 256) hidden < 2^31: loss, dh, dW and db against 64 bits, 2^15 rows at a time"""
    T, step = 2.0 if k else 1.0, 1 << 15
    base, w, b = R.make(step, vocab, hidden, BF16, 96, spread=0.02)
    h = base.repeat(-(-n // step), 1)[:n].contiguous()
    if k:
        values, index = (t.repeat(-(-n // step), 1)[:n].contiguous() for t in _teacher(step, vocab, k, 97, 0.3))
    else:
        y = _labels(n, vocab, 98, 0.4)
    leaves = [t.requires_grad_() for t in (h, w, b)]
    loss = (losses.linear_distillation(*leaves, values, index, temperature=T, reduction="none") if k else
            losses.linear_cross_entropy(*leaves, y, reduction="none"))
    dh, dw, db = torch.autograd.grad(loss, leaves, torch.ones(n, device="cuda"))
    h, w, b = (t.detach() for t in leaves)
    u, wd = R.half_step(BF16), w.double()
    want_w, each_w, size_w = (torch.zeros(vocab, hidden, dtype=torch.float64, device="cuda") for _ in range(3))
    want_b, each_b, size_b = (torch.zeros(vocab, dtype=torch.float64, device="cuda") for _ in range(3))
    for i in range(0, n, step):
        at = slice(i, min(i + step, n))
        if k:
            p, live, entropy = R.targets_distill(values[at], index[at], vocab, T)
        else:
            (p, live), entropy = R.targets_ce(y[at], vocab, -100), None
        if i < 2 * step or at.stop == n:
            want, err = R.reference(h[at], w, b, p, live, T, torch.ones(len(p), device="cuda"), entropy)
            R.assert_within("loss", loss[at], want[0], err[0])
            R.assert_within("dh", dh[at], want[1], err[1])
        # dW and db as R.reference has them, the sums' errors over all rows
        hd = h[at].double()
        z = (hd @ wd.t() + b.double()) / T
        lse = torch.logsumexp(z, 1)
        mag = z.abs().amax(1) + lse.abs()
        z_err = ((hidden + 2) * R.F32 * (hd.abs() @ wd.abs().t() + b.abs()) / T).amax(1) + 8 * R.F32 * mag
        q = (z - lse[:, None]).exp() * live[:, None]
        dz, s = T * (q - p), T * (q + p)
        dz_err = (2 * z_err + (16 + vocab / 64) * R.F32)[:, None] * s
        want_w += dz.t() @ hd
        each_w += (dz_err + u * dz.abs()).t() @ hd.abs()
        size_w += s.t() @ hd.abs()
        want_b += dz.sum(0)
        each_b += dz_err.sum(0)
        size_b += s.sum(0)
    R.assert_within("dw", dw, want_w, each_w + n * R.F32 * size_w + 1.01 * u * want_w.abs() + R.TINY[BF16])
    R.assert_within("db", db, want_b, each_b + (n + 4) * R.F32 * size_b + n * 2.0 ** -38 * T)


def test_ignore_index_inside_the_vocabulary():
    n, vocab = 300, 260
    h, w, b = R.make(n, vocab, 128, BF16, 44)
    y = _labels(n, vocab, 45)
    y[::3] = 5
    p, live = R.targets_ce(y, vocab, 5)
    assert not live.all()
    _check(h, w, b, lambda h, w, b: losses.linear_cross_entropy(h, w, b, y, ignore_index=5), p, live, 1.0, "mean", 5)


# ---------------------------------------------------------------- the C ABI itself
@pytest.mark.parametrize("n,vocab,hidden,ld_dh,ld_dw,k", [(50, 300, 64, 71, 68, 0), (100, 1000, 128, 128, 132, 5), (300, 1111, 128, 129, 136, 0),
                                                          (700, 4000, 384, 384, 388, 70), (1500, 257, 128, 128, 128, 0),
                                                          (300, 31111, 128, 129, 136, 0), (700, 24001, 128, 128, 132, 70), (5000, 3300, 128, 128, 128, 0), (4100, 257, 128, 128, 128, 3),
                                                          (300, 128111, 128, 129, 136, 0), (700, 85501, 128, 128, 132, 70)])
def test_c_abi_writes_only_its_outputs(n, vocab, hidden, ld_dh, ld_dw, k):
    """Row strides of the outputs, a workspace of exactly the size asked for and full of NaN, and untouched bytes around
    every output and behind the workspace; the same bits as the Python call."""
    import ctypes as C
    from clip_amd import _lib
    lib = _lib.load()
    h, w, b = R.make(n, vocab, hidden, BF16, 17)
    y = _labels(n, vocab, 18, 0.1)
    values, index = _teacher(n, vocab, max(k, 1), 19, 0.2)
    leaves = [t.clone().requires_grad_() for t in (h, w, b)]
    loss = losses.linear_distillation(*leaves, values, index, temperature=2.0) if k else losses.linear_cross_entropy(*leaves, y)
    want = torch.autograd.grad(loss, leaves)
    d = _lib.ClipLinear(_lib.PRECISION_BF16, n, hidden, vocab, h.data_ptr(), hidden, w.data_ptr(), hidden, b.data_ptr())
    GUARD = 4096

    def guarded(nbytes):
        t = torch.full((nbytes + 2 * GUARD,), 0xA5, dtype=torch.uint8, device="cuda")
        return t, t.data_ptr() + GUARD

    def intact(t, nbytes):
        return bool((t[:GUARD] == 0xA5).all()) and bool((t[GUARD + nbytes:] == 0xA5).all())
    st = torch.cuda.current_stream().cuda_stream
    need = C.c_int64()
    bufs = {}
    for name, size in (("row", 4 * n), ("lse", 8 * n), ("target", 4 * n * (2 * k + 1)), ("loss", 4), ("dh", 2 * n * ld_dh), ("dw", 2 * vocab * ld_dw),
                       ("db", 4 * vocab)):
        bufs[name] = (*guarded(size), size)
    at = {name: v[1] for name, v in bufs.items()}
    one = torch.ones((), device="cuda")
    for grad in (0, 1):
        _lib.check(lib.clip_linear_loss_workspace(C.byref(d), k, grad, C.byref(need)))
        work, base = guarded(need.value)
        work[GUARD:GUARD + need.value] = 0xFF          # NaN in every type
        if not grad:
            tail = (1, at["row"], at["lse"], at["target"], at["loss"], base, need.value, st)
            rc = lib.clip_linear_distill(C.byref(d), values.data_ptr(), index.data_ptr(), k, 2.0, *tail) if k else \
                lib.clip_linear_ce(C.byref(d), y.data_ptr(), -100, *tail)
        else:
            tail = (1, at["lse"], at["target"], one.data_ptr(), at["dh"], ld_dh, at["dw"], ld_dw, at["db"], base, need.value, st)
            rc = lib.clip_linear_distill_grad(C.byref(d), index.data_ptr(), k, 2.0, *tail) if k else \
                lib.clip_linear_ce_grad(C.byref(d), y.data_ptr(), -100, *tail)
        _lib.check(rc)
        torch.cuda.synchronize()
        assert intact(work, need.value)
    assert all(intact(t, size) for t, _, size in bufs.values())

    def rows(name, dtype, ld, cols):
        t, _, size = bufs[name]
        m = t[GUARD:GUARD + size].view(torch.int16).view(-1, ld)
        assert (m[:, cols:] == torch.tensor(0xA5A5 - 0x10000, dtype=torch.int16)).all(), name
        return m[:, :cols].contiguous().view(dtype)
    assert torch.equal(rows("dh", BF16, ld_dh, hidden), want[0]) and torch.equal(rows("dw", BF16, ld_dw, hidden), want[1])
    assert torch.equal(bufs["db"][0][GUARD:GUARD + 4 * vocab].view(F32), want[2])
    assert torch.equal(bufs["loss"][0][GUARD:GUARD + 4].view(F32)[0], loss.detach())
    # one output at a time
    for name in ("dh", "dw", "db"):
        bufs[name][0][GUARD:GUARD + bufs[name][2]] = 0xA5
        a = {x: (at[x] if x == name else None) for x in ("dh", "dw", "db")}
        tail = (1, at["lse"], at["target"], one.data_ptr(), a["dh"], ld_dh, a["dw"], ld_dw, a["db"], base, need.value, st)
        rc = lib.clip_linear_distill_grad(C.byref(d), index.data_ptr(), k, 2.0, *tail) if k else \
            lib.clip_linear_ce_grad(C.byref(d), y.data_ptr(), -100, *tail)
        _lib.check(rc)
    torch.cuda.synchronize()
    # dh and dW: the split of their long sums depends on what shares the workgroups, so a value may round to its neighbour
    for name, ld, ref in (("dh", ld_dh, want[0]), ("dw", ld_dw, want[1])):
        off = (rows(name, BF16, ld, hidden).float() - ref.float()).abs()
        assert (off <= 2 * R.half_step(BF16) * ref.float().abs() + 1e-6).all()
    assert torch.equal(bufs["db"][0][GUARD:GUARD + 4 * vocab].view(F32), want[2])


@pytest.mark.parametrize("k", [0, 5])
def test_c_abi_workspace_of_several_pieces(k):
    """a loss and its gradients whose pairs and score gradients are beyond one piece's bound: nothing is written behind a workspace
    of exactly the size asked for, full of NaN before; dbias, which is summed piece by piece, against 64 bits"""
    import ctypes as C
    from clip_amd import _lib
    lib = _lib.load()
    n, vocab, hidden, T = 1 << 17, 70001, 128, 2.0 if k else 1.0
    h, w, b = R.make(n, vocab, hidden, BF16, 93)
    if k:
        values, index = (t.repeat(n // 1024, 1) for t in _teacher(1024, vocab, k, 94, 0.2))
        index[::5] = -1
    else:
        y = _labels(n, vocab, 95, 0.4)
    d = _lib.ClipLinear(_lib.PRECISION_BF16, n, hidden, vocab, h.data_ptr(), hidden, w.data_ptr(), hidden, b.data_ptr())
    new = lambda *shape, dtype=F32: torch.empty(*shape, dtype=dtype, device="cuda")  # noqa: E731
    row, lse, target, total = new(n), new(n, 2), new(n, 2 * k + 1), new(())
    dh, dw, db = new(n, hidden, dtype=BF16), new(vocab, hidden, dtype=BF16), new(vocab)
    up = torch.ones((), device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    for grad in (0, 1):
        need = C.c_int64()
        _lib.check(lib.clip_linear_loss_workspace(C.byref(d), k, grad, C.byref(need)))
        work = torch.full((need.value + 8192,), 0xFF, dtype=torch.uint8, device="cuda")
        at = work.data_ptr() + 4096
        if not grad:
            tail = (2, row.data_ptr(), lse.data_ptr(), target.data_ptr(), total.data_ptr(), at, need.value, st)
            _lib.check(lib.clip_linear_distill(C.byref(d), values.data_ptr(), index.data_ptr(), k, T, *tail) if k else
                       lib.clip_linear_ce(C.byref(d), y.data_ptr(), -100, *tail))
        else:
            tail = (2, lse.data_ptr(), target.data_ptr(), up.data_ptr(), dh.data_ptr(), hidden, dw.data_ptr(), hidden, db.data_ptr(), at,
                    need.value, st)
            _lib.check(lib.clip_linear_distill_grad(C.byref(d), index.data_ptr(), k, T, *tail) if k else
                       lib.clip_linear_ce_grad(C.byref(d), y.data_ptr(), -100, *tail))
        torch.cuda.synchronize()
        assert (work[:4096] == 0xFF).all() and (work[4096 + need.value:] == 0xFF).all()
        del work
    leaves = [t.clone().requires_grad_() for t in (h, w, b)]
    loss = (losses.linear_distillation(*leaves, values, index, temperature=T, reduction="sum") if k else
            losses.linear_cross_entropy(*leaves, y, reduction="sum"))
    assert torch.equal(loss.detach(), total)
    for got, want in zip((dh, dw, db), torch.autograd.grad(loss, leaves)):
        assert torch.equal(got, want)
    # db = T sum (q - p): bounds as R.reference makes them, its sums taken over all rows
    want, each, size = (torch.zeros(vocab, dtype=torch.float64, device="cuda") for _ in range(3))
    for i in range(0, n, 4096):
        part = slice(i, i + 4096)
        p, live = R.targets_distill(values[part], index[part], vocab, T)[:2] if k else R.targets_ce(y[part], vocab, -100)
        z = (h[part].double() @ w.double().t() + b.double()) / T
        lse_ = torch.logsumexp(z, 1)
        mag = z.abs().amax(1) + lse_.abs()
        z_err = ((hidden + 2) * R.F32 * (h[part].double().abs() @ w.double().abs().t() + b.abs()) / T).amax(1) + 8 * R.F32 * mag
        q = (z - lse_[:, None]).exp() * live[:, None]
        want += T * (q - p).sum(0)
        s = T * (q + p)
        each += ((2 * z_err + (16 + vocab / 64) * R.F32)[:, None] * s).sum(0)
        size += s.sum(0)
    R.assert_within("db", db, want, each + (n + 4) * R.F32 * size + n * 2.0 ** -38 * T)


# ---------------------------------------------------------------- refusals
def test_refusals():
    h, w, b = R.make(4, 10, 64, BF16, 1)
    y = torch.zeros(4, dtype=torch.int64).cuda()
    ce, kd, top = losses.linear_cross_entropy, losses.linear_distillation, losses.topk_logits
    v, i = _teacher(4, 10, 3, 1)
    for err, call in [
            (TypeError, lambda: ce(h.float(), w.float(), b, y)), (TypeError, lambda: ce(h, w.half(), b, y)),
            (TypeError, lambda: ce(h, w, b.bfloat16(), y)), (TypeError, lambda: ce(h, w, b[:9], y)),
            (ValueError, lambda: ce(h[:, :32], w, b, y)), (ValueError, lambda: ce(h, w, b, y[:3])),
            (ValueError, lambda: ce(h, w, b, y.float())), (ValueError, lambda: ce(h, w, b, y, reduction="batchmean")),
            (RuntimeError, lambda: ce(h, w, b, y.cpu())), (RuntimeError, lambda: ce(h, w.cpu(), b, y)),
            (ValueError, lambda: ce(h[:, :32].contiguous(), w[:, :32].contiguous(), b, y)),
            (ValueError, lambda: kd(h, w, b, v, i, temperature=0.0)), (ValueError, lambda: kd(h, w, b, v, i, temperature=float("nan"))),
            (ValueError, lambda: kd(h, w, b, v, i.int())), (ValueError, lambda: kd(h, w, b, v[:, :2], i)),
            (ValueError, lambda: kd(h, w, b, v[:, :0], i[:, :0])), (ValueError, lambda: kd(h, w, b, v[:3], i[:3])),
            (ValueError, lambda: top(w, 0)), (ValueError, lambda: top(w, 65)), (TypeError, lambda: top(i, 2))]:
        with pytest.raises(err):
            call()
    leaf = h.requires_grad_()
    g, = torch.autograd.grad(ce(leaf, w, b, y), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.float().sum(), leaf)

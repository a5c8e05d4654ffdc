"""ops.distill_loss and its gradient against the formula in 64 bits.

Tolerances, u = 2^-24. An exponential exp((x - m) / T) of an argument of magnitude r is off by at most (2 r + 4) u of itself
(the rounded difference and product, the hardware's exponential); a sum of positive terms over at least 64 lanes by (V / 64 + 40) u. With
R the largest r of a row, a softmax value of the student is off by at most k = (4 R + V / 64 + 50) u of itself, one of the teacher's
by kt = (4 Rt + K + 50) u; logarithms of sums by the sums' relative error, and every sum of the loss's few terms by 8 u of the
magnitudes that meet in it. Results are rounded once more, half a step of their type; gradients below fp16's normal range by 2^-25, and
below fp32's by 2^-126 (the hardware's exponential gives zero there)."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24
INF = float("inf")


def reference(x, index, teacher, targets, tau, weight, ignore, upstream):
    """(row losses, their allowed errors, gradient of sum(upstream * rows), its allowed error before the last rounding), 64 bits, CPU."""
    x, index, t = x.detach().double().cpu(), index.cpu().long(), teacher.double().cpu()
    rows, vocab = x.shape
    up = upstream.double().cpu().expand(rows)
    counted = torch.ones(rows, dtype=torch.bool) if targets is None else targets.cpu().long() != ignore
    t = torch.where(index < 0, -INF, t)
    taught = (t.amax(1) > -INF) & (weight > 0)
    t = torch.where(taught[:, None], t, 0.0) / tau
    t = t - t.amax(1, keepdim=True)
    zt = t.exp().sum(1, keepdim=True)
    p = torch.where(taught[:, None], t.exp() / zt, 0.0)
    at = index.clamp(min=0)
    xm = x - x.amax(1, keepdim=True)

    def soft(tau):
        z = (xm / tau).exp().sum(1, keepdim=True)
        r = torch.where(xm > -INF, -xm / tau, 0.0).amax(1, keepdim=True)
        return xm / tau - z.log(), (4 * r + vocab / 64 + 50) * U

    lq, k = soft(tau)
    kt = (4 * torch.where(t > -INF, -t, 0.0).amax(1, keepdim=True) + t.shape[1] + 50) * U
    lp = t - zt.log()
    used = p > 0
    diff = torch.where(used, lp - lq.gather(1, at), 0.0)
    mags = torch.where(used, lp.abs() + lq.gather(1, at).abs() + 2 * lq.amax(1, keepdim=True).abs() + 2 * zt.log(), 0.0)
    row = weight * tau ** 2 * (p * diff).sum(1)
    err = weight * tau ** 2 * (p * (mags * (8 * U + kt) + kt + k + 4 * U)).sum(1)
    g = torch.where(taught[:, None], weight * tau * lq.exp(), 0.0)
    g_err = g * (2 * k + 8 * U)
    off = torch.zeros_like(g).scatter_add_(1, at, weight * tau * p)
    g, g_err = g - off, g_err + off * (kt + 8 * U)
    if weight < 1:
        y = torch.where(counted, targets.cpu().long(), 0)[:, None]
        lq, k = soft(1.0)
        row = row - (1 - weight) * lq.gather(1, y)[:, 0]
        err = err + (1 - weight) * ((8 * U) * (lq.gather(1, y).abs() + lq.amax(1, keepdim=True).abs()) + k + 4 * U)[:, 0]
        g = g + (1 - weight) * (lq.exp() - torch.zeros_like(g).scatter_(1, y, 1.0))
        g_err = g_err + (1 - weight) * (lq.exp() * (2 * k + 8 * U) + torch.zeros_like(g).scatter_(1, y, 8 * U))
    zero = torch.zeros((), dtype=torch.float64)
    c, u = counted, up[:, None]
    return torch.where(c, row, zero), torch.where(c, err, zero), torch.where(c[:, None], g * u, zero), torch.where(c[:, None], g_err * u.abs(), zero)


def near(got, want, err, what):
    assert got.shape == want.shape, what
    allowed = err + torch.finfo(got.dtype).eps / 2 * (want.abs() + err) * (1 + 2.0 ** -10) + (2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -125)
    got = got.detach().cpu().double()
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]) and torch.isfinite(got[~inf]).all(), what
    off = (got - want).abs()[~inf]
    assert (off <= allowed[~inf]).all(), f"{what}: off by {float((off - allowed[~inf]).max()):.3g} more than allowed"


def make(rows, vocab, k, dtype, seed, index=torch.int64, teacher="fp32", ignored=0.0, std=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g) * std).to(DT[dtype])
    idx = torch.stack([torch.randperm(vocab, generator=g)[:k] for _ in range(rows)]) if k <= vocab else torch.randint(0, vocab, (rows, k), generator=g)
    t = (torch.randn(rows, k, generator=g) * 2).sort(1, descending=True).values.to(DT[teacher])
    y = torch.where(torch.rand(rows, generator=g) < 0.6, idx[:, 0], torch.randint(0, vocab, (rows,), generator=g))
    y[torch.rand(rows, generator=g) < ignored] = -100
    return x.to(DEV), idx.to(index).to(DEV), t.to(DEV), y.to(index).to(DEV)


def check(x, idx, t, y, tau, weight, reduction="mean", scale=1.0, ignore=-100):
    from tandem_amd import ops

    how = dict(targets=y, temperature=tau, weight=weight, ignore_index=ignore, reduction=reduction)
    count = 1
    if reduction == "mean":
        count = x.shape[0] if y is None else max(1, int((y != ignore).sum()))
    row, err, g, g_err = reference(x, idx, t, y, tau, weight, ignore, torch.tensor(scale / count, dtype=torch.float64))
    loss, grad = ops.distill_loss_and_grad(x, idx, t, scale=scale, **how)
    near(grad, g, g_err + 4 * U * g.abs(), "gradient")
    alone = ops.distill_loss(x, idx, t, **how)  # a few long rows are split over their length: the sums' order may differ
    assert not alone.requires_grad
    for got in (loss, alone):
        if reduction == "none":
            near(got, row, err, "loss")
        else:
            near(got, row.sum() / count, (err.sum() + len(row) * U * row.abs().sum()) / count, "loss")
    assert torch.equal(alone, ops.distill_loss(x, idx, t, **how))
    again = ops.distill_loss_and_grad(x, idx, t, scale=scale, **how)
    assert torch.equal(loss, again[0]) and torch.equal(grad, again[1])
    return loss, grad


SIZES = [  # rows, vocab, k, dtype, columns, teacher
    (5, 1, 1, "fp32", torch.int64, "fp32"),
    (3, 2, 2, "bf16", torch.int32, "fp32"),
    (7, 7, 9, "fp16", torch.int64, "bf16"),
    (66, 63, 5, "bf16", torch.int64, "fp16"),
    (64, 256, 16, "fp32", torch.int64, "fp32"),
    (130, 256, 16, "bf16", torch.int64, "fp32"),
    (33, 257, 33, "fp16", torch.int32, "fp32"),
    (20, 1021, 64, "bf16", torch.int64, "bf16"),
    (20, 2048, 64, "fp32", torch.int64, "fp32"),
    (9, 4096, 65, "bf16", torch.int64, "fp32"),
    (9, 8191, 100, "fp32", torch.int64, "fp32"),
    (5, 16384, 256, "bf16", torch.int64, "fp32"),
    (5, 16391, 1024, "fp16", torch.int32, "fp32"),
    (4, 32003, 64, "bf16", torch.int64, "fp32"),
    (3, 50021, 33, "fp16", torch.int64, "fp32"),
    (3, 65536, 33, "fp32", torch.int64, "fp32"),
    (3, 65537, 33, "fp32", torch.int64, "fp32"),
    (2, 131072, 64, "bf16", torch.int64, "fp32"),
    (3, 131079, 64, "bf16", torch.int64, "fp32"),
    (2, 300000, 10, "fp32", torch.int64, "fp32"),
    (1200, 5000, 12, "bf16", torch.int64, "fp32"),
]


@pytest.mark.parametrize("tau,weight", [(1.0, 1.0), (2.0, 0.5), (1.0, 0.3), (1.5, 1.0), (0.5, 0.9), (2.0, 0.0)])
@pytest.mark.parametrize("rows,vocab,k,dtype,index,teacher", SIZES)
def test_loss_and_gradient(rows, vocab, k, dtype, index, teacher, tau, weight):
    x, idx, t, y = make(rows, vocab, k, dtype, 1, index, teacher, ignored=0.2 if weight < 1 else 0.0)
    check(x, idx, t, y if weight < 1 else None, tau, weight, scale=1024.0 if dtype == "fp16" else 1.0)


@pytest.mark.parametrize("tau", [0.75, 1.5, 1.7, 2.0])
@pytest.mark.parametrize("rows,vocab,k,dtype,index,teacher", [s for s in SIZES if s[1] > 2])
def test_two_temperatures_and_a_negative_scale(rows, vocab, k, dtype, index, teacher, tau):
    """Temperatures whose exponentials are powers of one, and others. A third power is off by three times 2 r / 3 + 2 (the hardware's
    exponential) and its two products, (2 r + 8) u: 4 u more than counted above, of the 40 u that sums have beyond V / 64, 20 of
    which no sum here needs (6 steps over lanes, 4 over waves, a vector's 8 and a step of the maximum's)."""
    x, idx, t, y = make(rows, vocab, k, dtype, 11, index, teacher, ignored=0.2)
    check(x, idx, t, y, tau, 0.4, "sum", scale=-64.0)
    x[0, vocab // 2] = 4000.0  # the exponent's terms are too large to be added up beforehand
    x[0, 0] = -INF
    check(x, idx, t, y, tau, 0.4, "none", scale=-64.0)


@pytest.mark.parametrize("rows,vocab,k,dtype", [(1024, 1500, 64, "fp32"), (1025, 1500, 64, "fp32"), (1025, 2049, 33, "fp32"), (1500, 5003, 9, "bf16"),
                                                (1025, 9001, 64, "fp16"), (1025, 9001, 65, "bf16"), (1025, 8193, 129, "fp16"), (256, 20011, 256, "bf16"),
                                                (255, 20011, 20, "bf16"), (260, 66003, 12, "fp16")])
def test_many_rows_and_rows_of_few_lanes(rows, vocab, k, dtype):
    """The sizes at which another number of lanes takes a row; loss alone, and with the gradient; a column named twice, and rows that
    have one entry or none."""
    x, idx, t, y = make(rows, vocab, k, dtype, 19, ignored=0.1)
    idx[5, 1] = idx[5, 0]
    idx[rows - 1, 1:] = -1
    idx[7] = -1
    check(x, idx, t, y, 2.0, 0.5, "mean", scale=256.0)
    check(x, idx, t, None, 1.0, 1.0, "none")


@pytest.mark.parametrize("rows", [1, 2, 31, 32, 33])
def test_the_loss_alone_of_a_few_long_rows(rows):
    for vocab, dtype, k in ((20001, "fp32", 70), (131072, "bf16", 64), (33000, "fp16", 1000)):
        x, idx, t, y = make(rows, vocab, k, dtype, 17, ignored=0.3)
        for reduction in ("none", "mean", "sum"):
            check(x, idx, t, y, 2.0, 0.5, reduction, scale=64.0)


@pytest.mark.parametrize("rows", [8191, 8193, 20000])
def test_many_rows_are_counted(rows):
    x, idx, t, y = make(rows, 40, 3, "fp32", 18, ignored=0.37)
    check(x, idx, t, y, 1.0, 0.5)


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_reductions_and_rows_that_do_not_count(reduction):
    x, idx, t, y = make(50, 700, 20, "fp32", 2, ignored=0.4)
    x[y == -100] = float("nan")  # a row that does not count may hold anything
    check(x.nan_to_num(0.0), idx, t, y, 2.0, 0.6, reduction)
    a, b = check_pair(x, idx, t, y, reduction), check_pair(x.nan_to_num(0.0), idx, t, y, reduction)
    assert all(torch.equal(i, j) for i, j in zip(a, b))
    nobody = torch.full_like(y, -100)
    loss, grad = check_pair(x, idx, t, nobody, reduction)
    assert (loss == 0).all() and (grad == 0).all()


def check_pair(x, idx, t, y, reduction):
    from tandem_amd import ops

    return ops.distill_loss_and_grad(x, idx, t, targets=y, temperature=2.0, weight=0.6, reduction=reduction)


def test_targets_that_only_say_which_rows_count():
    x, idx, t, y = make(30, 300, 8, "bf16", 3, ignored=0.5)
    check(x, idx, t, y, 1.5, 1.0)
    check(x, idx, t, torch.where(y == -100, 5, y), 1.5, 1.0, ignore=5)


@pytest.mark.parametrize("vocab,dtype", [(256, "fp32"), (3001, "bf16"), (40000, "fp16")])
def test_masks(vocab, dtype):
    """Student logits of -inf and of the type's lowest value where the teacher says nothing, entries without a column, teacher's logits
    of -inf, rows whose teacher says nothing at all, columns named twice and three times, the target among them."""
    x, idx, t, y = make(24, vocab, 12, dtype, 4)
    free = torch.ones(24, vocab, dtype=torch.bool, device=DEV).scatter_(1, idx, False).scatter_(1, y[:, None], False)
    drop = free & (torch.rand(24, vocab, generator=torch.Generator().manual_seed(5)).to(DEV) < 0.5)
    x[:8] = x[:8].masked_fill(drop[:8], -INF)
    x[8:16] = x[8:16].masked_fill(drop[8:16], torch.finfo(x.dtype).min)
    idx[3, 5:], t[4, 1:], t[5, :] = -1, -INF, -INF
    idx[6] = -7
    t[9, 3:] = torch.finfo(t.dtype).min
    idx[10, 4], idx[11, 1:3], idx[12, :] = idx[10, 2], idx[11, 0], y[12]
    for tau, weight in ((1.0, 1.0), (0.5, 0.5), (2.0, 0.5), (1.0, 0.5)):
        check(x, idx, t, y, tau, weight, scale=256.0 if dtype == "fp16" else 1.0)


def test_a_teacher_s_column_that_the_student_masks_costs_infinity():
    from tandem_amd import ops

    x, idx, t, y = make(4, 500, 6, "fp32", 6)
    x[1, idx[1, 2]] = -INF
    loss, grad = ops.distill_loss_and_grad(x, idx, t, reduction="none")
    assert torch.isinf(loss[1]) and torch.isfinite(loss[[0, 2, 3]]).all() and torch.isfinite(grad).all()
    check(x, idx, t, None, 1.0, 1.0, "none")


@pytest.mark.parametrize("dtype,shift", [("bf16", 3000.0), ("bf16", -2.0 ** 100), ("fp16", -60000.0), ("fp32", 1.0e30), ("bf16", 40.0)])
@pytest.mark.parametrize("vocab", [250, 3001, 40000, 100000])
def test_rows_far_from_zero(vocab, dtype, shift):
    """Softmax does not depend on a constant that all logits share: rows of two values of the type, `shift` and the next one up (or,
    where that is a step of more than 64, infinitely less likely ones), against the reference."""
    x, idx, t, y = make(6, vocab, 9, dtype, 16)
    low = torch.full((), shift, dtype=x.dtype, device=DEV)
    high = torch.nextafter(low.float() if dtype == "fp32" else low, torch.full((), INF, dtype=x.dtype, device=DEV))
    x = torch.where(x > 0, low, high)
    if float(high) - float(low) > 64:
        x = low.expand(6, vocab).contiguous()
    check(x, idx, t, y, 2.0, 0.5, scale=256.0)
    check(x, idx, t, None, 1.0, 1.0, scale=-256.0)


@pytest.mark.parametrize("vocab", [100, 9001, 70001])
def test_what_lies_outside_the_vocabulary_shows_and_stays_in_its_row(vocab):
    from tandem_amd import ops

    x, idx, t, y = make(12, vocab, 5, "fp32", 7)
    idx[1, 3], idx[2, 0], y[3], y[4], t[5, 1], x[6, 50], x[7] = vocab, 1 << 40, vocab, -1, float("nan"), float("nan"), -INF
    for weight in (0.5, 1.0):
        loss, grad = ops.distill_loss_and_grad(x, idx, t, targets=y, weight=weight, temperature=2.0, reduction="none")
        wrong = torch.zeros(12, dtype=torch.bool, device=DEV)
        wrong[[1, 2, 5, 6, 7] + ([3, 4] if weight < 1 else [])] = True
        assert torch.equal(torch.isnan(loss), wrong)
        assert torch.equal(torch.isnan(ops.distill_loss(x, idx, t, targets=y, weight=weight, temperature=2.0, reduction="none")), wrong)
        assert torch.isnan(grad[wrong]).all() and torch.isfinite(grad[~wrong]).all()


def test_a_row_that_the_teacher_says_nothing_about_is_zero_whatever_its_logits():
    from tandem_amd import ops

    for vocab in (200, 9001, 140000):
        x, idx, t, y = make(4, vocab, 5, "fp32", 15)
        x[1, 3], x[2, :], t[1:3] = float("nan"), -INF, -INF
        loss, grad = ops.distill_loss_and_grad(x, idx, t, reduction="none")
        assert (loss[1:3] == 0).all() and (grad[1:3] == 0).all() and (loss[[0, 3]] > 0).all()
        alone = ops.distill_loss(x, idx, t, reduction="none")
        assert (alone[1:3] == 0).all() and (alone[[0, 3]] > 0).all()


def test_rows_that_start_anywhere():
    from tandem_amd import ops

    g = torch.Generator().manual_seed(8)
    for dtype, lead in (("bf16", 1), ("bf16", 5), ("fp32", 3)):
        store = torch.randn(9 * 501 + 8, generator=g).to(DT[dtype]).to(DEV)
        x = store[lead:lead + 9 * 501].view(9, 501)
        _, idx, t, y = make(9, 501, 7, dtype, 9)
        check(x, idx, t, y, 2.0, 0.5)
        _, grad = ops.distill_loss_and_grad(x, idx, t)
        assert grad.data_ptr() % 16 == x.data_ptr() % 16
    for vocab in (40009, 131069):  # long rows, off the grid
        store = torch.randn(3 * vocab + 8, generator=g).bfloat16().to(DEV)
        _, idx, t, y = make(3, vocab, 7, "bf16", 9)
        check(store[3:3 + 3 * vocab].view(3, vocab), idx, t, y, 2.0, 0.5)


def test_autograd_in_more_dimensions_and_twice():
    from tandem_amd import ops

    x, idx, t, y = make(24, 333, 9, "fp32", 10, ignored=0.2)
    shaped = [v.view(4, 6, *v.shape[1:]) for v in (x, idx, t, y)]
    leaf = shaped[0].clone().requires_grad_()
    loss = ops.distill_loss(leaf, *shaped[1:], temperature=2.0, weight=0.5)
    want_loss, want = ops.distill_loss_and_grad(x, idx, t, y, temperature=2.0, weight=0.5)
    assert torch.equal(loss, want_loss)
    (first,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    assert torch.equal(first.view(24, 333), want)
    first.zero_()  # what was handed out belongs to the caller
    (second,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    assert torch.equal(second.view(24, 333), want)
    (third,) = torch.autograd.grad(loss * 3.0, leaf)
    assert torch.equal(third.view(24, 333), ops.distill_loss_and_grad(x, idx, t, y, temperature=2.0, weight=0.5, scale=3.0)[1])


def test_an_upstream_gradient_other_than_one():
    """fp16 with a scaled loss: the gradient is computed for the scaled loss, not scaled after its rounding."""
    from tandem_amd import ops

    x, idx, t, y = make(40, 2000, 9, "fp16", 11)
    leaf = x.clone().requires_grad_()
    (got,) = torch.autograd.grad(ops.distill_loss(leaf, idx, t) * 65536.0, leaf)
    assert torch.equal(got, ops.distill_loss_and_grad(x, idx, t, scale=65536.0)[1])
    rows = ops.distill_loss(leaf, idx, t, y, weight=0.5, reduction="none")
    up = torch.tensor([1.0, 2.0, 0.0, -1.5] * 10, device=DEV)
    (got,) = torch.autograd.grad(rows, leaf, up)
    _, _, g, g_err = reference(x, idx, t, y, 1.0, 0.5, -100, up)
    near(got, g, g_err + 4 * U * g.abs(), "gradient")
    ones = ops.distill_loss_and_grad(x, idx, t, y, weight=0.5, reduction="none")[1]
    assert torch.equal(got[0::4], ones[0::4]) and (got[2::4] == 0).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_a_scaled_loss_s_gradient_is_that_of_the_scale(dtype, reduction):
    """Loss scaling through autograd, for every type the bits of a call that is given the scale (a power of two); and again, retained."""
    from tandem_amd import ops

    for rows, vocab in ((40, 300), (70, 9001)):
        x, idx, t, y = make(rows, vocab, 7, dtype, 23, ignored=0.2)
        leaf = x.clone().requires_grad_()
        loss = ops.distill_loss(leaf, idx, t, y, temperature=2.0, weight=0.5, reduction=reduction)
        for scale in (4096.0, 1.0, -2.0):
            (got,) = torch.autograd.grad(loss.sum() * scale, leaf, retain_graph=True)
            assert torch.equal(got, ops.distill_loss_and_grad(x, idx, t, y, temperature=2.0, weight=0.5, reduction=reduction, scale=scale)[1]), (rows, scale)


def test_gradient_against_differences():
    """Central differences of the loss in fp32, step 2^-5 on logits of order 3: the third-order term is below h^2 / 6 times the third
    derivative, under 2 per row: 2^-11; the rounding of a loss below 16 (2^-20) over the step's 2^-4: 2^-16 each."""
    from tandem_amd import ops

    x, idx, t, y = make(2, 40, 5, "fp32", 12)
    how = dict(targets=y, temperature=2.0, weight=0.5, reduction="sum")
    _, grad = ops.distill_loss_and_grad(x, idx, t, **how)
    h = 2.0 ** -5
    for j in [int(idx[0, 0]), int(y[0]), 0, 39]:
        step = torch.zeros_like(x)
        step[0, j] = h
        d = (float(ops.distill_loss(x + step, idx, t, **how)) - float(ops.distill_loss(x - step, idx, t, **how))) / (2 * h)
        assert abs(d - float(grad[0, j])) < 2.0 ** -10


def test_no_rows():
    from tandem_amd import ops

    x, idx, t = torch.empty(0, 50, device=DEV), torch.empty(0, 4, device=DEV, dtype=torch.int64), torch.empty(0, 4, device=DEV)
    loss, grad = ops.distill_loss_and_grad(x, idx, t)
    assert float(loss) == 0.0 and grad.shape == (0, 50)
    assert ops.distill_loss_and_grad(x, idx, t, reduction="none")[0].shape == (0,)


@pytest.mark.parametrize("rows,vocab,dtype", [(300, 256, "fp32"), (70, 20000, "bf16")])
def test_a_captured_graph_replayed(rows, vocab, dtype):
    from tandem_amd import ops

    x, idx, t, y = make(rows, vocab, 8, dtype, 13, ignored=0.1)
    leaf = x.clone().requires_grad_()

    def step():
        loss = ops.distill_loss(leaf, idx, t, y, temperature=2.0, weight=0.5)
        return loss, *torch.autograd.grad(loss, leaf)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in (1, 2, 3):
        nx, _, _, ny = make(rows, vocab, 8, dtype, 20 + seed, ignored=0.3)
        with torch.no_grad():
            leaf.copy_(nx)
        y.copy_(ny)
        graph.replay()
        torch.cuda.synchronize()
        want = ops.distill_loss_and_grad(nx, idx, t, ny, temperature=2.0, weight=0.5)
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_two_streams_at_once():
    from tandem_amd import ops

    jobs = [(torch.cuda.Stream(), make(500, 3001, 8, "bf16", seed, ignored=0.1)) for seed in range(4)]
    torch.cuda.synchronize()
    got = []
    for stream, (x, idx, t, y) in jobs:
        with torch.cuda.stream(stream):
            got.append(ops.distill_loss_and_grad(x, idx, t, y, weight=0.5))
    torch.cuda.synchronize()
    for (_, (x, idx, t, y)), (loss, grad) in zip(jobs, got):
        want = ops.distill_loss_and_grad(x, idx, t, y, weight=0.5)
        assert torch.equal(loss, want[0]) and torch.equal(grad, want[1])


def test_refusals_on_the_gpu():
    from tandem_amd import ops

    x, idx, t, y = make(4, 30, 5, "fp32", 14)
    for call in (lambda: ops.distill_loss(x.double(), idx, t), lambda: ops.distill_loss(x.t(), idx, t), lambda: ops.distill_loss(x, idx.float(), t),
                 lambda: ops.distill_loss(x, idx[:3], t[:3]), lambda: ops.distill_loss(x, idx[:, :4], t), lambda: ops.distill_loss(x, idx, t, weight=0.5),
                 lambda: ops.distill_loss(x, idx, t, y[:3]), lambda: ops.distill_loss(x, idx, t, temperature=0.0),
                 lambda: ops.distill_loss(x, idx, t, y, weight=1.5), lambda: ops.distill_loss(x, idx, t, y, reduction="max"),
                 lambda: ops.distill_loss(x, idx.repeat(1, 300), t.repeat(1, 300)), lambda: ops.distill_loss(x, idx, t.cpu())):
        with pytest.raises(ValueError):
            call()

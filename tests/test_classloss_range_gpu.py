"""GPU: ``ops.linear_cross_entropy`` in fp32 where numbers of very different size meet: every row and class against the bound of its own size
(h, the sums' orders and the exactness of logits as in tests/test_classloss_gpu.py)."""
import pytest
import torch

from tests.test_classloss_gpu import DEV, _case, _exact

pytestmark = pytest.mark.gpu


def _logit_bound(x, w, lse):
    """Of each row: 2^-20 of its products' magnitudes (pairs of fp16 after one scale: 2^-21 of an element, or of its row's largest), the
    order of fp32 sums, the exponent and lse."""
    width = x.shape[1]
    mag = x.abs() @ w.abs().t()
    own = width * x.abs().max(1).values[:, None] * w.abs().max(1).values[None, :]
    return (2.0 ** -20 + (width / 8 + 8) * 2.0 ** -24) * mag.max(1).values + 2.0 ** -21 * own.max(1).values + 2.0 ** -21 * (lse.abs() + 2)


@pytest.mark.parametrize("rows,classes,width", [(200, 500, 64), (1500, 5003, 64), (20000, 1000, 40)])
def test_classes_of_low_probability(rows, classes, width):
    """fp32 gradients of classes whose probabilities are 1e-7 to 1e-14 in every row: right relative to themselves, down to 2^-50 of a row's
    weight (a step of the pair that holds the logits' gradient, whatever the tiles' orientation)."""
    from obman_train_amd import ops

    x, w, t, b = _case(rows, classes, width, torch.float32, True)
    low = torch.arange(0, classes, 7, device=DEV)
    b[low] = torch.linspace(-12, -30, len(low), device=DEV)
    t = torch.where(t % 7 == 0, t + 1, t) % classes
    t = torch.where(t % 7 == 0, t + 1, t)
    leaves = [v.requires_grad_() for v in (x, w, b)]
    dx, dw, db = torch.autograd.grad(ops.linear_cross_entropy(x, w, t, bias=b, reduction="sum"), leaves)
    _, lse, g, rx, rw, rb, xe, we, c, p = _exact(x, w, t, b, "sum")
    dz = _logit_bound(xe, we, lse)
    dg = 2.0 ** -21 * g.abs() + 4 * dz[:, None] * p + 2.0 ** -50
    sums = lambda n: (n / 8 + 8) * 2.0 ** -24 + 2.0 ** -20  # noqa: E731
    bw = dg.t() @ xe.abs() + sums(rows) * (g.abs().t() @ xe.abs())
    bx = dg @ we.abs() + sums(classes) * (g.abs() @ we.abs())
    assert ((dw.double() - rw).abs() <= bw).all(), float(((dw.double() - rw).abs() / bw).max())
    assert ((dx.double() - rx).abs() <= bx).all(), float(((dx.double() - rx).abs() / bx).max())


def _check_own_size(x, w, t, b, reduction):
    """Loss per row, dx and dw of a sum (or of random row weights) against bounds that know each row's and class's own size only."""
    from obman_train_amd import ops

    with torch.no_grad():
        loss = ops.linear_cross_entropy(x, w, t, bias=b, reduction="none")
    c = torch.ones(len(t), device=DEV)
    if reduction == "none":
        c = torch.randn(len(t), generator=torch.Generator().manual_seed(4)).to(DEV)
    leaves = [v.detach().requires_grad_() for v in (x, w, b)]
    out = ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2], reduction=reduction)
    dx, dw, db = torch.autograd.grad(out, leaves, grad_outputs=c if reduction == "none" else None)
    rl, lse, g, rx, rw, rb, xe, we, c, p = _exact(x, w, t, b, reduction, c)
    dz = _logit_bound(xe, we, lse)
    small = 2.0 ** -126 * 64  # where fp32 itself ends
    assert ((loss.double() - rl).abs() <= 4 * dz + 2.0 ** -23 * rl.abs()).all(), "loss"
    if reduction == "none":
        assert ((out.detach().double() - rl).abs() <= 4 * dz + 2.0 ** -23 * rl.abs()).all(), "loss"
    cm = c.abs()[:, None]
    # the exponential of a difference that is off by dz (at most everything) and the step of the logits' gradient
    off = torch.minimum(torch.expm1((4 * dz).clamp(max=50.0))[:, None] * p, torch.ones_like(p)) * cm
    dg = 2.0 ** -21 * g.abs() + off + 2.0 ** -50 * float(c.abs().max())
    sums = lambda n: (n / 8 + 8) * 2.0 ** -24 + 2.0 ** -20  # noqa: E731
    # dw sums rows: those of x are within 2^-22 of their own largest element, like the classes of w in dx
    xm, wm = xe.abs().max(1).values[:, None], we.abs().max(1).values[:, None]
    bx = dg @ we.abs() + sums(len(w)) * (g.abs() @ we.abs()) + 2.0 ** -22 * (g.abs() @ wm)
    bw = dg.t() @ xe.abs() + sums(len(x)) * (g.abs().t() @ xe.abs()) + 2.0 ** -22 * (g.abs().t() @ xm)
    for name, got, ref, bound in (("dx", dx, rx, bx), ("dw", dw, rw, bw), ("db", db, rb, (off + 2.0 ** -20 * g.abs()).sum(0))):
        far = (got.double() - ref).abs() - bound - 2.0 ** -23 * ref.abs() - small
        assert torch.isfinite(got).all() and float(far.max()) <= 0, (name, float(far.max()), int((far > 0).sum()))


SIZES = [(200, 500, 64), (129, 257, 65), (300, 33, 515), (70, 3001, 17), (1500, 5003, 64), (20000, 1000, 40)]


@pytest.mark.parametrize("rows,classes,width", SIZES)
@pytest.mark.parametrize("factor", [1e3, 1e6, 1e12])
@pytest.mark.parametrize("where", ["row", "class", "both", "small"])
def test_one_far_off_row_or_class(rows, classes, width, factor, where):
    """One row of x, or one class of w, that is larger than all others by far: the others keep their exactness.  "small": all but a few rows
    far below those few."""
    x, w, t, b = _case(rows, classes, width, torch.float32, True, 0.1)
    t[7] = 3  # the far-off row counts
    if where in ("row", "both"):
        x[7] *= factor
    if where in ("class", "both"):
        w[classes // 2] *= factor
    if where == "small":
        x[5:] /= factor
    _check_own_size(x, w, t, b, "sum")
    _check_own_size(x, w, t, b, "none")


def test_rows_of_zeros_and_ignored_rows_do_not_count_as_small():
    """Padding by zeros, and ignored rows whatever they hold, leave the bits of the others as they are."""
    from obman_train_amd import ops

    x, w, t, b = _case(150, 300, 40, torch.float32, True)
    want = ops.linear_cross_entropy(x.requires_grad_(), w, t, bias=b, reduction="none").detach()
    pad = torch.cat([x.detach(), torch.zeros(9, 40, device=DEV), torch.full((9, 40), 1e-30, device=DEV), torch.full((9, 40), 1e30, device=DEV)])
    labels = torch.cat([t, t[:9], torch.full((18,), -100, device=DEV)])
    got = ops.linear_cross_entropy(pad.requires_grad_(), w, labels, bias=b, reduction="none").detach()
    assert torch.equal(got[:150], want) and torch.isfinite(got).all() and not got[159:].any()


def test_far_off_rows_in_pieces_and_from_a_graph():
    """More of the logits' gradient than one piece holds, and a captured call whose replays go from one kind of operands to the other."""
    from obman_train_amd import ops

    x, w, t, b = _case(9000, 20011, 32, torch.float32, True, 0.1)
    x[11] *= 1e7
    leaves = [v.requires_grad_() for v in (x, w, b)]
    n = int((t != -100).sum())
    dx, dw, db = torch.autograd.grad(ops.linear_cross_entropy(x, w, t, bias=b), leaves)
    rw, rb = torch.zeros(20011, 32, dtype=torch.float64, device=DEV), torch.zeros(20011, dtype=torch.float64, device=DEV)
    for lo in range(0, 9000, 1500):
        s = slice(lo, lo + 1500)
        _, lse, g, gx, gw, gb, xe, we, c, p = _exact(x[s], w, t[s], b, "sum", torch.full((1500,), 1.0 / n, device=DEV))
        keep = torch.ones(len(gx), dtype=torch.bool, device=DEV)
        if lo == 0:
            keep[11] = False
        assert ((dx[s].double() - gx).abs()[keep] <= 2e-5 * (g.abs() @ we.abs())[keep] + 1e-12 / n).all(), lo
        rw += gw
        rb += gb
    few = rw.abs().max(1).values < 1e3 / n  # classes that the large row gives nothing
    assert int(few.sum()) > 20000 and float((dw.double() - rw)[few].norm() / rw[few].norm()) <= 2e-6
    assert float((db.double() - rb)[few].norm() / rb[few].norm()) <= 2e-6

    x, w, t, b = _case(300, 700, 40, torch.float32, True, 0.1)
    far = x.clone()
    far[3] *= 1e8

    def eager(x):
        leaves = [v.detach().clone().requires_grad_() for v in (x, w, b)]
        loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
        return [loss.detach()] + list(torch.autograd.grad(loss, leaves))

    want = [eager(x), eager(far)]
    static = [v.detach().clone().requires_grad_() for v in (x, w, b)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = ops.linear_cross_entropy(static[0], static[1], t, bias=static[2])
        out = [loss] + list(torch.autograd.grad(loss, static))
    for k in range(4):
        with torch.no_grad():
            static[0].copy_((x, far)[k % 2])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.detach(), r) for a, r in zip(out, want[k % 2])), k


@pytest.mark.parametrize("scale", [1e-34, 1e-30, 1e30])
def test_means_of_operands_far_from_one(scale):
    """Tiny features against a huge table and the other way round, averaged: what takes scales and average back together lies below fp32's normal
    numbers.  dx and dw are right to their bounds as at ordinary sizes."""
    from obman_train_amd import ops

    for rows, classes, width in ((90, 130, 40), (3001, 400, 24)):
        x, w, t, _ = _case(rows, classes, width, torch.float32)
        leaves = [v.requires_grad_() for v in (x * scale, w / scale)]
        dx, dw = torch.autograd.grad(ops.linear_cross_entropy(leaves[0], leaves[1], t), leaves)
        _, lse, g, rx, rw, _, xe, we, c, p = _exact(leaves[0], leaves[1], t, None, "mean")
        dg = 2.0 ** -21 * g.abs() + 4 * _logit_bound(xe, we, lse)[:, None] * p / rows + 2.0 ** -50 / rows
        sums = lambda n: (n / 8 + 8) * 2.0 ** -24 + 2.0 ** -20  # noqa: E731
        bx, bw = dg @ we.abs() + sums(classes) * (g.abs() @ we.abs()), dg.t() @ xe.abs() + sums(rows) * (g.abs().t() @ xe.abs())
        smallest = 2.0 ** -149  # fp32's last step, where a gradient of 1e-34 over 3 001 rows ends
        assert ((dx.double() - rx).abs() <= bx + smallest).all(), float(((dx.double() - rx).abs() / bx).max())
        assert ((dw.double() - rw).abs() <= bw + smallest).all(), float(((dw.double() - rw).abs() / bw).max())


def test_rows_of_zeros_beside_operands_near_the_end_of_fp32():
    """Features and table near 2^125: rows of zeros have the loss log V and finite gradients' rows, as any row of zeros."""
    import math

    from obman_train_amd import ops

    x, w, t, _ = _case(90, 130, 40, torch.float32)
    x[:-1] = 0.0
    x[-1] *= 1e37
    w *= 1e37
    with torch.no_grad():
        loss = ops.linear_cross_entropy(x, w, t, reduction="none")
    assert float((loss[:-1] - math.log(130)).abs().max()) <= 8 * 2.0 ** -24 * math.log(130)

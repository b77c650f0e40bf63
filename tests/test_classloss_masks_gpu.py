"""GPU: ``ops.linear_cross_entropy`` where whole blocks of classes are masked with a large negative number instead of -inf (the bounds are
those of tests/test_classloss_gpu.py: against the definition in 64 bits, element by element)."""
import math

import pytest
import torch

from tests.test_classloss_gpu import DEV, IGN, _bounds, _case, _check, _close, _exact, _h

pytestmark = pytest.mark.gpu
VALUES = [-1e9, -1e10, -1e12, -1e30, "lowest"]


def _value(dtype, value):
    return torch.finfo(dtype).min if value == "lowest" else value


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("value", VALUES)
@pytest.mark.parametrize("first,count", [(0, 32), (0, 128), (0, 256), (256, 256), (384, 300), (700, 128), (732, 96), (32, 796)])
def test_contiguous_masks(dtype, value, first, count):
    """Blocks as long as a wave's, a half tile's and a tile's classes, at the start, in the middle and at the end of the table, with both
    reductions over rows, and scored without gradients (few rows, and more)."""
    from obman_train_amd import ops

    x, w, t, b = _case(140, 828, 48, dtype, True, 0.1)
    left = torch.tensor([v for v in range(828) if not first <= v < first + count], device=DEV)
    t = torch.where(t == IGN, IGN, left[t.clamp(min=0) % len(left)])
    b[first:first + count] = _value(dtype, value)
    _check(x, w, t, b, "mean")
    _check(x, w, t, b, "none")
    for rows in (1, 3, 40, 140):
        rl, lse, g, *_rest, xe, we, c, p = _exact(x[:rows], w, t[:rows], b, "sum")
        with torch.no_grad():
            _close(ops.linear_cross_entropy(x[:rows], w, t[:rows], bias=b, reduction="none"), rl, _bounds(xe, we, g, p, c, dtype, lse)[0], torch.float32, rows)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("value", VALUES)
@pytest.mark.parametrize("rows", [3, 150])
def test_every_class_masked(dtype, value, rows):
    """All classes at one large negative number, which the products (below 32 in size: half a step of fp32 at 1e9) do not change: equal logits."""
    from obman_train_amd import ops

    classes = 700
    x, w, t, b = _case(rows, classes, 48, dtype, True)
    assert float((x.double() @ w.double().t()).abs().max()) < 32
    b.fill_(_value(dtype, value))
    with torch.no_grad():
        loss = ops.linear_cross_entropy(x, w, t, bias=b, reduction="none")
    # log2 of a sum of 700 ones in fp32, times log 2: some steps of 6.6
    want = torch.full_like(loss, math.log(classes))
    assert float((loss - want).abs().max()) <= 8 * 2.0 ** -24 * math.log(classes)
    leaves = [v.requires_grad_() for v in (x, w, b)]
    total = ops.linear_cross_entropy(x, w, t, bias=b, reduction="sum")
    assert abs(float(total.detach()) - rows * math.log(classes)) <= 8 * 2.0 ** -24 * rows * math.log(classes)
    g = torch.full((rows, classes), 1.0 / classes, dtype=torch.float64, device=DEV)
    g[torch.arange(rows, device=DEV), t] -= 1.0
    xe, we = x.detach().double(), w.detach().double()
    dg = (_h(dtype) + 2.0 ** -20) * g.abs() + 2.0 ** -36
    for got, ref, bound in zip(torch.autograd.grad(total, leaves), (g @ we, g.t() @ xe, g.sum(0)), (dg @ we.abs(), dg.t() @ xe.abs(), 2.0 ** -20 * g.abs().sum(0))):
        _close(got, ref, bound + 2.0 ** -20 * bound.max(), dtype, "gradient")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_either_kind_together(dtype):
    """Labels among the masked classes: a loss as large as the mask for those rows, the others as ever; gradients are finite."""
    from obman_train_amd import ops

    x, w, t, b = _case(140, 600, 48, dtype, True)
    t = 300 + t % 300
    b[:256] = -1e30
    t[::9] = 7
    mask = t == 7
    with torch.no_grad():
        loss = ops.linear_cross_entropy(x, w, t, bias=b, reduction="none")
    rl, lse, g, *_rest, xe, we, c, p = _exact(x, w, t, b, "sum")
    _close(loss[~mask], rl[~mask], _bounds(xe, we, g, p, c, dtype, lse)[0][~mask], torch.float32, "others")
    assert ((loss[mask].double() - rl[mask]).abs() <= 2.0 ** -23 * rl[mask]).all()
    leaves = [v.requires_grad_() for v in (x, w, b)]
    for got in torch.autograd.grad(ops.linear_cross_entropy(x, w, t, bias=b, reduction="sum"), leaves):
        assert torch.isfinite(got).all()


def test_large_logits():
    """Logits themselves beyond where the difference from the maximum is formed first: one-hot rows, the loss against 64 bits of the fp32 logits."""
    from obman_train_amd import ops

    g = torch.Generator().manual_seed(5)
    for size in (1e5, 3e6, 1e12, 1e30):
        x = torch.eye(64, 80) * size
        w = torch.randint(-8, 9, (300, 80), generator=g).float()
        t = torch.randint(300, (64,), generator=g)
        z = (x @ w.t()).double()  # exact: one product each
        z -= z.max(1, keepdim=True).values  # (64 bits at 8e12 end at 2^-10: the maximum out first, exactly)
        want = torch.logsumexp(z, 1) - z.gather(1, t[:, None])[:, 0]
        for rows in (64, 5):
            with torch.no_grad():
                got = ops.linear_cross_entropy(x[:rows].to(DEV), w.to(DEV), t[:rows].to(DEV), reduction="none").cpu().double()
            assert ((got - want[:rows]).abs() <= 2.0 ** -20 * (1 + want[:rows].abs())).all(), (size, rows)
        y = torch.cat([x, x])  # more rows than the direct path takes
        leaf = y.to(DEV).requires_grad_()
        loss = ops.linear_cross_entropy(leaf, w.to(DEV), torch.cat([t, t]).to(DEV), reduction="none")
        # operands in pairs: 2^-22 of the product of the largest
        assert ((loss.detach().cpu().double() - torch.cat([want, want])).abs() <= 2.0 ** -20 * 8 * size + 2.0 ** -20).all(), size
        assert torch.isfinite(torch.autograd.grad(loss.sum(), leaf)[0]).all()

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

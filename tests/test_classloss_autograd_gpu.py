"""GPU: what ``ops.linear_cross_entropy`` says to the kinds of differentiation that it does not have."""
import pytest
import torch
from torch.autograd import forward_ad

from tests.test_classloss_gpu import DEV, _case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("rows", [5, 150])
def test_forward_mode_is_refused_not_dropped(which, rows):
    """A tangent on any operand, with and without operands that require a gradient, inside and outside no_grad."""
    from obman_train_amd import ops

    x, w, t, b = _case(rows, 90, 24, torch.float32, True)
    want = ops.linear_cross_entropy(x, w, t, bias=b)
    with forward_ad.dual_level():
        args = [x, w, b]
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError):
            ops.linear_cross_entropy(args[0], args[1], t, bias=args[2])
        with torch.no_grad(), pytest.raises(NotImplementedError):
            ops.linear_cross_entropy(args[0], args[1], t, bias=args[2])
        args[(which + 1) % 3] = args[(which + 1) % 3].clone().requires_grad_()
        with pytest.raises(NotImplementedError):
            ops.linear_cross_entropy(args[0], args[1], t, bias=args[2])
        assert torch.equal(ops.linear_cross_entropy(x, w, t, bias=b), want)  # no tangent: as ever

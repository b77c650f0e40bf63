"""GPU: ``ops.linear_cross_entropy`` with many rows and many classes at once."""
import pytest
import torch

from tests.test_classloss_gpu import DEV, _bounds, _close, _exact

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,classes", [(1 << 21, 1 << 18), ((1 << 22) - 77, 140001)])
def test_more_tiles_than_one_launch_holds(rows, classes):
    """2^24 tiles of 128 rows x 256 classes, as many threads as a launch may not have: 1 024 different rows over and over have the bits of
    the call on those rows, labels in every part of the table among them."""
    from obman_train_amd import ops

    g = torch.Generator(device=DEV).manual_seed(1)
    x, w = (torch.randn(n, 8, generator=g, device=DEV).bfloat16() for n in (1024, classes))
    bias = torch.randn(classes, generator=g, device=DEV).bfloat16()
    t = (torch.arange(1024, device=DEV) * (classes - 1)) // 1023
    with torch.no_grad():
        want = ops.linear_cross_entropy(x, w, t, bias=bias, reduction="none")
        many = torch.arange(rows, device=DEV) % 1024
        got = ops.linear_cross_entropy(x[many], w, t[many], bias=bias, reduction="none")
        assert torch.equal(got, want[many])
        mean = ops.linear_cross_entropy(x[many], w, t[many], bias=bias)
    at = torch.arange(0, 1024, 31, device=DEV)
    rl, lse, gr, *_rest, xe, we, c, p = _exact(x[at], w, t[at], bias, "sum")
    _close(want[at], rl, _bounds(xe, we, gr, p, c, x.dtype, lse)[0], torch.float32, "loss")
    assert abs(float(mean) - float(got.double().mean())) <= 2.0 ** -23 * float(mean)

"""GPU: ``ops.linear_cross_entropy`` in an autocast region: features of an encoder that runs in bf16 against an fp32 table."""
import pytest
import torch

from tests.test_classloss_gpu import DEV, _case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("region", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [9, 150])
def test_operands_of_different_types(region, rows):
    from obman_train_amd import ops

    x, w, t, b = _case(rows, 300, 40, torch.float32, True, 0.1)
    half = [v.to(region).requires_grad_() for v in (x, w, b)]
    want = ops.linear_cross_entropy(half[0], half[1], t, bias=half[2])
    grads = torch.autograd.grad(want, half)
    for types in ((region, torch.float32, torch.float32), (torch.float32, region, region), (torch.float32, torch.float32, region)):
        leaves = [v.to(k).requires_grad_() for v, k in zip((x, w, b), types)]
        with pytest.raises(TypeError):
            ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
        with torch.autocast("cuda", dtype=region):
            loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
            with torch.no_grad():
                score = ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
        assert loss.dtype == torch.float32 and torch.equal(loss, want)
        with torch.no_grad():
            assert torch.equal(score, ops.linear_cross_entropy(half[0], half[1], t, bias=half[2]))
        for g, ref, leaf in zip(torch.autograd.grad(loss, leaves), grads, leaves):
            assert g.dtype == leaf.dtype and torch.equal(g.to(region), ref)


def test_operands_of_one_type_keep_it():
    """All fp32 stays fp32 in the region, and a type the operator does not have is refused there too."""
    from obman_train_amd import ops

    x, w, t, b = _case(150, 300, 40, torch.float32, True, 0.1)
    want = ops.linear_cross_entropy(x, w, t, bias=b)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.equal(ops.linear_cross_entropy(x, w, t, bias=b), want)
        for args in ((x.double(), w, b), (x.double(), w.double(), b.double())):
            with pytest.raises(TypeError):
                ops.linear_cross_entropy(args[0], args[1], t, bias=args[2])
    with torch.autocast("cpu", dtype=torch.bfloat16), pytest.raises(TypeError):
        ops.linear_cross_entropy(x.bfloat16(), w, t, bias=b)

"""GPU: ``ObmanAdam.grad_norm`` after steps that find no gradient."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_the_norm_is_of_the_last_step():
    from obman_train_amd.optim import ObmanAdam, clip_grad_norm_

    ps = [torch.nn.Parameter(torch.ones(n, device="cuda")) for n in (4, 9)]
    opt = ObmanAdam([dict(params=[p]) for p in ps], lr=1e-3, max_grad_norm=1.0)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    assert float(opt.grad_norm) == pytest.approx(13.0 ** 0.5)
    ps[1].grad = None
    opt.step()
    assert float(opt.grad_norm) == 2.0
    ps[0].grad = None
    before = [p.detach().clone() for p in ps]
    opt.step()
    assert float(opt.grad_norm) == 0.0 == float(clip_grad_norm_(ps, 1.0)) and opt.grad_norm.device == ps[0].device
    assert all(torch.equal(p, b) for p, b in zip(ps, before))
    opt = ObmanAdam(ps, lr=1e-3)
    opt.step()
    assert opt.grad_norm is None  # no limit, no norm

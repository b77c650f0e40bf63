"""GPU: ``trainer.GraphedTrainStep(max_grad_norm=...)``: clipping recorded with the step of an optimizer that does not clip by itself."""
import pytest
import torch

from tests.test_gradnorm_gpu import DEV, _Tiny

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["sgd", "adam"])
def test_a_recorded_step_clips_for_any_optimizer(name):
    from obman_train_amd.trainer import GraphedTrainStep, make_optimizer, train_step

    data = [{"x": torch.randn(8, 6, generator=torch.Generator().manual_seed(k)).to(DEV)} for k in range(4)]
    eager, free, model = _Tiny().to(DEV), _Tiny().to(DEV), _Tiny().to(DEV)
    eopt, fopt, opt = (make_optimizer(m, name, lr=1e-2, momentum=0.9) for m in (eager, free, model))
    step = GraphedTrainStep(model, opt, data[0], warmup=1, max_grad_norm=0.1)  # one real step, and the recording
    train_step(eager, eopt, data[0], max_grad_norm=0.1)
    train_step(free, fopt, data[0])
    for s in data:
        total = step(s)[0]
        torch.cuda.synchronize()
        want = train_step(eager, eopt, s, max_grad_norm=0.1)[0]
        assert float(total.detach()) == pytest.approx(float(want.detach()), rel=1e-5)
        train_step(free, fopt, s)
        for a, b in zip(model.parameters(), eager.parameters()):
            torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6)
            torch.testing.assert_close(a.grad, b.grad, rtol=1e-4, atol=1e-6)
    assert name == "adam" or any(float((a - b).detach().abs().max()) > 1e-3 for a, b in zip(free.parameters(), eager.parameters()))

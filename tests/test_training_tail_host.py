"""CPU: what the class loss, the gradient norm and clipping refuse without a GPU - host tensors, and bad arguments at the C-ABI, each
before anything is launched."""
import ctypes

import pytest
import torch


def test_host_tensors_are_refused():
    from obman_train_amd import _lib, ops, optim

    x, w, t = torch.zeros(3, 4), torch.zeros(5, 4), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(_lib.ObmanHipError):
        ops.linear_cross_entropy(x, w, t)
    with pytest.raises(ValueError):
        ops.linear_cross_entropy(x, w, t, reduction="avg")
    with pytest.raises(_lib.ObmanHipError):
        optim.grad_norm([x])
    p = torch.nn.Parameter(x)
    p.grad = torch.ones(3, 4)
    with pytest.raises(_lib.ObmanHipError):
        optim.clip_grad_norm_([p], 1.0)
    with pytest.raises(_lib.ObmanHipError):
        optim.ObmanAdam([p], max_grad_norm=1.0)
    with pytest.raises(ValueError):
        optim.ObmanAdam([p], max_grad_norm=-1.0)
    assert torch.equal(p.grad, torch.ones(3, 4))
    assert float(optim.clip_grad_norm_([torch.nn.Parameter(x)], 1.0)) == 0.0 and float(optim.grad_norm([])) == 0.0
    model = torch.nn.Linear(2, 2)
    from obman_train_amd.trainer import make_optimizer

    for name in ("adam", "rms", "sgd"):
        with pytest.raises(ValueError):
            make_optimizer(model, name, max_grad_norm=1.0)


def _params(**kw):
    from obman_train_amd import _lib

    base = dict(x=4096, w=4096, bias=None, target=4096, rows=10, classes=20, ignore_index=-100, width=8, type=0, target_wide=1, reduction=2)
    base.update(kw)
    return _lib.ClassLossParams(**base)


def _sizes(p, *flags):
    from obman_train_amd import _lib

    n = (ctypes.c_long * 3)()
    at = ctypes.addressof(n)
    status = _lib.lib().obman_class_loss_sizes(ctypes.addressof(p), *flags, at, at + 8, at + 16)
    return status, list(n)


@pytest.mark.parametrize("bad", [dict(rows=0), dict(rows=-1), dict(classes=0), dict(width=0), dict(width=16385), dict(rows=(1 << 22) + 1), dict(classes=(1 << 22) + 1),
                                 dict(type=3), dict(type=-1), dict(reduction=3), dict(reduction=-1), dict(target=None)])
def test_class_loss_arguments(bad):
    from obman_train_amd import _lib

    p = _params(**bad)
    at = ctypes.addressof(p)
    assert _sizes(p, 1, 1, 1, 1)[0] < 0
    assert _lib.lib().obman_class_loss_fwd(at, 4096, 4096, 4096, None) < 0
    assert _lib.lib().obman_class_loss_bwd(at, 4096, 4096, 4096, 4096, 4096, None, None) < 0


def test_class_loss_null_pointers_and_sizes():
    from obman_train_amd import _lib

    lib, p = _lib.lib(), _params()
    at = ctypes.addressof(p)
    assert lib.obman_class_loss_sizes(None, 0, 0, 0, 0, at, at, at) < 0 and lib.obman_class_loss_sizes(at, 0, 0, 0, 0, None, None, None) < 0
    for args in ((4096, None, 4096), (4096, 4096, None)):
        assert lib.obman_class_loss_fwd(at, *args, None) < 0
    for args in ((None, 4096, 4096), (4096, None, 4096), (4096, 4096, None)):
        assert lib.obman_class_loss_bwd(at, *args, 4096, None, None, None) < 0
    assert lib.obman_class_loss_bwd(at, 4096, 4096, 4096, None, None, None, None) == 0  # no gradient asked for: nothing to do
    for q in (_params(x=None), _params(w=None)):
        assert lib.obman_class_loss_fwd(ctypes.addressof(q), 4096, 4096, 4096, None) < 0
    status, (keep, fwd, bwd) = _sizes(_params(rows=1000, classes=5000, width=512), 1, 1, 1, 1)
    assert status == 0 and min(keep, fwd, bwd) > 0
    # what is kept is both operands (fp32: as two fp16 planes) and a few words a row, never rows x classes
    assert keep < 4 * 512 * (1024 + 5120) + 64 * 1024
    # a single row scored: block statistics only, whatever the table's size
    assert _sizes(_params(rows=1, classes=1 << 22, width=512, type=1), 0, 0, 0, 0)[1][1] < 1 << 20
    # the gradient of the logits exists in pieces: 4M rows x 64 050 classes in 16 bits would be 537 GB
    status, (_, _, bwd) = _sizes(_params(rows=64 * 64050, classes=64050, width=64, type=1), 1, 1, 1, 0)
    assert status == 0 and bwd < 12 << 30


def test_gradient_norm_arguments():
    from obman_train_amd import _lib

    lib = _lib.lib()
    ptr, n, kind = (ctypes.c_void_p * 2)(4096, None), (ctypes.c_long * 2)(5, 5), (ctypes.c_int * 2)(0, 0)
    a = [ctypes.addressof(v) for v in (ptr, n, kind)]
    assert lib.obman_grad_norm_ws_doubles(-1) < 0 and lib.obman_grad_norm_ws_doubles(0) > 0
    assert lib.obman_grad_norm(*a, 2, 2, 4096, 4096, None) < 0  # a tensor without memory
    assert lib.obman_grad_norm(*a, 1, 3, 4096, 4096, None) < 0  # no such norm
    assert lib.obman_grad_norm(*a, 1, 2, None, 4096, None) < 0 and lib.obman_grad_norm(*a, 1, 2, 4096, None, None) < 0
    assert lib.obman_grad_norm(None, None, None, 1, 2, 4096, 4096, None) < 0 and lib.obman_grad_norm(*a, -1, 2, 4096, 4096, None) < 0
    kind[0] = 3
    assert lib.obman_grad_norm(*a, 1, 2, 4096, 4096, None) < 0
    kind[0], n[0] = 0, -1
    assert lib.obman_grad_norm(*a, 1, 2, 4096, 4096, None) < 0
    n[0] = 5
    assert lib.obman_grad_clip(*a, 1, 2, -1.0, 4096, 4096, None) < 0 and lib.obman_grad_clip(*a, 1, 2, float("nan"), 4096, 4096, None) < 0
    assert lib.obman_adam_norm_partials(None, None, 1, 4096, 4096, None) < 0
    t = (_lib.AdamTensor * 1)()
    assert lib.obman_adam_step_clipped(ctypes.addressof(t), 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 4096, 1, 1.0, 4096, 4096, None) < 0  # no step counter
    assert lib.obman_adam_step_clipped(ctypes.addressof(t), 0, 1e-3, 0.9, 0.999, 1e-8, 0.0, 4096, 1, 1.0, 4096, 4096, None) < 0

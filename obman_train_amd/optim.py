"""The optimizer step of the training loop as ONE multi-tensor HIP kernel (``csrc/stepops.hip``, ``obman_adam_step``).

The reference builds ``torch.optim.Adam(model.parameters(), lr, weight_decay)`` (``traineval.py:112-116``) and calls ``step()`` once
per batch (``epochpass3d.py:86-91``).  ``ObmanAdam`` IS a ``torch.optim.Adam`` (constructor, ``param_groups``, ``state_dict`` /
``load_state_dict`` layout with ``step`` / ``exp_avg`` / ``exp_avg_sq`` per parameter - checkpoints written by either load into the
other), with ``step()`` replaced:

* every parameter that has a gradient is updated by one launch per <= 64 tensors (torch's fused Adam: three launches at 2.1 TB/s
  over the 350 MB it touches; this kernel streams 16-byte vectors of p, g, m, v);
* the per-parameter step counters live on the device (one fp32 array), so the step records into a hipGraph like torch's
  ``capturable=True`` form, without its per-step host work;
* ``max_grad_norm`` clips all gradients of all groups together by their global L2 norm (``clip_grad_norm_``'s rule) inside the
  same kernel: the norm is one pass over the gradients, the clipped values are never written (``grad_norm`` holds the norm);
* a parameter that carries a bf16 SHADOW (``attach_bf16_shadows``: the filters of a bf16-autocast encoder) gets
  ``shadow = bf16(p_new)`` written by the same kernel - the autocast encoder then reads the shadow
  (``ops.shadow_conv2d``) instead of launching one cast kernel per filter and step.
No CPU path: parameters must be fp32 ROCm tensors (``trainer.make_optimizer`` only builds this optimizer for such models).

``grad_norm`` and ``clip_grad_norm_`` are the same norm and clipping for any other optimizer (``csrc/gradnorm.hip``): lists of
fp32 / bf16 / fp16 gradients of any sizes, one or two launches per 192 tensors.
"""
import ctypes
import functools
import operator
from array import array

import torch
from torch.autograd.graph import increment_version

from . import _lib, ops

_is_none = functools.partial(operator.is_, None)
_GRAD_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_NORMS = {2.0: 2, 1.0: 1, float("inf"): 0}


def _norm_kind(norm_type):
    kind = _NORMS.get(float(norm_type))
    if kind is None:
        raise ValueError("norm_type must be 1, 2 or inf, got %r" % (norm_type,))
    return kind


def _same_device(tensors, what):
    """-> their device, their types (numbers of the C-ABI, one for each) and whether all are contiguous.  C-level maps instead of a walk in
    Python: the checks of 92 gradients would cost more than the kernels."""
    devices = set(map(torch.Tensor.get_device, tensors))
    if -1 in devices:
        raise _lib.ObmanHipError("%s must be ROCm device tensors (the HIP path has no CPU fallback)" % what)
    if len(devices) > 1:
        raise ValueError("%s must be on one device, got %s" % (what, ", ".join("cuda:%d" % d for d in sorted(devices))))
    dtypes = list(map(torch.Tensor.dtype.__get__, tensors))
    try:
        if dtypes.count(dtypes[0]) == len(dtypes):
            types = array("i", (_GRAD_TYPES[dtypes[0]],)) * len(dtypes)
        else:
            types = array("i", map(_GRAD_TYPES.__getitem__, dtypes))
    except KeyError as e:
        raise TypeError("%s must be fp32, bf16 or fp16, got %s" % (what, e.args[0])) from None
    contiguous = all(map(torch.Tensor.is_contiguous, tensors))
    if not contiguous and any(t.layout != torch.strided for t in tensors):
        raise TypeError("%s must be dense tensors" % what)
    return tensors[0].device, types, contiguous


def _norm_call(tensors, dev, types, norm_kind, max_norm=None):
    """One C-ABI call over dense tensors of one device: -> the norm, a 0-dim fp32 tensor on that device."""
    n = len(tensors)
    ptrs = array("Q", map(torch.Tensor.data_ptr, tensors))
    counts = array("q", map(torch.Tensor.numel, tensors))
    lib = _lib.lib()
    out = torch.empty((), dtype=torch.float32, device=dev)
    ws = torch.empty(lib.obman_grad_norm_ws_doubles(n), dtype=torch.float64, device=dev)  # of this call alone: recorded into a graph it is the graph's
    at = (ptrs.buffer_info()[0], counts.buffer_info()[0], types.buffer_info()[0])
    with ops._on_device(dev):
        if max_norm is None:
            _lib.check(lib.obman_grad_norm(*at, n, norm_kind, ws.data_ptr(), out.data_ptr(), ops._stream()), "obman_grad_norm")
        else:
            _lib.check(lib.obman_grad_clip(*at, n, norm_kind, max_norm, ws.data_ptr(), out.data_ptr(), ops._stream()), "obman_grad_clip")
    return out


def grad_norm(tensors, norm_type=2.0):
    """The norm of all elements of all ``tensors`` (gradients, fp32 / bf16 / fp16, mixed) as one vector: a 0-dim fp32 tensor on
    their device, without a host synchronisation.  ``norm_type`` 2, 1 or inf.  Summed in 64 bits in a fixed order: bit-reproducible.
    The result carries no derivative.  An empty list gives 0 (on the CPU); entries that are ``None`` (parameters without a gradient) are skipped."""
    kind = _norm_kind(norm_type)
    if isinstance(tensors, torch.Tensor):
        tensors = [tensors]
    tensors = [t for t in tensors if t is not None]
    if not tensors:
        return torch.zeros(())
    dev, types, contiguous = _same_device(tensors, "tensors")
    if not contiguous:
        tensors = [t if ops._is_dense(t) else t.detach().contiguous() for t in tensors]
    return _norm_call(tensors, dev, types, kind)


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """``torch.nn.utils.clip_grad_norm_`` on this package's kernels: every gradient of ``parameters`` is multiplied in place by
    ``min(1, max_norm / (norm + 1e-6))`` and the norm before clipping is returned (0-dim fp32 device tensor; nothing waits for it).

    A parameter listed twice, or two that share one gradient tensor, is counted and scaled once.  As in torch, a NaN norm makes the
    gradients NaN and an infinite one multiplies them by 0; ``error_if_nonfinite`` raises instead, before anything is scaled - it has
    to wait for the device and cannot be recorded into a graph.  ``ObmanAdam(max_grad_norm=...)`` does the same without writing the
    clipped gradients."""
    kind = _norm_kind(norm_type)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError("max_norm must not be negative or NaN, got %r" % (max_norm,))
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [g for p in parameters if (g := p.grad) is not None]
    if len(set(map(id, grads))) != len(grads):
        grads = list({id(g): g for g in grads}.values())
    if not grads:
        return torch.zeros(())
    dev, types, contiguous = _same_device(grads, "gradients")
    odd = [] if contiguous else [i for i, g in enumerate(grads) if not ops._is_dense(g)]
    for i in odd:
        if torch._debug_has_internal_overlap(grads[i]) == 1:
            raise ValueError("a gradient whose elements share memory (an expanded tensor) cannot be scaled in place")
    if error_if_nonfinite:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("clip_grad_norm_(error_if_nonfinite=True) reads the norm on the host: it cannot be recorded into a graph")
        norm = grad_norm(grads, norm_type)
        if not torch.isfinite(norm):
            raise RuntimeError("the total norm of order %s for gradients is non-finite, so it cannot be clipped" % (float(norm_type),))
    work = grads
    if odd:
        work = list(grads)
        for i in odd:
            work[i] = grads[i].detach().contiguous()
    norm = _norm_call(work, dev, types, kind, max_norm)
    if odd:
        with torch.no_grad():
            for i in odd:
                grads[i].copy_(work[i])
    increment_version(grads)
    return norm


class ObmanAdam(torch.optim.Adam):
    max_grad_norm = None  # read by every step; None = no clipping
    grad_norm = None  # 0-dim fp32 device tensor: the L2 norm of the last clipped step's gradients, before clipping

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, amsgrad=False, max_grad_norm=None, **kw):
        if max_grad_norm is not None and not float(max_grad_norm) >= 0.0:
            raise ValueError("max_grad_norm must not be negative or NaN, got %r" % (max_grad_norm,))
        if amsgrad or kw.get("maximize"):
            raise ValueError("ObmanAdam implements plain Adam (traineval.py:112-116): no amsgrad / maximize")
        kw.pop("fused", None)
        kw.pop("capturable", None)
        kw.pop("foreach", None)
        super().__init__(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, amsgrad=False, foreach=False, fused=False,
                         capturable=True)  # capturable: ``step`` entries are device tensors, as this kernel keeps them
        self.max_grad_norm = None if max_grad_norm is None else float(max_grad_norm)
        for group in self.param_groups:
            for p in group["params"]:
                if not p.is_cuda or p.dtype != torch.float32:
                    raise _lib.ObmanHipError("ObmanAdam needs fp32 ROCm parameters (there is no CPU path)")

    def __getstate__(self):  # copies and pickles keep the limit (torch's optimizers carry their groups and state only)
        return dict(super().__getstate__(), max_grad_norm=self.max_grad_norm)

    def _init_state(self, p):
        st = self.state[p]
        if "exp_avg" not in st:
            st["step"] = torch.zeros((), dtype=torch.float32, device=p.device)
            st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
            st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
        return st

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        lib = _lib.lib()
        work, devices = [], set()
        for gi, group in enumerate(self.param_groups):
            params = group["params"]
            grads = [p.grad for p in params]
            if any(map(_is_none, grads)):
                params = [p for p, g in zip(params, grads) if g is not None]
                grads = [g for g in grads if g is not None]
            if not params:
                continue
            if not hasattr(self, "_plans"):
                self._plans = {}
            cache = self._plans.get(gi)
            if cache is None or not self._refresh(cache, params, grads):
                cache = self._plans[gi] = self._build(params)
            b1, b2 = group["betas"]
            lr = group["lr"]
            if torch.is_tensor(lr):
                lr = float(lr)
            devices |= cache["devices"]
            work.append((cache["addr"], len(params), float(lr), float(b1), float(b2), float(group["eps"]), float(group["weight_decay"])))
        if not work:
            if self.max_grad_norm is not None:  # no gradient at all: their norm is 0, not the step's before
                self.grad_norm = torch.zeros((), device=self.param_groups[0]["params"][0].device)
            return loss
        if len(devices) > 1:
            if self.max_grad_norm is not None:
                raise ValueError("max_grad_norm needs all parameters on one device, got %s" % sorted(map(str, devices)))
            dev = torch.device("cuda", torch.cuda.current_device())
        else:
            dev, = devices
        with ops._on_device(dev):
            if self.max_grad_norm is not None:
                self._clipped(lib, work, dev, ops._stream())
            else:
                for args in work:
                    _lib.check(lib.obman_adam_step(*args, ops._stream()), "obman_adam_step")
        return loss

    def _clipped(self, lib, work, dev, stream):
        """The norm over every group's gradients, then each group's update on the clipped values.  Scratch of this call alone: recorded
        into a graph it belongs to the graph, and two graphs of one optimizer share nothing but the parameters."""
        lists = (ctypes.c_void_p * len(work))(*[w[0] for w in work])
        counts = (ctypes.c_int * len(work))(*[w[1] for w in work])
        total = sum(w[1] for w in work)
        ws = torch.empty(lib.obman_grad_norm_ws_doubles(total), dtype=torch.float64, device=dev)
        corr = torch.empty(2 * max(w[1] for w in work), dtype=torch.float32, device=dev)
        clip = torch.empty(2, dtype=torch.float32, device=dev)
        parts = ctypes.c_int(0)
        _lib.check(lib.obman_adam_norm_partials(ctypes.addressof(lists), ctypes.addressof(counts), len(work), ws.data_ptr(),
                                                ctypes.addressof(parts), stream), "obman_adam_norm_partials")
        first = parts.value
        if not first:
            clip.zero_()  # gradients without elements: their norm is 0
        for args in work:
            _lib.check(lib.obman_adam_step_clipped(*args, ws.data_ptr(), first, self.max_grad_norm, clip.data_ptr(), corr.data_ptr(), stream),
                       "obman_adam_step_clipped")
            first = 0
        self.grad_norm = clip[0]

    def _build(self, params):
        """The launch's descriptor table (host array of device pointers, seven words a tensor) for this set of parameters; everything but
        the gradient pointers is constant from step to step, so ``_refresh`` only rewrites those."""
        strides = list(map(torch.Tensor.stride, params))
        sts, shadows, grads = [], [], []
        for p, stride in zip(params, strides):
            g = p.grad
            if g.is_sparse:
                raise RuntimeError("ObmanAdam does not support sparse gradients")
            if not ops._is_dense(p):
                raise RuntimeError("ObmanAdam needs dense parameters (contiguous or channels_last)")
            st = self._init_state(p)
            if st["exp_avg"].stride() != stride:  # a state loaded from a checkpoint written with another layout
                st["exp_avg"] = torch.empty_like(p, memory_format=torch.preserve_format).copy_(st["exp_avg"])
                st["exp_avg_sq"] = torch.empty_like(p, memory_format=torch.preserve_format).copy_(st["exp_avg_sq"])
            step = st["step"]
            if not (torch.is_tensor(step) and step.is_cuda and step.dtype == torch.float32):
                st["step"] = torch.as_tensor(float(step), dtype=torch.float32, device=p.device)
            sh = getattr(p, "_obman_shadow", None)
            if sh is not None and sh.stride() != stride:
                sh = p._obman_shadow = ops.bf16_shadow(p.detach())  # the parameter was re-laid out (channels_last) after the shadow was made
                p._obman_shadow_version = p._version
            if g.stride() != stride:
                g = torch.empty_like(p, memory_format=torch.preserve_format).copy_(g)  # element order of the parameter
            sts.append(st)
            shadows.append(sh)
            grads.append(g)
        ms, vs, steps = ([st[key] for st in sts] for key in ("exp_avg", "exp_avg_sq", "step"))
        table = array("Q", bytes(56 * len(sts)))
        for word, tensors in enumerate((params, grads, ms, vs, None, steps)):
            if tensors is not None:
                table[word::7] = array("Q", map(torch.Tensor.data_ptr, tensors))
        table[4::7] = array("Q", (0 if sh is None else sh.data_ptr() for sh in shadows))
        table[6::7] = array("Q", map(torch.Tensor.numel, params))
        return {"table": table, "addr": table.buffer_info()[0], "devices": {p.device for p in params}, "params": list(params), "ptrs": table[0::7],
                "strides": strides, "states": sts, "ms": ms, "vs": vs, "steps": steps, "shadows": shadows, "grads": grads}

    def _refresh(self, cache, params, grads):
        """Same parameters, same storage, same state tensors as when the table was built?  Then only the gradient pointers change.
        Compared with C-level maps (a walk in Python over 92 parameters took 31 us of a step whose kernels take 80)."""
        def same(new, old):
            return all(map(operator.is_, new, old))

        if len(params) != len(cache["params"]) or not same(params, cache["params"]):
            return False
        strides, sts = cache["strides"], cache["states"]
        if array("Q", map(torch.Tensor.data_ptr, params)) != cache["ptrs"] or list(map(torch.Tensor.stride, params)) != strides:
            return False
        # load_state_dict, a replaced state or a re-created shadow: rebuild
        if not same(map(self.state.get, params), sts) or not same([getattr(p, "_obman_shadow", None) for p in params], cache["shadows"]):
            return False
        try:
            for key, old in (("exp_avg", cache["ms"]), ("exp_avg_sq", cache["vs"]), ("step", cache["steps"])):
                if not same(map(operator.itemgetter(key), sts), old):
                    return False
        except KeyError:
            return False
        if list(map(torch.Tensor.stride, grads)) != strides:
            grads = [g if g.stride() == s else torch.empty_like(p, memory_format=torch.preserve_format).copy_(g) for g, s, p in zip(grads, strides, params)]
        cache["table"][1::7] = array("Q", map(torch.Tensor.data_ptr, grads))
        cache["grads"] = grads  # the gradients stay referenced until the launch below has been enqueued
        return True


def attach_bf16_shadows(module):
    """Give every bias-free ``nn.Conv2d`` filter of ``module`` (the bf16-autocast encoder) a bf16 shadow in the filter's own memory
    order (``weight._obman_shadow``).  ``ObmanAdam.step`` keeps the shadows current; ``ops.shadow_conv2d`` reads them.  Call again
    after anything else writes the filters (``load_state_dict``, a broadcast): ``refresh_bf16_shadows``."""
    n = 0
    for m in module.modules():
        if isinstance(m, torch.nn.Conv2d) and m.bias is None and m.weight.is_cuda and m.weight.dtype == torch.float32:
            m.weight._obman_shadow = ops.bf16_shadow(m.weight.detach())
            m.weight._obman_shadow_version = m.weight._version
            n += 1
    return n


def refresh_bf16_shadows(module):
    for m in module.modules():
        if isinstance(m, torch.nn.Conv2d) and getattr(m.weight, "_obman_shadow", None) is not None:
            if m.weight._obman_shadow.stride() != m.weight.stride():
                m.weight._obman_shadow = ops.bf16_shadow(m.weight.detach())
            else:
                ops.bf16_shadow(m.weight.detach(), out=m.weight._obman_shadow)  # in place: a recorded graph keeps its address
            m.weight._obman_shadow_version = m.weight._version


def detach_bf16_shadows(module):
    for m in module.modules():
        if isinstance(m, torch.nn.Conv2d) and hasattr(m.weight, "_obman_shadow"):
            del m.weight._obman_shadow

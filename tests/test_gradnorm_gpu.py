"""GPU: ``optim.grad_norm`` / ``optim.clip_grad_norm_`` (csrc/gradnorm.hip) and the clipped optimizer step ``ObmanAdam(max_grad_norm=...)``
against their formulas in 64 bits.

The norm is summed in fp64 and rounded once to fp32: 2^-24 relative, 2^-23 asked for.  Clipping forms max_norm / (norm + 1e-6) in fp32 (the
norm's, the sum's and the quotient's rounding: 3 x 2^-24) and multiplies in fp32 (2^-24), then rounds to the gradient's type."""
import copy
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"fp32": [torch.float32], "bf16": [torch.bfloat16], "fp16": [torch.float16], "mixed": [torch.float32, torch.bfloat16, torch.float16]}


def _grads(sizes, kinds, seed=0, spread=3):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * 10.0 ** float(torch.rand((), generator=g) * -spread)).to(kinds[i % len(kinds)]).to(DEV) for i, n in enumerate(sizes)]


def _norm(grads, kind):
    flat = torch.cat([g.detach().double().flatten() for g in grads]) if grads else torch.zeros(0, dtype=torch.float64)
    return float(torch.linalg.vector_norm(flat, ord=kind)) if flat.numel() else 0.0


def _params(grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.zeros_like(g))
        p.grad = g
        out.append(p)
    return out


SIZES = {"one": [1], "empty_ones": [0, 5, 0, 1, 0], "small": [3, 4, 5, 1023, 8, 17], "edge": [4096, 4097, 8191, 8192, 8193, 32768, 1], "one_block": [32768],
         "layers": [9408, 64, 64, 36864, 589824, 2359296, 512, 515, 257, 132355, 3, 1], "many": [1 + 37 * i % 900 for i in range(500)], "large": [9000001, 7]}


@pytest.mark.parametrize("kind", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("name", sorted(SIZES))
def test_norm_and_clipping(name, types, kind):
    from obman_train_amd import optim

    grads = _grads(SIZES[name], TYPES[types])
    want = _norm(grads, kind)
    got = optim.grad_norm(grads, norm_type=kind)
    assert got.dtype == torch.float32 and got.shape == () and got.device == grads[0].device
    assert abs(float(got) - want) <= 2.0 ** -23 * want
    assert torch.equal(optim.grad_norm(grads, norm_type=kind), got)
    for max_norm in (want / 3, want * 3):
        clipped = [g.clone() for g in grads]
        versions = [g._version for g in clipped]
        total = optim.clip_grad_norm_(_params(clipped), max_norm, norm_type=kind)
        assert torch.equal(total, got)
        factor = min(1.0, max_norm / (float(got) + 1e-6))
        for before, after, v in zip(grads, clipped, versions):
            ref = before.double() * factor
            tiny = torch.finfo(before.dtype).smallest_normal * torch.finfo(before.dtype).eps
            bound = ref.abs() * (5 * 2.0 ** -24 + (torch.finfo(before.dtype).eps / 2 if before.dtype != torch.float32 else 0.0)) + tiny
            assert ((after.double() - ref).abs() <= bound).all()
            assert after._version > v
            if factor == 1.0:
                assert torch.equal(after, before)


@pytest.mark.parametrize("kind", [2.0, 1.0, math.inf])
def test_packed_at_every_offset(kind):
    """Gradients back to back in flat buffers (all-reduce buckets): any element alignment, and nothing beside them is touched."""
    from obman_train_amd import optim

    sizes = [1, 7, 30, 4095, 5, 9000, 33, 2, 16385]
    flats = [torch.randn(sum(sizes) + 2 * len(sizes) + 3, generator=torch.Generator().manual_seed(k)).to(t).to(DEV) for k, t in enumerate(TYPES["mixed"])]
    keep = [f.clone() for f in flats]
    grads, inside = [], [torch.zeros_like(f, dtype=torch.bool) for f in flats]
    for k, f in enumerate(flats):
        at = 1 + k
        for n in sizes:
            grads.append(f[at:at + n])
            inside[k][at:at + n] = True
            at += n + 1
    want = _norm(grads, kind)
    got = optim.clip_grad_norm_(_params(grads), want / 2, norm_type=kind)
    assert abs(float(got) - want) <= 2.0 ** -23 * want
    assert abs(_norm(grads, kind) - want / 2) <= 2.0 ** -8 * want
    for f, k, m in zip(flats, keep, inside):
        assert torch.equal(f[~m], k[~m])


def test_values_that_leave_fp32_and_non_finite_ones():
    from obman_train_amd import optim

    big = [torch.full((1000,), 3e30, device=DEV), torch.full((10,), 2e38, device=DEV)]
    want = _norm(big, 2.0)
    # the norm itself, sqrt(10) 2e38 = 6.3e38, leaves fp32 (3.4e38): its rounding is infinite
    assert want > torch.finfo(torch.float32).max and float(optim.grad_norm(big)) == math.inf
    assert abs(float(optim.grad_norm(big[:1])) - _norm(big[:1], 2.0)) <= 2.0 ** -23 * _norm(big[:1], 2.0)  # only the squares leave fp32
    small = [torch.full((1000,), 1e-30, device=DEV)]
    assert abs(float(optim.grad_norm(small)) - _norm(small, 2.0)) <= 2.0 ** -23 * _norm(small, 2.0)
    for n in (100, 200000):
        for kind in (2.0, 1.0, math.inf):
            for bad, total in ((math.nan, math.nan), (math.inf, math.inf), (-math.inf, math.inf)):
                g = [torch.ones(n, device=DEV), torch.ones(n // 3, device=DEV, dtype=torch.bfloat16)]
                g[1][n // 5] = bad
                got = float(optim.clip_grad_norm_(_params(g), 1.0, norm_type=kind))
                assert math.isnan(got) if math.isnan(total) else got == total
                ref = float("nan") if math.isnan(total) else 0.0
                assert torch.equal(g[0], torch.full_like(g[0], ref)) or math.isnan(ref) and torch.isnan(g[0]).all()
                g = [torch.ones(n, device=DEV)]
                g[0][3] = bad
                before = g[0].clone()
                with pytest.raises(RuntimeError):
                    optim.clip_grad_norm_(_params(g), 1.0, norm_type=kind, error_if_nonfinite=True)
                assert torch.equal(g[0].nan_to_num(7.0), before.nan_to_num(7.0))  # refused before anything was scaled
    assert float(optim.clip_grad_norm_(_params([torch.ones(4, device=DEV)]), 1.0, error_if_nonfinite=True)) == 2.0


def test_lists_and_layouts():
    from obman_train_amd import optim

    assert float(optim.grad_norm([])) == 0.0 and float(optim.grad_norm([None, None])) == 0.0
    p = torch.nn.Parameter(torch.zeros(3, device=DEV))
    assert float(optim.clip_grad_norm_([p], 1.0)) == 0.0 and float(optim.clip_grad_norm_([], 1.0)) == 0.0
    assert float(optim.grad_norm([torch.zeros(0, device=DEV)])) == 0.0
    g = torch.randn(6, 5, 4, 3, device=DEV)
    assert float(optim.grad_norm(g)) == float(optim.grad_norm([g]))
    layouts = [g.clone().contiguous(memory_format=torch.channels_last), torch.randn(40, 30, device=DEV).t(), torch.randn(50, 8, device=DEV)[:, ::2], torch.randn((), device=DEV)]
    want = _norm(layouts, 2.0)
    assert abs(float(optim.grad_norm(layouts)) - want) <= 2.0 ** -23 * want
    ref = [v.clone() for v in layouts]
    params = []
    for v in layouts:
        q = torch.nn.Parameter(v.clone(memory_format=torch.preserve_format))
        q.grad = v
        params.append(q)
    optim.clip_grad_norm_(params, want / 4)
    for v, r in zip(layouts, ref):
        assert torch.allclose(v, r / 4, rtol=1e-5, atol=0)
    # the same parameter twice, and two that share a gradient: counted and scaled once, as parameters() would list them
    a, b = torch.nn.Parameter(torch.zeros(9, device=DEV)), torch.nn.Parameter(torch.zeros(9, device=DEV))
    a.grad = b.grad = torch.full((9,), 2.0, device=DEV)
    assert float(optim.clip_grad_norm_([a, b, a], 3.0)) == 6.0
    assert torch.allclose(a.grad, torch.ones(9, device=DEV))
    # a generator, a single parameter, max_norm 0
    assert float(optim.clip_grad_norm_((q for q in [a]), 100.0)) == pytest.approx(3.0)
    optim.clip_grad_norm_(a, 0.0)
    assert not a.grad.any()


def test_refusals():
    from obman_train_amd import _lib, optim

    g = torch.ones(4, device=DEV)
    for bad in (0.0, 3.0, -1.0):
        with pytest.raises(ValueError):
            optim.grad_norm([g], norm_type=bad)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError):
            optim.clip_grad_norm_(_params([g]), bad)
        with pytest.raises(ValueError):
            optim.ObmanAdam(_params([g]), max_grad_norm=bad)
    with pytest.raises(_lib.ObmanHipError):
        optim.grad_norm([g, torch.ones(3)])
    for t in (torch.float64, torch.int32):
        with pytest.raises(TypeError):
            optim.grad_norm([g, torch.ones(3, device=DEV).to(t)])
    with pytest.raises(TypeError):
        optim.grad_norm([torch.eye(3, device=DEV).to_sparse()])
    p = torch.nn.Parameter(torch.zeros(4, 3, device=DEV))
    p.grad = torch.ones(1, 3, device=DEV).expand(4, 3)
    with pytest.raises(ValueError):
        optim.clip_grad_norm_([p], 1.0)
    assert float(optim.grad_norm([p.grad])) == pytest.approx(math.sqrt(12))


def _pair(shapes, seed, groups=1, **kw):
    from obman_train_amd.optim import ObmanAdam

    g = torch.Generator().manual_seed(seed)
    host = [torch.nn.Parameter(torch.randn(s, generator=g)) for s in shapes]
    dev = [torch.nn.Parameter(p.detach().clone().to(DEV)) for p in host]
    cut = lambda ps: [dict(params=ps[k::groups], lr=1e-3 * (k + 1)) for k in range(groups)]  # noqa: E731
    return host, dev, torch.optim.Adam(cut(host), **{k: v for k, v in kw.items() if k != "max_grad_norm"}), ObmanAdam(cut(dev), **kw)


@pytest.mark.parametrize("count,groups,weight_decay", [(1, 1, 0.0), (5, 2, 1e-2), (70, 1, 0.0), (330, 3, 0.0)])
def test_clipped_adam_is_clipping_and_adam(count, groups, weight_decay):
    """Against torch's clip_grad_norm_ + Adam on the host; gradients stay as they were, parameters without one are left out."""
    shapes = [(1 + 97 * i % 300, 1 + i % 7) for i in range(count)]
    host, dev, ref, opt = _pair(shapes, 1, groups, weight_decay=weight_decay, max_grad_norm=0.5)
    g = torch.Generator().manual_seed(2)
    for step in range(6):
        for i, (h, d) in enumerate(zip(host, dev)):
            gr = torch.randn(h.shape, generator=g) * (0.001 if step == 3 else 1.0)  # step 3 is under the limit when the set is small
            h.grad, d.grad = (None, None) if i % 5 == 4 and step % 2 else (gr.clone(), gr.to(DEV))
        kept = [None if d.grad is None else d.grad.clone() for d in dev]
        norm = torch.nn.utils.clip_grad_norm_([p for p in host], 0.5)
        ref.step()
        opt.step()
        assert abs(float(opt.grad_norm) - float(norm)) <= 1e-6 * float(norm)
        for d, k in zip(dev, kept):
            assert (d.grad is None and k is None) or torch.equal(d.grad, k)
    for h, d in zip(host, dev):
        torch.testing.assert_close(d.detach().cpu(), h.detach(), rtol=1e-5, atol=3e-6)
        assert float(opt.state[d]["step"]) == float(ref.state[h]["step"])


def test_clipped_adam_without_a_limit_reached_is_adam():
    """factor 1: the same bits as the unclipped kernel (g * 1 = g; the bias corrections are formed by the same expressions)."""
    from obman_train_amd.optim import ObmanAdam

    _, a, _, plain = _pair([(33, 5), (4097,), (1,)], 4, lr=1e-3)
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    clipped = ObmanAdam([dict(params=b, lr=1e-3)], lr=1e-3, max_grad_norm=1e6)
    g = torch.Generator().manual_seed(5)
    for _ in range(5):
        for x, y in zip(a, b):
            x.grad = torch.randn(x.shape, generator=g).to(DEV)
            y.grad = x.grad.clone()
        plain.step()
        clipped.step()
    assert plain.grad_norm is None
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    clipped.max_grad_norm = None  # may change between steps
    for x, y in zip(a, b):
        x.grad = torch.ones_like(x)
        y.grad = torch.ones_like(y)
    plain.step()
    clipped.step()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_clipped_adam_state_layouts_and_shadows():
    """A channels_last filter with a bf16 shadow, a gradient in another layout, a checkpoint taken and loaded, a state entry replaced."""
    from obman_train_amd import ops
    from obman_train_amd.optim import ObmanAdam

    p = torch.nn.Parameter(torch.randn(32, 16, 3, 3, device=DEV).contiguous(memory_format=torch.channels_last))
    p._obman_shadow = ops.bf16_shadow(p.detach())
    q = torch.nn.Parameter(p.detach().cpu().double().contiguous())
    opt, ref = ObmanAdam([p], lr=1e-2, max_grad_norm=1.0), torch.optim.Adam([q], lr=1e-2)
    g = torch.Generator().manual_seed(0)
    for step in range(4):
        gr = torch.randn(32, 16, 3, 3, generator=g)
        p.grad = gr.to(DEV) if step % 2 else gr.to(DEV).contiguous(memory_format=torch.channels_last)
        q.grad = gr.double()
        torch.nn.utils.clip_grad_norm_([q], 1.0)
        opt.step()
        ref.step()
        assert torch.equal(p._obman_shadow, p.detach().bfloat16())
        if step == 1:
            saved = copy.deepcopy(opt.state_dict())
            opt = ObmanAdam([p], lr=1e-2, max_grad_norm=1.0)
            opt.load_state_dict(saved)
        if step == 2:
            opt.state[p] = {k: v.clone() for k, v in opt.state[p].items()}
    torch.testing.assert_close(p.detach().cpu().double(), q.detach(), rtol=1e-5, atol=1e-6)
    assert float(opt.state[p]["step"]) == 4.0


def test_a_copied_optimizer_still_clips():
    from obman_train_amd.optim import ObmanAdam

    p = torch.nn.Parameter(torch.zeros(50, device=DEV))
    p.grad = torch.ones(50, device=DEV)
    opt = ObmanAdam([p], lr=1e-2, max_grad_norm=0.5)
    opt.step()
    twin = copy.deepcopy(opt)
    q = twin.param_groups[0]["params"][0]
    assert twin.max_grad_norm == 0.5 and q is not p
    for o, v in ((opt, p), (twin, q)):
        v.grad = torch.full((50,), 2.0, device=DEV)
        o.step()
    assert float(twin.grad_norm) == float(opt.grad_norm) == pytest.approx(2.0 * math.sqrt(50))
    assert torch.equal(p, q)


def test_clipping_in_a_graph():
    """Norm, clipping and the clipped step recorded together, two graphs alive, eager work between the replays."""
    from obman_train_amd import optim

    def build(seed):
        g = torch.Generator().manual_seed(seed)
        ps = [torch.nn.Parameter(torch.randn(n, generator=g).to(DEV)) for n in (5000, 77, 40001)]
        for p in ps:
            p.grad = torch.zeros_like(p)
        return ps, optim.ObmanAdam(ps, lr=1e-2, max_grad_norm=1.0)

    def feed(ps, k):
        g = torch.Generator().manual_seed(100 + k)
        for p in ps:
            p.grad.copy_(torch.randn(p.shape, generator=g))

    graphs = []
    for seed in (0, 1):
        ps, opt = build(seed)
        eps, eopt = build(seed)
        extra = [torch.randn(30000, device=DEV), torch.randn(11, device=DEV)]
        feed(ps, 0)
        opt.step()  # the state exists before the capture
        feed(eps, 0)
        eopt.step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step()
            norm = opt.grad_norm
            plain = optim.grad_norm([p.grad for p in ps], norm_type=math.inf)
            total = optim.clip_grad_norm_(ps, 0.25)
            again = optim.grad_norm([p.grad for p in ps])
        graphs.append((graph, ps, eps, eopt, norm, plain, total, again, opt))  # opt: its moments and counters are the graph's
        del extra
    for k in range(1, 5):
        for graph, ps, eps, eopt, norm, plain, total, again, _ in graphs:
            feed(ps, k)
            feed(eps, k)
            graph.replay()
            eopt.step()
            optim.grad_norm(_grads(SIZES["layers"], TYPES["mixed"], seed=k))
            torch.cuda.synchronize()
            assert torch.equal(norm, eopt.grad_norm) and all(torch.equal(a, b) for a, b in zip(ps, eps)), k
            assert float(plain) == max(float(p.grad.abs().max()) for p in eps)
            assert torch.equal(total, optim.clip_grad_norm_(eps, 0.25))
            assert all(torch.equal(a.grad, b.grad) for a, b in zip(ps, eps))
            assert float(again) == pytest.approx(0.25, rel=1e-4)


def test_within_the_limit_nothing_changes():
    """A factor of 1 leaves every bit, of many chunks and of the single block."""
    from obman_train_amd import optim

    for sizes in ([70000, 3, 40001], [5, 9]):
        grads = _grads(sizes, TYPES["mixed"])
        grads[0][1] = -0.0
        keep = [g.clone() for g in grads]
        norm = optim.clip_grad_norm_(_params(grads), 2.0 * _norm(grads, 2.0))
        assert float(norm) == pytest.approx(_norm(keep, 2.0), rel=1e-6)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(grads, keep))


def test_clipped_adam_with_gradients_without_elements():
    from obman_train_amd import optim

    ps = [torch.nn.Parameter(torch.zeros(0, 3, device=DEV)), torch.nn.Parameter(torch.zeros(0, device=DEV))]
    for p in ps:
        p.grad = torch.zeros_like(p)
    opt = optim.ObmanAdam(ps, max_grad_norm=1.0)
    for _ in range(2):
        opt.step()
        assert float(opt.grad_norm) == 0.0
    more = torch.nn.Parameter(torch.ones(7, device=DEV))
    more.grad = torch.full_like(more, 2.0)
    opt.add_param_group({"params": [more]})
    opt.step()
    assert float(opt.grad_norm) == pytest.approx(2.0 * math.sqrt(7.0), rel=1e-6)


def test_on_another_stream():
    from obman_train_amd import optim

    grads = _grads(SIZES["layers"], TYPES["mixed"])
    want = optim.grad_norm(grads)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [optim.grad_norm(grads) for _ in range(3)]
    other = optim.grad_norm(grads, norm_type=1.0)  # two calls under way at once
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(g, want) for g in got) and float(other) > 0


class _Tiny(torch.nn.Module):
    def __init__(self):
        super().__init__()
        torch.manual_seed(0)
        self.lin = torch.nn.Linear(6, 3)

    def forward(self, sample, **kw):
        loss = (self.lin(sample["x"]) * 100).square().mean()
        return loss, {}, {"total_loss": loss}


@pytest.mark.parametrize("name", ["adam", "rms", "sgd"])
def test_the_training_loop_clips(name):
    """train_step / epoch_pass with max_grad_norm for any optimizer, make_optimizer(max_grad_norm=...) for adam: torch's clipping and step."""
    from obman_train_amd.netscripts.epochpass3d import epoch_pass
    from obman_train_amd.trainer import make_optimizer, train_step

    data = [{"x": torch.randn(8, 6, generator=torch.Generator().manual_seed(k))} for k in range(3)]
    host = _Tiny()
    ref = {"adam": lambda ps: torch.optim.Adam(ps, lr=1e-2), "rms": lambda ps: torch.optim.RMSprop(ps, lr=1e-2), "sgd": lambda ps: torch.optim.SGD(ps, lr=1e-2, momentum=0.9)}[name](host.parameters())
    for s in data:
        ref.zero_grad()
        host(s)[0].backward()
        assert float(torch.nn.utils.clip_grad_norm_(host.parameters(), 0.1)) > 0.1
        ref.step()
    dev = [{"x": s["x"].to(DEV)} for s in data]

    def check(model):
        for a, b in zip(model.parameters(), host.parameters()):
            torch.testing.assert_close(a.detach().cpu(), b.detach(), rtol=1e-4, atol=1e-5)

    model = _Tiny().to(DEV)
    opt = make_optimizer(model, name, lr=1e-2, momentum=0.9)
    for s in dev:
        train_step(model, opt, s, max_grad_norm=0.1)
    check(model)
    model = _Tiny().to(DEV)
    epoch_pass(dev, model, 0, optimizer=make_optimizer(model, name, lr=1e-2, momentum=0.9), max_grad_norm=0.1)
    check(model)
    model = _Tiny().to(DEV)
    if name != "adam":
        with pytest.raises(ValueError):
            make_optimizer(model, name, max_grad_norm=0.1)
        return
    opt = make_optimizer(model, name, lr=1e-2, max_grad_norm=0.1)
    for s in dev:
        train_step(model, opt, s)
    check(model)
    assert float(opt.grad_norm) > 0.1


def test_a_recorded_training_step_clips():
    from obman_train_amd.trainer import GraphedTrainStep, make_optimizer, train_step

    data = [{"x": torch.randn(8, 6, generator=torch.Generator().manual_seed(k)).to(DEV)} for k in range(4)]
    eager, model = _Tiny().to(DEV), _Tiny().to(DEV)
    eopt, opt = make_optimizer(eager, lr=1e-2, max_grad_norm=0.1), make_optimizer(model, lr=1e-2, max_grad_norm=0.1)
    step = GraphedTrainStep(model, opt, data[0], restore_state=True)
    for s in data:
        train_step(eager, eopt, s)
        step(s)
        torch.cuda.synchronize()
        assert float(opt.grad_norm) == pytest.approx(float(eopt.grad_norm), rel=1e-5)
    for a, b in zip(model.parameters(), eager.parameters()):
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6)

"""GPU: ``ops.linear_cross_entropy`` (csrc/classloss.hip) against the definition in 64 bits, element by element.

Tolerances follow from the arithmetic (``_bounds``): h = eps / 2 of the 16-bit type is the rounding of the logits' gradient before its
two products and of each result; an fp32 operand is hi + lo in fp16, 2^-22 of an element after two roundings of 2^-12, and of the
tensor's largest 2^-39; a sum of n terms in fp32 is off by at most n 2^-24 of the sum of the magnitudes, of which the matrix
instruction's order leaves n / 8."""
import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IGN = -100


def _h(dtype):
    return 2.0 ** -21 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def _case(rows, classes, width, dtype, bias=False, ignored=0.0, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed + 7 * rows + 11 * classes + 13 * width)
    w = torch.randn(classes, width, generator=g) * (spread / math.sqrt(width))
    t = torch.randint(classes, (rows,), generator=g)
    x = torch.randn(rows, width, generator=g) + 0.5 * w[t]
    b = torch.randn(classes, generator=g) if bias else None
    if ignored:
        t[torch.rand(rows, generator=g) < ignored] = IGN
    mk = lambda v: None if v is None else v.to(dtype).to(DEV)  # noqa: E731
    return mk(x), mk(w), t.to(DEV), mk(b)


def _exact(x, w, t, b, reduction, g_rows=None, ignore=IGN):
    """loss (per row), dx, dw, db and what their bounds need, in float64 on the device; g_rows: weight of each row's loss."""
    x, w = x.detach().double(), w.detach().double()
    b = torch.zeros(w.shape[0], dtype=torch.float64, device=w.device) if b is None else b.detach().double()
    keep = t != ignore
    at = torch.where(keep, t, 0).long()
    x = torch.where(keep[:, None], x, 0.0)
    z = x @ w.t() + b
    lse = torch.logsumexp(z, 1)
    loss = torch.where(keep, lse - z.gather(1, at[:, None])[:, 0], 0.0)
    c = keep.double() if g_rows is None else torch.where(keep, g_rows.double(), 0.0)
    if reduction == "mean":
        c = c / max(1, int(keep.sum()))
    g = torch.exp(z - lse[:, None])
    p = g.clone()
    g.scatter_add_(1, at[:, None], -torch.ones_like(g[:, :1]))
    g = g * c[:, None]
    return loss, lse, g, (g @ w), (g.t() @ x), g.sum(0), x, w, c, p


def _bounds(x, w, g, p, c, dtype, lse):
    """Per-element bounds of the loss, dx, dw, db from the roundings named above."""
    width, classes, rows = x.shape[1], w.shape[0], x.shape[0]
    mag = x.abs() @ w.abs().t()  # of the products that make a logit
    split = 2.0 ** -20 if dtype == torch.float32 else 0.0
    tiny = 2.0 ** -37 * width * float(x.abs().max() * w.abs().max()) if dtype == torch.float32 else 0.0
    dz = (split + (width / 8 + 8) * 2.0 ** -24) * mag.max(1).values + tiny + 2.0 ** -21 * (lse.abs() + 2)  # [rows]: z, its exponent and lse
    h = _h(dtype)
    dg = h * g.abs() + 4 * dz[:, None] * p * c.abs()[:, None] + 2.0 ** -36 * float(c.abs().max()) * (dtype != torch.bfloat16)
    ax, aw = (classes / 8 + 8) * 2.0 ** -24 + split, (rows / 8 + 8) * 2.0 ** -24 + split
    bx = dg @ w.abs() + ax * (g.abs() @ w.abs())
    bw = dg.t() @ x.abs() + aw * (g.abs().t() @ x.abs())
    bb = (4 * dz[:, None] * p * c.abs()[:, None] + 2.0 ** -22 * g.abs()).sum(0)
    return 4 * dz, bx, bw, bb


def _close(got, want, bound, dtype, what):
    out = torch.finfo(dtype).eps / 2 * want.abs() + (torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps if dtype != torch.float32 else 1e-38)
    off = (got.double() - want).abs() - (bound + out) * 1.001
    assert got.dtype == dtype and torch.isfinite(got).all(), what
    assert float(off.max()) <= 0.0, "%s: %.3g over its bound at %d of %d" % (what, float(off.max()), int((off > 0).sum()), off.numel())


def _check(x, w, t, b, reduction, scale=1.0, g_rows=None):
    from obman_train_amd import ops

    leaves = [v.detach().requires_grad_() for v in (x, w, b) if v is not None]
    loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2] if b is not None else None, ignore_index=IGN, reduction=reduction)
    assert loss.dtype == torch.float32 and loss.shape == (t.shape if reduction == "none" else ())
    rows = None if g_rows is None else g_rows * scale
    seedg = (rows if rows is not None else torch.full_like(loss, scale)) if reduction == "none" else torch.full_like(loss, scale)
    grads = torch.autograd.grad(loss, leaves, grad_outputs=seedg)
    c = seedg if reduction == "none" else torch.full(t.shape, float(scale), device=t.device)
    rl, lse, g, dx, dw, db, xe, we, c, p = _exact(x, w, t, b, reduction, c)
    bl, bx, bw, bb = _bounds(xe, we, g, p, c, x.dtype, lse)
    kept = max(1, int((t != IGN).sum()))
    if reduction == "none":
        _close(loss.detach(), rl, bl, torch.float32, "loss")
    else:
        n = kept if reduction == "mean" else 1
        _close(loss.detach(), rl.sum() / n, bl.sum() / n, torch.float32, "loss")
    _close(grads[0], dx, bx, x.dtype, "dx")
    _close(grads[1], dw, bw, w.dtype, "dw")
    if b is not None:
        _close(grads[2], db, bb, b.dtype, "db")
    return loss, grads


SIZES = [(1, 1, 1), (1, 2, 3), (2, 33, 31), (127, 255, 32), (128, 256, 64), (129, 257, 65), (33, 1000, 515), (600, 778, 256), (5, 40, 3000), (257, 3001, 17)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,classes,width", SIZES)
def test_matches_the_definition(rows, classes, width, dtype):
    for bias, reduction, ignored in ((False, "mean", 0.0), (True, "mean", 0.3), (True, "sum", 0.0), (False, "none", 0.3)):
        x, w, t, b = _case(rows, classes, width, dtype, bias, ignored)
        # fp16 gradients of a mean over many rows are scaled up, as a training loop in fp16 scales its loss
        _check(x, w, t, b, reduction, scale=float(min(rows, 1024)) if dtype == torch.float16 and reduction == "mean" else 1.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_weights_per_row(dtype):
    """reduction "none" with a gradient for every row: signs, zeros, five orders of magnitude."""
    x, w, t, b = _case(200, 513, 96, dtype, True, 0.2)
    g = torch.Generator().manual_seed(3)
    rows = torch.randn(200, generator=g) * 10.0 ** torch.randint(-4, 2, (200,), generator=g)
    rows[::7] = 0.0
    _check(x, w, t, b, "none", g_rows=rows.to(DEV))
    _check(x, w, t, b, "none", g_rows=torch.zeros(200, device=DEV))


@pytest.mark.parametrize("dtype", TYPES)
def test_several_pieces_of_the_classes(dtype):
    """More classes x rows than one piece of the logits' gradient holds (512 MB): pieces add up in dx and follow each other in dw, db."""
    from obman_train_amd import ops

    rows, classes, width = (9000, 20011, 32) if dtype == torch.float32 else (16500, 20011, 32)
    x, w, t, b = _case(rows, classes, width, dtype, True, 0.1)
    leaves = [v.requires_grad_() for v in (x, w, b)]
    scale = 1024.0 if dtype == torch.float16 else 1.0
    loss = ops.linear_cross_entropy(x, w, t, bias=b)
    grads = torch.autograd.grad(loss * scale, leaves)
    n = int((t != IGN).sum())
    dw, db, total = torch.zeros(classes, width, dtype=torch.float64, device=DEV), torch.zeros(classes, dtype=torch.float64, device=DEV), 0.0
    bw, bb = torch.zeros_like(dw), torch.zeros_like(db)
    for lo in range(0, rows, 2000):
        s = slice(lo, lo + 2000)
        rl, lse, g, gx, gw, gb, xe, we, c, p = _exact(x[s], w, t[s], b, "sum", torch.full((len(t[s]),), scale / n, device=DEV))
        _, px, pw, pb = _bounds(xe, we, g, p, c, dtype, lse)
        total += float(rl.sum())
        _close(grads[0][s], gx, px, dtype, "dx from row %d" % lo)
        dw += gw; db += gb; bw += pw; bb += pb  # noqa: E702
    assert abs(float(loss.detach()) - total / n) <= 1e-6 * abs(total / n)
    _close(grads[1], dw, bw + rows / 8 * 2.0 ** -24 * bw, dtype, "dw")
    _close(grads[2], db, bb, dtype, "db")


@pytest.mark.parametrize("dtype,width", [(torch.bfloat16, 512), (torch.float32, 512)])
def test_the_most_rows_and_the_most_classes(dtype, width):
    """2^22 rows, then 2^22 classes, 512 wide: operands of 4 and 8 GB, whose later column blocks lie beyond 2^31 bytes and 2^32 elements of
    offset.  One more is refused."""
    from obman_train_amd import _lib, ops

    most, few = 1 << 22, 24
    g = torch.Generator(device=DEV).manual_seed(2)
    long = torch.empty(most, width, dtype=dtype, device=DEV)
    for lo in range(0, most, 1 << 19):
        long[lo:lo + (1 << 19)] = torch.randn(1 << 19, width, generator=g, device=DEV) * 0.2
    short = (torch.randn(few, width, generator=g, device=DEV) * 0.2).to(dtype)
    t = torch.randint(few, (most,), generator=g, device=DEV)
    t[::5] = IGN
    x, w = long.requires_grad_(), short.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, t, reduction="sum")
    gx, gw = torch.autograd.grad(loss, [x, w])
    dw, total, bw = torch.zeros(few, width, dtype=torch.float64, device=DEV), 0.0, torch.zeros(few, width, dtype=torch.float64, device=DEV)
    for lo in range(0, most, 1 << 17):
        s = slice(lo, lo + (1 << 17))
        rl, lse, gr, ex, ew, _, xe, we, c, p = _exact(x[s], w, t[s], None, "sum")
        _, px, pw, _ = _bounds(xe, we, gr, p, c, dtype, lse)
        total += float(rl.sum())
        dw += ew
        bw += pw
        if lo % (1 << 20) == 0 or lo + (1 << 17) == most:
            _close(gx[s], ex, px, dtype, "dx from row %d" % lo)
    assert abs(float(loss.detach()) - total) <= 1e-6 * total
    _close(gw, dw, bw * 1.01, dtype, "dw")
    del gx, gw
    # the same long operand as the table of classes
    rows = torch.randint(most, (few,), generator=g, device=DEV)
    loss = ops.linear_cross_entropy(w, x, rows, reduction="none")
    gw, gx = torch.autograd.grad(loss.sum(), [w, x])
    top, acc = torch.full((few,), -math.inf, dtype=torch.float64, device=DEV), torch.zeros(few, dtype=torch.float64, device=DEV)
    for lo in range(0, most, 1 << 17):
        z = w.detach().double() @ x[lo:lo + (1 << 17)].detach().double().t()
        new = torch.maximum(top, z.max(1).values)
        acc = acc * torch.exp(top - new) + torch.exp(z - new[:, None]).sum(1)
        top = new
    lse = top + acc.log()
    want = lse - (w.detach().double() * x.detach()[rows].double()).sum(1)
    assert float((loss.detach().double() - want).abs().max()) <= 2e-5
    for lo in (0, most // 2, most - 4096):
        s = slice(lo, lo + 4096)
        z = w.detach().double() @ x[s].detach().double().t()
        pr = torch.exp(z - lse[:, None])
        hot = (rows[:, None] == torch.arange(lo, lo + 4096, device=DEV)).double()
        ref, mag = (pr - hot).t() @ w.detach().double(), (pr + hot).t() @ w.detach().double().abs()
        out = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 2.0 ** -24
        assert ((gx[s].double() - ref).abs() <= (_h(dtype) + 1e-4 * (dtype == torch.float32)) * mag + out * ref.abs() + 2.0 ** -34 * float(w.detach().abs().max())).all(), lo
    assert torch.isfinite(gw).all()
    del gx, gw
    with pytest.raises(_lib.ObmanHipError):
        ops.linear_cross_entropy(torch.empty(most + 1, 1, dtype=dtype, device=DEV), short[:, :1].detach(), torch.zeros(most + 1, dtype=torch.int64, device=DEV))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,classes,width", [(1, 1, 1), (1, 778, 512), (3, 1000, 515), (32, 5003, 100), (31, 129, 7), (17, 300, 2048), (32, 300, 1030), (33, 300, 64), (64, 4099, 100), (65, 1000, 33), (128, 777, 512), (97, 5000, 260), (129, 300, 64)])
def test_scoring_without_gradients(rows, classes, width, dtype):
    from obman_train_amd import ops

    for bias, ignored in ((False, 0.0), (True, 0.3)):
        x, w, t, b = _case(rows, classes, width, dtype, bias, ignored)
        rl, lse, g, *_rest, xe, we, c, p = _exact(x, w, t, b, "sum")
        bound = _bounds(xe, we, g, p, c, dtype, lse)[0]
        _close(ops.linear_cross_entropy(x, w, t, bias=b, reduction="none"), rl, bound, torch.float32, "per row")
        kept = max(1, int((t != IGN).sum()))
        _close(ops.linear_cross_entropy(x, w, t, bias=b), rl.sum() / kept, bound.sum() / kept, torch.float32, "mean")
        _close(ops.linear_cross_entropy(x, w, t, bias=b, reduction="sum"), rl.sum(), bound.sum(), torch.float32, "sum")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [9, 150])
def test_ignored_rows_take_no_part_whatever_they_hold(dtype, rows):
    from obman_train_amd import ops

    x, w, t, b = _case(rows, 300, 40, dtype, True)
    t[2] = t[rows - 1] = IGN
    want = _check(x, w, t, b, "mean")
    for junk in (math.nan, math.inf, -math.inf):
        y = x.detach().clone()
        y[2], y[rows - 1, 3:] = junk, junk
        leaves = [y.requires_grad_(), w.detach().requires_grad_(), b.detach().requires_grad_()]
        loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
        grads = torch.autograd.grad(loss, leaves)
        assert torch.equal(loss, want[0])
        for a, e in zip(grads, want[1]):
            assert torch.equal(a, e)
        assert not grads[0][2].any() and not grads[0][rows - 1].any()
        with torch.no_grad():
            assert torch.allclose(ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2]), loss, rtol=1e-6, atol=0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_every_row_ignored(dtype, reduction):
    from obman_train_amd import ops

    x, w, t, b = _case(70, 90, 33, dtype, True)
    t.fill_(IGN)
    leaves = [v.requires_grad_() for v in (x, w, b)]
    loss = ops.linear_cross_entropy(x, w, t, bias=b, reduction=reduction)
    assert not loss.any()
    assert all(not g.any() for g in torch.autograd.grad(loss.sum(), leaves))
    with torch.no_grad():
        assert not ops.linear_cross_entropy(x[:5], w, t[:5], bias=b, reduction=reduction).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", ["-inf", "lowest"])
def test_masked_classes(dtype, value):
    from obman_train_amd import ops

    x, w, t, b = _case(140, 600, 48, dtype, True)
    mask = torch.ones(600, dtype=torch.bool, device=DEV)
    mask[t] = False
    b[mask] = -math.inf if value == "-inf" else torch.finfo(dtype).min
    leaves = [v.requires_grad_() for v in (x, w, b)]
    loss = ops.linear_cross_entropy(x, w, t, bias=b, reduction="sum")
    grads = torch.autograd.grad(loss, leaves)
    keep = ~mask
    new = torch.cumsum(keep, 0) - 1
    want = _check(x.detach(), w.detach()[keep], new[t], b.detach()[keep], "sum")
    assert torch.allclose(loss, want[0], rtol=1e-5)
    assert not grads[1][mask].any() and not grads[2][mask].any()
    h = 8 * _h(dtype)  # both sides round g, in other tiles, and their results
    for got, ref in ((grads[0], want[1][0]), (grads[1][keep], want[1][1]), (grads[2][keep], want[1][2])):
        assert float((got - ref).abs().max()) <= h * float(ref.float().abs().max()) + 1e-5 * float(ref.float().abs().max())
    # a row with nothing left has no loss: NaN by definition
    with torch.no_grad():
        nothing = torch.full_like(b, -math.inf)
        assert torch.isnan(ops.linear_cross_entropy(x, w, t, bias=nothing, reduction="none")).all()
        assert torch.isnan(ops.linear_cross_entropy(x[:3], w, t[:3], bias=nothing, reduction="none")).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [3, 140])
def test_a_label_outside_the_table_is_loud(dtype, rows):
    from obman_train_amd import ops

    for bad in (77, 1 << 40, -1):
        x, w, t, b = _case(rows, 77, 20, dtype)
        t[1] = bad
        with torch.no_grad():
            per_row = ops.linear_cross_entropy(x, w, t, reduction="none")
        assert torch.isnan(per_row[1]) and int(torch.isnan(per_row).sum()) == 1
        leaves = [x.requires_grad_(), w.requires_grad_()]
        loss = ops.linear_cross_entropy(x, w, t)
        gx, gw = torch.autograd.grad(loss, leaves)
        assert torch.isnan(loss) and torch.isnan(gx[1]).all() and torch.isnan(gw).any()


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(dtype):
    """Leading dimensions, int32 labels, another ignore_index, strided and misaligned operands: the bits of the contiguous call."""
    from obman_train_amd import ops

    x, w, t, b = _case(60, 130, 37, dtype, True)
    t[5] = 7

    def run(x, w, t, b, **kw):
        leaves = [v.detach().requires_grad_() for v in (x, w, b)]
        loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2], **kw)
        return [loss.detach()] + list(torch.autograd.grad(loss.sum(), leaves))

    want = run(x, w, t, b, ignore_index=7)
    odd = lambda v: torch.cat([v.flatten()[:1], v.flatten()])[1:].view(v.shape)  # noqa: E731 - one element off every alignment
    strided = lambda v: torch.stack([v, v], -1)[..., 0]  # noqa: E731
    for xx, ww, tt, bb in ((odd(x), odd(w), t, odd(b)), (strided(x), w.t().contiguous().t(), strided(t), strided(b)), (x, w, t.int(), b)):
        for got, ref in zip(run(xx, ww, tt, bb, ignore_index=7), want):
            assert torch.equal(got, ref)
    got = run(x.view(3, 20, 37), w, t.view(3, 20), b, ignore_index=7)
    assert got[1].shape == (3, 20, 37) and torch.equal(got[1].view(60, 37), want[1]) and torch.equal(got[2], want[2])
    with torch.no_grad():
        few = ops.linear_cross_entropy(x[:20], w, t[:20], bias=b, reduction="none")
        for xx, ww in ((odd(x[:20]), odd(w)), (strided(x[:20]), strided(w))):
            assert torch.equal(ops.linear_cross_entropy(xx, ww, t[:20].int(), bias=b, reduction="none"), few)


def test_only_the_gradients_asked_for_and_the_same_bits_twice():
    from obman_train_amd import ops

    x, w, t, b = _case(300, 700, 64, torch.bfloat16, True, 0.1)
    full = [v.detach().requires_grad_() for v in (x, w, b)]
    want = torch.autograd.grad(ops.linear_cross_entropy(full[0], full[1], t, bias=full[2]), full)
    for need in itertools.product((False, True), repeat=3):
        leaves = [v.detach().requires_grad_(n) for v, n in zip((x, w, b), need)]
        loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
        assert loss.requires_grad == any(need)
        if any(need):
            loss.backward()
        for v, n, ref in zip(leaves, need, want):
            assert (v.grad is not None) == n
            if n:  # (another set of gradients cuts the contractions otherwise: not the same bits)
                assert float((v.grad - ref).abs().max()) <= 2.0 ** -7 * float(ref.float().abs().max())
    again = torch.autograd.grad(ops.linear_cross_entropy(full[0], full[1], t, bias=full[2]), full)
    assert all(torch.equal(a, r) for a, r in zip(again, want))


def test_gradients_against_differences():
    from obman_train_amd import ops

    x, w, t, b = _case(40, 90, 24, torch.float32, True, 0.2)
    leaves = [v.requires_grad_() for v in (x, w, b)]
    grads = torch.autograd.grad(ops.linear_cross_entropy(*leaves[:2], t, bias=b, reduction="sum"), leaves)
    g = torch.Generator(device=DEV).manual_seed(1)
    step = 2.0 ** -7
    for k in range(3):
        u = torch.randn(leaves[k].shape, generator=g, device=DEV)
        with torch.no_grad():
            ends = []
            for s in (step, -step):
                v = [a.detach() + s * u if i == k else a.detach() for i, a in enumerate(leaves)]
                ends.append(ops.linear_cross_entropy(v[0], v[1], t, bias=v[2], reduction="none").double().sum())
        slope, want = float(ends[0] - ends[1]) / (2 * step), float((grads[k].double() * u).sum())
        # losses of size 40 x 5 are right to 2^-20 of it: 2e-4 / 2^-6; the cubic term is step^2 of the slope's size
        assert abs(slope - want) <= 0.02 + 1e-3 * abs(want), (k, slope, want)


def test_empty_batch_and_shared_leaf():
    from obman_train_amd import ops

    w = torch.randn(10, 4, device=DEV, requires_grad=True)
    x = torch.zeros(0, 4, device=DEV, requires_grad=True)
    t = torch.zeros(0, dtype=torch.int64, device=DEV)
    for reduction in ("mean", "sum"):
        loss = ops.linear_cross_entropy(x, w, t, reduction=reduction)
        assert float(loss.detach()) == 0.0
        loss.backward()
        assert x.grad.shape == (0, 4)
    assert ops.linear_cross_entropy(x, w, t, reduction="none").shape == (0,)
    # the table scored against itself: one leaf as both operands
    y, _, _, _ = _case(50, 50, 16, torch.float32)
    y.requires_grad_()
    t = torch.arange(50, device=DEV).roll(1)
    got = torch.autograd.grad(ops.linear_cross_entropy(y, y, t), y)[0]
    _, _, g, dx, dw, *_ = _exact(y, y, t, None, "mean")
    assert float((got - (dx + dw)).abs().max()) <= 1e-5 * float((dx + dw).abs().max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,classes,width", [(16500, 70, 33), (250, 16400, 64), (16641, 300, 300), (16385, 1, 5), (9001, 8003, 40), (66000, 4501, 40)])
def test_narrow_tables(rows, classes, width, dtype):
    """Widths that leave more of a 256 wide tile empty than of a 128 wide one, at sizes with tiles enough to mind; the last in pieces."""
    _check(*_case(rows, classes, width, dtype, True, 0.1), "mean", scale=float(rows))


@pytest.mark.parametrize("dtype", TYPES)
def test_backward_after_the_operands_changed(dtype):
    """The backward pass works on the forward pass's copies: features and table may be overwritten in between, and it may run twice."""
    from obman_train_amd import ops

    x, w, t, b = _case(300, 400, 48, dtype, True)
    for v in (x, w, b):
        v.requires_grad_()
    want = torch.autograd.grad(ops.linear_cross_entropy(x, w, t, b), (x, w, b))
    loss = ops.linear_cross_entropy(x, w, t, b)
    with torch.no_grad():
        x.zero_()
        w.mul_(-3.0)
    for _ in range(2):
        assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(loss, (x, w, b), retain_graph=True), want))
    with torch.no_grad():
        b.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):  # the bias is read again
        torch.autograd.grad(loss, (x, w, b))


def test_empty_batch_of_fixed_features():
    """No rows, and only the table learns: the loss is still differentiable and the gradients are zeros."""
    from obman_train_amd import ops

    x, t = torch.zeros(2, 0, 4, device=DEV), torch.zeros(2, 0, dtype=torch.int64, device=DEV)
    for reduction in ("mean", "sum", "none"):
        w, b = torch.randn(10, 4, device=DEV, requires_grad=True), torch.randn(10, device=DEV, requires_grad=True)
        loss = ops.linear_cross_entropy(x, w, t, b, reduction=reduction)
        assert loss.shape == ((2, 0) if reduction == "none" else ())
        loss.sum().backward()
        assert torch.equal(w.grad, torch.zeros_like(w)) and torch.equal(b.grad, torch.zeros_like(b))


@pytest.mark.parametrize("dtype", TYPES)
def test_weights_of_many_rows(dtype):
    """The largest weight decides the scale of all rows' gradients: in any block of 1024 rows, the last one among them; not from an
    ignored row."""
    for rows, at in ((8193, 8192), (9001, 0), (70001, 66666)):
        x, w, t, b = _case(rows, 40, 24, dtype, True, 0.1)
        g = torch.rand(rows, generator=torch.Generator().manual_seed(at)) + 0.5
        g[at], g[at - 5] = -3e3, math.inf
        t[at], t[at - 5] = 7, IGN
        _check(x, w, t, b, "none", g_rows=g.to(DEV))


def test_on_another_stream_and_replayed_from_a_graph():
    """A captured forward and backward replays to the eager results, with eager calls of other sizes between the replays."""
    from obman_train_amd import ops

    x, w, t, b = _case(500, 900, 80, torch.bfloat16, True, 0.1)
    nx, nw, nt, nb = _case(500, 900, 80, torch.bfloat16, True, 0.1, seed=5)

    def eager(x, w, t, b):
        leaves = [v.detach().clone().requires_grad_() for v in (x, w, b)]
        loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
        return [loss.detach()] + list(torch.autograd.grad(loss, leaves))

    want, other = eager(x, w, t, b), eager(nx, nw, nt, nb)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = eager(x, w, t, b)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, r) for a, r in zip(on_side, want))
    static = [v.clone() for v in (x, w, b)]
    labels = t.clone()
    leaves = [v.requires_grad_() for v in static]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = ops.linear_cross_entropy(leaves[0], leaves[1], labels, bias=leaves[2])
        out = [loss] + list(torch.autograd.grad(loss, leaves))
    for k in range(4):
        src, ref = ((x, w, t, b), want) if k % 2 == 0 else ((nx, nw, nt, nb), other)
        with torch.no_grad():
            for to, v in zip(static, (src[0], src[1], src[3])):
                to.copy_(v)
            labels.copy_(src[2])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.detach(), r) for a, r in zip(out, ref)), k
        eager(*_case(64, 100, 16, torch.float32, True))


@pytest.mark.parametrize("scale", [1e-30, 1e-15, 1e15])
def test_fp32_operands_far_from_one(scale):
    """fp32 operands are scaled by powers of two before they are split: tiny features against a huge table and the other way round."""
    x, w, t, b = _case(90, 130, 40, torch.float32, True)
    _check(x * scale, w / scale, t, b, "sum")


def test_the_first_call_of_a_process_may_be_captured():
    """Nothing is set up lazily in a way that a stream capture refuses: a fresh process records its first forward and backward."""
    import os
    import subprocess
    import sys

    code = """
import torch
from obman_train_amd import ops, optim
x, w = torch.randn(300, 32, device="cuda", requires_grad=True), torch.randn(500, 32, device="cuda", requires_grad=True)
t = torch.randint(500, (300,), device="cuda")
y, n = torch.randn(4, 32, device="cuda"), torch.randint(500, (4,), device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    loss = ops.linear_cross_entropy(x, w, t)
    grads = torch.autograd.grad(loss, [x, w])
    norm = optim.grad_norm(grads)
    with torch.no_grad():
        score = ops.linear_cross_entropy(y, w, n)
for _ in range(3):
    graph.replay()
    torch.cuda.synchronize()
eager = ops.linear_cross_entropy(x, w, t)
assert torch.equal(eager, loss) and all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(eager, [x, w]), grads))
assert torch.equal(norm, optim.grad_norm(grads))
with torch.no_grad():
    assert torch.equal(score, ops.linear_cross_entropy(y, w, n))
print("captured ok", flush=True)
"""
    root = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, env=dict(os.environ, PYTHONPATH=root), capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and "captured ok" in done.stdout, done.stdout[-2000:] + done.stderr[-2000:]


def test_refusals():
    from obman_train_amd import _lib, ops

    x, w, t, b = _case(6, 8, 4, torch.float32, True)
    f = ops.linear_cross_entropy
    with pytest.raises(_lib.ObmanHipError):
        f(x, w.cpu(), t)
    with pytest.raises(_lib.ObmanHipError):
        f(x, w, t, bias=[0.0])
    for args, kw in (((x, w.half(), t), {}), ((x.double(), w.double(), t), {}), ((x, w, t.float()), {}), ((x, w, t), dict(bias=b.half())), ((x, w, t.short()), {})):
        with pytest.raises(TypeError):
            f(*args, **kw)
    for args, kw in (((x, w, t), dict(reduction="max")), ((x, w[:, :3], t), {}), ((x, w, t[:5]), {}), ((x, w[0], t), {}), ((x, w, t), dict(bias=b[:5])),
                     ((x, w[:0], t), {}), ((x[:, :0], w[:, :0], t), {}), ((x, w, t.view(2, 3)), {})):
        with pytest.raises(ValueError):
            f(*args, **kw)
    leaves = x.detach().requires_grad_()
    g = torch.autograd.grad(f(leaves, w, t), leaves, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_correspondence_training_step():
    """The operators together as a training loop uses them: nearest template vertices (pairmin) as labels, the loss over the vertex table,
    its gradients clipped by their global norm inside the optimizer step, twice; against the same in float64 on the CPU."""
    from obman_train_amd import ops
    from obman_train_amd.optim import ObmanAdam

    g = torch.Generator().manual_seed(0)
    points, template = torch.randn(2, 90, 3, generator=g), torch.randn(1, 162, 3, generator=g).expand(2, -1, -1).contiguous()
    feats, lift, table, bias = torch.randn(2, 90, 3, generator=g), torch.randn(32, 3, generator=g), torch.randn(162, 32, generator=g) * 0.3, torch.zeros(162)
    _, idx, _, _ = ops.pairmin(points.to(DEV), template.to(DEV), want_y=False)
    ref_idx = torch.cdist(points.double(), template.double()).argmin(2)
    assert torch.equal(idx.cpu().long(), ref_idx)
    valid = torch.rand(2, 90, generator=g) > 0.2
    labels = torch.where(valid.to(DEV), idx, torch.full_like(idx, IGN))
    params = [torch.nn.Parameter(v.to(DEV)) for v in (lift, table, bias)]
    ref = [torch.nn.Parameter(v.double()) for v in (lift, table, bias)]
    opt, ropt = ObmanAdam(params, lr=1e-2, max_grad_norm=0.05), torch.optim.Adam(ref, lr=1e-2)
    for _ in range(2):
        loss = ops.linear_cross_entropy(feats.to(DEV) @ params[0].t(), params[1], labels, bias=params[2], ignore_index=IGN)
        opt.zero_grad()
        loss.backward()
        opt.step()
        rloss = torch.nn.functional.cross_entropy((feats.double() @ ref[0].t() @ ref[1].t() + ref[2]).view(-1, 162), torch.where(valid, ref_idx, IGN).view(-1), ignore_index=IGN)
        ropt.zero_grad()
        rloss.backward()
        rnorm = torch.nn.utils.clip_grad_norm_(ref, 0.05)
        ropt.step()
        assert abs(float(loss) - float(rloss)) <= 1e-5 * float(rloss)
        assert abs(float(opt.grad_norm) - float(rnorm)) <= 1e-5 * float(rnorm) and float(rnorm) > 0.05
    for p, r in zip(params, ref):
        # Adam divides by the gradient's own size: where that is near the rounding of the fp32 gradient, the step (1e-2) may differ
        off = (p.detach().cpu().double() - r.detach()).abs()
        assert float(off.median()) <= 1e-6 and float((off > 1e-4).double().mean()) < 0.01

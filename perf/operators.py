"""The operators of the training tail, as they are measured: the loss over a table of classes with its gradient, the global
gradient norm, clipping, and the clipped optimizer step.

``own`` false: the plain form in elementary torch operations (32 bits, 64 for long sums, rounded once at the end).  ``own`` true:
the calls a user makes of ``obman_train_amd``.  ``exact`` is the definition in 64 bits."""
import math
import random

import torch

own = False

IGNORE = -100
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
LOSS_SCALE = {"fp32": 1.0, "bf16": 1.0, "fp16": 4096.0}  # what a training loop in fp16 multiplies its loss by
ADAM = dict(lr=1e-4, beta1=0.9, beta2=0.999, eps=1e-8)  # the training loop's optimizer defaults


def listed():
    return [
        # one query feature scored against the hand template's 778 vertices: the smallest call, latency only
        dict(name="score_one_hand", op="score", rows=1, classes=778, width=512, type="bf16", bias=False, ignored=0.0),
        # one query feature against every vertex of a 25-patch, 2562-vertex sphere object: one read of the class table
        dict(name="score_one_object", op="score", rows=1, classes=64050, width=512, type="bf16", bias=False, ignored=0.0),
        # 64 samples x 21 joints labelled with hand vertices, from the 256-wide hidden layer of the hand head
        dict(name="train_hand", op="train", rows=1344, classes=778, width=256, type="fp32", bias=True, ignored=0.1),
        # odd everything: point features with their 3 coordinates (512 + 3), ragged class table, masked classes, padded rows
        dict(name="train_ragged", op="train", rows=4099, classes=10007, width=515, type="fp16", bias=True, ignored=0.3),
        # 32 samples x 600 object points against a 25-patch, 642-vertex object, in the training loop's default precision
        dict(name="train_patches", op="train", rows=19200, classes=16050, width=512, type="fp32", bias=False, ignored=0.1),
        # the same points against the 25 x 2562-vertex object in bf16: the largest
        dict(name="train_object", op="train", rows=19200, classes=64050, width=512, type="bf16", bias=False, ignored=0.1),
        # gradient norm of the hand and object heads alone (frozen encoder)
        dict(name="norm_heads", op="norm", tensors="heads", total=0, type="fp32", packed=False, norm="2"),
        # norm of a large half-precision gradient set
        dict(name="norm_large", op="norm", tensors="40", total=268435456, type="bf16", packed=False, norm="2"),
        # clipping of all gradients of the hand + object model
        dict(name="clip_model", op="clip", tensors="model", total=0, type="fp32", packed=False, norm="2"),
        # clipping of a large set in two types, tensors packed back to back as in an all-reduce bucket
        dict(name="clip_large", op="clip", tensors="180", total=120000001, type="mixed", packed=True, norm="2"),
        # the optimizer step of the hand + object model with its gradient clipped
        dict(name="adam_model", op="adam", tensors="model", total=0, type="fp32", packed=False, norm="2"),
        # the same for a large set of parameters
        dict(name="adam_large", op="adam", tensors="75", total=100000000, type="fp32", packed=False, norm="2"),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["score", "score", "train", "train", "train", "norm", "clip", "adam"])
    if op in ("score", "train"):
        while True:
            rows, classes, width = _log_int(rng, 1, 19200), _log_int(rng, 33, 64050), _log_int(rng, 16, 1100)
            if rng.random() < 0.5:
                width = (width + 7) // 8 * 8
            if rows * classes * width <= 19200 * 64050 * 512 // 2:
                break
        return dict(op=op, rows=rows, classes=classes, width=width, type=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    bias=rng.random() < 0.4, ignored=rng.choice([0.0, 0.1, 0.5]))
    total = _log_int(rng, 2000, 100000000)
    return dict(op=op, tensors=str(_log_int(rng, 1, 300)), total=total, type="fp32" if op == "adam" else rng.choice(["fp32", "bf16", "fp16", "mixed"]),
                packed=rng.random() < 0.4, norm="2" if op == "adam" else rng.choice(["2", "2", "inf"]))


# ------------------------------------------------------------------------------------------------ the gradients' tensor sizes
def _encoder_sizes():
    def block(cin, cout):
        down = [cin * cout, cout, cout] if cin != cout else []
        return [cin * cout * 9, cout, cout, cout * cout * 9, cout, cout] + down

    stages = [block(a, b) + block(b, b) for a, b in ((64, 64), (64, 128), (128, 256), (256, 512))]
    return [64 * 3 * 49, 64, 64] + sum(stages, []) + [512 * 1000, 1000]


def _head_sizes():
    dense = [(1024, 512), (256, 1024), (33, 256), (10, 256), (515, 515), (257, 515), (128, 257), (3, 128), (256, 512), (3, 256), (256, 512), (1, 256)]
    norms = [515, 515, 257, 257, 128, 128]
    return sum([[a * b, a] for a, b in dense], []) + norms


def _sizes(case):
    if case["tensors"] == "heads":
        return _head_sizes()
    if case["tensors"] == "model":
        return _encoder_sizes() + _head_sizes()
    count, total = int(case["tensors"]), case["total"]
    rng = random.Random(count * 1000003 + total)
    share = [rng.random() ** 3 + 1e-3 for _ in range(count)]
    sizes = [max(1, int(total * s / sum(share))) for s in share]
    sizes[0] += max(0, total - sum(sizes))
    return sizes


def _layout(case):
    """[(which buffer, offset, size)] and the buffers' lengths: tensors start at multiples of 128 elements (allocations of their
    own) or, packed, back to back at whatever offset that gives."""
    kinds = 2 if case["type"] == "mixed" else 1
    at, end = [], [0] * kinds
    for i, n in enumerate(_sizes(case)):
        at.append((i % kinds, end[i % kinds], n))
        end[i % kinds] += n if case["packed"] else (n + 127) // 128 * 128
    return at, end


def _buffer_types(case):
    return [torch.float32, torch.bfloat16] if case["type"] == "mixed" else [TYPES[case["type"]]]


# -------------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    rand = lambda *shape: torch.rand(*shape, generator=gen, device="cuda")  # noqa: E731
    if case["op"] in ("score", "train"):
        rows, classes, width, dtype = case["rows"], case["classes"], case["width"], TYPES[case["type"]]
        weight = randn(classes, width) * (2.0 / math.sqrt(width))
        target = torch.randint(classes, (rows,), generator=gen, device="cuda")
        feats = randn(rows, width) + 1.5 * weight[target]  # features of a model in training: the label stands out, not by far
        bias = None
        if case["bias"]:
            bias = 0.5 * randn(classes)
            masked = rand(classes) < 0.05  # classes that do not occur in this batch's objects
            masked[target] = False
            bias[masked] = -math.inf
            bias = bias.to(dtype)
        target[rand(rows) < case["ignored"]] = IGNORE  # padded or unmatched rows
        train = case["op"] == "train"
        return dict(case=case, x=feats.to(dtype).requires_grad_(train), w=weight.to(dtype).requires_grad_(train), t=target,
                    b=None if bias is None else bias.requires_grad_(train), scale=torch.tensor(LOSS_SCALE[case["type"]], device="cuda"))
    at, ends = _layout(case)
    grads = [torch.zeros(end, device="cuda") for end in ends]
    spread = torch.rand(len(at), generator=gen, device="cuda").mul(-3).tolist()  # layers' gradients differ in size by up to 10^3
    for (k, off, n), e in zip(at, spread):
        grads[k][off:off + n] = randn(n) * 10.0 ** e
    grads = [g.to(t) for g, t in zip(grads, _buffer_types(case))]
    state = dict(case=case, flat_g=grads, g=[grads[k][off:off + n] for k, off, n in at], max_norm=1.0)
    if case["op"] == "norm":
        return state
    flat_p = [torch.zeros_like(g) for g in grads]
    state["flat_p"] = flat_p
    if case["op"] == "adam":
        p, m, v = flat_p[0], torch.zeros_like(flat_p[0]), torch.zeros_like(flat_p[0])
        for _, off, n in at:
            p[off:off + n] = randn(n) * 0.02
            m[off:off + n] = randn(n) * 1e-3
            v[off:off + n] = randn(n).mul_(1e-3).square_()
        state.update(m=m, v=v, steps=10)
    state["params"] = []
    for (k, off, n), g in zip(at, state["g"]):
        q = torch.nn.Parameter(flat_p[k][off:off + n])
        q.grad = g
        state["params"].append(q)
    if case["op"] == "adam" and own:
        from obman_train_amd.optim import ObmanAdam

        opt = ObmanAdam(state["params"], lr=ADAM["lr"], betas=(ADAM["beta1"], ADAM["beta2"]), eps=ADAM["eps"], max_grad_norm=state["max_norm"])
        for (k, off, n), q in zip(at, state["params"]):  # a run that goes on: its moments and step counters are there
            opt.state[q] = dict(step=torch.tensor(float(state["steps"]), device="cuda"), exp_avg=state["m"][off:off + n], exp_avg_sq=state["v"][off:off + n])
        state["opt"] = opt
    return state


# ----------------------------------------------------------------------------------------------------------------- the calls
def run(state):
    return _own(state) if own else _plain(state)


def _own(state):
    case = state["case"]
    if case["op"] == "score":
        from obman_train_amd import ops

        with torch.no_grad():
            return ops.linear_cross_entropy(state["x"], state["w"], state["t"], bias=state["b"], ignore_index=IGNORE, reduction="none")
    if case["op"] == "train":
        from obman_train_amd import ops

        loss = ops.linear_cross_entropy(state["x"], state["w"], state["t"], bias=state["b"], ignore_index=IGNORE)
        leaves = [t for t in (state["x"], state["w"], state["b"]) if t is not None]
        return [loss.detach()] + list(torch.autograd.grad(loss, leaves, grad_outputs=state["scale"]))
    from obman_train_amd import optim

    if case["op"] == "norm":
        return optim.grad_norm(state["g"], norm_type=float(case["norm"]))
    if case["op"] == "clip":
        norm = optim.clip_grad_norm_(state["params"], state["max_norm"], norm_type=float(case["norm"]))
        return [norm] + state["flat_g"]
    state["opt"].step()
    return [state["opt"].grad_norm] + state["flat_p"] + [state["m"], state["v"]]


@torch.no_grad()
def _plain(state):
    case = state["case"]
    if case["op"] in ("score", "train"):
        return _plain_loss(state, case["op"] == "train")
    if case["norm"] == "inf":
        norm = torch.stack([g.abs().max().float() for g in state["flat_g"]]).max()
    else:
        norm = torch.stack([g.double().square().sum() for g in state["flat_g"]]).sum().sqrt().float()
    if case["op"] == "norm":
        return norm
    coef = (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    if case["op"] == "clip":
        state["flat_g"][0].copy_(state["flat_g"][0].float() * coef)
        if len(state["flat_g"]) > 1:
            state["flat_g"][1].copy_(state["flat_g"][1].float() * coef)
        return [norm] + state["flat_g"]
    g, p, m, v = state["flat_g"][0] * coef, state["flat_p"][0], state["m"], state["v"]
    state["steps"] += 1
    m += (1 - ADAM["beta1"]) * (g - m)
    v *= ADAM["beta2"]
    v += (1 - ADAM["beta2"]) * g * g
    denom = v.sqrt() / math.sqrt(1 - ADAM["beta2"] ** state["steps"]) + ADAM["eps"]
    p -= ADAM["lr"] / (1 - ADAM["beta1"] ** state["steps"]) * m / denom
    return [norm, p, m, v]


def _plain_loss(state, train):
    x, w, b, target = state["x"], state["w"], state["b"], state["t"]
    keep = target != IGNORE
    at = torch.where(keep, target, 0).unsqueeze(1)
    x32, w32 = x.float(), w.float()
    logits = x32 @ w32.t()
    if b is not None:
        logits += b.float()
    top = logits.amax(1, keepdim=True)
    picked = logits.gather(1, at)
    e = logits.sub_(top).exp_()
    total = e.sum(1, keepdim=True)
    loss = torch.where(keep, (total.log() + top - picked).squeeze(1), 0.0)
    if not train:
        return loss
    count = keep.sum().clamp(min=1)
    mean = (loss.double().sum() / count).float()
    g = e.div_(total)
    g.scatter_add_(1, at, torch.full_like(picked, -1.0))
    g *= (keep / count).float().unsqueeze(1) * state["scale"]
    grads = [(g @ w32).to(x.dtype), (g.t() @ x32).to(w.dtype)]
    if b is not None:
        grads.append(g.sum(0).to(b.dtype))
    return [mean] + grads


# ---------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] in ("score", "train"):
        rows, classes, width, size = case["rows"], case["classes"], case["width"], 4 if case["type"] == "fp32" else 2
        inputs = (rows * width + classes * width + (classes if case["bias"] else 0)) * size
        if case["op"] == "score":
            return dict(bytes=inputs + 12 * rows, flops=2.0 * rows * classes * width)
        return dict(bytes=2 * inputs + 8 * rows + 4, flops=6.0 * rows * classes * width)  # the logits and two products
    size = sum(n * (4 if t == torch.float32 else 2) for (_, _, n), t in
               zip(_layout(case)[0], (_buffer_types(case) * len(_sizes(case)))))
    count = sum(_sizes(case))
    if case["op"] == "norm":
        return dict(bytes=size + 4, flops=2.0 * count)
    if case["op"] == "clip":  # the norm needs every value before the first can be scaled, but 256 MB stay near: one read, one write
        return dict(bytes=2 * size + 4, flops=3.0 * count)
    return dict(bytes=7 * size + 4, flops=16.0 * count)


# ------------------------------------------------------------------------------------------------------ the definition, 64 bits
@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("score", "train"):
        return _exact_loss(case, s)
    parts = torch.cat([g.to(torch.float64).flatten() for g in s["flat_g"]])
    norm = torch.linalg.vector_norm(parts, ord=float(case["norm"]))
    if case["op"] == "norm":
        return norm
    scale = min(1.0, s["max_norm"] / (float(norm) + 1e-6))
    clipped = [g.to(torch.float64) * scale for g in s["flat_g"]]
    if case["op"] == "clip":
        return [norm] + clipped
    g, k = clipped[0], s["steps"] + 1
    m = ADAM["beta1"] * s["m"].double() + (1 - ADAM["beta1"]) * g
    v = ADAM["beta2"] * s["v"].double() + (1 - ADAM["beta2"]) * g.square()
    mhat, vhat = m / (1 - ADAM["beta1"] ** k), v / (1 - ADAM["beta2"] ** k)
    return [norm, s["flat_p"][0].double() - ADAM["lr"] * mhat / (vhat.sqrt() + ADAM["eps"]), m, v]


def _exact_loss(case, s):
    x, w, t = s["x"].detach().double(), s["w"].detach().double(), s["t"]
    b = torch.zeros(case["classes"], dtype=torch.float64, device=x.device) if s["b"] is None else s["b"].detach().double()
    valid = (t != IGNORE).double()
    n = max(1.0, float(valid.sum()))
    losses, dx, dw, db = [], [], torch.zeros_like(w), torch.zeros_like(b)
    step = max(1, (1 << 27) // case["classes"])
    for lo in range(0, case["rows"], step):
        xs, ts, keep = x[lo:lo + step], t[lo:lo + step].clamp(min=0), valid[lo:lo + step]
        logp = torch.log_softmax(torch.addmm(b, xs, w.t()), dim=1)
        losses.append(-logp[torch.arange(len(ts), device=ts.device), ts] * keep)
        if case["op"] == "train":
            d = logp.exp_()
            d[torch.arange(len(ts), device=ts.device), ts] -= 1.0
            d *= (keep * LOSS_SCALE[case["type"]] / n).unsqueeze(1)
            dx.append(d @ w)
            dw += d.t() @ xs
            db += d.sum(0)
    losses = torch.cat(losses)
    if case["op"] == "score":
        return losses
    return [losses.sum() / n, torch.cat(dx), dw] + ([] if s["b"] is None else [db])

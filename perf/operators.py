"""The measured operators: the global gradient norm with clipping, the Adam step that clips on the way, and the row lookup
with its gradient.

  clip    vegs_amd.optim.clip_grad_norm_      the norm of all gradients together, and the gradients scaled in place
  step    vegs_amd.optim.step_many            Adam over several optimizers, its gradients clipped by their global norm
  lookup  vegs_amd.embedding.lookup           rows of a shared table by index, scaled
  train   vegs_amd.embedding.lookup           the same with the gradients of the table and of the scales

With `own` false the same results come from elementary torch operations in 32 bits.
"""
import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i32": torch.int32, "i64": torch.int64}
# floats per Gaussian of a model's six tensors (position, the two SH tensors, opacity, scaling, rotation) and their rates
WIDTHS = (3, 3, 45, 1, 3, 4)
RATES = (1.6e-4, 2.5e-3, 1.25e-4, 5e-2, 1e-3, 1e-3)
POSE = (4, 3, 3)            # a box instance's pose correction: rotation, scale, translation
BETA1, BETA2 = 0.9, 0.999
CLIP_EPS = 1e-6             # max_norm / (norm + this), at most one


def listed():
    return [
        # the pose corrections of eight box instances: 24 tensors of three or four floats, all latency
        dict(name="clip_poses", op="clip", rows=0, boxes=0, box_rows=0, poses=8, grad="f32", norm="2", active=True),
        # the dynamic part of a frame: five instance models of 8196 Gaussians and eight poses, 54 tensors that fit the cache
        dict(name="clip_instances", op="clip", rows=0, boxes=5, box_rows=8196, poses=8, grad="f32", norm="2", active=True),
        # gradients held in 16 bits, an odd number of rows, the largest magnitude as the norm
        dict(name="clip_bf16_inf", op="clip", rows=300001, boxes=0, box_rows=0, poses=0, grad="bf16", norm="inf", active=True),
        # the street model of two million Gaussians in a step whose norm stays below the bound: the usual step of a run
        dict(name="clip_model", op="clip", rows=2000000, boxes=0, box_rows=0, poses=0, grad="f32", norm="2", active=False),
        # six pose optimizers stepped together, clipped
        dict(name="step_poses", op="step", rows=0, boxes=0, box_rows=0, poses=6, active=True),
        # the whole model with an instance and three poses: five optimizers, 21 tensors, 118 M values
        dict(name="step_model", op="step", rows=2000000, boxes=1, box_rows=8196, poses=3, active=True),
        # one image's code out of a table of a few hundred
        dict(name="lookup_one", op="lookup", ids=1, table=500, width=32, data="f32", out="f32", index="i64", scale="none", skew=0.0),
        # the SH coefficients of two million Gaussians from a codebook, each with its own gain
        dict(name="lookup_sh", op="lookup", ids=2000000, table=8192, width=45, data="f32", out="f32", index="i32", scale="row", skew=0.5),
        # token rows of a 16-bit table of 32000, scaled by the root of the width
        dict(name="lookup_tokens", op="lookup", ids=16384, table=32000, width=2048, data="bf16", out="bf16", index="i64", scale="one", skew=1.0),
        # a batch of views takes its frames' corrections, ten floats each, and gives their gradients back
        dict(name="train_frames", op="train", ids=100, table=1000, width=10, data="f32", out="f32", index="i64", scale="row", skew=0.0),
        # a training step through the SH codebook
        dict(name="train_sh", op="train", ids=2000000, table=8192, width=45, data="f32", out="f32", index="i32", scale="row", skew=0.5),
        # a training step on token rows: few rows hit, some of them thousands of times, the rest of the gradient is zeros
        dict(name="train_tokens", op="train", ids=16384, table=32000, width=1024, data="bf16", out="bf16", index="i64", scale="one", skew=1.0),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("clip", "step", "lookup", "train"))
    if op in ("clip", "step"):
        kind = rng.choice(("poses", "boxes", "model"))
        # (a step returns three tensors for each of its own: at most 21 of them)
        boxes = rng.randint(1, 5 if op == "clip" else 2 if kind == "boxes" else 1)
        case = dict(op=op, rows=_log(rng, 1000, 1500000) if kind == "model" else 0,
                    boxes=boxes if kind != "poses" else 0, box_rows=_log(rng, 50, 12000),
                    poses=rng.randint(1, 8 if op == "clip" else 6 if kind == "poses" else 3))
        if op == "clip":
            case.update(grad=rng.choice(("f32", "f32", "bf16", "f16")), norm=rng.choice(("2", "2", "inf")))
        case["active"] = rng.random() < 0.7
        return case
    data = rng.choice(("f32", "f32", "bf16", "f16"))
    width = _log(rng, 1, 2500)
    # at most 40 M looked-up values and as many in the table
    return dict(op=op, ids=_log(rng, 1, min(2000000, 40000000 // width)), table=_log(rng, 16, min(60000, 40000000 // width)),
                width=width, data=data, out=rng.choice((data, "f32")), index=rng.choice(("i32", "i64")),
                scale=rng.choice(("none", "one", "row")), skew=rng.choice((0.0, 0.5, 1.0)))


def _shapes(case):
    """[(shape, learning rate)] of each optimizer: the static model, the instances' models, the poses."""
    out = []
    for rows in [case["rows"]] * (case["rows"] > 0) + [case["box_rows"]] * case["boxes"]:
        out.append([((rows, w), lr) for w, lr in zip(WIDTHS, RATES)])
    return out + [[((w,), 5e-3) for w in POSE]] * case["poses"]


def _gradient(shape, gen):
    """Gradients as a backward leaves them: magnitudes spread over decades, a third of the rows (not seen) exactly zero."""
    g = torch.randn(shape, device=DEV, generator=gen) * 10.0 ** (-3.0 * torch.rand((1,), device=DEV, generator=gen))
    if len(shape) > 1:
        g *= torch.rand((shape[0], 1), device=DEV, generator=gen) > 0.33
    return g


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    if case["op"] in ("clip", "step"):
        groups = _shapes(case)
        grads = [[_gradient(s, gen).to(TYPES[case.get("grad", "f32")]) for s, _ in group] for group in groups]
        flat = [g for group in grads for g in group]
        norm = case.get("norm", "2")
        top = [g.abs().max().float() if norm == "inf" else g.float().norm() for g in flat]
        size = float(torch.stack(top).max() if norm == "inf" else torch.stack(top).norm())
        max_norm = size * (0.37 if case["active"] else 2.5)
        if case["op"] == "clip":
            params = [torch.empty_like(g) for g in flat]
            for p, g in zip(params, flat):
                p.grad = g
            # where the clipping changes the gradients, each pass begins with the ones that a step leaves: copied anew
            return dict(case=case, params=params, grads=flat, fresh=[g.clone() for g in flat] if case["active"] else None,
                        max_norm=max_norm)
        opts = []
        for group, gs in zip(groups, grads):
            ps = [torch.nn.Parameter(torch.randn(s, device=DEV, generator=gen)) for s, _ in group]
            opt = torch.optim.Adam([{"params": [p], "lr": lr} for p, (_, lr) in zip(ps, group)], lr=0.0,
                                   betas=(BETA1, BETA2), eps=1e-15 if group[0][0] != (4,) else 1e-8)
            for p, g in zip(ps, gs):
                p.grad = g
                opt.state[p] = {"step": torch.tensor(100.0), "exp_avg": 0.1 * _gradient(g.shape, gen),
                                "exp_avg_sq": _gradient(g.shape, gen) ** 2 * 0.01 + 1e-12}
            opts.append(opt)
        return dict(case=case, opts=opts, max_norm=max_norm)
    n, k, w = case["ids"], case["table"], case["width"]
    table = torch.randn((k, w), device=DEV, generator=gen).to(TYPES[case["data"]])
    u = torch.rand((n,), device=DEV, generator=gen, dtype=torch.float64)
    # skew 0: all rows alike; towards 1: rows as words or codes occur, a few of them most of the time
    rank = k * u if case["skew"] == 0 else (k + 1.0) ** u - 1.0 if case["skew"] == 1 else k * u ** 2
    place = torch.randperm(k, device=DEV, generator=gen)
    ids = place[rank.long().clamp(0, k - 1)]
    ids = torch.where(torch.rand((n,), device=DEV, generator=gen) < 0.01, -1, ids).to(TYPES[case["index"]])   # "no row"
    scale = None
    if case["scale"] == "one":
        scale = math.sqrt(w)
    elif case["scale"] == "row":
        scale = torch.exp(0.3 * torch.randn((n,), device=DEV, generator=gen))
    state = dict(case=case, table=table, ids=ids, scale=scale)
    if case["op"] == "train":
        state["grad"] = torch.randn((n, w), device=DEV, generator=gen).to(TYPES[case["out"]])
        state["wanted"] = [table.requires_grad_(True)] + ([scale.requires_grad_(True)] if case["scale"] == "row" else [])
    return state


def _plain_norm(grads, norm):
    if norm == "inf":
        return torch.stack([g.float().abs().max() for g in grads]).max()
    return torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()


def _plain_adam(opts, coef):
    groups = [g for opt in opts for g in opt.param_groups]
    ps = [g["params"][0] for g in groups]
    state = [opt.state[g["params"][0]] for opt in opts for g in opt.param_groups]
    steps, m, v = ([s[k] for s in state] for k in ("step", "exp_avg", "exp_avg_sq"))
    torch._foreach_add_(steps, 1)
    times = [t.item() for t in steps]
    grads = torch._foreach_mul([p.grad for p in ps], coef)
    torch._foreach_mul_(m, BETA1)
    torch._foreach_add_(m, torch._foreach_mul(grads, 1 - BETA1))
    torch._foreach_mul_(v, BETA2)
    torch._foreach_add_(v, torch._foreach_mul(torch._foreach_mul(grads, grads), 1 - BETA2))
    denom = torch._foreach_div(torch._foreach_sqrt(v), [math.sqrt(1 - BETA2 ** t) for t in times])
    torch._foreach_add_(denom, [g["eps"] for g in groups])
    update = torch._foreach_div(m, denom)
    torch._foreach_sub_(ps, torch._foreach_mul(update, [g["lr"] / (1 - BETA1 ** t) for g, t in zip(groups, times)]))


@torch.no_grad()
def _plain_lookup(state):
    ids = state["ids"].long()
    there = (ids >= 0).unsqueeze(1)
    rows = state["table"].float()[ids.clamp(min=0)]
    scale = state["scale"]
    if scale is None:
        scale = 1.0
    if isinstance(scale, torch.Tensor):
        scale = scale.unsqueeze(1)
    out = torch.where(there, rows * scale, 0.0).to(TYPES[state["case"]["out"]])
    if state["case"]["op"] == "lookup":
        return [out]
    g = torch.where(there, state["grad"].float(), 0.0)
    d_table = torch.zeros(state["table"].shape, device=DEV)
    d_table.index_add_(0, ids.clamp(min=0), g * scale)
    got = [out, d_table.to(state["table"].dtype)]
    if isinstance(scale, torch.Tensor):
        got.append((g * rows).sum(1))
    return got


def _state_of(opts):
    ps = [g["params"][0] for opt in opts for g in opt.param_groups]
    state = [opt.state[g["params"][0]] for opt in opts for g in opt.param_groups]
    return [p.detach() for p in ps] + [s["exp_avg"] for s in state] + [s["exp_avg_sq"] for s in state]


def run(state):
    case = state["case"]
    if case["op"] == "clip":
        if state["fresh"] is not None:
            torch._foreach_copy_(state["grads"], state["fresh"])
        if own:
            from vegs_amd import optim
            norm = optim.clip_grad_norm_(state["params"], state["max_norm"],
                                         norm_type=math.inf if case["norm"] == "inf" else 2.0)
        else:
            norm = _plain_norm(state["grads"], case["norm"])
            coef = (state["max_norm"] / (norm + CLIP_EPS)).clamp(max=1.0)
            torch._foreach_copy_(state["grads"], torch._foreach_mul([g.float() for g in state["grads"]], coef))
        return [norm] + state["grads"]
    if case["op"] == "step":
        if own:
            from vegs_amd import optim
            norm = optim.step_many(state["opts"], max_grad_norm=state["max_norm"])
        else:
            with torch.no_grad():
                norm = _plain_norm([g["params"][0].grad for opt in state["opts"] for g in opt.param_groups], "2")
                _plain_adam(state["opts"], (state["max_norm"] / (norm + CLIP_EPS)).clamp(max=1.0))
        return [norm] + _state_of(state["opts"])
    if not own:
        return _plain_lookup(state)
    from vegs_amd import embedding
    out = embedding.lookup(state["table"], state["ids"], state["scale"], dtype=TYPES[case["out"]])
    if case["op"] == "lookup":
        return [out]
    return [out.detach()] + list(torch.autograd.grad(out, state["wanted"], state["grad"]))


def _size(kind):
    return 4 if kind in ("f32", "i32") else 8 if kind == "i64" else 2


def work(case):
    if case["op"] in ("clip", "step"):
        n = sum(math.prod(s) for group in _shapes(case) for s, _ in group)
        if case["op"] == "step":
            return {"bytes": 28.0 * n, "flops": 17.0 * n}           # four arrays read, three written
        size = _size(case["grad"])
        return {"bytes": size * n * (2.0 if case["active"] else 1.0), "flops": 3.0 * n}
    n, k, w = case["ids"], case["table"], case["width"]
    values = n * w
    used = min(k, n)             # rows that can be read at all
    moved = values * _size(case["out"]) + used * w * _size(case["data"]) + n * _size(case["index"])
    moved += n * 4 if case["scale"] == "row" else 0
    flops = values if case["scale"] != "none" else 0
    if case["op"] == "train":
        moved += values * _size(case["out"]) + k * w * _size(case["data"])
        flops += values * (1 + (case["scale"] != "none") + 2 * (case["scale"] == "row"))
        moved += n * 4 if case["scale"] == "row" else 0
    return {"bytes": float(moved), "flops": float(flops)}


def _number(x):
    return torch.tensor(x, dtype=torch.float64, device=DEV)


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] in ("clip", "step"):
            opts = state.get("opts", [])
            ps = [g["params"][0] for opt in opts for g in opt.param_groups]
            grads = [p.grad for p in ps] if opts else state["grads"]
            parts = [g.to(torch.float64).reshape(-1) for g in grads]
            if case.get("norm") == "inf":
                norm = max(float(torch.maximum(x.max(), -x.min())) for x in parts)
            else:
                norm = math.sqrt(math.fsum(float(torch.dot(x, x)) for x in parts))
            factor = min(1.0, state["max_norm"] / (norm + CLIP_EPS))
            if not opts:
                return [_number(norm)] + [(factor * x).reshape(g.shape) for x, g in zip(parts, grads)]
            kinds = ([], [], [])
            for opt in opts:
                for group in opt.param_groups:
                    p = group["params"][0]
                    st = opt.state[p]
                    t = float(st["step"]) + 1
                    g = p.grad.double() * factor
                    m = BETA1 * st["exp_avg"].double() + (1 - BETA1) * g
                    v = BETA2 * st["exp_avg_sq"].double() + (1 - BETA2) * g ** 2
                    m_hat, v_hat = m / (1 - BETA1 ** t), v / (1 - BETA2 ** t)
                    kinds[0].append(p.detach().double() - group["lr"] * m_hat / (v_hat ** 0.5 + group["eps"]))
                    kinds[1].append(m)
                    kinds[2].append(v)
            return [_number(norm)] + kinds[0] + kinds[1] + kinds[2]
        ids, table, scale = state["ids"].long(), state["table"].detach().double(), state["scale"]
        n, k = ids.shape[0], table.shape[0]
        padded = torch.cat((table, torch.zeros_like(table[:1])))           # the row of "no row"
        ids = torch.where(ids < 0, k, ids)
        rows = padded.index_select(0, ids)
        by_row = isinstance(scale, torch.Tensor)
        s = scale.detach().double().reshape(n, 1) if by_row else torch.full((n, 1), scale or 1.0, dtype=torch.float64, device=DEV)
        out = [rows * s]
        if case["op"] == "train":
            g = state["grad"].double()
            if by_row:
                d_scale = torch.linalg.vecdot(g, rows)
            order = torch.argsort(ids, stable=True)
            del rows
            sums = torch.cat((torch.zeros_like(g[:1]), torch.cumsum((g * s).index_select(0, order), 0)))
            ends = torch.searchsorted(ids[order], torch.arange(k + 1, device=DEV), right=False)
            out.append(sums[ends[1:]] - sums[ends[:-1]])
            if by_row:
                out.append(d_scale)
        return out


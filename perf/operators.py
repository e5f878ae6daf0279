"""The vocabulary operators and the clipping of many gradients: cases, plain forms and the framework's calls.

Three operators: the softmax cross entropy of a linear layer over a large vocabulary with its gradients (kind "xent"), the lookup of
token embeddings and the gradient of the table ("embed", "embed_grad"), and the global norm of many gradient tensors with the clipping
by it ("clip").  ``run`` computes them with elementary torch operations, or calls vision_transformers_torch_xla_amd.ops where
``own`` is true."""
import math

import torch

own = False

DEVICE = "cuda"
IGNORE = -100
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}

# parameter shapes of a plain transformer of the given width and depth, the way this repository's models have them
def _layer_shapes(width, depth, classes):
    shapes = [(classes, width), (classes,), (1, 197, width), (1, 1, width), (width, 3, 16, 16), (width,), (width,), (width,)]
    for _ in range(depth):
        shapes += [(3 * width, width), (3 * width,), (width, width), (width,), (4 * width, width), (4 * width,), (width, 4 * width)] + [(width,)] * 5
    return shapes


def listed():
    return [
        # one image's class scores during serving: the latency of the smallest call
        {"name": "xent_eval_1x1000x192", "kind": "xent", "t": 1, "v": 1000, "d": 192, "grad": False, "bias": True, "smoothing": 0.0, "ignored": 0.0},
        # a training step of a head with 21843 classes over one batch of pooled features
        {"name": "xent_train_512x21843x768", "kind": "xent", "t": 512, "v": 21843, "d": 768, "grad": True, "bias": True, "smoothing": 0.1, "ignored": 0.0},
        # prediction of visual tokens: 128 images of 196 positions, the positions that were not masked are not counted
        {"name": "xent_train_25088x8192x768", "kind": "xent", "t": 25088, "v": 8192, "d": 768, "grad": True, "bias": False, "smoothing": 0.0, "ignored": 0.4},
        # a language model's training step, odd vocabulary: the largest case
        {"name": "xent_train_8192x100003x2048", "kind": "xent", "t": 8192, "v": 100003, "d": 2048, "grad": True, "bias": False, "smoothing": 0.0, "ignored": 0.02},
        # perplexity of a held-out text: losses alone
        {"name": "xent_eval_2047x50021x1024", "kind": "xent", "t": 2047, "v": 50021, "d": 1024, "grad": False, "bias": False, "smoothing": 0.0, "ignored": 0.01},
        # the token of a decoding step
        {"name": "embed_1x8192x768", "kind": "embed", "t": 1, "v": 8192, "d": 768, "type": "bf16", "hot": True},
        # the tokens of a training batch
        {"name": "embed_65536x50021x1024", "kind": "embed", "t": 65536, "v": 50021, "d": 1024, "type": "bf16", "hot": True},
        # the gradient of the table: words of a text, one of them padding
        {"name": "embed_grad_16384x50021x768", "kind": "embed_grad", "t": 16384, "v": 50021, "d": 768, "type": "bf16", "hot": True, "padding": 0.2},
        # the same for visual tokens into an fp32 gradient: 512 images of 196 positions, every row is hit
        {"name": "embed_grad_100352x8192x768", "kind": "embed_grad", "t": 100352, "v": 8192, "d": 768, "type": "f32", "hot": False, "padding": 0.0},
        # a probe that trains a head and two norms: few small tensors
        {"name": "clip_6_small", "kind": "clip", "count": 6, "width": 192, "total": 0, "type": "f32", "clipped": True},
        # the gradients of a transformer of width 384 with 12 layers
        {"name": "clip_152_w384", "kind": "clip", "count": 152, "width": 384, "total": 0, "type": "f32", "clipped": True},
        # a large model's gradients in two types, of many sizes
        {"name": "clip_400_mixed", "kind": "clip", "count": 400, "width": 0, "total": 600000000, "type": "mixed", "clipped": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["xent", "xent", "xent", "embed", "embed_grad", "clip"])
    if kind == "xent":
        while True:
            t, v, d = _log(rng, 1, 32768), _log(rng, 2, 131072), 8 * _log(rng, 2, 512)
            if t * v * d <= 1.6e12 and t * v <= 8e8 and v * d <= 3e8:
                break
        return {"kind": kind, "t": t, "v": v, "d": d, "grad": rng.random() < 0.7, "bias": rng.random() < 0.5, "smoothing": rng.choice([0.0, 0.1]),
                "ignored": rng.choice([0.0, 0.1, 0.5])}
    if kind in ("embed", "embed_grad"):
        while True:
            t, v, d = _log(rng, 1, 131072), _log(rng, 2, 131072), 8 * _log(rng, 2, 512)
            if t * d <= 1.3e8 and v * d <= 2e8:
                break
        case = {"kind": kind, "t": t, "v": v, "d": d, "type": rng.choice(["bf16", "f32"]), "hot": rng.random() < 0.5}
        if kind == "embed_grad":
            case["padding"] = rng.choice([0.0, 0.3])
        return case
    return {"kind": kind, "count": _log(rng, 1, 400), "width": 0, "total": _log(rng, 2000, 400000000), "type": rng.choice(["f32", "bf16", "mixed"]),
            "clipped": rng.random() < 0.8}


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _tokens(g, t, v, hot):
    """Token numbers: all alike, or a few of them most of the time as words are (the share of a token falls with its rank)."""
    u = torch.rand(t, generator=g, device=DEVICE, dtype=torch.float64)
    rank = (torch.exp(u * math.log(v + 1.0)) - 1.0 if hot else u * v).long().clamp_(0, v - 1)
    step = 7919 if math.gcd(7919, v) == 1 else 1
    return rank * step % v


def _clip_sizes(case, seed):
    if case["width"]:
        if case["count"] == 6:
            w = case["width"]
            return [(1000, w), (1000,), (w,), (w,), (w,), (w,)]
        return _layer_shapes(case["width"], (case["count"] - 8) // 12, 1000)
    n = case["count"]
    share = torch.rand(n, generator=torch.Generator().manual_seed(n * 7 + case["total"] % 1000003)) ** 4 + 1e-4       # a few large, many small
    sizes = (share / share.sum() * case["total"]).long().clamp_(min=1).tolist()
    return [(s,) for s in sizes]


def prepare(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    state = {"case": case, "kind": kind}
    if kind == "xent":
        t, v, d = case["t"], case["v"], case["d"]
        target = _tokens(g, t, v, True)
        # features of a model that has learned something: the target's class direction on top of noise
        w = torch.randn(v, d, generator=g, device=DEVICE) * (2.0 / math.sqrt(d))
        x = torch.randn(t, d, generator=g, device=DEVICE)
        x += w[target] * (torch.rand(t, 1, generator=g, device=DEVICE) * 2.0)
        if case["ignored"]:
            target[torch.rand(t, generator=g, device=DEVICE) < case["ignored"]] = IGNORE
        state.update(x=x.bfloat16(), w=w.bfloat16(), target=target,
                     b=(torch.randn(v, generator=g, device=DEVICE) * 0.5).bfloat16() if case["bias"] else None)
    elif kind in ("embed", "embed_grad"):
        t, v, d, dt = case["t"], case["v"], case["d"], TYPES[case["type"]]
        ids = _tokens(g, t, v, case["hot"])
        if kind == "embed":
            state.update(ids=ids, table=torch.randn(v, d, generator=g, device=DEVICE).to(dt))
        else:
            if case["padding"]:
                ids[torch.rand(t, generator=g, device=DEVICE) < case["padding"]] = v - 1
            state.update(ids=ids, dout=torch.randn(t, d, generator=g, device=DEVICE).bfloat16(), padding=v - 1 if case["padding"] else None)
    else:
        shapes = _clip_sizes(case, seed)
        types = [TYPES[case["type"]] if case["type"] != "mixed" else (torch.bfloat16 if i % 3 else torch.float32) for i in range(len(shapes))]
        grads = [(torch.randn(s, generator=g, device=DEVICE) * 0.01).to(dt) for s, dt in zip(shapes, types)]
        count = sum(t.numel() for t in grads)
        norm = 0.01 * math.sqrt(count)          # near the norm that the gradients have
        # the clipped gradients go to buffers of their own, one for each type, so that every pass finds the same gradients
        flat, out = {}, []
        for dt in sorted(set(types), key=str):
            flat[str(dt)] = torch.zeros(sum(_room(math.prod(s)) for s, u in zip(shapes, types) if u == dt), dtype=dt, device=DEVICE)
        at = dict.fromkeys(flat, 0)
        for s, dt in zip(shapes, types):
            first, n = at[str(dt)], math.prod(s)
            out.append(flat[str(dt)][first:first + n].view(s))
            at[str(dt)] += _room(n)
        state.update(grads=grads, out=out, flat=flat, max_norm=0.37 * norm if case["clipped"] else 4.0 * norm)
    return state


def _room(n):
    return (n + 63) // 64 * 64          # a tensor's place in a flat buffer starts at a multiple of 64 values


def _scale(d):
    return math.sqrt(d)


def run(state):
    if own:
        return _run_own(state)
    return {"xent": _plain_xent, "embed": _plain_embed, "embed_grad": _plain_embed_grad, "clip": _plain_clip}[state["kind"]](state)


def _run_own(state):
    from vision_transformers_torch_xla_amd import ops
    case, kind = state["case"], state["kind"]
    if kind == "xent":
        r = ops.linear_xent(state["x"], state["w"], state["target"], bias=state["b"], smoothing=case["smoothing"], ignore_index=IGNORE,
                            reduction="mean", want_grad=case["grad"])
        out = {"loss": r.loss, "rows": r.rows}
        if case["grad"]:
            out.update(dx=r.dx, dw=r.dweight)
            if case["bias"]:
                out["db"] = r.dbias
        return out
    if kind == "embed":
        return ops.embedding_fwd(state["ids"], state["table"], scale=_scale(case["d"]))
    if kind == "embed_grad":
        return ops.embedding_bwd(state["dout"], state["ids"], case["v"], scale=_scale(case["d"]), padding_idx=state["padding"],
                                 out_dtype=TYPES[case["type"]])
    norm = ops.clip_grads(state["grads"], state["max_norm"], out=state["out"])
    return {"norm": norm, "grads": state["flat"]}


def _plain_xent(state):
    case = state["case"]
    x, w, target = state["x"].float(), state["w"].float(), state["target"]
    v, eps = case["v"], case["smoothing"]
    z = x @ w.t()
    if state["b"] is not None:
        z = z + state["b"].float()
    top = z.max(dim=1, keepdim=True).values
    lse = top + torch.log(torch.exp(z - top).sum(dim=1, keepdim=True))
    counted = target != IGNORE
    at = torch.where(counted, target, torch.zeros_like(target)).unsqueeze(1)
    rows = lse[:, 0] - (1.0 - eps) * z.gather(1, at)[:, 0] - (eps / v) * z.sum(dim=1)
    rows = torch.where(counted, rows, torch.zeros_like(rows))
    count = counted.sum()
    loss = rows.sum() / count.clamp(min=1)
    out = {"loss": loss, "rows": rows}
    if case["grad"]:
        dz = torch.exp(z - lse) - eps / v
        dz.scatter_add_(1, at, torch.full_like(lse, -(1.0 - eps)))
        dz = dz * (counted / count.clamp(min=1)).unsqueeze(1)
        out.update(dx=(dz @ w).to(torch.bfloat16), dw=(dz.t() @ x).to(torch.bfloat16))
        if state["b"] is not None:
            out["db"] = dz.sum(dim=0).to(torch.bfloat16)
    return out


def _plain_embed(state):
    table = state["table"]
    return (table[state["ids"]].float() * _scale(state["case"]["d"])).to(table.dtype)


def _plain_embed_grad(state):
    case, ids = state["case"], state["ids"]
    dout = state["dout"].float()
    if state["padding"] is not None:
        dout = dout * (ids != state["padding"]).unsqueeze(1)
    grad = torch.zeros(case["v"], case["d"], dtype=torch.float32, device=ids.device)
    grad.index_add_(0, ids, dout)
    return (grad * _scale(case["d"])).to(TYPES[case["type"]])


def _plain_clip(state):
    grads = state["grads"]
    norm = torch.sqrt(torch.stack([t.float().square().sum() for t in grads]).sum())
    coef = torch.clamp(state["max_norm"] / (norm + 1e-6), max=1.0)
    [to.copy_(t.float() * coef) for t, to in zip(grads, state["out"])]
    return {"norm": norm, "grads": state["flat"]}


def work(case):
    kind = case["kind"]
    if kind == "xent":
        t, v, d = case["t"], case["v"], case["d"]
        reads = 2.0 * (t * d + v * d) + 8.0 * t + (2.0 * v if case["bias"] else 0.0)
        writes = 4.0 * t + 4.0 + (2.0 * (t * d + v * d) + (2.0 * v if case["bias"] else 0.0) if case["grad"] else 0.0)
        return {"bytes": reads + writes, "flops": (6.0 if case["grad"] else 2.0) * t * v * d}
    if kind in ("embed", "embed_grad"):
        t, v, d = case["t"], case["v"], case["d"]
        size = 2.0 if case["type"] == "bf16" else 4.0
        if kind == "embed":
            return {"bytes": 8.0 * t + size * (min(t, v) * d + t * d), "flops": 1.0 * t * d}
        return {"bytes": 8.0 * t + 2.0 * t * d + size * v * d, "flops": 1.0 * t * d}
    sizes = [math.prod(s) for s in _clip_sizes(case, 0)]
    per = [4.0 if case["type"] == "f32" or (case["type"] == "mixed" and i % 3 == 0) else 2.0 for i in range(len(sizes))]
    return {"bytes": sum(2.0 * n * b for n, b in zip(sizes, per)), "flops": 3.0 * sum(sizes)}


def exact(case, seed):
    """The operators from their definitions in 64 bits; the cross entropy goes through the rows in blocks, from log-probabilities."""
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "xent":
        x, w, target = s["x"].double(), s["w"].double(), s["target"]
        t, v, eps = case["t"], case["v"], case["smoothing"]
        counted = torch.nonzero(target != IGNORE)[:, 0]
        n = max(1, counted.numel())
        rows = torch.zeros(t, dtype=torch.float64, device=x.device)
        dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros(v, dtype=torch.float64, device=x.device)
        block = max(1, min(t, 200000000 // v))
        for part in counted.split(block):
            q = torch.full((part.numel(), v), eps / v, dtype=torch.float64, device=x.device)        # the target distribution
            q[torch.arange(part.numel(), device=x.device), target[part]] += 1.0 - eps
            z = x[part] @ w.t()
            if s["b"] is not None:
                z += s["b"].double()
            logp = torch.log_softmax(z, dim=1)
            rows[part] = -(q * logp).sum(dim=1)
            if case["grad"]:
                dz = (logp.exp() - q) / n
                dx[part] = dz @ w
                dw += dz.t() @ x[part]
                db += dz.sum(dim=0)
        out = {"loss": rows.sum() / n, "rows": rows}
        if case["grad"]:
            out.update(dx=dx, dw=dw)
            if s["b"] is not None:
                out["db"] = db
        return out
    if kind == "embed":
        return s["table"].double().index_select(0, s["ids"]) * case["d"] ** 0.5
    if kind == "embed_grad":
        keep = torch.nonzero(s["ids"] != s["padding"])[:, 0] if s["padding"] is not None else torch.arange(case["t"], device=s["ids"].device)
        grad = torch.zeros(case["v"], case["d"], dtype=torch.float64, device=s["ids"].device)
        for part in keep.split(16384):
            grad.index_add_(0, s["ids"][part], s["dout"][part].double())
        return grad * case["d"] ** 0.5
    total = sum(float(t.double().pow(2).sum()) for t in s["grads"]) ** 0.5
    coef = min(1.0, s["max_norm"] / (total + 1e-6))
    flat = {}
    for t in s["grads"]:
        flat.setdefault(str(t.dtype), []).append(torch.nn.functional.pad(t.double().reshape(-1) * coef, (0, _room(t.numel()) - t.numel())))
    return {"norm": torch.tensor(total, dtype=torch.float64), "grads": {k: torch.cat(v) for k, v in flat.items()}}

"""Measured cases of the operators that train the tables and norms around a decoder.

Each case runs one operator once, in two forms: elementary fp32 torch operations
(``own = False``) or the framework's entry points (``own = True``):

* ``loss``   -- cross entropy of hidden states against a vocabulary projection, with
  the gradients of the hidden states and of the projection;
* ``embed``  -- scaled embedding lookup and the gradient of its table;
* ``norm``   -- layer norm, forward and backward with the weight's and bias's gradient;
* ``clip``   -- global norm of many gradient tensors, and clipping by it.
"""

import math
import random

import torch

own = False

IGNORE = -100
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # a short answer through the smoke model's head: launch latency
        {"name": "loss tiny", "op": "loss", "tokens": 61, "hidden": 512, "vocab": 4096, "valid": 0.8,
         "reduction": "mean"},
        # ragged everything, a signed weight per token (a policy-gradient step), prompts masked out
        {"name": "loss ragged", "op": "loss", "tokens": 777, "hidden": 1000, "vocab": 50001, "valid": 0.6,
         "reduction": "none"},
        # a supervised micro-batch of the 8B-shaped config, a quarter of it prompt
        {"name": "loss batch", "op": "loss", "tokens": 8192, "hidden": 4096, "vocab": 151936, "valid": 0.75,
         "reduction": "mean"},
        # a short prompt through the smoke model's table
        {"name": "embed tiny", "op": "embed", "tokens": 64, "hidden": 512, "vocab": 4096, "dtype": "bf16",
         "scale": 22.627416997969522, "pad": 0.0, "into": False},
        # a padded micro-batch, fp32 table with odd rows, the gradient added to one that is there;
        # two fifths of the tokens are the same padding token
        {"name": "embed ragged into", "op": "embed", "tokens": 24571, "hidden": 1001, "vocab": 50001, "dtype": "fp32",
         "scale": 0.5, "pad": 0.4, "into": True},
        # a micro-batch of the 8B-shaped config, the whole table's gradient
        {"name": "embed batch", "op": "embed", "tokens": 8192, "hidden": 4096, "vocab": 151936, "dtype": "bf16",
         "scale": 1.0, "pad": 0.0, "into": False},
        # one small image in the vision tower
        {"name": "norm tiny", "op": "norm", "rows": 256, "hidden": 1152, "dtype": "bf16"},
        # odd rows, fp32 master weights
        {"name": "norm odd", "op": "norm", "rows": 5003, "hidden": 1001, "dtype": "fp32"},
        # a batch of large images in the vision tower
        {"name": "norm batch", "op": "norm", "rows": 65536, "hidden": 1152, "dtype": "bf16"},
        # a few small gradients, clipped into the optimizer's buffer: launch latency
        {"name": "clip tiny", "op": "clip", "tensors": 12, "total": 10007, "layout": 3, "dtype": "fp32", "out": True},
        # the LoRA gradients of the 8B-shaped config (36 layers, seven linears, rank 16), below the limit
        {"name": "clip lora", "op": "clip", "tensors": 504, "total": 43646976, "layout": 0, "dtype": "fp32",
         "out": False},
        # the bf16 gradients of a small fully trained model, clipped into fp32 optimizer buffers
        {"name": "clip full", "op": "clip", "tensors": 220, "total": 600000011, "layout": 5, "dtype": "bf16",
         "out": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("loss", "embed", "norm", "clip"))
    if op == "loss":
        hidden = rng.choice((_log(rng, 64, 4096), 8 * _log(rng, 8, 512)))
        vocab = _log(rng, 1000, 151936)
        return {"op": op, "tokens": _log(rng, 1, 8192), "hidden": min(hidden, 4096), "vocab": vocab,
                "valid": rng.choice((1.0, 0.75, 0.5, 0.1)), "reduction": rng.choice(("mean", "none"))}
    if op == "embed":
        hidden = rng.choice((_log(rng, 64, 4096), 8 * _log(rng, 8, 512)))
        return {"op": op, "tokens": _log(rng, 1, 24576), "hidden": min(hidden, 4096), "vocab": _log(rng, 1000, 151936),
                "dtype": rng.choice(("bf16", "bf16", "fp32", "fp16")), "scale": rng.choice((1.0, 0.5, 11.25)),
                "pad": rng.choice((0.0, 0.2, 0.6)), "into": rng.random() < 0.4}
    if op == "norm":
        hidden = rng.choice((_log(rng, 64, 8192), 8 * _log(rng, 8, 1024)))
        rows = min(_log(rng, 1, 65536), max(1, 75000000 // hidden))
        return {"op": op, "rows": rows, "hidden": hidden, "dtype": rng.choice(("bf16", "bf16", "fp32", "fp16"))}
    total = _log(rng, 1000, 300000000)
    return {"op": op, "tensors": min(_log(rng, 1, 1000), total // 8), "total": total, "layout": rng.randrange(1, 1 << 20),
            "dtype": rng.choice(("fp32", "bf16")), "out": rng.random() < 0.6}


def _tensor_sizes(case):
    """Sizes of the gradient tensors: the LoRA factors of the 8B-shaped config
    (layout 0), else a few large tensors and many small ones, odd sizes among them."""
    if case["layout"] == 0:
        dims = [(4096, 4096), (4096, 1024), (4096, 1024), (4096, 4096), (4096, 12288), (4096, 12288), (12288, 4096)]
        return [16 * d for _ in range(36) for pair in dims for d in pair]
    rng = random.Random(case["layout"])
    n, total = case["tensors"], case["total"]
    weight = [math.exp(rng.uniform(0.0, 6.0)) for _ in range(n)]
    whole = sum(weight)
    sizes = [max(1, int(total * w / whole)) for w in weight]
    sizes[0] = max(1, sizes[0] + total - sum(sizes))
    return sizes


def _valid_tokens(case):
    return max(1, int(round(case["tokens"] * case["valid"])))


def _touched_rows(case):
    """Expected number of distinct rows among the ids that ``prepare`` draws."""
    pads = int(case["tokens"] * case["pad"])
    edge = torch.linspace(0, 1, case["vocab"] + 1, dtype=torch.float64) ** (1 / 3)
    some = 1 - (1 - edge.diff()) ** (case["tokens"] - pads)
    return float(some.sum()) + (float(1 - some[-1]) if pads else 0.0)


def work(case):
    op = case["op"]
    if op == "loss":
        T, H, V, n = case["tokens"], case["hidden"], case["vocab"], _valid_tokens(case)
        # hidden states of the trained tokens and the projection in, their gradients out (all T rows of
        # the hidden states' gradient are written); three products
        return {"bytes": 2 * n * H + 2 * T * H + 4 * V * H + 8 * T, "flops": 6 * n * H * V}
    if op == "embed":
        T, H, V, e = case["tokens"], case["hidden"], case["vocab"], _SIZE[case["dtype"]]
        rows = _touched_rows(case)
        # lookup: the touched rows in, T rows out; gradient: dy in, and the whole table or the touched rows in and out
        table = 2 * rows * H * e if case["into"] else V * H * e
        return {"bytes": (rows + T) * H * e + T * H * e + table + 16 * T, "flops": 2 * T * H}
    if op == "norm":
        n = case["rows"] * case["hidden"] * _SIZE[case["dtype"]]
        # forward: x in, y out; backward: x and dy in, dx out
        return {"bytes": 5 * n, "flops": 20 * case["rows"] * case["hidden"]}
    n, e = case["total"], _SIZE[case["dtype"]]
    return {"bytes": n * e + (4 * n if case["out"] else 0), "flops": 3 * n}


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    op = case["op"]
    s = {"case": case}
    if op == "loss":
        T, H, V, n = case["tokens"], case["hidden"], case["vocab"], _valid_tokens(case)
        s["h"] = randn(T, H).to(torch.bfloat16)                                  # normed hidden states
        s["w"] = (randn(V, H) * (2.5 / math.sqrt(H))).to(torch.bfloat16)         # logits of a few units
        t = (V * rand(T) ** 3).long().clamp_(max=V - 1)                          # frequent and rare tokens
        t[torch.randperm(T, generator=g, device="cuda")[n:]] = IGNORE
        s["targets"] = t
        s["g"] = randn(T) / T if case["reduction"] == "none" else None           # advantage of each token
    elif op == "embed":
        T, H, V, dt = case["tokens"], case["hidden"], case["vocab"], _TYPES[case["dtype"]]
        s["table"] = (randn(V, H) * 0.05).to(dt)
        ids = (V * rand(T) ** 3).long().clamp_(max=V - 1)
        ids[: int(T * case["pad"])] = V - 1                                      # left padding, one row's worth of it
        s["ids"] = ids
        s["dy"] = randn(T, H).to(dt)
        s["out"] = randn(V, H).to(dt) if case["into"] else None
    elif op == "norm":
        R, H, dt = case["rows"], case["hidden"], _TYPES[case["dtype"]]
        s["x"] = (randn(R, H) * (0.5 + rand(R, 1)) + 0.5 * randn(R, 1)).to(dt)
        s["w"] = (1 + 0.1 * randn(H)).to(dt)
        s["b"] = (0.1 * randn(H)).to(dt)
        s["dy"] = randn(R, H).to(dt)
    else:
        sizes = _tensor_sizes(case)
        flat = s["flat"] = randn(sum(sizes)).mul_(1e-3).to(_TYPES[case["dtype"]])
        s["grads"] = list(flat.split(sizes))                                     # views, at any alignment
        expect = 1e-3 * math.sqrt(flat.numel())
        s["out_flat"] = s["out"] = None
        s["max_norm"] = 2.0 * expect
        if case["out"]:
            s["out_flat"] = torch.empty(flat.numel(), device="cuda", dtype=torch.float32)
            s["out"] = list(s["out_flat"].split(sizes))
            s["max_norm"] = 0.25 * expect
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    op = s["case"]["op"]
    if op == "loss":
        from graspo_b200.ops.cross_entropy import linear_cross_entropy_grads

        return linear_cross_entropy_grads(s["h"], s["w"], s["targets"], grad=s["g"], ignore_index=IGNORE,
                                          reduction=s["case"]["reduction"])
    if op == "embed":
        from graspo_b200.ops.embedding import embedding, embedding_grad

        y = embedding(s["ids"], s["table"], scale=s["case"]["scale"])
        return y, embedding_grad(s["dy"], s["ids"], s["table"].shape[0], scale=s["case"]["scale"], out=s["out"])
    if op == "norm":
        from graspo_b200.ops.layer_norm import layer_norm_backward, layer_norm_forward

        y, mean, rstd = layer_norm_forward(s["x"], s["w"], s["b"], 1e-6)
        return (y, *layer_norm_backward(s["dy"], s["x"], s["w"], mean, rstd))
    from graspo_b200.ops.grad_clip import clip_grad_norm_

    norm = clip_grad_norm_(s["grads"], s["max_norm"], out=s["out"])
    return norm, s["out_flat"] if s["out"] is not None else s["flat"]


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "loss":
        h, w, t = s["h"].float(), s["w"].float(), s["targets"]
        live = t != IGNORE
        at = t.clamp(min=0)[:, None]
        logits = h @ w.T
        top = logits.amax(-1, keepdim=True)
        e = torch.exp(logits - top)
        z = e.sum(-1, keepdim=True)
        per_token = torch.where(live, (z.log() + top - logits.gather(1, at))[:, 0], 0.0)
        if case["reduction"] == "mean":
            count = live.sum().clamp(min=1)
            loss, scale = per_token.sum() / count, live / count
        else:
            loss, scale = per_token, torch.where(live, s["g"], 0.0)
        p = e / z
        p.scatter_add_(1, at, torch.full_like(at, -1, dtype=p.dtype))
        p *= scale[:, None]
        return loss, (p @ w).to(s["h"].dtype), (p.T @ h).to(s["w"].dtype)
    if op == "embed":
        table, ids, dy = s["table"], s["ids"], s["dy"]
        y = (table[ids].float() * case["scale"]).to(table.dtype)
        if s["out"] is None:
            grad = torch.zeros(table.shape, device=table.device, dtype=torch.float32)
            grad.index_add_(0, ids, dy.float() * case["scale"])
            return y, grad.to(table.dtype)
        grad = s["out"].float()
        grad.index_add_(0, ids, dy.float() * case["scale"])
        return y, s["out"].copy_(grad)
    if op == "norm":
        x, w, dy = s["x"].float(), s["w"].float(), s["dy"].float()
        c = x - x.mean(-1, keepdim=True)
        rstd = 1.0 / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-6)
        n = c * rstd
        y = n * w + s["b"].float()
        a = dy * w
        dx = rstd * (a - a.mean(-1, keepdim=True) - n * (a * n).mean(-1, keepdim=True))
        dt = s["x"].dtype
        return y.to(dt), dx.to(dt), (dy * n).sum(0).to(dt), dy.sum(0).to(dt)
    norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
    coef = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    if s["out"] is None:
        [g.copy_(g.float() * coef) for g in s["grads"]]
        return norm, s["flat"]
    [o.copy_(g.float() * coef) for o, g in zip(s["out"], s["grads"])]
    return norm, s["out_flat"]


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "loss":
        h, w, t = s["h"], s["w"].double(), s["targets"]
        T = t.numel()
        rows = (t != IGNORE).nonzero()[:, 0]
        weight = torch.full((T,), 1.0 / rows.numel(), dtype=torch.float64, device="cuda") \
            if case["reduction"] == "mean" else s["g"].double()
        loss = torch.zeros(T, dtype=torch.float64, device="cuda")
        dh = torch.zeros(h.shape, dtype=torch.float64, device="cuda")
        dw = torch.zeros(w.shape, dtype=torch.float64, device="cuda")
        for r in rows.split(1024):
            hr = h[r].double()
            logp = torch.log_softmax(hr @ w.T, -1)
            pick = (torch.arange(r.numel(), device="cuda"), t[r])
            loss[r] = -logp[pick]
            d = logp.exp_()
            d[pick] -= 1.0
            d *= weight[r, None]
            dh[r] = d @ w
            dw.addmm_(d.T, hr)
        return (loss.sum() / rows.numel() if case["reduction"] == "mean" else loss), dh, dw
    if op == "embed":
        ids, dy = s["ids"], s["dy"].double() * case["scale"]
        y = s["table"].index_select(0, ids).double() * case["scale"]
        order = torch.argsort(ids, stable=True)
        used, count = torch.unique_consecutive(ids[order], return_counts=True)
        end = count.cumsum(0)
        run = torch.cumsum(dy[order], 0)
        upto = run[end - 1]
        sums = upto - torch.cat([torch.zeros_like(upto[:1]), upto[:-1]])
        grad = s["out"].double() if case["into"] else torch.zeros(s["table"].shape, dtype=torch.float64, device="cuda")
        grad[used] += sums
        return y, grad
    if op == "norm":
        x, w, dy = s["x"].double(), s["w"].double(), s["dy"].double()
        var, mean = torch.var_mean(x, -1, keepdim=True, correction=0)
        sd = torch.sqrt(var + 1e-6)
        n = (x - mean) / sd
        H = x.shape[-1]
        a = dy * w
        dx = (H * a - a.sum(-1, keepdim=True) - n * (a * n).sum(-1, keepdim=True)) / (H * sd)
        return torch.addcmul(s["b"].double(), n, w), dx, torch.einsum("rh,rh->h", dy, n), dy.sum(0)
    norm = torch.linalg.vector_norm(s["flat"], dtype=torch.float64)
    coef = min(1.0, s["max_norm"] / (float(norm) + 1e-6))
    out = s["flat"].to(torch.float64).mul_(coef)
    return norm, out

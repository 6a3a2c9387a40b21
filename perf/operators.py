"""Performance cases of the operators around a training step's products: the vocabulary loss in pieces, layer norm, rotary
positions, and the global gradient norm with clipping.

    ce    softmax cross entropy of ``hidden @ weight.T`` over a large vocabulary, with the gradients of both
    norm  layer norm, forward and (in training) backward with the gradients of weight and bias
    rope  rotary positions of queries and keys, forward and (in training) backward
    clip  global 2-norm of many gradient tensors, and the clipped gradients written to the flat buffers of an optimizer

`own` selects the framework's operators; otherwise `run` computes them in elementary torch operations, in 32 bits (angles and
the norm's sum in 64).
"""
import math
import random

import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MOST_PRODUCT = 8192 * 50048 * 1024          # rows x vocabulary x hidden of the largest loss
MOST_NORM = 16384 * 1024                    # elements of the largest layer norm
MOST_ROPE = 65537 * 10 * 128                # elements of the largest rotation
MOST_CLIP = 200_000_000                     # elements of the largest gradient list


def _ce(rows, vocab, hidden, train, reduction, ignored, **more):
    return dict(kind="ce", rows=rows, vocab=vocab, hidden=hidden, train=train, reduction=reduction, ignored=ignored, **more)


def _norm(rows, dim, dtype, train, affine=True, **more):
    return dict(kind="norm", rows=rows, dim=dim, dtype=dtype, train=train, affine=affine, **more)


def _rope(batch, seq, heads, kv_heads, head_dim, rotary_dim, interleaved, dtype, train, layout, start, scaling="none", factor=1.0, **more):
    return dict(kind="rope", batch=batch, seq=seq, heads=heads, kv_heads=kv_heads, head_dim=head_dim, rotary_dim=rotary_dim, interleaved=interleaved, dtype=dtype,
                train=train, layout=layout, start=start, scaling=scaling, factor=factor, **more)


def _clip(tensors, elements, dtype, limit, **more):
    return dict(kind="clip", tensors=tensors, elements=elements, dtype=dtype, limit=limit, **more)


def listed():
    return [
        # validation: the losses of the last, short window of a small model, one by one (latency)
        _ce(37, 10112, 448, False, "none", 0.0, name="ce_eval_short"),
        # one sequence of the flagship width with the presets' vocabulary
        _ce(4096, 10112, 576, True, "mean", 0.1, name="ce_train_10k"),
        # odd sizes throughout, each row's loss with a gradient of its own (weighted tokens)
        _ce(2049, 30011, 711, True, "none", 0.1, name="ce_train_odd"),
        # the largest tokenizer under the widest preset, two sequences
        _ce(8192, 50048, 1024, True, "mean", 0.02, name="ce_train_50k"),
        # a short prompt through a norm (latency)
        _norm(64, 448, "bf16", False, name="norm_infer_short"),
        # four sequences at the widest preset's width
        _norm(16384, 1024, "bf16", True, name="norm_train"),
        # fp32 residual stream of an odd width
        _norm(5001, 2305, "fp32", True, name="norm_train_odd"),
        # one token for each of sixteen sequences, far into long contexts (latency)
        _rope(16, 1, 22, 2, 64, 16, False, "bf16", False, "packed", 1_000_000, "yarn", 32.0, name="rope_decode_far"),
        # the flagship's heads, a quarter of each rotated, queries and keys as views of one packed projection
        _rope(4, 4096, 22, 2, 64, 16, False, "bf16", True, "packed", 0, name="rope_train"),
        # one long document, neighbouring pairs, whole heads, head-major tensors
        _rope(1, 65537, 8, 2, 128, 128, True, "bf16", True, "heads", 0, "ntk", 8.0, name="rope_train_long"),
        # the vectors and small matrices of an adapter (latency)
        _clip(24, 30_000, "fp32", 1.0, name="clip_small"),
        # a whole model's gradients, matrices in bf16 and the rest in fp32
        _clip(300, 200_000_000, "mixed", 1.0, name="clip_large"),
    ]


def draw(rng):
    log_int = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    kind = rng.choice(["ce", "ce", "norm", "norm", "rope", "rope", "clip"])
    train = rng.random() < 0.7
    if kind == "ce":
        while True:
            rows, vocab, hidden = log_int(1, 16384), log_int(1000, 50048), log_int(64, 2048)
            if rng.random() < 0.5:
                hidden = (hidden + 63) // 64 * 64
            if rows * vocab * hidden <= MOST_PRODUCT and rows * vocab <= 8192 * 50048:
                return _ce(rows, vocab, hidden, train, rng.choice(["mean", "sum", "none"]), rng.choice([0.0, 0.05, 0.5]))
    if kind == "norm":
        while True:
            rows, dim = log_int(1, 65536), log_int(32, 16384)
            if rng.random() < 0.5:
                dim = (dim + 31) // 32 * 32
            if rows * dim <= MOST_NORM:
                return _norm(rows, dim, rng.choice(["bf16", "bf16", "fp32", "fp16"]), train, rng.random() < 0.8)
    if kind == "rope":
        while True:
            batch, seq, kv_heads, head_dim = rng.choice([1, 2, 3, 8, 32]), log_int(1, 65536), rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 128, 256])
            heads, rotary_dim = kv_heads * rng.choice([1, 3, 4, 7]), rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4])
            if batch * seq * (heads + kv_heads) * head_dim <= MOST_ROPE:
                return _rope(batch, seq, heads, kv_heads, head_dim, rotary_dim, rng.random() < 0.5, rng.choice(["bf16", "bf16", "fp16", "fp32"]), train,
                             rng.choice(["packed", "heads", "plain"]), rng.choice([0, 0, log_int(1, 2_000_000)]), *rng.choice([("none", 1.0), ("linear", 4.0), ("ntk", 8.0), ("yarn", 16.0)]))
    elements = log_int(5_000, MOST_CLIP)
    return _clip(min(log_int(1, 600), elements // 8), elements, rng.choice(["fp32", "bf16", "mixed"]), rng.choice([1.0, 1.0, 1e9]))


# ---- inputs -----------------------------------------------------------------------------------------------------------------
def _frequencies(c):
    """Angles per position of the rotated pairs, in 64 bits, and the factor on the result."""
    r, theta, s = c["rotary_dim"], 1e7, c["factor"]
    if c["scaling"] == "ntk" and r > 2:
        theta *= s ** (r / (r - 2))
    f = theta ** -(torch.arange(0, r, 2, dtype=torch.float64) / r)
    if c["scaling"] == "linear":
        f = f / s
    if c["scaling"] == "yarn":                                     # pairs that turn often in the trained length stay, slow ones are stretched
        turns = 4096 * f / (2 * math.pi)
        keep = ((turns.log() - math.log(1.0)) / (math.log(32.0) - math.log(1.0))).clamp(0, 1)
        f = f * keep + f / s * (1 - keep)
        return f, 0.1 * math.log(s) + 1
    return f, 1.0


def _sizes(c):
    """Sizes of a list of gradients: a few large ones hold most of the elements, as matrices do beside vectors."""
    r = random.Random(c["tensors"] * 1_000_003 + c["elements"])
    weight = [math.exp(r.gauss(0, 2)) for _ in range(c["tensors"])]
    return [max(1, int(c["elements"] * w / sum(weight))) for w in weight]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, device=DEVICE, generator=gen)
    s = dict(case=case)
    if case["kind"] == "ce":
        T, V, h = case["rows"], case["vocab"], case["hidden"]
        s["weight"] = normal(V, h).mul_(2.4 / math.sqrt(h)).to(torch.bfloat16)
        s["target"] = torch.randint(0, V, (T,), device=DEVICE, generator=gen)
        row = s["weight"][s["target"]].float()                     # hidden states that know something of their target
        s["hidden"] = (normal(T, h) + 6.0 * row / row.square().sum(-1, keepdim=True)).to(torch.bfloat16)
        s["target"] = s["target"].masked_fill(torch.rand(T, device=DEVICE, generator=gen) < case["ignored"], -100)
        s["upstream"] = torch.rand(T, device=DEVICE, generator=gen) if case["reduction"] == "none" else torch.ones((), device=DEVICE)
        if case["train"]:
            s["hidden"].requires_grad_()
            s["weight"].requires_grad_()
    elif case["kind"] == "norm":
        dtype = TYPES[case["dtype"]]
        s["x"] = (normal(case["rows"], case["dim"]) * 2 + 0.5).to(dtype)
        s["dy"] = normal(case["rows"], case["dim"]).to(dtype)
        s["weight"] = 1 + 0.2 * normal(case["dim"]) if case["affine"] else None
        s["bias"] = 0.2 * normal(case["dim"]) if case["affine"] else None
        if case["train"]:
            for name in ("x", "weight", "bias"):
                if s[name] is not None:
                    s[name].requires_grad_()
    elif case["kind"] == "rope":
        B, S, H, K, D, dtype = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["head_dim"], TYPES[case["dtype"]]
        if case["layout"] == "packed":                             # queries, keys and values of a token side by side
            packed = normal(B, S, H + 2 * K, D).to(dtype)
            s["q"], s["k"] = packed[:, :, :H], packed[:, :, H:H + K]
        elif case["layout"] == "heads":
            s["q"], s["k"] = normal(B, H, S, D).to(dtype).transpose(1, 2), normal(B, K, S, D).to(dtype).transpose(1, 2)
        else:
            s["q"], s["k"] = normal(B, S, H, D).to(dtype), normal(B, S, K, D).to(dtype)
        first = torch.randint(0, case["start"] + 1, (B, 1), device=DEVICE, generator=gen)      # each sequence has come to a place of its own
        s["positions"] = first + torch.arange(S, device=DEVICE)
        f, s["magnitude"] = _frequencies(case)
        s["frequencies"] = f.to(DEVICE)
        s["dq"], s["dk"] = normal(B, S, H, D).to(dtype), normal(B, S, K, D).to(dtype)
        if case["train"]:
            s["q"], s["k"] = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
    else:
        sizes, kinds = _sizes(case), ["fp32", "bf16"]
        large = sorted(sizes)[len(sizes) // 2]
        s["grads"], s["out"], s["flat"] = [], [], {}
        kind = [case["dtype"] if case["dtype"] != "mixed" else "bf16" if n > large else "fp32" for n in sizes]
        for name in kinds:
            mine = [(n + 7) // 8 * 8 for n, t in zip(sizes, kind) if t == name]
            if mine:
                s["flat"][name] = torch.zeros(sum(mine), device=DEVICE, dtype=TYPES[name])
        at = dict.fromkeys(kinds, 0)
        scale = (10 ** (-3 * torch.rand(len(sizes), device=DEVICE, generator=gen))).tolist()
        for n, t, a in zip(sizes, kind, scale):
            g = torch.empty(n, device=DEVICE, dtype=TYPES[t]).normal_(0, a, generator=gen)
            s["grads"].append(g.view(-1, 16) if n % 16 == 0 else g)
            s["out"].append(s["flat"][t][at[t]:at[t] + n].view_as(s["grads"][-1]))
            at[t] += (n + 7) // 8 * 8
    return s


# ---- the operators in elementary operations -------------------------------------------------------------------------------------
def _plain_ce(s, c):
    h, w, target = s["hidden"].float(), s["weight"].float(), s["target"]
    valid = target != -100
    at = target.clamp_min(0)[:, None]
    logits = h @ w.t()
    top = logits.amax(-1, keepdim=True)
    e = (logits - top).exp()
    total = e.sum(-1, keepdim=True)
    losses = (top + total.log() - logits.gather(1, at))[:, 0] * valid
    count = valid.sum().clamp_min(1)
    loss = losses if c["reduction"] == "none" else losses.sum(dtype=torch.float64).float() if c["reduction"] == "sum" else (losses.sum(dtype=torch.float64) / count).float()
    if not c["train"]:
        return loss
    g = s["upstream"] * valid / (count if c["reduction"] == "mean" else 1)
    dz = (e / total).scatter_add(1, at, torch.full_like(top, -1.0)) * g[:, None]
    return loss, (dz @ w).to(s["hidden"].dtype), (dz.t() @ h).to(s["weight"].dtype)


def _plain_norm(s, c):
    x, dtype = s["x"].float(), s["x"].dtype
    centred = x - x.mean(-1, keepdim=True)
    rstd = (centred.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    hat = centred * rstd
    y = (hat * s["weight"] + s["bias"] if c["affine"] else hat).to(dtype)
    if not c["train"]:
        return y
    dy = s["dy"].float()
    g = dy * s["weight"] if c["affine"] else dy
    dx = (rstd * (g - g.mean(-1, keepdim=True) - hat * (g * hat).mean(-1, keepdim=True))).to(dtype)
    return (y, dx, (dy * hat).sum(0), dy.sum(0)) if c["affine"] else (y, dx)


def _turn(x, cos, sin, r, interleaved):
    xf = x.float()
    a, b = (xf[..., 0:r:2], xf[..., 1:r:2]) if interleaved else (xf[..., :r // 2], xf[..., r // 2:r])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([turned, xf[..., r:]], -1).to(x.dtype)


def _plain_rope(s, c):
    angle = s["positions"].double()[..., None, None] * s["frequencies"]
    cos, sin = (angle.cos() * s["magnitude"]).float(), (angle.sin() * s["magnitude"]).float()
    r, pairs = c["rotary_dim"], c["interleaved"]
    q, k = _turn(s["q"], cos, sin, r, pairs), _turn(s["k"], cos, sin, r, pairs)
    return (q, k, _turn(s["dq"], cos, -sin, r, pairs), _turn(s["dk"], cos, -sin, r, pairs)) if c["train"] else (q, k)


def _plain_clip(s, c):
    norm = torch.stack([g.double().square().sum() for g in s["grads"]]).sum().sqrt().float()
    factor = (c["limit"] / (norm + 1e-6)).clamp(max=1.0)
    [o.copy_(g.float() * factor) for o, g in zip(s["out"], s["grads"])]
    return norm, s["flat"]


# ---- the framework's operators ----------------------------------------------------------------------------------------------------
def _own_ce(s, c):
    from q38.losses import vocabulary_cross_entropy
    loss = vocabulary_cross_entropy(s["weight"], s["hidden"], s["target"], reduction=c["reduction"])
    if not c["train"]:
        return loss
    return loss.detach(), *torch.autograd.grad(loss, [s["hidden"], s["weight"]], s["upstream"])


def _own_norm(s, c):
    from q38 import ops
    y = ops.layer_norm(s["x"], s["weight"], s["bias"], eps=1e-5)
    if not c["train"]:
        return y
    return y.detach(), *torch.autograd.grad(y, [t for t in (s["x"], s["weight"], s["bias"]) if t is not None], s["dy"])


def _own_rope(s, c):
    from q38 import ops
    q, k = ops.rotary(s["q"], s["k"], s["positions"], s["frequencies"], magnitude=s["magnitude"], interleaved=c["interleaved"])
    if not c["train"]:
        return q, k
    return q.detach(), k.detach(), *torch.autograd.grad([q, k], [s["q"], s["k"]], [s["dq"], s["dk"]])


def _own_clip(s, c):
    from q38 import ops
    return ops.clip_grad_norm(s["grads"], c["limit"], out=s["out"]), s["flat"]


def run(state):
    c = state["case"]
    if own:
        return {"ce": _own_ce, "norm": _own_norm, "rope": _own_rope, "clip": _own_clip}[c["kind"]](state, c)
    with torch.no_grad():
        return {"ce": _plain_ce, "norm": _plain_norm, "rope": _plain_rope, "clip": _plain_clip}[c["kind"]](state, c)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------
def work(case):
    c, size = case, {"bf16": 2, "fp16": 2, "fp32": 4}
    if c["kind"] == "ce":
        T, V, h = c["rows"], c["vocab"], c["hidden"]
        operands = 2 * h * (T + V)
        return {"bytes": operands * (2 if c["train"] else 1) + 12 * T, "flops": 2.0 * T * V * h * (3 if c["train"] else 1)}
    if c["kind"] == "norm":
        n = c["rows"] * c["dim"]
        return {"bytes": n * size[c["dtype"]] * (4 if c["train"] else 2) + 8 * c["dim"] * c["affine"] * (2 if c["train"] else 1), "flops": n * (20.0 if c["train"] else 8.0)}
    if c["kind"] == "rope":
        n = c["batch"] * c["seq"] * (c["heads"] + c["kv_heads"]) * c["head_dim"]
        return {"bytes": n * size[c["dtype"]] * (4 if c["train"] else 2) + 8 * c["batch"] * c["seq"], "flops": 3.0 * n * c["rotary_dim"] / c["head_dim"] * (2 if c["train"] else 1)}
    sizes = _sizes(c)
    large = sorted(sizes)[len(sizes) // 2]
    each = lambda n: size[c["dtype"]] if c["dtype"] != "mixed" else 2 if n > large else 4
    return {"bytes": 2.0 * sum(n * each(n) for n in sizes), "flops": 3.0 * sum(sizes)}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------------
def exact(case, seed):
    s, c = prepare(case, seed), case
    with torch.no_grad():
        if c["kind"] == "ce":
            h, w = s["hidden"].double(), s["weight"].double()
            losses, dh, dw = [], [], torch.zeros_like(w)
            valid = s["target"] >= 0
            share = s["upstream"].double() * valid / (max(1, int(valid.sum())) if c["reduction"] == "mean" else 1)
            for o in range(0, h.shape[0], 2048):
                p = slice(o, o + 2048)
                logp = torch.log_softmax(h[p] @ w.T, -1)
                pick = torch.nn.functional.one_hot(s["target"][p].clamp(min=0), w.shape[0])
                losses.append(-(logp.gather(1, s["target"][p].clamp(min=0)[:, None])[:, 0]) * valid[p])
                if c["train"]:
                    dz = logp.exp_().sub_(pick).mul_(share[p, None])
                    dh.append(dz @ w)
                    dw += dz.T @ h[p]
            losses = torch.cat(losses)
            loss = losses if c["reduction"] == "none" else losses.sum() if c["reduction"] == "sum" else losses.sum() / max(1, int(valid.sum()))
            return (loss, torch.cat(dh), dw) if c["train"] else loss
        if c["kind"] == "norm":
            x = s["x"].double()
            var, mean = torch.var_mean(x, -1, unbiased=False, keepdim=True)
            hat = (x - mean) / torch.sqrt(var + 1e-5)
            w = s["weight"].double() if c["affine"] else torch.ones((), device=x.device, dtype=torch.float64)
            y = hat * w + (s["bias"].double() if c["affine"] else 0)
            if not c["train"]:
                return y
            dy = s["dy"].double()
            dhat = dy * w
            n = x.shape[-1]
            dx = (n * dhat - dhat.sum(-1, keepdim=True) - hat * (dhat * hat).sum(-1, keepdim=True)) / (n * torch.sqrt(var + 1e-5))
            return (y, dx, torch.einsum("td,td->d", dy, hat), dy.sum(0)) if c["affine"] else (y, dx)
        if c["kind"] == "rope":
            r = c["rotary_dim"]
            angle = s["positions"].double()[:, :, None, None] * s["frequencies"]

            def turned(x, sign):
                out = x.double().clone()
                first, second = (slice(0, r, 2), slice(1, r, 2)) if c["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
                z = torch.complex(out[..., first], out[..., second]) * torch.polar(torch.full_like(angle, s["magnitude"]), sign * angle)
                out[..., first], out[..., second] = z.real, z.imag
                return out

            both = turned(s["q"], 1), turned(s["k"], 1)
            return (*both, turned(s["dq"], -1), turned(s["dk"], -1)) if c["train"] else both
        flat = {name: torch.zeros(t.shape, device=t.device, dtype=torch.float64) for name, t in s["flat"].items()}
        norm = math.sqrt(sum(torch.linalg.vector_norm(g, dtype=torch.float64).item() ** 2 for g in s["grads"]))
        for o, g in zip(s["out"], s["grads"]):
            name = next(n for n, t in s["flat"].items() if t.dtype == g.dtype)
            flat[name][o.storage_offset():o.storage_offset() + g.numel()] = g.double().flatten() * min(1.0, c["limit"] / (norm + 1e-6))
        return torch.tensor(norm, dtype=torch.float64), flat

"""The operators for deep residual graph networks and large sets of answers, as cases that can be timed and checked.

    norms   y = x + scale * sigmoid(gate) * N_post(branch), h = N_pre(y): the end of one block and the norm before the next,
            forward, or forward and backward; with `checkpoint` the backward pass sees its inputs through 8-bit checkpoints
    keep8   an activation kept in 8 bits, and the weight gradient of a Linear layer from it
    scores  log probabilities of given tokens with entropy and the top alternatives, forward, or forward and backward

`run` computes them with elementary torch operations in 32 bits, or, with `own` true, through `cpp_extension.ops`.  `exact` is
the definition in 64 bits."""
import os
import sys

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
_EPS = 1e-5
_BLOCK = 32              # features that share one step of an 8-bit checkpoint


def _ops():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "schemanet-pytorch_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from cpp_extension import ops
    return ops


# ----------------------------------------------------------------------------------------------------------------- cases
def _norms(graphs, n, width, dtype, norm="layer", gate=True, scale=True, post=True, pre=True, train=False, checkpoint=False, name=None):
    case = dict(op="norms", graphs=graphs, n=n, width=width, dtype=dtype, norm=norm, gate=gate, scale=scale, post=post, pre=pre,
                train=train, checkpoint=checkpoint)
    return dict(case, name=name) if name else case


def _keep8(rows, inputs, outputs, dtype, restore, name=None):
    case = dict(op="keep8", rows=rows, inputs=inputs, outputs=outputs, dtype=dtype, restore=restore)
    return dict(case, name=name) if name else case


def _scores(rows, tokens, dtype, top, train, masked, name=None):
    case = dict(op="scores", rows=rows, tokens=tokens, dtype=dtype, top=top, train=train, masked=masked)
    return dict(case, name=name) if name else case


def listed():
    return [
        # four sequences, one new token each, between two blocks of width 1024: latency
        _norms(0, 4, 1024, "bf16", name="norms_tokens4_1024_bf16"),
        # a batch of 64 instance graphs of up to 196 vertices, width 256, in training
        _norms(64, 196, 256, "fp32", train=True, name="norms_graphs64x196_256_fp32_train"),
        # an odd width and an odd number of rows, RMS norms, no gate
        _norms(0, 1537, 1111, "fp16", norm="rms", gate=False, train=True, name="norms_rows1537_1111_fp16_train"),
        # a long training batch of a wide model
        _norms(0, 32768, 4096, "bf16", norm="rms", train=True, name="norms_rows32768_4096_bf16_train"),
        # the 101 class graphs of 1024 vertices, width 256, in training with 8-bit checkpoints
        _norms(101, 1024, 256, "fp32", train=True, checkpoint=True, name="norms_graphs101x1024_256_fp32_train8"),
        # the input of the instance graphs' Linear, kept, restored, and its weight gradient
        _keep8(12544, 256, 256, "fp32", True, name="keep8_rows12544_256x256_fp32"),
        # odd sizes: a ragged batch into 1000 classes
        _keep8(4999, 387, 1000, "bf16", True, name="keep8_rows4999_387x1000_bf16"),
        # a wide feed-forward layer over a long batch
        _keep8(32768, 2048, 8192, "bf16", False, name="keep8_rows32768_2048x8192_bf16"),
        # the answer for one image among 1000 classes: latency
        _scores(1, 1000, "fp32", 5, False, False, name="scores_rows1_1000_fp32"),
        # the class scores of a training batch
        _scores(256, 100, "fp32", 0, True, False, name="scores_rows256_100_fp32_train"),
        # sixteen next tokens out of a large vocabulary with padded entries
        _scores(16, 131072, "bf16", 20, False, True, name="scores_rows16_131072_bf16"),
        # token scores of a training batch, an odd vocabulary
        _scores(4096, 32769, "bf16", 0, True, True, name="scores_rows4096_32769_bf16_train"),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(["norms", "keep8", "scores"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "norms":
        train = rng.random() < 0.6
        width = _spread(rng, 8, 4096)
        if rng.random() < 0.4:
            width = max(16, width // 16 * 16)
        most = 32768 * 4096 // (2 if dtype == "fp32" else 1) // width
        rows = _spread(rng, 1, min(most, 65536))
        graphs = rng.choice([0, 0, 3, 17, 64]) if rows >= 64 else 0
        pre, post = rng.choice([(True, True), (True, True), (True, False), (False, True)])
        return _norms(graphs, rows // graphs if graphs else rows, width, dtype, rng.choice(["layer", "rms"]), rng.random() < 0.7,
                      rng.random() < 0.7, post, pre, train, train and rng.random() < 0.5)
    if op == "keep8":
        return _keep8(_spread(rng, 64, 32768), _spread(rng, 16, 2048), _spread(rng, 16, 4096), dtype, rng.random() < 0.5)
    if rng.random() < 0.5:
        tokens = _spread(rng, 2, 131072)
        return _scores(_spread(rng, 1, 64), tokens, dtype, min(tokens, rng.choice([1, 3, 5, 8, 20, 32])), False, rng.random() < 0.5)
    tokens = _spread(rng, 2, 32768)
    rows = _spread(rng, 1, 2048)
    return _scores(rows, tokens, dtype, 0, True, rng.random() < 0.5)


# ---------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t = _TYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=g, device="cuda") * std + mean

    s = dict(case=case)
    if case["op"] == "norms":
        lead = (case["graphs"], case["n"]) if case["graphs"] else (case["n"],)
        e = case["width"]
        columns = torch.exp(normal(e, std=0.5))                     # features of unequal size, as trained networks have them
        s["x"] = (normal(*lead, e, std=2.0) * columns + 0.3).to(t)
        s["branch"] = (normal(*lead, e) * columns - 0.1).to(t)
        s["gate"] = normal(*lead, e, std=1.5).to(t) if case["gate"] else None
        s["scale"] = normal(e, std=0.1, mean=0.5).to(t) if case["scale"] else None
        bias = case["norm"] == "layer"
        s["post"] = (normal(e, std=0.2, mean=1.0).to(t), normal(e, std=0.1).to(t) if bias else None) if case["post"] else None
        s["pre"] = (normal(e, std=0.2, mean=1.0).to(t), normal(e, std=0.1).to(t) if bias else None) if case["pre"] else None
        s["n_valid"] = None
        if case["graphs"]:
            s["n_valid"] = torch.randint(case["n"] // 2, case["n"] + 1, (case["graphs"],), generator=g, device="cuda").to(torch.int32)
        if case["train"]:
            s["dy"] = normal(*lead, e, std=1e-2).to(t)
            s["dh"] = normal(*lead, e, std=1e-2).to(t) if case["pre"] else None
            if own:
                for k in ("x", "branch", "gate", "scale"):
                    if s[k] is not None:
                        s[k].requires_grad_(True)
                for k in ("post", "pre"):
                    for p in s[k] or ():
                        if p is not None:
                            p.requires_grad_(True)
    elif case["op"] == "keep8":
        r, i, o = case["rows"], case["inputs"], case["outputs"]
        x = normal(r, i) * torch.exp(normal(i, std=0.5))
        s["x"] = (x * torch.sigmoid(1.7 * x)).to(t)                 # what a smooth activation hands to the next Linear
        s["dy"] = normal(r, o, std=1e-2).to(t)
    else:
        r, v = case["rows"], case["tokens"]
        x = normal(r, v, std=2.0) + 3.0 * normal(1, v)
        if case["masked"]:
            x[:, v - v // 50:] = float("-inf")                      # entries that pad the vocabulary
        s["logits"] = x.to(t)
        s["target"] = torch.randint(0, max(1, v - v // 50), (r,), generator=g, device="cuda")
        if case["train"]:
            s["target"][torch.rand(r, generator=g, device="cuda") < 0.1] = -100      # padded positions
            s["d_log_probs"] = normal(r, std=1.0 / r, mean=-1.0 / r)
            s["d_entropy"] = normal(r, std=0.1 / r)
            if own:
                s["logits"].requires_grad_(True)
    return s


# ----------------------------------------------------------------------------------------------------------- plain forms
def _checkpoint(x):
    """x in 8-bit integers times one power of two for every 32 features: the values that are kept, in x's working type."""
    e = x.shape[-1]
    pad = (-e) % _BLOCK
    v = torch.nn.functional.pad(x, (0, pad)).reshape(*x.shape[:-1], (e + pad) // _BLOCK, _BLOCK)
    top = v.abs().amax(-1, keepdim=True)
    m, p = torch.frexp(top)                                          # top = m 2^p, 0.5 <= m < 1
    k = (p - 7 + (m >= 127.5 / 128).to(p.dtype)).clamp(min=-125, max=121)
    step = torch.ldexp(torch.ones_like(top), k)
    q = torch.round(torch.ldexp(v, -k)).clamp(-127, 127)
    kept = torch.where(top > 0, q * step, torch.zeros_like(v))
    return kept.reshape(*x.shape[:-1], e + pad)[..., :e]


def _statistics(v, norm):
    mean = v.mean(-1, keepdim=True) if norm == "layer" else torch.zeros_like(v[..., :1])
    return mean, torch.rsqrt(((v - mean) ** 2).mean(-1, keepdim=True) + _EPS)


def _norm_gradient(d, unit, rstd, norm):
    """gradient of unit = (v - mean) rstd with respect to v"""
    out = d - unit * (d * unit).mean(-1, keepdim=True)
    if norm == "layer":
        out = out - d.mean(-1, keepdim=True)
    return out * rstd


def _plain_norms(s):
    case = s["case"]
    norm, t = case["norm"], _TYPES[case["dtype"]]
    f32 = lambda v: None if v is None else v.float()        # noqa: E731
    x, f, z, scale = f32(s["x"]), f32(s["branch"]), f32(s["gate"]), f32(s["scale"])
    lead = x.shape[:-1]
    valid = None
    if s["n_valid"] is not None:
        valid = (torch.arange(lead[1], device=x.device)[None, :] < s["n_valid"][:, None])[..., None]

    def forward(x, f, z, first=None, second=None):
        sig = None if z is None else 1.0 / (1.0 + torch.exp(-z))
        unit1 = p = f
        if case["post"]:
            first = _statistics(f, norm) if first is None else first
            unit1 = (f - first[0]) * first[1]
            p = unit1 * s["post"][0].float()
            if s["post"][1] is not None:
                p = p + s["post"][1].float()
        a = p if sig is None else p * sig
        y = x + (a if scale is None else a * scale)
        unit2 = h = None
        if case["pre"]:
            second = _statistics(y, norm) if second is None else second
            unit2 = (y - second[0]) * second[1]
            h = unit2 * s["pre"][0].float()
            if s["pre"][1] is not None:
                h = h + s["pre"][1].float()
        return sig, first, unit1, p, y, second, unit2, h

    sig, first, unit1, p, y, second, unit2, h = forward(x, f, z)
    keep = (lambda v: v) if valid is None else (lambda v: torch.where(valid, v, torch.zeros_like(v)))
    out = [keep(y).to(t)] + ([keep(h).to(t)] if case["pre"] else [])
    if not case["train"]:
        return out
    if case["checkpoint"]:
        sig, _, unit1, p, _, _, unit2, _ = forward(_checkpoint(x), _checkpoint(f), None if z is None else _checkpoint(z), first, second)
    dy = keep(s["dy"].float())
    rows = tuple(range(x.dim() - 1))
    weights = []
    if case["pre"]:
        dh = keep(s["dh"].float())
        weights.append((dh * unit2).sum(rows).to(t))
        if s["pre"][1] is not None:
            weights.append(dh.sum(rows).to(t))
        dy = dy + _norm_gradient(dh * s["pre"][0].float(), unit2, second[1], norm)
    dp = dy if scale is None else dy * scale
    grads = [keep(dy).to(t)]
    dz = None
    if sig is not None:
        dz = keep(dp * p * sig * (1 - sig)).to(t)
        dp = dp * sig
    dscale = None
    if scale is not None:
        dscale = (dy * p if sig is None else dy * p * sig)
        dscale = keep(dscale).sum(rows).to(t)
    dp = keep(dp)
    df = dp
    if case["post"]:
        weights.append(keep(dp * unit1).sum(rows).to(t))
        if s["post"][1] is not None:
            weights.append(dp.sum(rows).to(t))
        df = _norm_gradient(dp * s["post"][0].float(), unit1, first[1], norm)
    grads.append(keep(df).to(t))
    return out + grads + [v for v in (dz, dscale) if v is not None] + weights


def _plain_keep8(s):
    t = _TYPES[s["case"]["dtype"]]
    kept = _checkpoint(s["x"].float())
    dy = s["dy"].float()
    out = [torch.matmul(dy.t(), kept).to(t), dy.sum(0).to(t)]
    return out + ([kept.to(t)] if s["case"]["restore"] else [])


def _plain_scores(s):
    case = s["case"]
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    shifted = x - torch.where(torch.isinf(top), torch.zeros_like(top), top)
    weight = torch.exp(shifted)
    total = weight.sum(-1, keepdim=True)
    log_p = shifted - torch.log(total)
    p = weight / total
    finite = torch.where(p > 0, log_p, torch.zeros_like(log_p))
    entropy = -(p * finite).sum(-1)
    used = s["target"] != -100
    at = s["target"].clamp(min=0)[:, None]
    log_probs = torch.where(used, log_p.gather(-1, at)[:, 0], torch.zeros_like(entropy))
    out = [log_probs, entropy]
    if case["top"]:
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :case["top"]].clone()
        out += [log_p.gather(-1, order), order]
    if case["train"]:
        d = torch.where(used, s["d_log_probs"], torch.zeros_like(entropy))[:, None]
        grad = -p * (d + s["d_entropy"][:, None] * (finite + entropy[:, None]))
        out.append(grad.scatter_add(-1, at, d).to(s["logits"].dtype))
    return out


# ------------------------------------------------------------------------------------------------------- the framework's
def _own_norms(s):
    ops, case = _ops(), s["case"]
    y, h = ops.gated_residual_norms(s["x"], s["branch"], gate=s["gate"], scale=s["scale"], post=s["post"], pre=s["pre"], norm=case["norm"],
                                    eps=_EPS, n_valid=s["n_valid"], checkpoint8=case["checkpoint"])
    out = [y] + ([h] if case["pre"] else [])
    if not case["train"]:
        return out
    leaves = [s["x"], s["branch"], s["gate"], s["scale"]]
    for k in ("pre", "post"):
        leaves += list(s[k] or ())
    leaves = [v for v in leaves if v is not None]
    grads = torch.autograd.grad(out, leaves, [s["dy"]] + ([s["dh"]] if case["pre"] else []))
    return [v.detach() for v in out] + list(grads)


def _own_keep8(s):
    ops = _ops()
    kept = ops.checkpoint8(s["x"])
    out = list(ops.checkpoint8_weight_grad(s["dy"], kept))
    return out + ([kept.restore()] if s["case"]["restore"] else [])


def _own_scores(s):
    case = s["case"]
    got = _ops().label_log_probs(s["logits"], s["target"], topk=case["top"])
    out = [got.log_probs, got.entropy]
    if case["top"]:
        out += [got.top_log_probs, got.top_ids]
    if case["train"]:
        grad, = torch.autograd.grad((got.log_probs, got.entropy), s["logits"], (s["d_log_probs"], s["d_entropy"]))
        out = [v.detach() for v in out] + [grad]
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norms": _own_norms, "keep8": _own_keep8, "scores": _own_scores}[op](state)
    with torch.no_grad():
        return {"norms": _plain_norms, "keep8": _plain_keep8, "scores": _plain_scores}[op](state)


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    b = _SIZE[case["dtype"]]
    if case["op"] == "norms":
        rows = max(1, case["graphs"]) * case["n"]
        if case["graphs"]:
            rows = rows * 3 // 4                     # rows behind a graph's last vertex are written (zeros), not read
        cells = rows * case["width"]
        reads, writes = 2 + case["gate"], 1 + case["pre"]
        flops = 12 + 8 * case["post"] + 8 * case["pre"]
        if case["train"]:
            reads, writes, flops = reads + 1 + case["pre"], writes + 2 + case["gate"], 3 * flops
        pad = (max(1, case["graphs"]) * case["n"] - rows) * case["width"]
        return {"bytes": b * (cells * (reads + writes) + pad * writes), "flops": flops * cells}
    if case["op"] == "keep8":
        r, i, o = case["rows"], case["inputs"], case["outputs"]
        return {"bytes": b * (r * i * (1 + case["restore"]) + r * o + i * o + o), "flops": 2 * r * i * o + r * o + 4 * r * i}
    cells = case["rows"] * case["tokens"]
    return {"bytes": b * cells * (1 + case["train"]) + case["rows"] * (16 + 12 * case["top"]), "flops": (6 + 6 * case["train"]) * cells}


# ----------------------------------------------------------------------------------------------------------------- exact
def _kept64(x):
    blocks = []
    for start in range(0, x.shape[-1], _BLOCK):
        v = x[..., start:start + _BLOCK]
        top = v.abs().amax(-1, keepdim=True)
        # the smallest power of two with top < 127.5 step: start one below log2 and step up while it is too small
        step = torch.exp2(torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top)))) - 7)
        for _ in range(3):
            step = torch.where(top >= 127.5 * step, 2 * step, step)
        step = step.clamp(min=2.0 ** -125, max=2.0 ** 121)
        blocks.append((v / step).round().clamp(-127, 127) * step)
    return torch.cat(blocks, -1)


def _exact_norms(case, s):
    norm, checkpoint = case["norm"], case["checkpoint"]
    up = lambda v: None if v is None else v.detach().double()      # noqa: E731
    x, f, z, scale = up(s["x"]), up(s["branch"]), up(s["gate"]), up(s["scale"])
    post, pre = [tuple(up(p) for p in s[k]) if s[k] is not None else None for k in ("post", "pre")]
    if s["n_valid"] is not None:                                    # the rows that count, as one list
        index = (torch.arange(case["n"], device=x.device)[None, :] < s["n_valid"][:, None]).reshape(-1).nonzero()[:, 0]
    else:
        index = torch.arange(x.shape[0], device=x.device)
    width = x.shape[-1]
    take = lambda v: None if v is None else v.reshape(-1, width)[index]       # noqa: E731

    def back(v, like):
        full = torch.zeros(like.numel() // width, width, dtype=v.dtype, device=v.device)
        full[index] = v
        return full.reshape(like.shape)

    leaves = [take(x), take(f), take(z), scale] + [p for k in (pre, post) for p in (k or ())]
    leaves = [None if v is None else v.clone().requires_grad_(case["train"] and not checkpoint) for v in leaves]
    xr, fr, zr, sc = leaves[:4]
    rest = leaves[4:]
    pre = (rest.pop(0), rest.pop(0)) if pre is not None else None
    post = (rest.pop(0), rest.pop(0)) if post is not None else None

    def unit(v):
        c = v - v.mean(-1, keepdim=True) if norm == "layer" else v
        return c / torch.sqrt(c.square().mean(-1, keepdim=True) + _EPS)

    def affine(u, w):
        return u * w[0] if w[1] is None else u * w[0] + w[1]

    with torch.set_grad_enabled(case["train"] and not checkpoint):
        p = fr if post is None else affine(unit(fr), post)
        y = p if zr is None else p * torch.sigmoid(zr)
        y = xr + (y if sc is None else y * sc)
        h = None if pre is None else affine(unit(y), pre)
    out = [back(y.detach(), s["x"])] + ([back(h.detach(), s["x"])] if h is not None else [])
    if not case["train"]:
        return out
    dy, dh = take(up(s["dy"])), take(up(s["dh"]))
    full = [s["x"], s["branch"], s["gate"]]
    if not checkpoint:
        asked = [v for v in leaves if v is not None]
        grads = list(torch.autograd.grad([y] + ([h] if h is not None else []), asked, [dy] + ([dh] if h is not None else [])))
        per_row = sum(v is not None for v in full)
        return out + [back(v, s["x"]) for v in grads[:per_row]] + grads[per_row:]
    # the backward pass at the kept values, with the row statistics of the forward pass
    centre = (lambda v: v.mean(-1, keepdim=True)) if norm == "layer" else (lambda v: torch.zeros_like(v[..., :1]))
    spread = lambda v: torch.sqrt((v - centre(v)).square().mean(-1, keepdim=True) + _EPS)      # noqa: E731
    mean1, sd1, mean2, sd2 = centre(fr), spread(fr), centre(y), spread(y)
    xk, fk, zk = _kept64(xr), _kept64(fr), None if zr is None else _kept64(zr)
    gate = torch.ones_like(xk) if zk is None else torch.sigmoid(zk)
    one = torch.ones(width, dtype=xk.dtype, device=xk.device)
    by = one if sc is None else sc
    u1 = (fk - mean1) / sd1
    pk = fk if post is None else affine(u1, post)
    u2 = (xk + by * gate * pk - mean2) / sd2
    tail = []
    total = dy
    if pre is not None:
        tail.append((dh * u2).sum(0))
        if pre[1] is not None:
            tail.append(dh.sum(0))
        d = dh * pre[0]
        total = dy + (d - centre(d) - u2 * (d * u2).mean(-1, keepdim=True)) / sd2
    dpk = total * by * gate
    df = dpk
    if post is not None:
        tail.append((dpk * u1).sum(0))
        if post[1] is not None:
            tail.append(dpk.sum(0))
        d = dpk * post[0]
        df = (d - centre(d) - u1 * (d * u1).mean(-1, keepdim=True)) / sd1
    grads = [back(total, s["x"]), back(df, s["x"])]
    if zk is not None:
        grads.append(back(total * by * pk * gate * (1 - gate), s["x"]))
    if sc is not None:
        grads.append((total * gate * pk).sum(0))
    return out + grads + tail


def _exact_keep8(case, s):
    x, dy = s["x"].detach().double(), s["dy"].double()
    kept = _kept64(x)
    dw = torch.zeros(case["outputs"], case["inputs"], dtype=torch.float64, device=x.device)
    for start in range(0, case["rows"], 4096):
        dw += dy[start:start + 4096].t().contiguous() @ kept[start:start + 4096]
    return [dw, dy.sum(0)] + ([kept] if case["restore"] else [])


def _exact_scores(case, s):
    x = s["logits"].detach().double()
    log_p = x - torch.logsumexp(x, -1, keepdim=True)
    p = torch.exp(log_p)
    entropy = -torch.where(p > 0, p * log_p, torch.zeros_like(p)).sum(-1)
    used = s["target"] != -100
    safe = torch.where(used, s["target"], torch.zeros_like(s["target"]))
    rows = torch.arange(case["rows"], device=x.device)
    out = [torch.where(used, log_p[rows, safe], torch.zeros_like(entropy)), entropy]
    if case["top"]:
        taken = torch.zeros_like(x, dtype=torch.bool)
        place = torch.arange(case["tokens"], device=x.device).expand_as(x)
        ids = []
        for _ in range(case["top"]):                                 # the largest, the lowest index among equals
            best = torch.where(taken, torch.full_like(x, float("-inf")), x).amax(-1, keepdim=True)
            first = torch.where((x == best) & ~taken, place, case["tokens"]).amin(-1)
            ids.append(first)
            taken[rows, first] = True
        ids = torch.stack(ids, -1)
        out += [log_p.gather(-1, ids), ids]
    if case["train"]:
        d = torch.where(used, s["d_log_probs"].double(), torch.zeros_like(entropy))
        grad = -p * d[:, None]
        grad[rows, safe] += d
        surprise = torch.where(p > 0, log_p, torch.zeros_like(log_p)) + entropy[:, None]
        grad -= s["d_entropy"].double()[:, None] * p * surprise
        out.append(grad)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "keep8":
            return _exact_keep8(case, s)
        if case["op"] == "scores":
            return _exact_scores(case, s)
    return _exact_norms(case, s)

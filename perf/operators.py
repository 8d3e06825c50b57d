"""Measured cases of the attention-block training operators, with their plain forms.

Three operators, as a training or inference program of this package uses them:

  attention   softmax(scale * Q K^T + bias) V over the tokens of a feature map (or of a sequence of slices: a map of
              height 1), with a learned bias per head looked up by the bucket of the relative position; keys may be masked.
              "train" is the forward pass and the gradients of Q, K, V and the bias table, "infer" the forward pass alone.
  residual    y = x + scale * gate * norm_post(f),  z = norm_pre(y): the end of one residual branch fused with the norm in
              front of the next; "train" returns every gradient too.
  clip        the global norm of a list of gradients, and either the gradients scaled in place to a largest norm or an AdamW
              step that takes the clipped gradients.

`run` computes the plain form from elementary torch operations while `own` is false, and calls this package otherwise."""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_ADAM = {"lr": 1e-3, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 1e-4}


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def _attention(name, mode, dtype, batch, heads, dim, height, width, buckets, queries=0, keys=0, masked=False, packed=False):
    keys = keys or height * width
    case = dict(op="attention", mode=mode, dtype=dtype, batch=batch, heads=heads, dim=dim, height=height, width=width,
                buckets=buckets, queries=queries or keys, keys=keys, masked=masked, packed=packed)
    return dict(case, name=name) if name else case


def _residual(name, mode, dtype, images, tokens, channels, post, pre, gated):
    case = dict(op="residual", mode=mode, dtype=dtype, images=images, tokens=tokens, channels=channels, post=post, pre=pre,
                gated=gated)
    return dict(case, name=name) if name else case


def _clip(name, mode, dtype, model, elements, tensors):
    case = dict(op="clip", mode=mode, dtype=dtype, model=model, elements=elements, tensors=tensors)
    return dict(case, name=name) if name else case


def listed():
    return [
        # the classification head of the default model: 300x300 images leave a 10x10 map of 384 channels in 8 heads
        _attention("head_train_bf16", "train", "bf16", 128, 8, 48, 10, 10, 16, packed=True),
        # the same head at the reference's default batch in fp32
        _attention("head_train_fp32", "train", "fp32", 16, 8, 48, 10, 10, 16, packed=True),
        # attention over the 38x38 map of stride 8, images of different sizes padded to one (some keys masked)
        _attention("map38_train_bf16", "train", "bf16", 4, 8, 64, 38, 38, 16, masked=True),
        # the 75x75 map of stride 4: the longest sequence a decoder level has
        _attention("map75_train_bf16", "train", "bf16", 1, 4, 32, 75, 75, 32),
        # one new slice against a long series, for a batch of volumes
        _attention("slice_infer_bf16", "infer", "bf16", 8, 8, 64, 1, 16384, 32, queries=1),
        # one query over one short volume: nothing but latency
        _attention("slice_infer_fp32", "infer", "fp32", 1, 8, 48, 1, 155, 32, queries=1),
        # the head's residual with its squeeze-excite style gate, default batch
        _residual("head_residual_bf16", "train", "bf16", 128, 100, 384, "layer", "layer", True),
        # widest expanded activation of the trunk, one fp32 image at a time on the odd 19x19 map
        _residual("wide_residual_fp32", "train", "fp32", 1, 361, 2304, None, "rms", False),
        # a large batch of 38x38 maps at a width of a power of two
        _residual("large_residual_bf16", "train", "bf16", 32, 1444, 1024, "rms", "rms", False),
        # one token in inference
        _residual("token_residual_bf16", "infer", "bf16", 1, 1, 384, "rms", "layer", False),
        # every parameter of the default model, clipped in place (gradients are views of one exchange buffer)
        _clip("model_clip_fp32", "scale", "fp32", "trunk", 10_900_000, 430),
        # fine-tuning the attention head alone: clipped AdamW step
        _clip("head_adamw_fp32", "adamw", "fp32", "head", 810_240, 22),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("attention", "attention", "slices", "residual", "residual", "clip"))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    if kind == "attention":
        height, width = _log_int(rng, 1, 75), _log_int(rng, 2, 75)
        heads, dim = rng.choice((1, 3, 4, 8, 12)), rng.choice((8, 16, 24, 32, 48, 64, 96, 128))
        pairs, budget = (height * width) ** 2, 4.1e9        # pairs x width of a head, as in the largest listed case
        if heads * pairs * dim > budget:
            heads, dim = 4, 32
        most = max(1, min(128, int(min(1.3e8, budget / dim) / (heads * pairs)), int(6e6 / (heads * height * width * dim))))
        return _attention(None, rng.choice(("train", "train", "infer")), dtype, _log_int(rng, 1, most), heads, dim, height,
                          width, rng.choice((8, 16, 32)), masked=rng.random() < 0.5, packed=rng.random() < 0.5)
    if kind == "slices":
        width = _log_int(rng, 1, 16384)
        heads, dim = rng.choice((1, 4, 8, 12)), rng.choice((16, 32, 48, 64, 128))
        most = max(1, min(16, int(1.3e5 * 64 * 8 / (width * heads * dim))))
        keys = max(1, width - rng.randrange(0, 1 + width // 4))
        return _attention(None, "infer", dtype, _log_int(rng, 1, most), heads, dim, 1, width, rng.choice((16, 32, 64)),
                          queries=min(keys, rng.choice((1, 1, 1, 2, 5, 16))), keys=keys, masked=rng.random() < 0.5)
    if kind == "residual":
        channels = rng.choice((_log_int(rng, 8, 4096), 8 * _log_int(rng, 2, 512), rng.choice((24, 136, 384, 1024, 2304))))
        rows = _log_int(rng, 1, max(2, int(4.7e7 * (1 if dtype == "bf16" else 0.5) / channels)))
        images = rng.choice((1, _log_int(rng, 1, min(rows, 128))))
        return _residual(None, rng.choice(("train", "train", "infer")), dtype, images, max(1, rows // images), channels,
                         rng.choice((None, "rms", "layer")), rng.choice(("rms", "layer")), rng.random() < 0.5)
    if rng.random() < 0.4:
        return _clip(None, "adamw", "fp32", "head", _log_int(rng, 1000, 8_000_000), rng.randrange(1, 25))
    return _clip(None, "scale", dtype, "list", _log_int(rng, 100, 20_000_000), _log_int(rng, 1, 450))


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _bucket_index(height, width, buckets):
    """Bucket of every offset (dy, dx) between two positions of a map, flattened over (2 height - 1)(2 width - 1): half the
    buckets of an axis for each direction, half of those exact and the rest logarithmic up to a distance of 128."""
    def axis(n):
        if n == 1:
            return torch.zeros(1, dtype=torch.int64), 1
        d = torch.arange(-(n - 1), n, dtype=torch.float64)
        half, exact = buckets // 2, buckets // 4
        far = exact + ((d.abs().clamp(min=exact) / exact).log() / math.log(128 / exact) * (half - exact)).floor()
        b = torch.where(d.abs() < exact, d.abs(), far.clamp(max=half - 1))
        return (b + half * (d > 0)).to(torch.int64), 2 * half
    by, _ = axis(height)
    bx, nx = axis(width)
    return (by[:, None] * nx + bx[None, :]).reshape(-1)


def _sizes(case):
    """Element counts of the parameters: a few large matrices, many vectors, odd lengths among them."""
    n, total = case["tensors"], case["elements"]
    share = [1.0 / (1 + i % 29) ** 2 for i in range(n)]
    sizes = [max(1, int(total * s / sum(share))) for s in share]
    return sizes


def _split(flat, sizes):
    return list(torch.split(flat, sizes))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    if case["op"] == "attention":
        B, H, D, Lq, Lk = (case[k] for k in ("batch", "heads", "dim", "queries", "keys"))
        train = case["mode"] == "train"
        index = _bucket_index(case["height"], case["width"], case["buckets"])
        table = normal(int(index.max()) + 1, H, scale=0.5)
        mask = None
        if case["masked"]:
            length = torch.randint(Lk // 2, Lk + 1, (B, 1), generator=g, device="cuda")
            mask = torch.arange(Lk, device="cuda")[None, :] < length
            if B > 1:
                mask[B // 2] = False        # an image that was all padding
        s = dict(case=case, index=index.cuda(), table=table, mask=mask, q_start=Lk - Lq)
        if case["packed"] and Lq == Lk:
            s["qkv"] = normal(B, Lk, 3, H, D, dtype=dt).requires_grad_(train)
        else:
            s.update(q=normal(B, Lq, H, D, dtype=dt).requires_grad_(train), k=normal(B, Lk, H, D, dtype=dt).requires_grad_(train),
                     v=normal(B, Lk, H, D, dtype=dt).requires_grad_(train))
        if train:
            table.requires_grad_()
            s["dout"] = normal(B, Lq, H, D, dtype=dt)
        if own:
            from mia_amd.relpos import RelativePositionBuckets
            s["plan"] = RelativePositionBuckets.from_index(case["height"], case["width"], index, device="cuda")
        return s
    if case["op"] == "residual":
        N, T, C = case["images"], case["tokens"], case["channels"]
        train = case["mode"] == "train"
        s = dict(case=case, x=normal(N, T, C, dtype=dt), f=(normal(N, T, C) * 2 + 0.5).to(dt))
        s["scale"] = normal(C, scale=0.1) + 0.2
        if case["gated"]:
            s["gate"] = torch.sigmoid(normal(N, C))
        for which in ("post", "pre"):
            if case[which]:
                s[which + "_weight"] = 1 + normal(C, scale=0.1)
            if case[which] == "layer":
                s[which + "_bias"] = normal(C, scale=0.1)
        if train:
            for name in _residual_leaves(s):
                s[name].requires_grad_()
            s["dy"], s["dz"] = normal(N, T, C, dtype=dt), normal(N, T, C, dtype=dt)
        return s
    sizes = _sizes(case)
    total = sum(sizes)
    flat = normal(total, scale=0.05, dtype=dt)
    s = dict(case=case, flat=flat, grads=_split(flat, sizes), max_norm=1.0)
    if case["mode"] == "adamw":
        s["p_flat"] = normal(total, scale=0.05)
        s["params"] = _split(s["p_flat"], sizes)
        if own:
            from mia_amd.optim import AdamW
            s["leaves"] = [torch.nn.Parameter(p) for p in s["params"]]
            for p, grad in zip(s["leaves"], s["grads"]):
                p.grad = grad
            s["optimizer"] = AdamW(s["leaves"], max_grad_norm=s["max_norm"], **_ADAM)
        else:
            s["m"], s["v"] = [torch.zeros_like(p) for p in s["params"]], [torch.zeros_like(p) for p in s["params"]]
            s["step"] = 0
    return s


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if op == "attention":
        return _own_attention(state) if own else _plain_attention(state)
    if op == "residual":
        return _own_residual(state) if own else _plain_residual(state)
    return _own_clip(state) if own else _plain_clip(state)


def _own_attention(s):
    from mia_amd.relpos import relpos_attention, relpos_self_attention
    if s["case"]["mode"] == "infer":
        with torch.no_grad():
            if "qkv" in s:
                return {"out": relpos_self_attention(s["qkv"], s["table"], s["plan"], key_mask=s["mask"])}
            return {"out": relpos_attention(s["q"], s["k"], s["v"], s["table"], s["plan"], key_mask=s["mask"], q_start=s["q_start"])}
    if "qkv" in s:
        out = relpos_self_attention(s["qkv"], s["table"], s["plan"], key_mask=s["mask"])
        dqkv, dtable = torch.autograd.grad(out, (s["qkv"], s["table"]), s["dout"])
        return {"out": out.detach(), "dqkv": dqkv, "dtable": dtable}
    out = relpos_attention(s["q"], s["k"], s["v"], s["table"], s["plan"], key_mask=s["mask"], q_start=s["q_start"])
    dq, dk, dv, dtable = torch.autograd.grad(out, (s["q"], s["k"], s["v"], s["table"]), s["dout"])
    return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv, "dtable": dtable}


def _offsets(case, q_start, device):
    """Flat offset index [Lq, Lk] of every (query, key) pair."""
    H, W = case["height"], case["width"]
    i = torch.arange(case["queries"], device=device) + q_start
    j = torch.arange(case["keys"], device=device)
    dy = j[None, :] // W - i[:, None] // W + (H - 1)
    dx = j[None, :] % W - i[:, None] % W + (W - 1)
    return dy * (2 * W - 1) + dx


@torch.no_grad()
def _plain_attention(s):
    case = s["case"]
    q, k, v = s["qkv"].unbind(2) if "qkv" in s else (s["q"], s["k"], s["v"])
    dt = q.dtype
    q, k, v = (t.float().transpose(1, 2).contiguous() for t in (q, k, v))        # [B, heads, L, D]
    scale = 1.0 / math.sqrt(case["dim"])
    off = _offsets(case, s["q_start"], q.device)
    bias = s["table"].t()[:, s["index"]][:, off]                                 # [heads, Lq, Lk]
    p = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale).add_(bias)
    if s["mask"] is not None:
        p.masked_fill_(~s["mask"][:, None, None, :], -math.inf)
    m = p.amax(-1, keepdim=True)
    p.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total == 0, 1.0, total))
    out = torch.matmul(p, v).transpose(1, 2).to(dt).contiguous()
    if case["mode"] == "infer":
        return {"out": out}
    do = s["dout"].float().transpose(1, 2).contiguous()
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    ds = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds.sub_((ds * p).sum(-1, keepdim=True)).mul_(p)
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q) * scale
    # bias gradient: sum over the batch, then over the pairs of one offset, then over the offsets of one bucket
    heads, n_off = case["heads"], s["index"].numel()
    per_off = torch.zeros(heads, n_off, dtype=torch.float64, device=q.device)
    per_off.index_add_(1, off.reshape(-1), ds.sum(0, dtype=torch.float64).reshape(heads, -1))
    dtable = torch.zeros(s["table"].shape, dtype=torch.float64, device=q.device)
    dtable.index_add_(0, s["index"], per_off.t().contiguous())
    grads = [t.transpose(1, 2).to(dt) for t in (dq, dk, dv)]
    if "qkv" in s:
        return {"out": out, "dqkv": torch.stack(grads, 2), "dtable": dtable.float()}
    return {"out": out, "dq": grads[0].contiguous(), "dk": grads[1].contiguous(), "dv": grads[2].contiguous(),
            "dtable": dtable.float()}


def _residual_leaves(s):
    return [n for n in ("x", "f", "scale", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias") if n in s]


def _own_residual(s):
    from mia_amd.block_norm import gated_residual_norm
    kw = {n: s[n] for n in ("scale", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias") if n in s}
    kw.update(post=s["case"]["post"], pre=s["case"]["pre"], eps=1e-6)
    if s["case"]["mode"] == "infer":
        with torch.no_grad():
            y, z = gated_residual_norm(s["x"], s["f"], **kw)
        return {"y": y, "z": z}
    y, z = gated_residual_norm(s["x"], s["f"], **kw)
    names = _residual_leaves(s)
    grads = torch.autograd.grad((y, z), [s[n] for n in names], (s["dy"], s["dz"]))
    return dict(zip(["d" + n for n in names], grads), y=y.detach(), z=z.detach())


def _norm(t, kind):
    """-> (normalised t, 1 / deviation) over the last axis."""
    if kind == "layer":
        t = t - t.mean(-1, keepdim=True)
    r = (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    return t * r, r


def _norm_grad(dhat, hat, r, kind):
    g = dhat - hat * (dhat * hat).mean(-1, keepdim=True)
    return (g - dhat.mean(-1, keepdim=True) if kind == "layer" else g) * r


@torch.no_grad()
def _plain_residual(s):
    case = s["case"]
    post, pre, dt = case["post"], case["pre"], s["x"].dtype
    x, f = s["x"].float(), s["f"].float()
    u, fhat = f, None
    if post:
        fhat, fr = _norm(f, post)
        u = fhat * s["post_weight"] + s.get("post_bias", 0.0)
    a = s["scale"] * s["gate"][:, None, :] if "gate" in s else s["scale"]
    y = x + a * u
    yhat, yr = _norm(y, pre)
    z = yhat * s["pre_weight"] + s.get("pre_bias", 0.0)
    got = {"y": y.to(dt), "z": z.to(dt)}
    if case["mode"] == "infer":
        return got
    dz = s["dz"].float()
    dy = s["dy"].float() + _norm_grad(dz * s["pre_weight"], yhat, yr, pre)
    du = dy * a
    got["dx"] = dy.to(dt)
    got["df"] = (_norm_grad(du * s["post_weight"], fhat, fr, post) if post else du).to(dt)
    per_image = (dy * u).sum(1, dtype=torch.float64)
    got["dscale"] = (per_image * s["gate"] if "gate" in s else per_image).sum(0).float()
    if "gate" in s:
        got["dgate"] = (per_image * s["scale"]).float()
    if post:
        got["dpost_weight"] = (du * fhat).sum((0, 1), dtype=torch.float64).float()
    if post == "layer":
        got["dpost_bias"] = du.sum((0, 1), dtype=torch.float64).float()
    got["dpre_weight"] = (dz * yhat).sum((0, 1), dtype=torch.float64).float()
    if pre == "layer":
        got["dpre_bias"] = dz.sum((0, 1), dtype=torch.float64).float()
    return got


def _own_clip(s):
    if s["case"]["mode"] == "scale":
        from mia_amd.optim import clip_grads_
        return {"norm": clip_grads_(s["grads"], s["max_norm"]), "grads": s["flat"]}
    opt = s["optimizer"]
    opt.step()
    return {"norm": opt.grad_norm, "p": s["p_flat"], "m": [opt.state[p]["exp_avg"] for p in s["leaves"]],
            "v": [opt.state[p]["exp_avg_sq"] for p in s["leaves"]]}


@torch.no_grad()
def _plain_clip(s):
    norm = torch.stack([g.double().square().sum() for g in s["grads"]]).sum().sqrt()
    factor = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    if s["case"]["mode"] == "scale":
        [g.copy_(g.float() * factor) for g in s["grads"]]
        return {"norm": norm.float(), "grads": s["flat"]}
    s["step"] += 1
    b1, b2 = _ADAM["betas"]
    size, root = _ADAM["lr"] / (1 - b1 ** s["step"]), math.sqrt(1 - b2 ** s["step"])
    [_plain_adamw(p, g * factor, m, v, b1, b2, size, root) for p, g, m, v in zip(s["params"], s["grads"], s["m"], s["v"])]
    return {"norm": norm.float(), "p": s["p_flat"], "m": s["m"], "v": s["v"]}


def _plain_adamw(p, g, m, v, b1, b2, size, root):
    p.mul_(1 - _ADAM["lr"] * _ADAM["weight_decay"])
    m.add_((g - m) * (1 - b1))
    v.mul_(b2).add_(g * g * (1 - b2))
    p.sub_(size * m / (v.sqrt() / root + _ADAM["eps"]))


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    train = case["mode"] == "train"
    if case["op"] == "attention":
        B, H, D, Lq, Lk = (case[k] for k in ("batch", "heads", "dim", "queries", "keys"))
        q, kv = B * Lq * H * D * es, B * Lk * H * D * es
        pairs = B * H * Lq * Lk
        index = _bucket_index(case["height"], case["width"], case["buckets"])
        small = index.numel() * 4 + (int(index.max()) + 1) * H * 4 * (2 if train else 1) + (B * Lk if case["masked"] else 0)
        if not train:
            return {"bytes": 2 * q + 2 * kv + small, "flops": 4 * pairs * D}
        return {"bytes": 4 * q + 4 * kv + small, "flops": 14 * pairs * D}
    if case["op"] == "residual":
        rows, C = case["images"] * case["tokens"], case["channels"]
        n = rows * C
        small = 4 * C * (1 + (case["images"] if case["gated"] else 0) + sum({"layer": 2, "rms": 1}.get(case[w], 0) for w in ("post", "pre")))
        if not train:
            return {"bytes": 4 * n * es + small, "flops": 12 * n}
        return {"bytes": 8 * n * es + 2 * small, "flops": 45 * n}
    n = sum(_sizes(case))
    if case["mode"] == "scale":
        return {"bytes": 2 * n * es, "flops": 3 * n}
    return {"bytes": 28 * n, "flops": 16 * n}


# ------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ------------------------------------------------------------------------------------------------
@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "residual": _exact_residual, "clip": _exact_clip}[case["op"]](s)


def _exact_attention(s):
    """Head by head and image by image; the bias gradient by sorting the pairs' buckets."""
    case = s["case"]
    q, k, v = (t.detach().double() for t in (s["qkv"].unbind(2) if "qkv" in s else (s["q"], s["k"], s["v"])))
    B, H, W, Lq, Lk = case["batch"], case["heads"], case["width"], case["queries"], case["keys"]
    if B * H > 2048:
        return None
    pos_q, pos_k = s["q_start"] + torch.arange(Lq, device="cuda"), torch.arange(Lk, device="cuda")
    rel_y = torch.div(pos_k, W, rounding_mode="floor").unsqueeze(0) - torch.div(pos_q, W, rounding_mode="floor").unsqueeze(1)
    rel_x = torch.remainder(pos_k, W).unsqueeze(0) - torch.remainder(pos_q, W).unsqueeze(1)
    bucket = s["index"].reshape(2 * case["height"] - 1, 2 * W - 1)[rel_y + case["height"] - 1, rel_x + W - 1]
    table = s["table"].detach().double()
    train = case["mode"] == "train"
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    dtable = torch.zeros_like(table)
    if train:
        order = bucket.reshape(-1).argsort(stable=True)
        found, count = torch.unique_consecutive(bucket.reshape(-1)[order], return_counts=True)
        ends = count.cumsum(0)
    for h in range(H):
        ds_all = torch.zeros(Lq, Lk, dtype=torch.float64, device="cuda")
        for b in range(B):
            scores = q[b, :, h] @ k[b, :, h].T / math.sqrt(case["dim"]) + table[bucket, h]
            w = torch.softmax(scores, 1)
            if s["mask"] is not None:
                keep = s["mask"][b]
                if not bool(keep.any()):
                    continue
                w = torch.softmax(torch.where(keep[None, :], scores, torch.full_like(scores, -math.inf)), 1)
            out[b, :, h] = w @ v[b, :, h]
            if train:
                go = s["dout"][b, :, h].double()
                dw = go @ v[b, :, h].T
                ds = w * (dw - (go * out[b, :, h]).sum(1, keepdim=True))
                ds_all += ds
                dv[b, :, h] = w.T @ go
                dq[b, :, h] = ds @ k[b, :, h] / math.sqrt(case["dim"])
                dk[b, :, h] = ds.T @ q[b, :, h] / math.sqrt(case["dim"])
        if train:
            running = torch.cat((torch.zeros(1, dtype=torch.float64, device="cuda"), ds_all.reshape(-1)[order].cumsum(0)))
            dtable[found, h] = running[ends] - running[ends - count]
    if not train:
        return {"out": out}
    if "qkv" in s:
        return {"out": out, "dqkv": torch.stack((dq, dk, dv), 2), "dtable": dtable}
    return {"out": out, "dq": dq, "dk": dk, "dv": dv, "dtable": dtable}


def _exact_residual(s):
    """The forward formula written out in float64; the gradients are its derivatives as autograd forms them."""
    names = _residual_leaves(s)
    t = {n: s[n].detach().double().requires_grad_(_trains(s)) for n in names}

    def normed(a, kind, which):
        if kind is None:
            return a
        mean = a.mean(-1, keepdim=True) if kind == "layer" else 0.0
        var = ((a - mean) ** 2).mean(-1, keepdim=True)
        r = (a - mean) / torch.sqrt(var + 1e-6) * t[which + "_weight"]
        return r + t[which + "_bias"] if kind == "layer" else r

    with torch.enable_grad():
        branch = normed(t["f"], s["case"]["post"], "post") * t["scale"]
        if "gate" in t:
            branch = branch * t["gate"].unsqueeze(1)
        y = t["x"] + branch
        z = normed(y, s["case"]["pre"], "pre")
        if not _trains(s):
            return {"y": y, "z": z}
        grads = torch.autograd.grad((y, z), [t[n] for n in names], (s["dy"].double(), s["dz"].double()))
    return dict(zip(["d" + n for n in names], grads), y=y.detach(), z=z.detach())


def _trains(s):
    return s["case"]["mode"] == "train"


def _exact_clip(s):
    g = s["flat"].double()
    norm = torch.linalg.vector_norm(g)
    g = g * min(1.0, s["max_norm"] / (float(norm) + 1e-6))
    if s["case"]["mode"] == "scale":
        return {"norm": norm, "grads": g}
    b1, b2 = _ADAM["betas"]
    m, v = (1 - b1) * g, (1 - b2) * g ** 2
    p = s["p_flat"].double() * (1 - _ADAM["lr"] * _ADAM["weight_decay"])
    p = p - _ADAM["lr"] * (m / (1 - b1)) / (torch.sqrt(v / (1 - b2)) + _ADAM["eps"])
    sizes = _sizes(s["case"])
    return {"norm": norm, "p": p, "m": _split(m, sizes), "v": _split(v, sizes)}

"""Attention with a relative position bias in float64 from its formula, with the bound of what fp32 / bf16 arithmetic may be off.

Bounds. fp32: every product or sum of n terms is off by at most n 2^-24 of its largest magnitude; a score of at most ~16 in
size from D products, its exponential, and a sum over L terms give `c32 = 8 (D + 64) + L` roundings of 2^-24 relative to
the largest output. bf16 inputs are exact. `dv` and `dk` allow for P and dS rounded once (half a step, 2^-8 of each) as matrix
operands, `out` and `dq` to two numbers (2^-16 of each is left), results are rounded once; dQ starts from row sums D of an output kept
to 2^-16 of its terms:
  out: 2^-16 P |v| + 2^-8 |out|          dV: 2^-8 (P^T |dO| + |dV|)
  dK:  2^-8 (scale |dS|^T |q| + |dK|)    dQ: 2^-16 scale |dS| |k| + 2^-8 |dQ| + scale 2^-16 (|dO| . (|out| + P |v|)) (P |k|)
dV and dK of weights held as two numbers have 2^-8 of their first term again, `dv_split` and `dk_split`:
  dV: 2^-8 (2^-8 P^T |dO| + |dV|)        dK: 2^-8 (2^-8 scale |dS|^T |q| + |dK|)
The table's gradient is fp32 in both: c32 2^-24 times the sum of |dS| of its bucket."""
import numpy as np
import torch

H = 2.0 ** -8


def dropout_factors(seed, shape, p):
    """1/(1-p) or 0 for element number i = 0 .. of the array, by the library's counter-based rule."""
    n = int(np.prod(shape))
    with np.errstate(over="ignore"):
        z = np.arange(n, dtype=np.uint64) + np.uint64(seed) * np.uint64(0x9E3779B97F4A7C15) + np.uint64(0xD1B54A32D192ED03)
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        z = z ^ (z >> np.uint64(31))
    u = (z >> np.uint64(40)).astype(np.float32) * np.float32(1.0 / 16777216.0)
    return torch.from_numpy(np.where(u >= np.float32(p), 1.0 / (1.0 - p), 0.0)).reshape(shape)


def offsets(height, width, Lq, Lk, q_start):
    i, j = torch.arange(Lq) + q_start, torch.arange(Lk)
    dy = j[None, :] // width - i[:, None] // width + height - 1
    dx = j[None, :] % width - i[:, None] % width + width - 1
    return dy * (2 * width - 1) + dx


def formula(q, k, v, table, plan, mask=None, scale=None, q_start=0, dout=None, drop=None):
    """q [B,Lq,h,D], k, v [B,Lk,h,D], table [buckets,h] (any type, CPU). -> ({name: value}, {name: bound}); gradients too
    when dout is given. drop: factors [B,h,Lq,Lk]."""
    half = q.dtype == torch.bfloat16
    B, Lq, heads, D = q.shape
    Lk = k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    q, k, v = (t.detach().cpu().double().permute(0, 2, 1, 3) for t in (q, k, v))
    keep = torch.ones(B, Lk, dtype=torch.bool) if mask is None else mask.cpu().bool()
    k = torch.where(keep[:, None, :, None], k, 0.0)     # what a masked row holds does not exist
    v = torch.where(keep[:, None, :, None], v, 0.0)
    index = plan.index.cpu().long()
    off = offsets(plan.height, plan.width, Lq, Lk, q_start)
    bucket = index[off]
    s = scale * (q @ k.transpose(2, 3)) + table.detach().cpu().double()[bucket].permute(2, 0, 1)
    s = torch.where(keep[:, None, None, :], s, -np.inf)
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(m == -np.inf, 0.0, m))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    pd = p if drop is None else p * drop
    out = pd @ v
    eps = 2.0 ** -24 * (8 * (D + 64) + Lk)
    back = lambda t: t.permute(0, 2, 1, 3)      # noqa: E731
    got, tol = {"out": back(out)}, {}
    pv = pd @ v.abs()
    tol["out"] = back((H * (H * pv + out.abs()) if half else 0.0) + eps * (1e-30 + pv.max()) * torch.ones_like(out))
    if dout is None:
        return got, tol
    do = dout.detach().cpu().double().permute(0, 2, 1, 3)
    dv = pd.transpose(2, 3) @ do
    dp = do @ v.transpose(2, 3)
    if drop is not None:
        dp = dp * drop
    row = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - row)
    dq, dk = scale * ds @ k, scale * ds.transpose(2, 3) @ q
    eq = 2.0 ** -24 * (8 * (D + 64) + Lk + Lq)
    size = (p * (dp.abs() + row.abs()))     # what dS is the difference of
    one = torch.ones_like
    tol["dv"] = back((H * (pd.transpose(2, 3) @ do.abs() + dv.abs()) if half else 0.0) + eq * (1e-30 + (pd.transpose(2, 3) @ do.abs()).max()) * one(dv))
    kk, qq = scale * size @ k.abs(), scale * size.transpose(2, 3) @ q.abs()
    tol["dk"] = back((H * (scale * ds.abs().transpose(2, 3) @ q.abs() + dk.abs()) if half else 0.0) + eq * (1e-30 + qq.max()) * one(dk))
    vo, ko = pd.transpose(2, 3) @ do.abs(), scale * ds.abs().transpose(2, 3) @ q.abs()
    tol["dv_split"] = back((H * (H * vo + dv.abs()) if half else 0.0) + eq * (1e-30 + vo.max()) * one(dv))
    tol["dk_split"] = back((H * (H * ko + dk.abs()) if half else 0.0) + eq * (1e-30 + qq.max()) * one(dk))
    slack = (do.abs() * (out.abs() + pv)).sum(-1, keepdim=True) * (p @ k.abs()) * scale
    tol["dq"] = back((H * (H * scale * ds.abs() @ k.abs() + dq.abs() + H * slack * (1 + H)) if half else 0.0) + eq * (1e-30 + kk.max()) * one(dq))
    dt, da = torch.zeros(plan.num_buckets, heads, dtype=torch.float64), torch.zeros(plan.num_buckets, heads, dtype=torch.float64)
    flat = bucket.reshape(-1)
    dt.index_add_(0, flat, ds.sum(0).reshape(heads, -1).t())
    da.index_add_(0, flat, size.sum(0).reshape(heads, -1).t())
    got.update(dq=back(dq), dk=back(dk), dv=back(dv), dtable=dt)
    tol["dtable"] = eq * (1e-30 + da)
    return got, tol

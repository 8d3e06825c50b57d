"""Norms before and after a residual branch fused with its gate and its residual scale, on the gfx950 kernels of
csrc/blocknorm.hip."""
import torch

from ._lib import lib
from .ops import _DT, _p, _stream, first_derivative_only, on_device

_KINDS = {None: 0, "rms": 1, "layer": 2}


class GatedResidualNormFn(torch.autograd.Function):
    """record: whether autograd records the call (forward itself cannot see it); the statistics are kept only then."""

    @staticmethod
    def forward(ctx, x, f, scale, gate, w1, b1, w2, b2, post, pre, eps, record):
        x, f = x.contiguous(), f.contiguous()
        scale, gate, w1, b1, w2, b2 = [t if t is None else t.contiguous() for t in (scale, gate, w1, b1, w2, b2)]
        C, n = x.shape[-1], x.numel()
        images = 1 if gate is None else gate.shape[0]
        rows = n // (images * C) if n else 0
        y = torch.empty_like(x)
        z = torch.empty_like(x) if pre else None
        stats = torch.empty((images * rows, 4), dtype=torch.float32, device=x.device) if record and any(ctx.needs_input_grad) else None
        if rows:
            with on_device(x.device):
                lib().mia_blocknorm_fwd(_DT[x.dtype], _p(x), _p(f), images, rows, C, _p(scale), _p(gate), post, _p(w1), _p(b1),
                                        pre, _p(w2), _p(b2), eps, _p(y), _p(z), _p(stats), _stream())
        ctx.meta = (images, rows, C, post, pre)
        ctx.save_for_backward(x, f, scale, gate, w1, b1, w2, b2, stats)
        ctx.set_materialize_grads(False)
        return y, z

    @staticmethod
    def backward(ctx, dy, dz):
        first_derivative_only("gated_residual_norm")
        x, f, scale, gate, w1, b1, w2, b2, stats = ctx.saved_tensors
        images, rows, C, post, pre = ctx.meta
        ds, dg, dw1, db1, dw2, db2 = [t if t is None else torch.empty_like(t) for t in (scale, gate, w1, b1, w2, b2)]
        dx, df = torch.empty_like(x), torch.empty_like(f)
        if rows == 0 or (dy is None and dz is None):
            return (*[t if t is None else t.zero_() for t in (dx, df, ds, dg, dw1, db1, dw2, db2)], None, None, None, None)
        if dy is not None:
            dy = dy.contiguous()
        if dz is not None:
            dz = dz.contiguous()
        lb = lib()
        nws = lb.mia_blocknorm_ws_floats(images, rows, C, 1 if gate is not None else 0)
        ws = torch.empty((nws,), dtype=torch.float32, device=x.device)
        with on_device(x.device):
            lb.mia_blocknorm_bwd(_DT[x.dtype], _p(dy), _p(dz), _p(x), _p(f), _p(stats), images, rows, C, _p(scale), _p(gate), post,
                                 _p(w1), _p(b1), pre, _p(w2), _p(ws), nws, _p(dx), _p(df), _p(ds), _p(dg), _p(dw1), _p(db1),
                                 _p(dw2), _p(db2), _stream())
        return dx, df, ds, dg, dw1, db1, dw2, db2, None, None, None, None


def gated_residual_norm(x, f, scale=None, gate=None, post=None, post_weight=None, post_bias=None, pre="rms", pre_weight=None,
                        pre_bias=None, eps=1e-6):
    """The end of one residual branch and the norm in front of the next one, in one pass over the data:

        u = norm_post(f)                 (f itself for post=None)
        y = x + scale * gate * u
        z = norm_pre(y)                  (None for pre=None)

    x, f [..., C]: the residual stream and the branch's output, fp32 or bf16, the same shape and type. scale [C] and gate
    [x.shape[0], C] (one row per image, broadcast over its tokens) are optional; post and pre name the norms, "rms" or
    "layer", each with a weight [C] and optionally a bias [C] (population variance over C, eps added to it). Parameters and
    gate are fp32. All arithmetic is fp32: z is formed from y before y is rounded to the tensors' type. Returns (y, z);
    differentiable in every tensor. C <= 8192."""
    if post not in _KINDS or pre not in _KINDS:
        raise ValueError(f"norms are 'rms', 'layer' or None (got post={post!r}, pre={pre!r})")
    dtype, shape = x.dtype, x.shape
    if dtype not in _DT or f.dtype != dtype:
        raise TypeError(f"x and f are both fp32 or both bf16 (got {dtype}, {f.dtype})")
    if len(shape) < 1 or f.shape != shape:
        raise ValueError(f"x and f have one shape [..., C] (got {tuple(shape)}, {tuple(f.shape)})")
    C = shape[-1]
    if not 1 <= C <= 8192:
        raise ValueError(f"C must be 1..8192 (got {C})")
    for kind, w, b, which in ((post, post_weight, post_bias, "post"), (pre, pre_weight, pre_bias, "pre")):
        if (kind is None) != (w is None) or (kind is None and b is not None):
            raise ValueError(f"{which}={kind!r} needs {'no weight and no bias' if kind is None else which + '_weight'}")
    if gate is not None and len(shape) < 2:
        raise ValueError("a gate needs x of at least two dimensions")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative (got {eps})")
    device = x.get_device()
    for name, t, want in (("scale", scale, (C,)), ("gate", gate, (shape[0], C)), ("post_weight", post_weight, (C,)), ("post_bias", post_bias, (C,)),
                          ("pre_weight", pre_weight, (C,)), ("pre_bias", pre_bias, (C,))):
        if t is None:
            continue
        if t.shape != want or t.dtype != torch.float32:
            raise ValueError(f"{name} must be fp32 {want} (got {t.dtype} {tuple(t.shape)})")
        if t.get_device() != device:
            raise RuntimeError(f"gated_residual_norm needs its tensors on one MI355X device; there is no CPU path ({name} on {t.device}, x on {x.device})")
    if device < 0 or f.get_device() != device:
        raise RuntimeError(f"gated_residual_norm needs its tensors on one MI355X device; there is no CPU path (x on {x.device}, f on {f.device})")
    return GatedResidualNormFn.apply(x, f, scale, gate, post_weight, post_bias, pre_weight, pre_bias, _KINDS[post], _KINDS[pre],
                                     float(eps), torch.is_grad_enabled())

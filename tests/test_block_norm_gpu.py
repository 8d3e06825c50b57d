"""Residual branch end fused with its norms, on the gfx950 kernels, against the formula in float64.

Tolerances. All arithmetic is fp32 on the given inputs, so an element is off by at most a few tens of roundings (sums of a row
are formed as trees of depth <= 10 over <= 16 serial additions a lane; norm, affine and residual add about ten more): 64 * 2^-24 of
the tensor's largest magnitude, to which a bf16 output adds half a step, 2^-8 of itself. A parameter gradient adds terms of
order 1 and random sign over the rows: its partial sums stay below ~4 sqrt(rows) and no more than 64 additions follow each
other in one lane, so it is off by at most 64 * 4 * 2^-24 * sqrt(rows), or that share of its own largest magnitude."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import mia_amd  # noqa: E402,F401
from mia_amd.block_norm import gated_residual_norm  # noqa: E402

F32, BF16 = torch.float32, torch.bfloat16
NAMES = ("x", "f", "scale", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias")


def _formula(t, post, pre, eps):
    def norm(a, kind, w, b):
        if kind is None:
            return a
        m = a.mean(-1, keepdim=True) if kind == "layer" else 0.0
        o = (a - m) / torch.sqrt(((a - m) ** 2).mean(-1, keepdim=True) + eps) * w
        return o if b is None else o + b
    u = norm(t["f"], post, t.get("post_weight"), t.get("post_bias"))
    if "scale" in t:
        u = u * t["scale"]
    if "gate" in t:
        u = u * t["gate"].view(t["gate"].shape[0], *[1] * (u.dim() - 2), -1)
    y = t["x"] + u
    return y, norm(y, pre, t.get("pre_weight"), t.get("pre_bias")) if pre else None


def _inputs(shape, dtype, post, pre, scale, gate, bias, seed):
    g = torch.Generator().manual_seed(seed)
    C = shape[-1]
    t = {"x": torch.randn(shape, generator=g).to(dtype), "f": (torch.randn(shape, generator=g) * 2 + 0.5).to(dtype)}
    if scale:
        t["scale"] = torch.randn(C, generator=g) * 0.3
    if gate:
        t["gate"] = torch.rand(shape[0], C, generator=g)
    for which, kind in (("post", post), ("pre", pre)):
        if kind:
            t[which + "_weight"] = 1 + 0.2 * torch.randn(C, generator=g)
            if bias:
                t[which + "_bias"] = 0.2 * torch.randn(C, generator=g)
    dy, dz = torch.randn(shape, generator=g).to(dtype), torch.randn(shape, generator=g).to(dtype)
    return t, dy, dz


def _close(got, want, tol_abs, name):
    tol = tol_abs + (2.0 ** -8 * want.abs() if got.dtype == BF16 else 0.0)
    err = (got.double().cpu() - want).abs()
    assert torch.all(err <= tol), f"{name}: off by {(err - tol).max().item():.3g} more than allowed (largest value {want.abs().max():.3g})"


def _check(shape, dtype, post, pre, scale=True, gate=False, bias=True, use=("y", "z"), seed=0, eps=1e-6, make=lambda t: t):
    t, dy, dz = _inputs(shape, dtype, post, pre, scale, gate, bias, seed)
    ref = {k: v.double().requires_grad_() for k, v in t.items()}
    y64, z64 = _formula(ref, post, pre, eps)
    outs64, gs64 = [], []
    if "y" in use:
        outs64.append(y64), gs64.append(dy.double())
    if "z" in use and pre:
        outs64.append(z64), gs64.append(dz.double())
    names = list(ref)
    want = torch.autograd.grad(outs64, [ref[n] for n in names], gs64, allow_unused=True)
    mine = {k: make(v.cuda()).requires_grad_() for k, v in t.items()}
    kw = {k: v for k, v in mine.items() if k not in ("x", "f")}
    y, z = gated_residual_norm(mine["x"], mine["f"], post=post, pre=pre, eps=eps, **kw)
    assert y.shape == y64.shape and y.dtype == dtype and (z is None) == (pre is None)
    eps32 = 64 * 2.0 ** -24
    _close(y.detach(), y64.detach(), eps32 * y64.abs().max(), "y")
    if pre:
        # z divides by the row's deviation, which small rows can make large
        _close(z.detach(), z64.detach(), eps32 * max(1.0, float(z64.detach().abs().max())), "z")
    outs, gs = [], []
    if "y" in use:
        outs.append(y), gs.append(make(dy.cuda()))
    if "z" in use and pre:
        outs.append(z), gs.append(make(dz.cuda()))
    got = torch.autograd.grad(outs, [mine[n] for n in names], gs)
    rows = t["x"].numel() // shape[-1]
    for n, g, w in zip(names, got, want):
        w = torch.zeros_like(ref[n]) if w is None else w
        assert g.shape == t[n].shape and g.dtype == t[n].dtype
        top = float(w.abs().max())
        _close(g, w, eps32 * (top if n in ("x", "f") else 4 * max(math.sqrt(rows), top)), "d" + n)


KINDS = [(None, "rms"), ("rms", "layer"), ("layer", "rms"), ("layer", "layer"), ("rms", None)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("C", [1, 7, 24, 136, 384, 512, 520, 1000, 1024, 1030, 2304, 2100, 4096, 4100, 8192, 8191])
def test_widths(C, dtype):
    """Every row layout: wave or workgroup a row, vectors or single elements, the last channels of each."""
    if C == 1:      # a layer norm of one channel is constant: its true gradients are zero
        _check((3, 5, 1), dtype, "rms", "rms", gate=True, eps=0.5)
    else:
        _check((3, 5, C), dtype, "layer", "layer", gate=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("post,pre", KINDS)
@pytest.mark.parametrize("scale,gate,bias", [(True, False, True), (False, False, False), (False, True, True), (True, True, False)])
def test_kinds(post, pre, scale, gate, bias, dtype):
    _check((4, 33, 136), dtype, post, pre, scale, gate, bias)


@pytest.mark.parametrize("shape", [(1, 1, 384), (1, 384), (384,), (5, 384), (2, 10, 10, 384), (1, 4999, 64), (130, 3, 48), (700, 1, 24)])
@pytest.mark.parametrize("gate", [False, True])
def test_rows(shape, gate):
    if gate and len(shape) < 2:
        pytest.skip("a gate needs images")
    _check(shape, F32, "rms", "layer", gate=gate, seed=1)


@pytest.mark.parametrize("use", [("y",), ("z",)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_output_unused(use, dtype):
    _check((2, 9, 72), dtype, "layer", "rms", gate=True, use=use)


def test_gates_of_many_images():
    """More images than a grid has second or third dimensions."""
    _check((70000, 1, 8), F32, "rms", "layer", gate=True)


def test_views_of_any_layout():
    """Strided inputs and gradients, and rows that are not aligned to 16 bytes."""
    def odd(t):
        if t.dim() == 1:
            return torch.cat((torch.zeros(1, dtype=t.dtype, device=t.device), t))[1:].detach()
        return torch.stack((t, t), -1)[..., 0].detach()
    for dtype in (F32, BF16):
        _check((3, 7, 64), dtype, "rms", "layer", gate=True, make=odd)
    x = torch.randn(6 * 40 + 1, device="cuda")[1:].view(6, 40)
    w = torch.ones(40, device="cuda")
    y, z = gated_residual_norm(x, x, pre_weight=w)
    assert torch.equal(y, x + x)


def test_extreme_rows():
    """Rows of zeros (the deviation is sqrt(eps)), of one large value, and rows that are not finite stay among themselves."""
    x = torch.randn(8, 96)
    f = torch.randn(8, 96)
    x[0] = 0; f[0] = 0
    x[1] = 1e15
    f[2, 5] = float("inf")
    x[3, 7] = float("nan")
    w = torch.ones(96)
    y, z = gated_residual_norm(x.cuda(), f.cuda(), post="layer", post_weight=w.cuda(), pre="layer", pre_weight=w.cuda())
    good = [0, 4, 5, 6, 7]
    t = {"x": x[good].double(), "f": f[good].double(), "post_weight": w.double(), "pre_weight": w.double()}
    y64, z64 = _formula(t, "layer", "layer", 1e-6)
    _close(y[good], y64, 64 * 2.0 ** -24 * y64.abs().max(), "y")
    _close(z[good], z64, 64 * 2.0 ** -24 * z64.abs().max(), "z")
    assert int((z[0] != 0).sum()) == 0 and bool(torch.isnan(z[2:4]).all()) and bool(torch.isfinite(z[1]).all())


def test_empty_and_no_grad():
    w = torch.ones(16, device="cuda", requires_grad=True)
    x = torch.zeros(0, 5, 16, device="cuda", requires_grad=True)
    y, z = gated_residual_norm(x, x, pre_weight=w)
    assert y.shape == z.shape == x.shape
    gx, gw = torch.autograd.grad((y.sum() + z.sum()), (x, w))
    assert gx.shape == x.shape and int((gw != 0).sum()) == 0
    a = torch.randn(2, 3, 16, device="cuda")
    with torch.no_grad():
        y1, z1 = gated_residual_norm(a, a, pre_weight=w)
    y2, z2 = gated_residual_norm(a, a, pre_weight=w)
    assert torch.equal(y1, y2) and torch.equal(z1, z2) and not z1.requires_grad and z2.requires_grad


def test_difference_quotient():
    """The gradients along a random direction against a central difference of the operator itself (fp32: the quotient of a
    function of size ~S over a step h is off by 2^-22 S / h + h^2, 3e-3 of it at h = 1e-2 for the sums here)."""
    t, dy, dz = _inputs((3, 4, 40), F32, "layer", "rms", True, True, True, 5)
    mine = {k: v.cuda().requires_grad_() for k, v in t.items()}

    def value(d):
        y, z = gated_residual_norm(d["x"], d["f"], post="layer", pre="rms", **{k: v for k, v in d.items() if k not in ("x", "f")})
        return (y.double() * dy.cuda().double()).sum() + (z.double() * dz.cuda().double()).sum()
    grads = torch.autograd.grad(value(mine), list(mine.values()))
    g = torch.Generator().manual_seed(6)
    for name, grad in zip(mine, grads):
        d = torch.randn(t[name].shape, generator=g).cuda()
        d = d / d.norm()
        with torch.no_grad():
            hi, lo = dict(mine), dict(mine)
            hi[name], lo[name] = mine[name] + 1e-2 * d, mine[name] - 1e-2 * d
            quotient = float(value(hi) - value(lo)) / 2e-2
        along = float((grad * d).double().sum())
        assert abs(quotient - along) <= 1e-2 * max(1.0, abs(along)), name


def test_repeatable_streams_and_capture():
    t, dy, dz = _inputs((8, 50, 384), BF16, "layer", "layer", True, True, True, 7)
    mine = {k: v.cuda().requires_grad_() for k, v in t.items()}
    dy, dz = dy.cuda(), dz.cuda()

    def step():
        y, z = gated_residual_norm(mine["x"], mine["f"], post="layer", pre="layer", **{k: v for k, v in mine.items() if k not in ("x", "f")})
        return [y.detach(), z.detach(), *torch.autograd.grad((y, z), list(mine.values()), (dy, dz))]
    first = [t.clone() for t in step()]
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(first, g))
    graph = torch.cuda.CUDAGraph()
    cap = torch.cuda.Stream()
    cap.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(cap):
        step()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=cap):
        static = step()
    keep = mine["x"].detach().clone()
    for k in range(4):
        with torch.no_grad():
            mine["x"].copy_(keep * (1 + k))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(static, eager)), k


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("shape", [(1, 361, 2304), (128, 100, 384), (3, 40, 64), (300, 7, 136), (2, 5000, 1024)])
def test_column_sums_are_added_up_exactly(shape, gated):
    """Without norms the gradient of the scale is a plain sum of dy * f over the rows (of the gate, over its image's). Whole numbers of up to 2^9
    leave the few rows of a workgroup exact (63 rows of products below 2^18), the sum over workgroups needs more than 24 bits: it may
    cost the result's own rounding, 2^-24."""
    g = torch.Generator().manual_seed(8)
    C, rows = shape[-1], shape[0] * shape[1]
    f, dy = (torch.randint(300, 512, shape, generator=g).float() for _ in range(2))
    scale = torch.ones(C).cuda().requires_grad_()
    gate = torch.ones(shape[0], C).cuda().requires_grad_() if gated else None
    y, _ = gated_residual_norm(torch.zeros(shape).cuda(), f.cuda(), scale=scale, gate=gate, pre=None)
    per_image = (f.double() * dy.double()).sum(1)
    got = torch.autograd.grad(y, [scale] + [gate] * gated, dy.cuda())
    _close(got[0], per_image.sum(0), 2.0 ** -24 * per_image.sum(0).abs(), "dscale")
    if gated:
        _close(got[1], per_image, 2.0 ** -24 * per_image.abs(), "dgate")
    assert float(per_image.sum(0).min()) > 2 ** 23 or rows < 200

"""Attention with a learned relative position bias on the gfx950 kernels against the formula in float64; the bounds are
derived in relpos_formula.py."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import mia_amd  # noqa: E402,F401
from mia_amd.relpos import RelativePositionBuckets, relpos_attention, relpos_self_attention  # noqa: E402
from relpos_formula import dropout_factors, formula  # noqa: E402

F32, BF16 = torch.float32, torch.bfloat16


def _compare(got, want, tol, where=""):
    assert not torch.isnan(got).any() or torch.isnan(want).any(), where
    err = (got.double().cpu() - want).abs()
    assert torch.all(err <= tol), f"{where}: off by {err.max():.3g} where {tol.reshape(-1)[int((err - tol).argmax())]:.3g} is allowed (largest {want.abs().max():.3g})"


def _inputs(B, Lq, Lk, heads, D, dtype, buckets, seed):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(B, n, heads, D, generator=g).to(dtype) for n in (Lq, Lk, Lk))
    return q, k, v, torch.randn(buckets, heads, generator=g), torch.randn(B, Lq, heads, D, generator=g).to(dtype)


def _check(plan, B=2, heads=2, D=16, dtype=F32, Lq=None, Lk=None, q_start=0, mask=None, scale=None, seed=0, drop=0.0, packed=False,
           place=lambda t: t.cuda()):
    Lk = plan.height * plan.width if Lk is None else Lk
    Lq = Lk if Lq is None else Lq
    q, k, v, table, dout = _inputs(B, Lq, Lk, heads, D, dtype, plan.num_buckets, seed)
    factors = dropout_factors(1234, (B, heads, Lq, Lk), drop) if drop else None
    want, tol = formula(q, k, v, table, plan, mask, scale, q_start, dout, factors)
    t = table.cuda().requires_grad_()
    kw = dict(key_mask=mask.cuda() if mask is not None else None, scale=scale, dropout_p=drop, seed=1234)
    if packed:
        qkv = place(torch.stack((q, k, v), 2)).requires_grad_()
        out = relpos_self_attention(qkv, t, plan, **kw)
        dqkv, dt = torch.autograd.grad(out, (qkv, t), place(dout))
        assert dqkv.shape == qkv.shape
        got = {"out": out, "dq": dqkv[:, :, 0], "dk": dqkv[:, :, 1], "dv": dqkv[:, :, 2], "dtable": dt}
    else:
        mine = [place(x).requires_grad_() for x in (q, k, v)]
        out = relpos_attention(*mine, t, plan, q_start=q_start, **kw)
        grads = torch.autograd.grad(out, (*mine, t), place(dout))
        got = dict(zip(("out", "dq", "dk", "dv", "dtable"), (out, *grads)))
        with torch.no_grad():       # the forward pass alone gives the same bits
            assert torch.equal(relpos_attention(*mine, t, plan, q_start=q_start, **kw), out)
    for name, value in got.items():
        assert value.dtype == (F32 if name == "dtable" else dtype) and value.shape == want[name].shape, name
        _compare(value.detach(), want[name], tol[name], name)


MAPS = [(1, 1), (1, 2), (2, 1), (3, 5), (10, 10), (1, 63), (1, 64), (1, 65), (1, 200), (7, 30), (2, 129), (19, 19), (130, 2)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("height,width", MAPS)
def test_maps(height, width, dtype):
    _check(RelativePositionBuckets(height, width, 8, 16), dtype=dtype, D=24)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [8, 16, 24, 32, 40, 48, 56, 64, 72, 96, 104, 128])
def test_head_widths(D, dtype):
    _check(RelativePositionBuckets(9, 11, 16, 32), D=D, heads=3, dtype=dtype, packed=True)


@pytest.mark.parametrize("D", [32, 48, 64, 128])
def test_two_columns_a_wave(D):
    """Enough images and heads for the variant that gives a wave 32 queries (or keys)."""
    _check(RelativePositionBuckets(10, 10, 16, 32), B=65, heads=8, D=D, dtype=BF16, packed=True)


def test_long_map():
    _check(RelativePositionBuckets(38, 38, 16, 64), B=1, heads=2, D=64, dtype=BF16)
    _check(RelativePositionBuckets(2, 700, 16, 64), B=1, heads=1, D=32, dtype=BF16)


def _masks(B, Lk, seed):
    g = torch.Generator().manual_seed(seed)
    m = torch.rand(B, Lk, generator=g) < 0.6
    m[0] = False                                # nothing left
    m[1] = torch.arange(Lk) < Lk // 2           # a padded tail, whole tiles of it
    m[2] = False
    m[2, Lk - 1] = True                         # one key
    return m


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("height,width", [(1, 5), (10, 10), (1, 300), (13, 17)])
def test_masks(height, width, dtype):
    _check(RelativePositionBuckets(height, width, 8, 32), B=5, D=32, dtype=dtype, mask=_masks(5, height * width, 3))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Lq,Lk,q_start", [(1, 155, 154), (1, 1, 0), (5, 300, 100), (16, 700, 684), (70, 33, 200), (1, 900, 0)])
def test_queries_anywhere(Lq, Lk, q_start, dtype):
    _check(RelativePositionBuckets(1, 1000, 32, 128), Lq=Lq, Lk=Lk, q_start=q_start, D=48, dtype=dtype)
    if Lk <= 33 * 31:
        _check(RelativePositionBuckets(33, 31, 16, 32), Lq=Lq, Lk=Lk, q_start=q_start, D=16, dtype=dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Lq,Lk,B,heads", [(1, 4096, 2, 3), (1, 16383, 1, 8), (3, 5001, 3, 1), (20, 2049, 1, 2)])
def test_split_over_the_keys(Lq, Lk, B, heads, dtype):
    plan = RelativePositionBuckets(1, 16384, 32, 128)
    mask = torch.rand(B, Lk, generator=torch.Generator().manual_seed(4)) < 0.9
    mask[0] = torch.arange(Lk) >= Lk - 70       # whole splits without a key
    if B > 2:
        mask[2] = False
    _check(plan, B=B, heads=heads, Lq=Lq, Lk=Lk, q_start=Lk - Lq, D=64, dtype=dtype, mask=mask)
    _check(plan, B=B, heads=heads, Lq=Lq, Lk=Lk, q_start=Lk - Lq, D=64, dtype=dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [8, 32, 40, 64, 96, 128])
@pytest.mark.parametrize("Lq", [1, 2, 15, 16, 17])
def test_few_queries(Lq, D, dtype):
    """Both sides of the border between the two forward kernels, over ends inside a chunk of keys, on maps of several rows."""
    plan = RelativePositionBuckets(9, 37, 8, 16)
    g = torch.Generator().manual_seed(Lq)
    for Lk, q_start in ((333, 316), (65, 0)):
        _check(plan, Lq=Lq, Lk=Lk, q_start=q_start, D=D, dtype=dtype)
        mask = torch.rand(3, Lk, generator=g) < 0.5
        mask[0] = False
        mask[1, :64] = False
        _check(plan, B=3, Lq=Lq, Lk=Lk, q_start=q_start, D=D, dtype=dtype, mask=mask, drop=0.2)


@pytest.mark.parametrize("heads,D,dtype", [(8, 64, BF16), (6, 64, BF16), (7, 32, BF16), (4, 64, F32)])
def test_few_queries_of_neighbouring_heads(heads, D, dtype):
    """Enough keys for the variants whose waves read several heads."""
    B, Lk = -(-9000 // (heads * (4100 // (64 if dtype == BF16 else 32)))), 4100
    mask = torch.arange(Lk)[None, :] < torch.randint(1, Lk + 1, (B, 1), generator=torch.Generator().manual_seed(18))
    mask[0] = False
    _check(RelativePositionBuckets(1, 4200, 32, 128), B=B, heads=heads, Lq=2, Lk=Lk, q_start=Lk - 2, D=D, dtype=dtype, mask=mask)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scale_and_dropout(dtype):
    plan = RelativePositionBuckets(8, 12, 8, 16)
    _check(plan, scale=1.0, D=16, dtype=dtype)
    _check(plan, scale=0.01, D=64, dtype=dtype)
    _check(plan, drop=0.3, D=48, dtype=dtype, packed=True)
    _check(RelativePositionBuckets(1, 150, 8, 16), drop=0.1, Lq=40, q_start=90, D=32, dtype=dtype)


def test_split_with_dropout():
    _check(RelativePositionBuckets(1, 3000, 8, 16), drop=0.25, Lq=1, q_start=2999, D=32, B=1, heads=2)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_memory_layouts(dtype):
    plan = RelativePositionBuckets(5, 9, 8, 16)

    def heads_first(t):
        return t.cuda().transpose(1, 2).contiguous().transpose(1, 2)

    def unaligned(t):
        flat = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = t.reshape(-1).cuda()
        return flat[1:].view(t.shape)

    def strided(t):
        wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 3, dtype=t.dtype, device="cuda")
        wide[..., :t.shape[-1]] = t.cuda()
        return wide[..., :t.shape[-1]]
    for place in (heads_first, unaligned, strided):
        _check(plan, D=24, dtype=dtype, place=place)
        _check(plan, D=24, dtype=dtype, place=place, packed=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("height,width,D", [(1, 2, 8), (10, 10, 48), (1, 300, 32)])
def test_keys_with_a_common_part(height, width, D, dtype):
    """What all keys share drops out of the gradient of the queries: it must not come back through rounded weights."""
    plan = RelativePositionBuckets(height, width, 8, 16)
    n = height * width
    q, k, v, table, dout = _inputs(3, n, n, 2, D, dtype, plan.num_buckets, 16)
    k = (k.float() + 20.0).to(dtype)
    q = (q.float() * 0.05).to(dtype)
    mine = [t.cuda().requires_grad_() for t in (q, k, v, table)]
    want, tol = formula(q, k, v, table, plan, dout=dout)
    out = relpos_attention(*mine, plan)
    for name, value in zip(("out", "dq", "dk", "dv", "dtable"), (out.detach(), *torch.autograd.grad(out, mine, dout.cuda()))):
        _compare(value, want[name], tol[name], name)


@pytest.mark.parametrize("height,width", [(7, 30), (1, 500), (3, 97)])
def test_bias_gradient_repeats(height, width):
    """One bucket per offset over several tiles of queries: every single sum has the same bits each time."""
    plan = RelativePositionBuckets.from_index(height, width, torch.arange((2 * height - 1) * (2 * width - 1)))
    n = height * width
    q, k, v, table, dout = _inputs(8, n, n, 4, 32, BF16, plan.num_buckets, 17)
    mine = [t.cuda().requires_grad_() for t in (q, k, v, table)]
    dout = dout.cuda()
    first = torch.autograd.grad(relpos_attention(*mine, plan), mine, dout)
    for _ in range(6):
        assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(relpos_attention(*mine, plan), mine, dout)))


def test_custom_buckets():
    """One bucket for every offset, one for all, and buckets that no offset falls into."""
    g = torch.Generator().manual_seed(5)
    for index, n in ((torch.arange(13 * 17), None), (torch.zeros(13 * 17, dtype=torch.long), None), (torch.randint(0, 50, (13 * 17,), generator=g), 60)):
        plan = RelativePositionBuckets.from_index(7, 9, index, n)
        _check(plan, D=32)
        _check(plan, D=32, dtype=BF16)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_what_masked_keys_hold_does_not_matter(dtype):
    plan = RelativePositionBuckets(6, 12, 8, 16)
    q, k, v, table, dout = _inputs(2, 72, 72, 2, 32, dtype, plan.num_buckets, 6)
    mask = torch.rand(2, 72, generator=torch.Generator().manual_seed(7)) < 0.7
    results = []
    for junk in (0.0, float("nan"), float("inf"), torch.finfo(dtype).min):
        kj, vj = k.clone(), v.clone()
        kj[~mask], vj[~mask] = junk, junk
        mine = [t.cuda().requires_grad_() for t in (q, kj, vj, table)]
        out = relpos_attention(*mine, plan, key_mask=mask.cuda())
        results.append([out.detach(), *torch.autograd.grad(out, mine, dout.cuda())])
    for r in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], r))
    assert int((results[0][2][~mask.cuda()] != 0).sum()) == 0 and int((results[0][3][~mask.cuda()] != 0).sum()) == 0


def test_extreme_table_entries():
    """A bucket at the type's lowest value is out-scored by every other one but still a score; one at -inf forbids its pairs, and a
    query whose pairs are all forbidden gives zeros."""
    plan = RelativePositionBuckets(1, 70, 8, 16)
    q, k, v, table, dout = _inputs(1, 70, 70, 2, 16, F32, 8, 8)
    for low in (torch.finfo(F32).min, float("-inf")):
        t = table.clone()
        t[0] = low                  # distance 0: the query's own token
        t[1] = low
        want, tol = formula(q, k, v, t, plan)
        _compare(relpos_attention(q.cuda(), k.cuda(), v.cuda(), t.cuda(), plan), want["out"], tol["out"])
    every = torch.full_like(table, torch.finfo(F32).min)
    got = relpos_attention(q.cuda(), k.cuda(), v.cuda(), every.cuda(), plan)
    # all scores are equal at that size: the mean of the values, and the gradients of that
    mine = [t.cuda().requires_grad_() for t in (q, k, v, every)]
    want, tol = formula(q, k, v, every, plan, dout=dout)
    for name, grad in zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(relpos_attention(*mine, plan), mine, dout.cuda())):
        _compare(grad, want[name], tol[name], name)
    _compare(got, v.double().mean(1, keepdim=True).expand_as(v), torch.full(v.shape, 1e-6, dtype=torch.float64))
    none = torch.full_like(table, float("-inf"))
    mine = [t.cuda().requires_grad_() for t in (q, k, v, none)]
    out = relpos_attention(*mine, plan)
    assert int((out != 0).sum()) == 0
    assert all(int((g != 0).sum()) == 0 for g in torch.autograd.grad(out, mine, dout.cuda()))


def test_not_finite_inputs_stay_in_their_rows():
    plan = RelativePositionBuckets(1, 80, 8, 16)
    q, k, v, table, _ = _inputs(2, 80, 80, 1, 16, F32, 8, 9)
    q[0, 3, 0, 5] = float("nan")
    out = relpos_attention(q.cuda(), k.cuda(), v.cuda(), table.cuda(), plan).cpu()
    assert bool(torch.isnan(out[0, 3]).all())
    q[0, 3, 0, 5] = 0.0
    want, tol = formula(q, k, v, table, plan)
    out[0, 3], want["out"][0, 3] = 0.0, 0.0
    _compare(out, want["out"], tol["out"])


def test_empty():
    plan = RelativePositionBuckets(1, 8, 8, 16)
    table = torch.zeros(8, 2, device="cuda", requires_grad=True)
    for B, Lq, Lk in ((0, 4, 4), (2, 0, 4), (2, 4, 0)):
        q, k, v = (torch.ones(B, n, 2, 16, device="cuda", requires_grad=True) for n in (Lq, Lk, Lk))
        out = relpos_attention(q, k, v, table, plan)
        assert out.shape == q.shape and int((out != 0).sum()) == 0
        assert all(int((g != 0).sum()) == 0 and g.shape == t.shape for g, t in zip(torch.autograd.grad(out.sum(), (q, k, v, table)), (q, k, v, table)))


def test_only_some_gradients():
    plan = RelativePositionBuckets(4, 5, 8, 16)
    q, k, v, table, dout = _inputs(2, 20, 20, 2, 16, BF16, plan.num_buckets, 10)
    mine = [t.cuda().requires_grad_() for t in (q, k, v, table)]
    full = torch.autograd.grad(relpos_attention(*mine, plan), mine, dout.cuda())
    for i in range(4):
        some = [t.detach().requires_grad_(j == i) for j, t in enumerate(mine)]
        (got,) = torch.autograd.grad(relpos_attention(*some, plan), some[i], dout.cuda())
        assert torch.equal(got, full[i])


def test_difference_quotient():
    """Along random directions the gradients agree with a central difference of the operator (fp32, values of order 30 over a
    step of 1e-2: the quotient is good to about 1e-3)."""
    plan = RelativePositionBuckets(3, 4, 8, 16)
    q, k, v, table, dout = _inputs(1, 12, 12, 2, 16, F32, plan.num_buckets, 11)
    mine = [t.cuda().requires_grad_() for t in (q, k, v, table)]
    value = lambda ts: (relpos_attention(*ts, plan).double() * dout.cuda().double()).sum()     # noqa: E731
    grads = torch.autograd.grad(value(mine), mine)
    g = torch.Generator().manual_seed(12)
    for i, grad in enumerate(grads):
        d = torch.randn(mine[i].shape, generator=g).cuda()
        d = d / d.norm()
        with torch.no_grad():
            hi, lo = list(mine), list(mine)
            hi[i], lo[i] = mine[i] + 1e-2 * d, mine[i] - 1e-2 * d
            quotient = float(value(hi) - value(lo)) / 2e-2
        along = float((grad * d).double().sum())
        assert abs(quotient - along) <= 5e-3 * max(1.0, abs(along)), i


def test_offsets_past_32_bits():
    """Images more than 2^31 elements apart, as in a slice of a long cache."""
    plan = RelativePositionBuckets(1, 100, 8, 16)
    q, k, v, table, _ = _inputs(2, 3, 100, 2, 16, BF16, 8, 13)
    far = 1 << 31
    store = torch.empty(far + 100 * 2 * 16, dtype=BF16, device="cuda")
    out = []
    for k_, v_ in ((k, v),):
        kc = store.as_strided((2, 100, 2, 16), (far, 32, 16, 1))
        kc.copy_(k_)
        out.append(relpos_attention(q.cuda(), kc, v_.cuda(), table.cuda(), plan, q_start=97))
        keep = kc.clone()
        vc = kc
        vc.copy_(v_)
        out.append(relpos_attention(q.cuda(), keep, vc, table.cuda(), plan, q_start=97))
    want, tol = formula(q, k, v, table, plan, q_start=97)
    for o in out:
        _compare(o, want["out"], tol["out"])


@pytest.mark.parametrize("Lq", [2, 40])
def test_tokens_past_32_bits(Lq):
    """Tokens so far apart that the last ones lie more than 2^31 elements (2^32 bytes) behind the first."""
    plan = RelativePositionBuckets(1, 150, 8, 16)
    q, k, v, table, dout = _inputs(1, Lq, 150, 1, 16, BF16, 8, 19)
    apart = (1 << 24) - 8
    store = torch.empty(149 * apart + 32, dtype=BF16, device="cuda")
    kc, vc = (store[i:].as_strided((1, 150, 1, 16), (16, apart, 16, 1)) for i in (0, 16))
    kc.copy_(k), vc.copy_(v)
    mine = [q.cuda().requires_grad_(), kc.requires_grad_(), vc.requires_grad_(), table.cuda().requires_grad_()]
    want, tol = formula(q, k, v, table, plan, q_start=100, dout=dout)
    out = relpos_attention(*mine, plan, q_start=100)
    for name, value in zip(("out", "dq", "dk", "dv", "dtable"), (out.detach(), *torch.autograd.grad(out, mine, dout.cuda()))):
        _compare(value, want[name], tol[name], name)


def test_repeatable_streams_and_capture():
    plan = RelativePositionBuckets(12, 12, 16, 32)
    q, k, v, table, dout = _inputs(4, 144, 144, 4, 48, BF16, plan.num_buckets, 14)
    mine = [t.cuda().requires_grad_() for t in (q, k, v, table)]
    dout = dout.cuda()
    mask = (torch.rand(4, 144, generator=torch.Generator().manual_seed(15)) < 0.8).cuda()

    def step():
        out = relpos_attention(*mine, plan, key_mask=mask)
        return [out.detach(), *torch.autograd.grad(out, mine, dout)]
    first = [t.clone() for t in step()]
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, step()))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in got for a, b in zip(first, r))
    graph, cap = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    cap.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(cap):
        step()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=cap):
        static = step()
    keep, keep_t = mine[0].detach().clone(), mine[3].detach().clone()
    for n in range(4):
        with torch.no_grad():
            mine[0].copy_(keep * (1 + 0.5 * n))
            mine[3].copy_(keep_t * (1 - 0.2 * n))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(static, eager)), n


@pytest.mark.parametrize("height,width,B,D,drop", [(10, 10, 8, 48, 0.0), (10, 10, 3, 16, 0.2), (1, 300, 2, 32, 0.0), (17, 19, 2, 64, 0.0), (9, 11, 4, 128, 0.0)])
def test_key_gradients_hold_the_weights_twice(height, width, B, D, drop):
    """bf16: dK and dV carry no rounding of P and dS beyond their own last one, where a sum over many queries nearly cancels too."""
    plan = RelativePositionBuckets(height, width, 8, 16)
    n = height * width
    q, k, v, table, dout = _inputs(B, n, n, 4, D, BF16, plan.num_buckets, 21)
    mine = [t.cuda().requires_grad_() for t in (q, k, v, table)]
    want, tol = formula(q, k, v, table, plan, dout=dout, drop=dropout_factors(1234, (B, 4, n, n), drop) if drop else None)
    grads = torch.autograd.grad(relpos_attention(*mine, plan, dropout_p=drop, seed=1234), mine, dout.cuda())
    _compare(grads[1], want["dk"], tol["dk_split"], "dk")
    _compare(grads[2], want["dv"], tol["dv_split"], "dv")


def _variants():
    from relpos_variants import VARIANTS
    return [pytest.param(p, id="-".join(map(str, p))) for p in VARIANTS]


@pytest.mark.parametrize("problem", _variants())
def test_every_layout_of_the_kernels(problem):
    """Each choice of columns, splits and heads of a workgroup, with masks and with dropout (see relpos_variants.py)."""
    from relpos_variants import VARIANTS, layout
    dtype, B, heads, Lq, Lk, D, height, width, q_start = problem
    for direction, want in VARIANTS[problem].items():
        assert layout(direction, *problem[:6]) == want
    mask = torch.rand(B, Lk, generator=torch.Generator().manual_seed(22)) < 0.8
    mask[0] = False
    if B > 1:
        mask[1] = torch.arange(Lk) < Lk // 2
    plan = RelativePositionBuckets(height, width, 16, 64)
    _check(plan, B=B, heads=heads, Lq=Lq, Lk=Lk, q_start=q_start, D=D, dtype=(F32, BF16)[dtype], mask=mask, drop=0.1 if B * heads * Lq * Lk < 1 << 23 else 0.0)
    if B * heads * Lq * Lk < 1 << 22:
        _check(plan, B=B, heads=heads, Lq=Lq, Lk=Lk, q_start=q_start, D=D, dtype=(F32, BF16)[dtype])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_bias_gradient_over_more_than_1024_key_blocks(dtype):
    _check(RelativePositionBuckets(1, 65800, 32, 128), B=1, heads=1, Lq=70, Lk=65700, q_start=65700, D=16, dtype=dtype)
    _check(RelativePositionBuckets(256, 257, 16, 64), B=1, heads=1, Lq=70, Lk=65700, q_start=30000, D=8, dtype=dtype)


@pytest.mark.parametrize("height,width,Lq", [(1, 64, 64), (8, 8, 64), (1, 1088, 64), (32, 34, 64)])
def test_bias_gradient_is_added_up_exactly(height, width, Lq):
    """With equal scores over a power of two of keys every weight is exact, and with small whole numbers in v and dout so are dS
    (multiples of 2^-12) and the sum of an offset over a tile. What is left is the addition over images, tiles and offsets, whose
    terms do not cancel here (odd dx against even) and need more than 24 bits: it may cost the result's own rounding, 2^-24."""
    index = torch.arange((2 * height - 1) * (2 * width - 1)) % (2 * width - 1) % 2      # whether dx is even
    plan = RelativePositionBuckets.from_index(height, width, index)
    B, L, g = 100, height * width, torch.Generator().manual_seed(23)
    keep = torch.arange(L) >= L - 64            # 64 keys that exist: weights of 1/64
    sign = 1.0 - 2.0 * (torch.arange(L) % 2)
    v = torch.randint(-3, 4, (B, L, 2, 8), generator=g).float()
    v[..., 0] = 7.0 * sign[None, :, None]
    dout = torch.randint(-3, 4, (B, Lq, 2, 8), generator=g).float()
    dout[..., 0] = 7.0 * sign[None, :Lq, None]
    q, k = torch.zeros(B, Lq, 2, 8), torch.randn(B, L, 2, 8, generator=g)
    table = torch.zeros(2, 2)
    mask = keep.expand(B, L)
    want, _ = formula(q, k, v, table, plan, mask, dout=dout)
    assert float(want["dtable"].abs().min()) * 2 ** 12 > 2 ** 25
    t = table.cuda().requires_grad_()
    out = relpos_attention(q.cuda(), k.cuda(), v.cuda(), t, plan, key_mask=mask.cuda())
    (got,) = torch.autograd.grad(out, t, dout.cuda())
    _compare(got, want["dtable"], 2.0 ** -24 * want["dtable"].abs() + 1e-9, "dtable")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Lq", [3, 70])
def test_shared_heads_and_broadcast_inputs(Lq, dtype):
    """Keys and values shared by the heads, by the batch, queries shared by the tokens (strides of zero): read where they lie, and their
    gradients are the sums over what shares them. (Such a sum of n rounded gradients is off by n of their bounds and its own rounding.)"""
    plan = RelativePositionBuckets(6, 15, 8, 16)
    q, k, v, table, dout = _inputs(2, Lq, 90, 4, 24, dtype, plan.num_buckets, 24)
    for dims in ((2,), (0,), (0, 2), (0, 1)):
        one = [t[tuple(slice(0, 1) if d in dims else slice(None) for d in range(4))] for t in (q, k, v)]
        wide = [t.expand(2, n, 4, 24) for t, n in zip(one, (Lq, 90, 90))]
        want, tol = formula(*wide, table, plan, q_start=90 - Lq, dout=dout)
        mine = [t.cuda().requires_grad_() for t in one]
        out = relpos_attention(*(t.expand(2, n, 4, 24) for t, n in zip(mine, (Lq, 90, 90))), table.cuda(), plan, q_start=90 - Lq)
        _compare(out.detach(), want["out"], tol["out"], "out")
        for name, t, got in zip(("dq", "dk", "dv"), mine, torch.autograd.grad(out, mine, dout.cuda())):
            total, slack = (x.sum(dims, keepdim=True) for x in (want[name], tol[name]))
            size = want[name].abs().sum(dims, keepdim=True)
            n = 2 * 4 * 90
            _compare(got, total, slack + (2.0 ** -8 * total.abs() if dtype == BF16 else 0.0) + n * 2.0 ** -24 * size, name)

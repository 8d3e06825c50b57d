"""Relative position buckets, and the refusals of the attention's entry points, without a GPU."""
import ctypes
from array import array

import pytest
import torch

import mia_amd
from mia_amd.relpos import RelativePositionBuckets, relpos_attention, relpos_self_attention
from relpos_formula import formula, offsets

P = ctypes.c_void_p(4096)


def test_axis_buckets():
    plan = RelativePositionBuckets(1, 400, 32, 128, device="cpu")
    b = {d: int(plan.index[d + 399]) for d in range(-399, 400)}
    assert plan.num_buckets == 32 and [b[-d] for d in range(8)] == list(range(8)) and [b[d] for d in range(1, 8)] == list(range(17, 24))
    assert b[8] == 24 and b[-8] == 8 and b[127] == 31 and b[399] == 31 and b[-128] == 15
    far = [b[-d] for d in range(8, 400)]
    assert far == sorted(far) and set(far) == set(range(8, 16))
    assert [b[d] - 16 for d in range(1, 400)] == [b[-d] for d in range(1, 400)]


def test_map_buckets_and_sorted_lists():
    plan = RelativePositionBuckets(5, 9, 8, 16, device="cpu")
    rows, cols = RelativePositionBuckets(1, 5, 8, 16, device="cpu").index, RelativePositionBuckets(1, 9, 8, 16, device="cpu").index
    assert plan.num_buckets == 64
    for dy in range(-4, 5):
        for dx in range(-8, 9):
            o = (dy + 4) * 17 + dx + 8
            assert int(plan.index[o]) == int(rows[dy + 4]) * 8 + int(cols[dx + 8])
    assert int(plan.start[-1]) == plan.index.numel() and sorted(plan.order.tolist()) == list(range(plan.index.numel()))
    for k in range(64):
        members = plan.order[plan.start[k]:plan.start[k + 1]].long()
        assert bool((plan.index[members] == k).all())


def test_offset_numbers():
    off = offsets(3, 4, 12, 12, 0)
    assert off[0, 0] == 2 * 7 + 3 and off[0, 11] == 4 * 7 + 6 and off[11, 0] == 0 and off[3, 4] == 3 * 7 + 0
    assert torch.equal(offsets(3, 4, 2, 12, 5), off[5:7])


def test_bucket_refusals():
    for kw in (dict(height=0, width=3), dict(height=2, width=1025), dict(height=3, width=3, num_buckets=6),
               dict(height=3, width=3, num_buckets=32, max_distance=8), dict(height=1, width=1 << 28)):
        with pytest.raises(ValueError):
            RelativePositionBuckets(device="cpu", **kw)
    for index, n, err in ((torch.zeros(24, dtype=torch.long), None, ValueError), (torch.full((25,), -1), None, ValueError),
                          (torch.arange(25), 20, ValueError), (torch.zeros(25), None, TypeError)):
        with pytest.raises(err):
            RelativePositionBuckets.from_index(3, 3, index, n, device="cpu")
    assert RelativePositionBuckets.from_index(3, 3, torch.arange(25).view(5, 5), 40, device="cpu").num_buckets == 40


def test_formula_against_autograd():
    """The oracle's hand-written gradients are those of its forward pass."""
    g = torch.Generator().manual_seed(0)
    plan = RelativePositionBuckets(2, 4, 4, 8, device="cpu")
    q, k, v = (torch.randn(2, n, 3, 8, generator=g, dtype=torch.float64) for n in (5, 7, 7))
    table = torch.randn(plan.num_buckets, 3, generator=g, dtype=torch.float64)
    dout = torch.randn(2, 5, 3, 8, generator=g, dtype=torch.float64)
    mask = torch.tensor([[1, 1, 0, 1, 1, 0, 1], [0] * 7]).bool()
    want, _ = formula(q, k, v, table, plan, mask, q_start=2, dout=dout)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, table)]
    s = torch.einsum("bihd,bjhd->bhij", leaves[0], leaves[1]) * 8 ** -0.5 + leaves[3][plan.index.long()[offsets(2, 4, 5, 7, 2)]].permute(2, 0, 1)
    p = torch.softmax(torch.where(mask[:, None, None, :], s, -1e30), -1) * mask[:, None, None, :]
    out = torch.einsum("bhij,bjhd->bihd", p, leaves[2])
    assert torch.allclose(out, want["out"], atol=1e-12)
    for name, grad in zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(out, leaves, dout)):
        assert torch.allclose(grad, want[name], atol=1e-12), name


def _fwd(dtype=0, q=P, strides=None, B=1, heads=2, Lq=5, Lk=9, D=16, bias=P, height=3, width=3, q_start=0, scale=0.25, pdrop=0.0, ws=None, n=0):
    st = array("q", strides or [80, 32, 16] * 3)
    mia_amd.lib().mia_relpos_fwd(dtype, q, P, P, st.buffer_info()[0], B, heads, Lq, Lk, D, bias, height, width, q_start, None, scale, pdrop, 0,
                                 None, ws, n, P, None, None, None)


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=5), "bad dtype"), (dict(B=0), "bad shape"), (dict(Lk=0), "bad shape"), (dict(D=12), "multiple of 8"), (dict(D=136), "multiple of 8"),
    (dict(height=0), "bad map"), (dict(height=2, width=1030, Lk=9), "bad map"), (dict(height=1, width=1 << 29), "too many offsets"), (dict(height=1, width=(1 << 26) + 1), "too many offsets"),
    (dict(B=1 << 20, heads=16, Lq=9), "too many workgroups"),
    (dict(Lk=10), "do not fit"), (dict(q_start=5), "do not fit"), (dict(q_start=-1), "do not fit"), (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(pdrop=1.0), "dropout"), (dict(bias=None), "null"), (dict(q=ctypes.c_void_p(4104)), "16 bytes"),
    (dict(strides=[80, 32, 16, 80, 32, 16, 80, 33, 16]), "16 bytes"), (dict(dtype=1, strides=[80, 32, 16, 80, 32, 12, 80, 32, 16]), "16 bytes"),
    (dict(Lq=1, Lk=4096, height=1, width=4096), "workspace")])
def test_forward_entry_refuses(kw, match):
    with pytest.raises(mia_amd.MiaError, match=match):
        _fwd(**kw)


def test_backward_entry_refuses():
    lib = mia_amd.lib()
    st = array("q", [80, 32, 16] * 3)
    need = lib.mia_relpos_bwd_ws_floats(0, 1, 2, 5, 9, 16, 3, 3, 1)
    assert need > lib.mia_relpos_bwd_ws_floats(0, 1, 2, 5, 9, 16, 3, 3, 0) > 0

    def bwd(dout=P, stat=P, order=P, buckets=3, n=need, dq=P, dtype=0, low=None):
        a = st.buffer_info()[0]
        lib.mia_relpos_bwd(dtype, P, P, P, a, dout, P, low, stat, 1, 2, 5, 9, 16, P, 3, 3, 0, None, 0.25, 0.0, 0, None, order, P, buckets, P, n, dq, P, P, a,
                           P, None)
    for kw, match in ((dict(dout=None), "null"), (dict(stat=None), "null"), (dict(order=None), "bucket lists"), (dict(buckets=0), "bucket lists"),
                      (dict(n=need - 1), "too small"), (dict(dtype=1), "out_low"), (dict(dtype=1, low=ctypes.c_void_p(4100)), "16 bytes"), (dict(dq=ctypes.c_void_p(4100)), "16 bytes")):
        with pytest.raises(mia_amd.MiaError, match=match):
            bwd(**kw)
    with pytest.raises(mia_amd.MiaError, match="null"):
        lib.mia_relpos_bias(None, P, 3, 3, 2, 1.0, P, None)
    with pytest.raises(mia_amd.MiaError, match="bad arguments"):
        lib.mia_relpos_bias(P, P, 3, 3, 2, 0.0, P, None)


def test_wrapper_refuses():
    plan = RelativePositionBuckets(3, 3, 4, 8, device="cpu")
    q, k = torch.zeros(2, 4, 3, 16), torch.zeros(2, 9, 3, 16)
    table = torch.zeros(16, 3)
    for kw, err, match in (
            (dict(), RuntimeError, "no CPU path"),
            (dict(q=q.bfloat16()), TypeError, "all fp32 or all bf16"),
            (dict(q=q[0]), ValueError, "must be"),
            (dict(v=k[:, :8]), ValueError, "belong together"),
            (dict(q=q[:, :, :2]), ValueError, "belong together"),
            (dict(q_start=6), ValueError, "do not fit"),
            (dict(q_start=-1), ValueError, "do not fit"),
            (dict(table=torch.zeros(16, 2)), ValueError, "table must be"),
            (dict(table=table.double()), ValueError, "table must be"),
            (dict(key_mask=torch.ones(2, 8).bool()), ValueError, "key_mask"),
            (dict(key_mask=torch.ones(2, 9)), ValueError, "key_mask"),
            (dict(scale=0.0), ValueError, "scale"), (dict(scale=float("nan")), ValueError, "scale"),
            (dict(dropout_p=1.0), ValueError, "dropout")):
        args = dict(q=q, k=k, v=k, table=table, buckets=plan)
        args.update(kw)
        with pytest.raises(err, match=match):
            relpos_attention(**args)
    with pytest.raises(ValueError, match="multiple of 8"):
        relpos_attention(torch.zeros(1, 2, 1, 12), torch.zeros(1, 2, 1, 12), torch.zeros(1, 2, 1, 12), torch.zeros(16, 1), plan)
    with pytest.raises(ValueError, match="must be"):
        relpos_self_attention(torch.zeros(2, 4, 3, 16), table, plan)
    with pytest.raises(RuntimeError, match="no CPU path"):
        relpos_self_attention(torch.zeros(2, 4, 3, 3, 16), table, plan)


def test_every_layout_of_the_kernels_is_tested():
    from relpos_variants import BF16, F32, FORWARD, KEYS, QUERIES, VARIANTS, layout
    seen = set()
    for problem, want in VARIANTS.items():
        dtype, B, heads, Lq, Lk, D, height, width, q_start = problem
        assert Lk <= height * width and q_start + Lq <= height * width
        assert {direction: layout(direction, *problem[:6]) for direction in want} == want, problem
        seen |= {(direction, dtype, *want[direction]) for direction in want}
    both = (False, True)
    assert seen >= {(d, BF16, cols, split, 0) for d in (FORWARD, QUERIES, KEYS) for cols in (1, 2) for split in both}
    assert seen >= {(d, F32, 1, split, 0) for d in (FORWARD, QUERIES, KEYS) for split in both}
    assert seen >= {(FORWARD, BF16, 0, split, few) for split in both for few in (1, 2)} | {(FORWARD, F32, 0, split, few) for split in both for few in (1, 4)}


def test_plan_entry_refuses():
    lib, plan = mia_amd.lib(), (ctypes.c_int * 3)()
    for args in ((3, 0, 1, 1, 5, 5, 16, plan), (-1, 0, 1, 1, 5, 5, 16, plan), (0, 2, 1, 1, 5, 5, 16, plan), (0, 0, 1, 1, 5, 5, 16, None)):
        with pytest.raises(mia_amd.MiaError, match="bad arguments"):
            lib.mia_relpos_plan(*args)
    for args in ((0, 5, 5, 16), (1, 0, 5, 16), (1, 5, 0, 16), (1, 5, 5, 12), (1, 5, 5, 136)):
        with pytest.raises(mia_amd.MiaError, match="bad shape"):
            lib.mia_relpos_plan(0, 0, 1, *args, plan)


@pytest.mark.parametrize("dtype,B,heads,height,width,D", [(1, 1, 4, 75, 75, 32), (0, 1, 4, 75, 75, 32), (1, 1, 4, 38, 38, 64), (1, 4, 8, 38, 38, 64), (0, 1, 2, 128, 128, 64),
                                                          (1, 1, 4, 1, 4096, 64), (1, 128, 8, 10, 10, 48), (0, 1, 1, 700, 2, 16)])
def test_workspace_of_the_bias_gradient(dtype, B, heads, height, width, D):
    """A key block keeps room for the offsets that its queries reach, not once more for every range that its walk is split into:
    what the ranges add is their ends alone."""
    lib, plan, L = mia_amd.lib(), (ctypes.c_int * 3)(), height * width
    lib.mia_relpos_plan(2, dtype, B, heads, L, L, D, plan)
    cols, splits = plan[0], plan[1]
    span = lambda n: n - 1 + (-(-(n - 1) // width) * (width - 1) if height > 1 else 0)     # noqa: E731  (offsets between n tokens)
    blocks = -(-L // (64 * cols))
    rows = blocks * (span(L) + splits * (span(128) + span(64 * cols) + 2))
    n_off = (2 * height - 1) * (2 * width - 1)
    want = lambda table: lib.mia_relpos_bwd_ws_floats(dtype, B, heads, L, L, D, height, width, table)      # noqa: E731
    assert want(1) - want(0) <= heads * n_off + B * heads * rows + 4

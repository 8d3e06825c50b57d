"""Global gradient norm and clipping on the gfx950 kernels against the formula in float64.

Tolerances: the norm is a sum of squares in double, rounded once to fp32 (2^-24 relative) after a double square root; the
oracle's float64 sum differs by far less. A scaled gradient is one fp32 product with a factor that is itself rounded to fp32
(2 * 2^-24), and for bf16 one more rounding (2^-8)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import mia_amd  # noqa: E402,F401
from mia_amd.optim import AdamW, clip_grad_norm_, clip_grads_, grad_norm  # noqa: E402

F32, BF16 = torch.float32, torch.bfloat16


def _grads(sizes, dtypes, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale).to(dt).cuda() for n, dt in zip(sizes, dtypes)]


def _norm64(grads):
    return math.sqrt(sum(float(g.double().cpu().square().sum()) for g in grads))


def _check(grads, max_norm):
    before = [g.double().cpu() for g in grads]
    want = math.sqrt(sum(float(b.square().sum()) for b in before))
    got = clip_grads_(grads, max_norm)
    assert got.shape == () and got.dtype == F32
    assert abs(float(got) - want) <= 2.0 ** -23 * want
    factor = min(1.0, max_norm / (want + 1e-6))
    for g, b in zip(grads, before):
        tol = 3 * 2.0 ** -24 + (2.0 ** -8 if g.dtype == BF16 else 0.0)
        # the smallest bf16 / fp32 subnormal step is far below these values
        assert torch.all((g.double().cpu() - b * factor).abs() <= tol * (b * factor).abs() + 1e-40)


@pytest.mark.parametrize("sizes", [[1], [3], [0, 5, 0], [8191, 8192, 8193], [1, 2, 3, 4, 5, 6, 7, 8, 9, 63, 64, 65], [100003],
                                   [7] * 523, [3_000_001, 17, 1]])
@pytest.mark.parametrize("kind", ["fp32", "bf16", "mixed"])
def test_clip_matches_formula(sizes, kind):
    dtypes = [F32 if kind == "fp32" or (kind == "mixed" and i % 2) else BF16 for i in range(len(sizes))]
    _check(_grads(sizes, dtypes, 1), 0.37)
    _check(_grads(sizes, dtypes, 2, scale=1e-9), 0.37)     # below the limit: untouched


def test_untouched_when_below_the_limit_is_bitwise():
    g = _grads([1000, 37], [F32, BF16], 3, scale=1e-3)
    b = [t.clone() for t in g]
    clip_grads_(g, 10.0)
    assert all(torch.equal(x, y) for x, y in zip(g, b))


@pytest.mark.parametrize("offset", range(8))
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views_of_one_buffer_with_any_alignment(offset, dtype):
    """Views into an exchange buffer start anywhere, and the elements around them stay as they are."""
    flat = torch.randn(50_000, generator=torch.Generator().manual_seed(4)).to(dtype).cuda()
    keep = flat.clone()
    views = [flat[offset:offset + 1], flat[offset + 3:offset + 20_000], flat[offset + 20_001:offset + 20_007], flat[offset + 21_000:offset + 49_001]]
    _check(views, 2.0)
    inside = torch.zeros_like(flat, dtype=torch.bool)
    for a, b in ((0, 1), (3, 20_000), (20_001, 20_007), (21_000, 49_001)):
        inside[offset + a:offset + b] = True
    assert torch.equal(flat[~inside], keep[~inside]) and not torch.equal(flat[inside], keep[inside])


def test_squares_outside_fp32():
    """Squares of 1e30 overflow fp32 and those of 1e-30 vanish in it; the norm does neither."""
    for scale in (1e30, 1e-30):
        g = _grads([5000, 11], [F32, BF16], 5, scale=scale)
        want = _norm64(g)
        assert abs(float(grad_norm(g)) - want) <= 2.0 ** -23 * want
    g = _grads([5000], [F32], 6, scale=1e30)
    _check(g, 1.0)


def test_not_finite():
    g = _grads([100, 100], [F32, F32], 7)
    g[0][3] = float("inf")
    n = clip_grads_(g, 1.0)
    assert math.isinf(float(n))
    assert torch.isnan(g[0][3]) and int((g[1] != 0).sum()) == 0      # factor 0, and 0 * inf, as torch's clipping leaves them
    g = _grads([100, 100], [F32, BF16], 8)
    g[1][99] = float("nan")
    assert math.isnan(float(clip_grads_(g, 1.0))) and bool(torch.isnan(g[0]).all())


def test_layouts_and_duplicates():
    x = torch.randn(2, 3, 4, 5, device="cuda").to(memory_format=torch.channels_last)
    _check([x, torch.randn(6, 4, device="cuda").t()], 0.5)
    with pytest.raises(ValueError, match="twice"):
        clip_grads_([x, x], 1.0)
    with pytest.raises(TypeError, match="fp32 or bf16"):
        clip_grads_([x.half()], 1.0)
    with pytest.raises(RuntimeError, match="one MI355X device"):
        clip_grads_([x, torch.zeros(3)], 1.0)
    s = torch.randn(4, 6, device="cuda")[:, ::2]
    assert abs(float(grad_norm([s])) - _norm64([s])) <= 2.0 ** -23 * _norm64([s])


def test_same_bits_every_time():
    a, b = _grads([1_000_003, 5, 77], [F32, BF16, F32], 9), _grads([1_000_003, 5, 77], [F32, BF16, F32], 9)
    assert torch.equal(clip_grads_(a, 1.0), clip_grads_(b, 1.0)) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_two_streams_and_a_captured_call():
    """Calls on two streams have workspaces of their own; a captured call follows new gradients at every replay."""
    lists = [_grads([400_000, 33], [F32, F32], s) for s in (10, 11)]
    want = [_norm64(g) for g in lists]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for g, s in zip(lists, streams):
        with torch.cuda.stream(s):
            got.append(clip_grads_(g, 1.0))
    torch.cuda.synchronize()
    assert all(abs(float(n) - w) <= 2.0 ** -23 * w for n, w in zip(got, want))
    static = _grads([70_001, 3], [F32, BF16], 12)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grads_(static, 0.5)
    for seed in range(13, 17):
        new = _grads([70_001, 3], [F32, BF16], seed)
        for s, n in zip(static, new):
            s.copy_(n)
        graph.replay()
        eager = clip_grads_(new, 0.5)
        torch.cuda.synchronize()
        assert torch.equal(norm, eager) and all(torch.equal(s, n) for s, n in zip(static, new))


def _params(seed, sizes=(700, 33, 5000)):
    g = torch.Generator().manual_seed(seed)
    ps = [torch.nn.Parameter(torch.randn(n, generator=g).cuda()) for n in sizes]
    for p in ps:
        p.grad = torch.randn(p.shape, generator=g).cuda()
    return ps


def test_clip_grad_norm_takes_parameters():
    ps = _params(20) + [torch.nn.Parameter(torch.zeros(3, device="cuda"))]
    want = _norm64([p.grad for p in ps[:3]])
    assert abs(float(clip_grad_norm_(ps, 1.0)) - want) <= 2.0 ** -23 * want
    after = _norm64([p.grad for p in ps[:3]])
    assert abs(after - want / (want + 1e-6)) < 1e-6
    assert clip_grad_norm_(ps[0], 100.0).shape == ()


@pytest.mark.parametrize("grad_scale", [1.0, 0.25])
def test_adamw_with_clipping_equals_clip_then_step(grad_scale):
    """One update from gradients clipped on the fly against clipping them first: the factor reaches the update as one fp32
    number in both, so the difference is one rounding of the gradient; two groups count towards one norm."""
    a, b = _params(21), _params(21)
    keep = [p.grad.clone() for p in a]
    oa = AdamW([{"params": a[:1]}, {"params": a[1:], "lr": 3e-3}], max_grad_norm=0.7)
    ob = AdamW([{"params": b[:1]}, {"params": b[1:], "lr": 3e-3}])
    for step in range(3):
        oa.step(grad_scale=grad_scale)
        saved = [p.grad.clone() for p in b]
        for p in b:
            p.grad.mul_(grad_scale)
        n = clip_grad_norm_(b, 0.7)
        ob.step()
        for p, s in zip(b, saved):
            p.grad.copy_(s)
        assert abs(float(oa.grad_norm) - float(n)) <= 2.0 ** -22 * float(n)
        for x, y in zip(a, b):
            # an update is at most ~lr large and its relative error a few fp32 roundings
            assert (x - y).abs().max() <= 3e-3 * 1e-5 + 2.0 ** -23 * y.abs().max()
            assert (oa.state[x]["exp_avg"] - ob.state[y]["exp_avg"]).abs().max() <= 1e-6 * ob.state[y]["exp_avg"].abs().max()
    assert all(torch.equal(p.grad, k) for p, k in zip(a, keep))      # the gradients are only read


def test_adamw_below_the_limit_is_the_plain_step():
    a, b = _params(22), _params(22)
    AdamW(a, max_grad_norm=1e9).step()
    AdamW(b).step()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_captured_training_step_with_clipping():
    """GraphedTrainStep over an optimizer that clips follows the eager trajectory bit for bit."""
    import copy
    from mia_amd.graphs import GraphedTrainStep
    from mia_amd.head_ops import CrossEntropyLoss
    from mia_amd.src.model import FoundationModel
    torch.manual_seed(0)
    model = FoundationModel(backbone="efficientnet_b3", pretrained=False, dropout=0.2, classification_heads={"d": 4}).cuda().train()
    for m in model.modules():
        if isinstance(m, torch.nn.Dropout):
            m.p = 0.0
    other = copy.deepcopy(model)
    xs = [torch.randn(4, 3, 64, 64, device="cuda") for _ in range(3)]
    ys = [torch.randint(0, 4, (4,), device="cuda") for _ in range(3)]
    crit = CrossEntropyLoss()
    opt_e = AdamW(model.parameters(), lr=1e-3, max_grad_norm=0.5)
    opt_g = AdamW(other.parameters(), lr=1e-3, max_grad_norm=0.5)
    step = GraphedTrainStep(other, "classification", "d", crit, opt_g, xs[0], ys[0])
    for x, y in zip(xs, ys):
        opt_e.zero_grad(set_to_none=True)
        loss = crit(model(x, "classification", "d"), y)
        loss.backward()
        opt_e.step()
        got = step(x, y)
        torch.cuda.synchronize()
        assert torch.equal(got, loss) and torch.equal(opt_e.grad_norm, opt_g.grad_norm) and float(opt_e.grad_norm) > 0.5
        for p, q in zip(model.parameters(), other.parameters()):
            assert torch.equal(p, q)


@pytest.mark.parametrize("max_grad_norm", [None, 0.5])
def test_adamw_without_the_autograd_module(monkeypatch, max_grad_norm):
    """The optimizer's own check of its parameters: the same steps, and a transposed gradient made contiguous."""
    import mia_amd._lib as _lib
    from mia_amd import _proto, optim
    a, b = _params(24, (70, 4000)), _params(24, (70, 4000))
    for ps in (a, b):
        ps.append(torch.nn.Parameter(torch.ones(6, 5, device="cuda")))
        ps[-1].grad = torch.arange(30.0, device="cuda").view(5, 6).t()
    first, second = AdamW(a, max_grad_norm=max_grad_norm), AdamW(b, max_grad_norm=max_grad_norm)
    first.step()
    monkeypatch.setattr(_lib, "_nodes", None)
    monkeypatch.setattr(_proto, "autograd_digest", lambda: "another")
    monkeypatch.setattr(optim, "_update_check", None)
    second.step()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def _rank(rank, port, q):
    try:
        import copy
        import faulthandler
        import os
        import torch.distributed as dist
        faulthandler.dump_traceback_later(100, exit=True)
        os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
        dist.init_process_group("gloo", rank=rank, world_size=2)
        from mia_amd.ddp import GradReducer
        torch.manual_seed(3)
        net = torch.nn.Sequential(torch.nn.Linear(20, 30), torch.nn.Tanh(), torch.nn.Linear(30, 5))
        data = [torch.randn(8, 20) * (1 + 3 * r) for r in range(2)]
        ref = copy.deepcopy(net).double()
        (0.5 * sum(ref(x.double()).square().sum() for x in data)).backward()      # the mean of the ranks' gradients
        want = math.sqrt(sum(float(p.grad.square().sum()) for p in ref.parameters()))
        own = copy.deepcopy(net).double()
        own(data[rank].double()).square().sum().backward()
        alone = math.sqrt(sum(float(p.grad.square().sum()) for p in own.parameters()))
        net.cuda()
        red = GradReducer(net.parameters(), bucket_bytes=1 << 10)
        opt = AdamW(net.parameters(), lr=1e-3, max_grad_norm=0.5)
        red.zero_grad()
        net(data[rank].cuda()).square().sum().backward()
        red.finish()
        opt.step()
        inside = float(opt.grad_norm)
        got = float(clip_grad_norm_(net.parameters(), 0.5))
        after = _norm64([p.grad for p in net.parameters()])
        dist.destroy_process_group()
        q.put((rank, want, alone, inside, got, after, [p.detach().cpu().numpy() for p in net.parameters()]))
    except Exception:
        import traceback
        q.put((rank, traceback.format_exc()[-1500:]))


def test_norm_of_exchanged_gradients():
    """Behind GradReducer the norm is that of the averaged gradients, the same on both ranks, and so is the step. (fp32 gradients of two
    small layers: a few sums of at most 30 terms, 100 * 2^-24 of the norm.)"""
    import socket
    import torch.multiprocessing as mp
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    ranks = [ctx.Process(target=_rank, args=(r, port, q)) for r in range(2)]
    for p in ranks:
        p.start()
    try:
        res = sorted((q.get(timeout=110) for _ in ranks), key=lambda r: r[0])
    finally:
        for p in ranks:
            p.join(timeout=20)
            if p.is_alive():
                p.kill()
    assert all(len(r) > 2 for r in res), [r[1] for r in res if len(r) == 2]
    for _, want, alone, inside, got, after, _ in res:
        assert abs(inside - want) <= 100 * 2.0 ** -24 * want and inside == got and abs(alone - want) > 0.1 * want and want > 0.5
        assert abs(after - 0.5 * want / (want + 1e-6)) < 1e-6
    assert res[0][3] == res[1][3] and all((a == b).all() for a, b in zip(res[0][-1], res[1][-1]))


def test_overlapping_gradients_are_refused():
    """Their common elements would be scaled twice, by workgroups that race; neighbours in one buffer are fine."""
    flat = torch.randn(1000, device="cuda")
    keep = flat.clone()
    for a, b in ((flat[:600], flat[599:]), (flat, flat[10:20]), (flat[300:], flat[:301]), (flat.view(10, 100)[2:4], flat[250:260])):
        with pytest.raises(ValueError, match="overlap"):
            clip_grads_([a, torch.zeros(3, device="cuda"), b], 0.1)
    assert torch.equal(flat, keep)
    want = _norm64([flat])
    assert abs(float(clip_grads_([flat[600:], flat[:600], flat[5:5]], 1e9)) - want) <= 2.0 ** -23 * want

"""The new operators together, as the attention head and a training step use them, against plain torch on the CPU in float64.

Bounds: an output or gradient passes through about ten fp32 products of at most 512 terms, each off by at most 512 * 2^-24 =
3e-5 of its largest magnitude: 3e-4 of each tensor's largest magnitude for outputs; gradients pass through twice as many, 1e-3
with the sums over the batch's tokens."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

import mia_amd  # noqa: E402,F401
from mia_amd.graphs import GraphedForward, GraphedTrainStep  # noqa: E402
from mia_amd.head_ops import CrossEntropyLoss  # noqa: E402
from mia_amd.heads import MultiHeadAttentionClassifier  # noqa: E402
from mia_amd.optim import AdamW, clip_grad_norm_  # noqa: E402
from mia_amd.src.model import FoundationModel  # noqa: E402
from position_head import PositionHead  # noqa: E402
from seeding import randn, seeded_state_dict  # noqa: E402


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).abs().max() / b.abs().max().clamp_min(1e-30))


def _pair(C, heads, n, buckets, norm, seed, distance=16):
    ref = PositionHead(C, heads, n, buckets=buckets, distance=distance, norm=norm)
    sd = seeded_state_dict(ref, seed)
    if buckets:
        sd["relative_position_table"] = randn(seed + 1, buckets * buckets, heads)
    if norm:
        sd["residual_scale"] = 1 + 0.3 * randn(seed + 2, C)
    mine = MultiHeadAttentionClassifier(C, heads, n, 0.0, relative_position_buckets=buckets, relative_position_distance=distance, residual_norm=norm)
    assert set(mine.state_dict()) == set(sd)
    ref.load_state_dict(sd)
    mine.load_state_dict(sd)
    return ref.double().train(), mine.cuda().train()


@pytest.mark.parametrize("C,heads,hw,buckets,norm", [
    (384, 8, (10, 10), 16, "rms"), (64, 8, (3, 5), 8, "layer"), (96, 3, (1, 9), 8, None), (64, 1, (5, 1), 0, "rms"), (64, 4, (19, 17), 8, "layer")])
def test_head_and_clipped_step(C, heads, hw, buckets, norm):
    """Forward, backward, gradients clipped to a norm, in one run; the last map has more tokens than the default path takes."""
    ref, mine = _pair(C, heads, 4, buckets, norm, 51)
    x = randn(52, 3, C, *hw)
    xr, xm = x.double().requires_grad_(), x.permute(0, 2, 3, 1).contiguous().cuda().requires_grad_()
    out_r, out_m = ref(xr), mine(xm)
    assert rel(out_m, out_r) < 3e-4
    g = randn(53, *out_r.shape)
    out_r.backward(g.double())
    out_m.backward(g.cuda())
    assert rel(xm.grad.permute(0, 3, 1, 2), xr.grad) < 1e-3
    want = dict(ref.named_parameters())
    for k, p in mine.named_parameters():
        if k == "key.bias" and not buckets:
            assert p.grad.abs().max().item() < 1e-5
        elif k != "key.bias":
            assert rel(p.grad, want[k].grad) < 1e-3, k
    # the key bias has no gradient (a softmax does not see it): both sides hold noise there
    mine.key.bias.grad.zero_()
    ref.key.bias.grad.zero_()
    norm_r = torch.nn.utils.clip_grad_norm_(ref.parameters(), 0.5)
    keep = [p.grad.clone() for p in mine.parameters()]
    opt = AdamW(mine.parameters(), lr=1e-3, max_grad_norm=0.5)
    other = copy.deepcopy(mine)
    for p, grad in zip(other.parameters(), keep):
        p.grad = grad.clone()
    opt_other = AdamW(other.parameters(), lr=1e-3)
    norm_m = clip_grad_norm_(list(other.parameters()), 0.5)
    assert abs(float(norm_m) / float(norm_r) - 1) < 1e-3 and float(norm_r) > 0.5
    for p, q in zip(other.parameters(), ref.parameters()):
        assert rel(p.grad, q.grad) < 2e-3 or float(q.grad.abs().max()) == 0
    opt.step()          # scales inside the update: the gradients stay, the parameters are those of a clipped step
    opt_other.step()
    assert all(torch.equal(p.grad, grad) for p, grad in zip(mine.parameters(), keep))
    assert torch.equal(opt.grad_norm, norm_m)
    for p, q in zip(mine.parameters(), other.parameters()):
        assert rel(p, q) < 1e-6


def test_zero_table_is_the_default_head():
    """A head loaded from a checkpoint without a table starts as it was."""
    torch.manual_seed(3)
    plain = MultiHeadAttentionClassifier(384, 8, 4, 0.0).cuda().eval()
    biased = MultiHeadAttentionClassifier(384, 8, 4, 0.0, relative_position_buckets=16).cuda().eval()
    missing, unexpected = biased.load_state_dict(plain.state_dict(), strict=False)
    assert missing == ["relative_position_table"] and not unexpected
    x = torch.randn(4, 10, 10, 384, device="cuda")
    with torch.no_grad():
        assert rel(biased(x), plain(x)) < 1e-4
        assert rel(biased(x.bfloat16()), plain(x)) < 3e-2


def _model(dtype, dropout):
    torch.manual_seed(0)
    m = FoundationModel(pretrained=False, dropout=dropout, classification_heads={"d": 4}, compute_dtype=dtype, relative_position_buckets=16,
                        residual_norm="rms").cuda().train()
    for mod in m.modules():
        if isinstance(mod, torch.nn.Dropout):
            mod.p = dropout
    return m


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_training_step_captured(dtype):
    """Captured and replayed with eager steps of the same model in between, on three learning rates: bit for bit the eager run."""
    eager = _model(dtype, 0.0)
    graphed = copy.deepcopy(eager)
    crit = CrossEntropyLoss()
    opt_e = AdamW(eager.parameters(), lr=1e-3, max_grad_norm=1.0)
    opt_g = AdamW(graphed.parameters(), lr=1e-3, max_grad_norm=1.0)
    g = torch.Generator(device="cuda").manual_seed(1)
    xs = [torch.randn(4, 3, 96, 96, generator=g, device="cuda") for _ in range(4)]
    ys = [torch.randint(0, 4, (4,), generator=g, device="cuda") for _ in range(4)]
    step = GraphedTrainStep(graphed, "classification", "d", crit, opt_g, xs[0], ys[0])
    for i, (x, y) in enumerate(zip(xs, ys)):
        for opt in (opt_e, opt_g):
            opt.param_groups[0]["lr"] = 1e-3 * (1 + i)
        opt_e.zero_grad(set_to_none=True)
        loss = crit(eager(x, "classification", "d"), y)
        loss.backward()
        opt_e.step()
        assert torch.equal(step(x, y), loss.detach()), i
        torch.cuda.synchronize()
    for (k, p), q in zip(eager.named_parameters(), graphed.parameters()):
        assert torch.equal(p, q), k
    table = eager.classification_layers["d"].relative_position_table
    assert bool(table.any()) and bool(torch.isfinite(table).all())


def test_inference_captured():
    m = _model("bf16", 0.2).eval()
    with torch.no_grad():
        m.classification_layers["d"].relative_position_table.normal_()
    xs = [torch.randn(2, 3, 96, 96, device="cuda") for _ in range(3)]
    g = GraphedForward(m, "classification", "d", xs[0])
    with torch.no_grad():
        for x in xs:
            assert torch.equal(g(x), m(x, "classification", "d"))


def test_dropout_in_the_head():
    m = _model("fp32", 0.3)
    x = torch.randn(2, 3, 96, 96, device="cuda")
    outs = []
    for seed in (1, 1, 2):
        torch.manual_seed(seed)
        outs.append(m(x, "classification", "d").detach())
    assert torch.equal(outs[0], outs[1]) and not torch.equal(outs[0], outs[2])


def test_second_derivatives_are_refused():
    from mia_amd.block_norm import gated_residual_norm
    from mia_amd.relpos import RelativePositionBuckets, relpos_self_attention
    plan = RelativePositionBuckets(2, 3, 8, 16)
    qkv = torch.randn(1, 6, 3, 2, 8, device="cuda", requires_grad=True)
    out = relpos_self_attention(qkv, torch.zeros(64, 2, device="cuda"), plan)
    with pytest.raises(RuntimeError, match="relpos_attention has no second derivative"):
        torch.autograd.grad(out.sum(), qkv, create_graph=True)
    x = torch.randn(3, 16, device="cuda", requires_grad=True)
    _, z = gated_residual_norm(x, x.detach(), pre="rms", pre_weight=torch.ones(16, device="cuda"))
    with pytest.raises(RuntimeError, match="gated_residual_norm has no second derivative"):
        torch.autograd.grad(z.square().sum(), x, create_graph=True)


def test_nothing_is_kept_without_gradients():
    """Parameters that ask for gradients under no_grad: the same results and no more memory than the result itself."""
    from mia_amd.block_norm import gated_residual_norm
    from mia_amd.relpos import RelativePositionBuckets, relpos_self_attention
    plan = RelativePositionBuckets(8, 8, 8, 16)
    qkv = torch.randn(16, 64, 3, 4, 32, device="cuda").bfloat16().requires_grad_()
    table, w = torch.randn(64, 4, device="cuda", requires_grad=True), torch.ones(128, device="cuda", requires_grad=True)
    x = torch.randn(16, 64, 128, device="cuda").bfloat16().requires_grad_()

    def run():
        a = relpos_self_attention(qkv, table, plan)
        return (a, *gated_residual_norm(x, a.view(16, 64, 128), pre="rms", pre_weight=w))
    kept = run()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    with torch.no_grad():
        plain = run()
    assert torch.cuda.memory_allocated() - before == 3 * 16 * 64 * 128 * 2
    assert all(torch.equal(a, b) for a, b in zip(kept, plain)) and not any(t.requires_grad for t in plain)


def _block(dtype):
    from mia_amd.block_norm import gated_residual_norm
    from mia_amd.relpos import RelativePositionBuckets, relpos_attention
    plan = RelativePositionBuckets(5, 7, 8, 16)
    g = torch.Generator().manual_seed(5)
    x = torch.randn(3, 35, 64, generator=g).cuda().to(dtype).requires_grad_()
    table, w, s = (t.cuda().requires_grad_() for t in (torch.randn(64, 4, generator=g), 1 + torch.randn(64, generator=g), torch.randn(64, generator=g)))

    def run(x):
        h = x.view(3, 35, 4, 16)
        a = relpos_attention(h, h * 0.5, h + 1, table, plan)
        y, z = gated_residual_norm(x, a.reshape(3, 35, 64), scale=s, pre="layer", pre_weight=w)
        return y + z
    return run, x, (x, table, w, s)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_inside_checkpoints_and_hooks(dtype):
    """Recomputed in the backward, with saved tensors moved to the host and back, and twice through one graph: the same bits."""
    from torch.utils.checkpoint import checkpoint
    run, x, leaves = _block(dtype)
    dout = torch.randn(3, 35, 64, device="cuda").to(dtype)
    out = run(x)
    want = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(out, leaves, dout)))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out, leaves, dout)
    for reentrant in (False, True):
        for t in leaves:
            t.grad = None
        checkpoint(run, x, use_reentrant=reentrant).backward(dout)
        assert all(torch.equal(a, t.grad) for a, t in zip(want, leaves)), reentrant
    with torch.autograd.graph.save_on_cpu():
        out = run(x)
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(out, leaves, dout)))


def test_inputs_changed_in_between_are_noticed():
    run, x, leaves = _block(torch.float32)
    out = run(x)
    with torch.no_grad():
        leaves[2].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_two_threads_backward():
    """Two backward passes at once, each of its own graph over the same leaves."""
    import threading
    run, x, leaves = _block(torch.bfloat16)
    dout = torch.randn(3, 35, 64, device="cuda").bfloat16()
    want = torch.autograd.grad(run(x), leaves, dout)
    torch.cuda.synchronize()
    got = {}

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(8):
                got[i] = torch.autograd.grad(run(x), leaves, dout)
        torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(a, b) for i in range(2) for a, b in zip(want, got[i]))


def _elsewhere(kind):
    """Saved-tensor hooks that bring the same values back in another layout."""
    def strided(t):
        return torch.stack((t, t), -1)[..., 0]

    def unaligned(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)

    def reversed_dims(t):
        return t.permute(*reversed(range(t.dim()))).contiguous().permute(*reversed(range(t.dim())))
    if kind in ("cpu", "pinned"):
        return torch.autograd.graph.save_on_cpu(pin_memory=kind == "pinned")
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), {"strided": strided, "unaligned": unaligned, "reversed": reversed_dims}[kind])


@pytest.mark.parametrize("kind", ["cpu", "pinned", "strided", "unaligned", "reversed"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_saved_tensors_come_back_in_another_layout(dtype, kind):
    """Views that the kernels read in place (slices of a packed projection, heads first) and every other saved tensor: what a hook
    returns is read as it lies, not as the forward's tensors lay."""
    from mia_amd.block_norm import gated_residual_norm
    from mia_amd.relpos import RelativePositionBuckets, relpos_attention, relpos_self_attention
    plan = RelativePositionBuckets(5, 9, 8, 16)
    g = torch.Generator().manual_seed(31)
    qkv = torch.randn(2, 45, 3, 4, 16, generator=g).to(dtype).cuda().requires_grad_()
    table = torch.randn(64, 4, generator=g).cuda().requires_grad_()
    mask = (torch.rand(2, 45, generator=g) < 0.7).cuda()
    w, s, b = (torch.randn(64, generator=g).cuda().requires_grad_() for _ in range(3))
    gate = torch.rand(2, 64, generator=g).cuda().requires_grad_()
    dout = torch.randn(2, 45, 4, 16, generator=g).to(dtype).cuda()

    def sliced():
        return relpos_attention(*qkv.unbind(2), table, plan, key_mask=mask)

    def heads_first():
        return relpos_attention(*(t.transpose(1, 2).contiguous().transpose(1, 2) for t in qkv.unbind(2)), table, plan, key_mask=mask)

    def packed():
        return relpos_self_attention(qkv, table, plan, key_mask=mask)

    def norm():
        y, z = gated_residual_norm(qkv[:, :, 0].reshape(2, 45, 64), qkv[:, :, 1].reshape(2, 45, 64), scale=s, gate=gate, post="layer", post_weight=w,
                                   post_bias=b, pre="rms", pre_weight=w)
        return (y + z).view(2, 45, 4, 16)
    for run, leaves in ((sliced, (qkv, table)), (heads_first, (qkv, table)), (packed, (qkv, table)), (norm, (qkv, w, s, b, gate))):
        want = torch.autograd.grad(run(), leaves, dout)
        with _elsewhere(kind):
            out = run()
        got = torch.autograd.grad(out, leaves, dout)
        assert all(torch.equal(a, c) for a, c in zip(want, got)), run.__name__


def test_saved_tensors_that_come_back_wrong_are_refused():
    run, x, leaves = _block(torch.float32)
    dout = torch.randn(3, 35, 64, device="cuda")
    for unpack in (lambda t: t.bfloat16(), lambda t: t.cpu(), lambda t: t[:1], lambda t: t.reshape(-1)[:1]):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            out = run(x)
        with pytest.raises(RuntimeError, match="came back from its hooks"):
            torch.autograd.grad(out, leaves, dout)


def test_forward_mode_is_refused():
    """A tangent would be lost; tensors without one are taken inside a dual level."""
    from torch.autograd import forward_ad
    from mia_amd.optim import clip_grads_, grad_norm
    run, x, leaves = _block(torch.float32)
    want = run(x)
    g = torch.randn(10, device="cuda")
    with forward_ad.dual_level():
        assert torch.equal(run(x), want)
        dual = forward_ad.make_dual(x.detach(), torch.ones_like(x))
        for call in (lambda: run(dual), lambda: grad_norm([g, forward_ad.make_dual(g, g)]), lambda: clip_grads_([forward_ad.make_dual(g, g)], 1.0)):
            with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
                call()
    with pytest.raises(RuntimeError):
        torch.func.jvp(run, (x.detach(),), (torch.ones_like(x),))


def test_tracing_is_refused():
    from torch.fx.experimental.proxy_tensor import make_fx
    from mia_amd.block_norm import gated_residual_norm
    from mia_amd.optim import clip_grads_
    from mia_amd.relpos import RelativePositionBuckets, relpos_self_attention
    plan = RelativePositionBuckets(2, 3, 8, 16)
    table, w = torch.zeros(64, 2, device="cuda"), torch.ones(8, device="cuda")
    x = torch.randn(1, 6, 3, 2, 8, device="cuda")
    for function in (lambda t: relpos_self_attention(t, table, plan), lambda t: gated_residual_norm(t, t, pre_weight=w)[1], lambda t: clip_grads_([t], 1.0)):
        for trace in (lambda f: torch.jit.trace(f, (x,), check_trace=False), lambda f: make_fx(f)(x)):
            with pytest.raises(RuntimeError, match="cannot be traced"):
                trace(function)
        assert bool(torch.isfinite(function(x)).all())


def test_plans_built_in_inference_mode_serve_training():
    """A head's first map may come under inference_mode; its plan, also copied and pickled with the head, is then used in training."""
    import io
    torch.manual_seed(4)
    head = MultiHeadAttentionClassifier(64, 4, 3, 0.0, relative_position_buckets=8, residual_norm="rms").cuda()
    with torch.no_grad():
        head.relative_position_table.normal_()
    x = torch.randn(2, 5, 6, 64, device="cuda")
    with torch.inference_mode():
        want = head.eval()(x)
    buffer = io.BytesIO()
    torch.save(head, buffer)
    buffer.seek(0)
    grads = []
    for other in (head, copy.deepcopy(head), torch.load(buffer, weights_only=False)):
        assert torch.equal(other.eval()(x), want)
        loss = other.train()(x).square().sum()
        grads.append(torch.autograd.grad(loss, list(other.parameters()), allow_unused=True))
    for g in grads[1:]:
        assert all((a is None and b is None) or torch.equal(a, b) for a, b in zip(grads[0], g))
    assert all(g is not None for g in grads[0])

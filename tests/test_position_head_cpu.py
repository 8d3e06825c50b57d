"""The attention head's optional position bias and residual norm: what they add to a model, and what they refuse."""
import pytest

import mia_amd  # noqa: F401
from mia_amd.heads import MultiHeadAttentionClassifier
from mia_amd.src.model import FoundationModel, create_foundation_model

NEW = ["relative_position_table", "residual_norm_bias", "residual_norm_weight", "residual_scale"]


def _keys(head):
    return [k for k in head.state_dict() if not k.startswith(("cbam", "classifier", "query", "key", "value", "output_projection"))]


def test_state_dict_keys():
    assert _keys(MultiHeadAttentionClassifier(64, 8, 2)) == []
    assert _keys(MultiHeadAttentionClassifier(64, 8, 2, relative_position_buckets=8)) == NEW[:1]
    assert sorted(_keys(MultiHeadAttentionClassifier(64, 8, 2, residual_norm="rms"))) == NEW[2:]
    full = MultiHeadAttentionClassifier(64, 8, 2, relative_position_buckets=8, residual_norm="layer")
    assert sorted(_keys(full)) == NEW
    assert full.relative_position_table.shape == (64, 8) and not full.relative_position_table.any()
    assert bool((full.residual_scale == 1).all())


@pytest.mark.parametrize("kw,match", [
    (dict(relative_position_buckets=6), "multiple of 4"), (dict(relative_position_buckets=2), "multiple of 4"),
    (dict(relative_position_buckets=16, relative_position_distance=4), "beyond its quarter"), (dict(residual_norm="batch"), "residual_norm")])
def test_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        MultiHeadAttentionClassifier(64, 8, 2, **kw)


def test_head_width_is_refused_only_with_the_bias():
    MultiHeadAttentionClassifier(60, 5, 2)
    with pytest.raises(ValueError, match="multiple of 8"):
        MultiHeadAttentionClassifier(60, 5, 2, relative_position_buckets=8)


def test_model_options():
    kw = dict(pretrained=False, classification_heads={"a": 2})
    m = FoundationModel(relative_position_buckets=8, residual_norm="rms", **kw)
    m.add_classification_head("b", 3)
    for name in "ab":
        assert sorted(_keys(m.classification_layers[name])) == [NEW[0], *NEW[2:]]
    assert _keys(FoundationModel(**kw).classification_layers["a"]) == []
    with pytest.raises(ValueError, match="use_attention"):
        FoundationModel(use_attention=False, residual_norm="rms", **kw)
    config = {"model": {"backbone": "efficientnet_b3", "pretrained": False, "dropout": 0.2, "relative_position_buckets": 16, "residual_norm": "layer"},
              "classification_datasets": [{"name": "a", "classes": ["x", "y"]}]}
    m = create_foundation_model(config)
    assert sorted(_keys(m.classification_layers["a"])) == NEW
    assert m.classification_layers["a"].relative_position_table.shape == (256, 8)
    del config["model"]["relative_position_buckets"], config["model"]["residual_norm"]
    assert _keys(create_foundation_model(config).classification_layers["a"]) == []


def test_nodes_are_those_of_this_tree(monkeypatch):
    """The C++ module that makes the operators' calls was compiled against this header and this torch, or is refused."""
    import mia_amd._lib as _lib
    from mia_amd import _proto
    assert _lib.nodes().digest() == _proto.autograd_digest()
    monkeypatch.setattr(_lib, "_nodes", None)
    monkeypatch.setattr(_proto, "autograd_digest", lambda: "another")
    with pytest.raises(ImportError, match="another header or another torch"):
        _lib.nodes()


@pytest.mark.parametrize("height,width", [(1, 5), (4, 1), (3, 7), (12, 2)])
def test_plan_of_a_map(height, width):
    """One table serves maps of every size, a single row among them; the buckets are those of a loop over the pairs."""
    import torch
    from position_head import PositionHead
    head = MultiHeadAttentionClassifier(64, 8, 2, relative_position_buckets=8, relative_position_distance=9)
    ref = PositionHead(64, 8, 2, buckets=8, distance=9)
    with torch.no_grad():
        ref.relative_position_table.copy_(torch.arange(64 * 8, dtype=torch.float32).reshape(64, 8))
    plan = head.position_plan(height, width, "cpu")
    assert plan is head.position_plan(height, width, "cpu") and plan.num_buckets == 64
    from relpos_formula import offsets
    n = height * width
    bucket = plan.index.long()[offsets(height, width, n, n, 0)]
    assert torch.equal(ref.relative_position_table[bucket].permute(2, 0, 1), ref.bias(height, width))


def _node_calls(shape=(1, 4, 2, 8)):
    """The operators' C++ entry points on host tensors, past the wrappers' checks: what is refused is refused before any work. Each call
    takes the tensor that stands in its first place; `others` are its further differentiable places."""
    import torch
    from mia_amd._lib import nodes
    t, index = torch.zeros(shape), torch.zeros(7, dtype=torch.int32)
    table, w = torch.zeros(3, 2), torch.ones(8)
    attend = lambda q=t, k=t, v=t, tab=table: nodes().relpos(q, k, v, tab, index, index, index, None, 1, 4, 3, 0.35, 0, 0.0, 0, 0)     # noqa: E731
    norm = lambda x=t, f=t, s=None, w2=w: nodes().residual(x, f, s, None, None, None, w2, None, 0, 1, 1e-6)        # noqa: E731
    return [(attend, "q", t), (attend, "k", t), (attend, "v", t), (attend, "tab", table), (norm, "x", t), (norm, "f", t), (norm, "s", w), (norm, "w2", w),
            (lambda g=t: nodes().grad_norm([g]), "g", t), (lambda g=t: nodes().grad_clip([g], 1.0), "g", t)]


@pytest.mark.parametrize("which", range(10))
def test_forward_mode_is_refused(which):
    import torch
    from torch.autograd import forward_ad
    call, place, t = _node_calls()[which]
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
            call(**{place: forward_ad.make_dual(t, torch.ones_like(t))})


@pytest.mark.parametrize("which", [0, 4, 8, 9])
def test_tracing_is_refused(which):
    """A traced program would hold the allocation of the results and none of the kernels."""
    import torch
    from torch.fx.experimental.proxy_tensor import make_fx
    call, place, t = _node_calls()[which]

    def function(x):
        out = call(**{place: x})
        return out[0] if isinstance(out, tuple) else out
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(function, (t,), check_trace=False)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(function)(t)


def test_another_torch_makes_the_module_stale(monkeypatch):
    """The build that an ImportError asks for compiles the module where its digest is another one, though no file is newer."""
    import importlib.util
    import os
    import torch
    spec = importlib.util.spec_from_file_location("mia_build_again", os.path.join(os.path.dirname(mia_amd.__file__), "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    made = []
    monkeypatch.setattr(build.subprocess, "check_call", lambda cmd, *a, **k: made.append(cmd))
    monkeypatch.setattr(build.os.path, "getmtime", lambda path: 0.0)
    assert build.build_autograd(verbose=False) == build.autograd_module_path() and not made
    monkeypatch.setattr(torch, "__version__", torch.__version__ + ".another")
    build.build_autograd(verbose=False)
    assert len(made) == 1 and build.autograd_module_path() in made[0]

"""Refusals of the gradient norm / clipping entry points that need no GPU, and the host-side layout checks."""
import ctypes

import pytest
import torch

import mia_amd
from mia_amd import optim


def _table(sizes, null=()):
    n = len(sizes)
    ptrs = (ctypes.c_void_p * n)(*[None if i in null else 4096 * (i + 1) for i in range(n)])
    return n, ptrs, (ctypes.c_longlong * n)(*sizes)


def test_entry_points_refuse_bad_tables():
    lib = mia_amd.lib()
    n, ptrs, sizes = _table([10, 20])
    need = lib.mia_grad_norm_ws_doubles(n, sizes)
    assert need >= 2
    some = ctypes.c_void_p(4096)
    with pytest.raises(mia_amd.MiaError, match="null workspace"):
        lib.mia_grad_norm(n, ptrs, None, sizes, 1.0, 1.0, None, need, some, None)
    with pytest.raises(mia_amd.MiaError, match="too small"):
        lib.mia_grad_clip(n, ptrs, None, sizes, 1.0, some, need - 1, some, None)
    with pytest.raises(mia_amd.MiaError, match="max_norm"):
        lib.mia_grad_norm(n, ptrs, None, sizes, 1.0, -1.0, some, need, some, None)
    with pytest.raises(mia_amd.MiaError, match="bad dtype"):
        lib.mia_grad_norm(n, ptrs, (ctypes.c_int * 2)(0, 7), sizes, 1.0, 1.0, some, need, some, None)
    n, ptrs, sizes = _table([10, 20], null=(1,))
    with pytest.raises(mia_amd.MiaError, match="null pointer"):
        lib.mia_grad_norm(n, ptrs, None, sizes, 1.0, 1.0, some, need, some, None)
    n, ptrs, sizes = _table([10, -1])
    with pytest.raises(mia_amd.MiaError, match="negative size"):
        lib.mia_grad_clip(n, ptrs, None, sizes, 1.0, some, need, some, None)
    with pytest.raises(mia_amd.MiaError, match="aligned"):
        lib.mia_grad_clip(1, (ctypes.c_void_p * 1)(4098), None, (ctypes.c_longlong * 1)(4), 1.0, some, need, some, None)
    n, ptrs, sizes = _table([10])
    with pytest.raises(mia_amd.MiaError, match="norm_and_factor"):
        lib.mia_adamw_step_clipped(n, ptrs, ptrs, ptrs, ptrs, sizes, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 1.0, None, None, None)


def test_workspace_grows_with_entries():
    lib = mia_amd.lib()
    one = lib.mia_grad_norm_ws_doubles(1, (ctypes.c_longlong * 1)(5))
    many = lib.mia_grad_norm_ws_doubles(1000, (ctypes.c_longlong * 1000)(*[5] * 1000))
    long = lib.mia_grad_norm_ws_doubles(1, (ctypes.c_longlong * 1)(300 << 30))
    assert lib.mia_grad_norm_ws_doubles(0, None) >= 1 and many > one and long > one


def test_host_wrappers_refuse():
    with pytest.raises(RuntimeError, match="no CPU path"):
        optim.grad_norm([torch.zeros(4)])
    with pytest.raises(RuntimeError, match="no CPU path"):
        optim.clip_grads_([torch.zeros(4)], 1.0)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            optim.clip_grads_([torch.zeros(4)], bad)
        with pytest.raises(ValueError, match="max_norm"):
            optim.AdamW([torch.nn.Parameter(torch.zeros(2))], max_grad_norm=bad)
    with pytest.raises(ValueError, match="dense"):
        optim.clip_grads_([torch.zeros(4, 6)[:, ::2]], 1.0)
    assert float(optim.clip_grads_([], 1.0)) == 0 and float(optim.grad_norm([])) == 0


def test_dense_layouts():
    t = torch.zeros(2, 3, 4, 5)
    assert optim._dense(t) and optim._dense(t.to(memory_format=torch.channels_last)) and optim._dense(t.permute(3, 1, 0, 2))
    assert optim._dense(t[:, :1, :1, :1].contiguous()) and optim._dense(torch.zeros(())) and optim._dense(t[1:])
    assert not optim._dense(t[:, 1:]) and not optim._dense(t[..., ::2]) and not optim._dense(torch.zeros(3, 1).expand(3, 4))


@pytest.fixture
def without_the_module(monkeypatch):
    """As where _mia_autograd is missing or was built against another torch."""
    import mia_amd._lib as _lib
    from mia_amd import _proto
    monkeypatch.setattr(_lib, "_nodes", None)
    monkeypatch.setattr(_proto, "autograd_digest", lambda: "another")
    monkeypatch.setattr(optim, "_update_check", None, raising=False)


def test_adamw_does_not_need_the_autograd_module(without_the_module):
    """A step gets as far as the check of its parameters; the clipping functions say what is missing."""
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.ones(4)
    for kw in ({}, {"max_grad_norm": 1.0}):
        for _ in range(2):
            with pytest.raises(RuntimeError, match="contiguous fp32 parameters on an MI355X device"):
                optim.AdamW([p], **kw).step()
    with pytest.raises(ImportError, match="another header or another torch"):
        optim.clip_grad_norm_([p], 1.0)

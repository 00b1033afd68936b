"""Argument checks of fused.add_rmsnorm and add_rmsnorm_quant (no GPU: every
error is raised before a launch)."""

from __future__ import annotations

import pytest
import torch

from kda import _lib, fused


@pytest.mark.parametrize("call", [fused.add_rmsnorm, fused.add_rmsnorm_quant])
def test_argument_checks(call):
    x = torch.zeros(3, 64)
    with pytest.raises(ValueError):
        call(torch.zeros(()))
    with pytest.raises(ValueError):
        call(torch.zeros(3, 0))
    with pytest.raises(ValueError):
        call(x, torch.zeros(1, 64))  # no broadcast
    with pytest.raises(TypeError):
        call(x, x.half())
    with pytest.raises(ValueError):
        call(x, x, torch.zeros(3, 64))
    with pytest.raises(TypeError):
        call(x, x, torch.zeros(64, dtype=torch.bfloat16))
    with pytest.raises(TypeError):
        call(x.half(), x.half(), torch.zeros(64, dtype=torch.bfloat16))
    with pytest.raises(TypeError):
        call(torch.zeros(3, 64, dtype=torch.int32))
    for eps in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError):
            call(x, x, None, eps)
    with pytest.raises(RuntimeError, match="GPU"):
        call(x, x)


@pytest.mark.parametrize("call", [fused.add_rmsnorm, fused.add_rmsnorm_quant])
@pytest.mark.parametrize("which", ["x", "residual", "weight"])
def test_a_tangent_is_refused_not_lost(call, which):
    args = {"x": torch.ones(3, 64), "residual": torch.ones(3, 64), "weight": torch.ones(64)}
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            call(**{**args, which: dual})
        with pytest.raises(RuntimeError, match="GPU"):  # a level alone changes nothing
            call(**args)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda t: call(**{**args, which: t})[0], (args[which],), (args[which],))


def test_quant_argument_checks():
    with pytest.raises(TypeError):
        fused.add_rmsnorm_quant(torch.zeros(3, 64, dtype=torch.float64))
    for width, group in ((96, 64), (64, 16), (64, 0), (1024, 512), (64, -32)):
        with pytest.raises((ValueError, RuntimeError)):
            fused.add_rmsnorm_quant(torch.zeros(2, width), group_size=group)


def test_entry_points_reject_bad_arguments():
    lib = _lib.load()
    a, bad = 4096, _lib.KDA_ERR_INVALID_ARGUMENT

    def fwd(x=a, r=a, h=a, y=a, f32=0, rows=4, width=64, eps=1e-6, dtype=2):
        return lib.kda_add_rmsnorm_fwd(x, r, a, f32, h, y, rows, width, eps, dtype, None)

    for kw in (dict(x=None), dict(y=None), dict(h=None), dict(rows=0), dict(width=0), dict(width=-1), dict(eps=0.0),
               dict(dtype=9), dict(dtype=3, f32=1), dict(rows=1 << 40, width=1 << 40)):
        assert fwd(**kw) == bad, kw
    assert fwd(rows=1 << 31) == _lib.KDA_ERR_UNSUPPORTED

    def quant(group, width=192, dtype=2, q=a):
        return lib.kda_add_rmsnorm_quant(a, None, None, 0, None, q, a, group, 4, width, 1e-6, dtype, None)

    for kw in (dict(group=128), dict(group=16), dict(group=0), dict(group=64, dtype=3), dict(group=64, q=None)):
        assert quant(**kw) == bad, kw

    need = lib.kda_add_rmsnorm_bwd_workspace_bytes(100, 64, 2)
    assert need > 0 and lib.kda_add_rmsnorm_bwd_workspace_bytes(0, 64, 2) == 0

    def bwd(ws=a, nbytes=need, dy=a, dw=a):
        return lib.kda_add_rmsnorm_bwd(a, a, 0, dy, None, a, dw, 100, 64, 1e-6, 2, ws, nbytes, None)

    assert bwd(ws=None) == _lib.KDA_ERR_WORKSPACE and bwd(nbytes=need - 1) == _lib.KDA_ERR_WORKSPACE
    assert bwd(ws=a + 4) == bad and bwd(dy=None) == bad


def test_a_weight_gradient_wider_than_its_launch_is_refused():
    # 1024 threads for 64 columns, fewer than 2^32 in a launch
    lib, a, width = _lib.load(), 4096, 1 << 28
    need = lib.kda_add_rmsnorm_bwd_workspace_bytes(1, width, 2)
    assert lib.kda_add_rmsnorm_bwd(a, a, 0, a, None, a, a, 1, width, 1e-6, 2, a, need, None) == _lib.KDA_ERR_UNSUPPORTED

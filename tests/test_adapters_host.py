"""Argument checks of adapters (no GPU: every error is raised before a launch)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from kda import _lib
from kda import adapters
from kda.adapters import AdapterStack, KDALayerAdapters, adapter_linear
from kda.adapters import row_pieces
from kda.layer import KDALayerWeights, kda_attention_forward
from tests._inputs import layer_weights


def _stack(n=2, rank=4, d_in=8, d_out=6, dtype=torch.float32):
    return AdapterStack(torch.zeros(n, rank, d_in, dtype=dtype), torch.zeros(n, d_out, rank, dtype=dtype))


def test_stack_checks():
    z = torch.zeros
    for a, b in ((z(2, 4), z(2, 6, 4)), (z(2, 4, 8), z(3, 6, 4)), (z(2, 4, 8), z(2, 6, 5)), (z(0, 4, 8), z(0, 6, 4)),
                 (z(1, 257, 8), z(1, 6, 257))):
        with pytest.raises(ValueError):
            AdapterStack(a, b)
    with pytest.raises(TypeError):
        AdapterStack(z(2, 4, 8), z(2, 6, 4).half())
    with pytest.raises(TypeError):
        AdapterStack(z(2, 4, 8).double(), z(2, 6, 4).double())
    for scaling in (z(3), z(2).double()):
        with pytest.raises(ValueError):
            AdapterStack(z(2, 4, 8), z(2, 6, 4), scaling)


def test_call_checks():
    x, w, bias, ids = torch.zeros(3, 5, 8), torch.zeros(6, 8), torch.zeros(6), torch.zeros(3, dtype=torch.long)
    call = lambda x=x, w=w, bias=bias, stack=_stack(), ids=ids: adapter_linear(x, w, bias, stack, ids)  # noqa: E731
    for kw in (dict(x=torch.zeros(8)), dict(x=torch.zeros(3, 5, 0)), dict(w=torch.zeros(6, 7)), dict(bias=torch.zeros(5)),
               dict(stack=_stack(d_in=9)), dict(stack=_stack(d_out=7)), dict(ids=ids[:2]), dict(ids=ids[:, None].repeat(1, 4)),
               dict(ids=torch.tensor(0))):
        with pytest.raises(ValueError):
            call(**kw)
    for kw in (dict(x=x.double()), dict(w=w.half()), dict(bias=bias.half()), dict(stack=_stack(dtype=torch.bfloat16)),
               dict(ids=ids.float())):
        with pytest.raises(TypeError):
            call(**kw)
    with pytest.raises(RuntimeError, match="backward"):
        call(w=w.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="backward"):
        stack = _stack()
        stack.a.requires_grad_()
        call(stack=stack)
    with pytest.raises(RuntimeError, match="GPU"):
        call()


@pytest.mark.parametrize("which", ["x", "weight", "bias", "a", "b", "scaling"])
def test_a_tangent_is_refused_not_lost(which):
    t = {"x": torch.ones(3, 8), "weight": torch.ones(6, 8), "bias": torch.ones(6), "a": torch.ones(2, 4, 8),
         "b": torch.ones(2, 6, 4), "scaling": torch.ones(2)}

    def call(**kw):
        t2 = {**t, **kw}
        return adapter_linear(t2["x"], t2["weight"], t2["bias"], AdapterStack(t2["a"], t2["b"], t2["scaling"]),
                              torch.zeros(3, dtype=torch.long))

    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(t[which], torch.ones_like(t[which]))
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            call(**{which: dual})
        with pytest.raises(RuntimeError, match="GPU"):  # a level alone changes nothing
            call()


def test_layer_checks():
    weights = layer_weights(128, 1, 128, 128, dtype=torch.float32)
    w = KDALayerWeights(**weights)
    x = torch.zeros(2, 3, 128)
    with pytest.raises(ValueError, match="together"):
        kda_attention_forward(w, x, adapters=KDALayerAdapters())
    with pytest.raises(ValueError, match="together"):
        kda_attention_forward(w, x, adapter_ids=torch.zeros(2, dtype=torch.long))
    with pytest.raises(ValueError, match="adapter_ids"):
        kda_attention_forward(w, x, adapters=KDALayerAdapters(), adapter_ids=torch.zeros(3, dtype=torch.long))


def test_entry_point_rejects_bad_arguments():
    lib, p = _lib.load(), 4096

    def args(**kw):
        fields = dict(x=p, weight=None, a=p, b=p, bias=None, scaling=None, ids=p, y=p, workspace=p, workspace_bytes=1 << 30, rows=4,
                      span=1, d_in=8, d_out=8, rank=4, adapters=2, dtype=2, ids_are_int64=1)
        return _lib.AdapterArgs(**{**fields, **kw})

    def call(**kw):
        d = args(**kw)
        return lib.kda_adapter_linear(ctypes.addressof(d), None)

    for kw in (dict(x=None), dict(a=None), dict(b=None), dict(ids=None), dict(y=None), dict(rows=0), dict(span=0),
               dict(rows=1 << 31), dict(d_in=0), dict(d_in=1 << 24), dict(d_out=0), dict(rank=0), dict(rank=257),
               dict(adapters=0), dict(dtype=3), dict(workspace=p + 4)):
        assert call(**kw) == _lib.KDA_ERR_INVALID_ARGUMENT, kw
    assert lib.kda_adapter_linear(None, None) == _lib.KDA_ERR_INVALID_ARGUMENT
    d = args()
    need = lib.kda_adapter_linear_workspace_bytes(ctypes.addressof(d))
    assert need > 0
    assert call(workspace=None) == _lib.KDA_ERR_WORKSPACE and call(workspace_bytes=need - 1) == _lib.KDA_ERR_WORKSPACE
    # the product with the weight: for few aligned 16-bit rows
    few = dict(weight=p, d_in=64, rows=20)

    def takes(**kw):
        d = args(**{**few, **kw})  # lives as long as its address is used
        return lib.kda_adapter_linear_takes_weight(ctypes.addressof(d))

    assert takes() == 1 and takes(rows=32) == 1 and takes(dtype=1) == 1 and takes(span=15) == 1
    for kw in (dict(rows=33), dict(dtype=0), dict(span=16), dict(d_in=96), dict(x=p + 8), dict(weight=p + 2), dict(a=p + 4)):
        assert takes(**kw) == 0 and call(**{**few, **kw}) == _lib.KDA_ERR_UNSUPPORTED, kw
    d, plain = args(**few), args(**{**few, "weight": None})
    assert lib.kda_adapter_linear_workspace_bytes(ctypes.addressof(d)) > \
        lib.kda_adapter_linear_workspace_bytes(ctypes.addressof(plain))
    d = args(rank=300)
    assert lib.kda_adapter_linear_workspace_bytes(ctypes.addressof(d)) == 0


@pytest.mark.parametrize("rows,span,most", [(1, 1, 1), (10, 1, 3), (10, 3, 4), (10, 4, 4), (25, 7, 15), (25, 10, 4), (30, 10, 3),
                                            (9, 100, 2), (5, 100, 100), (1 << 33, 1 << 31, 1 << 27), ((1 << 30) + 1, 6, 1 << 28)])
def test_rows_are_taken_in_pieces_of_whole_ids_or_inside_one(rows, span, most):
    at = 0
    for first, n, first_id in row_pieces(rows, span, most):
        assert first == at and 1 <= n <= most
        for m in {0, 1, n // 2, n - 1} if n > 1 else {0}:  # the piece's own rule for row m's id
            assert (first + m) // span == first_id + m // span
        at += n
    assert at == rows


def test_a_launch_never_gets_more_rows_than_it_holds():
    # 512 threads for 32 rows, fewer than 2^32 of them
    lib, p = _lib.load(), 4096
    d = _lib.AdapterArgs(p, None, p, p, None, None, p, p, p, 1 << 30, 1 << 28, 16, 8, 8, 4, 2, 2, 1)
    assert lib.kda_adapter_linear(ctypes.addressof(d), None) == _lib.KDA_ERR_UNSUPPORTED
    assert adapters.PIECE_ROWS < 1 << 28


def test_adding_to_a_product_rejects_bad_arguments():
    lib, p, bad = _lib.load(), 4096, _lib.KDA_ERR_INVALID_ARGUMENT

    def call(product=p, weight=None, rows=40, workspace=p):
        d = _lib.AdapterArgs(p, weight, p, p, None, None, p, p, workspace, 1 << 30, rows, 1, 64, 8, 4, 2, 2, 1)
        return lib.kda_adapter_linear_add(ctypes.addressof(d), product, None)

    assert call(product=None) == bad and call(product=p + 2) == bad and call(rows=0) == bad
    assert call(weight=p, rows=20) == bad and call(weight=p) == _lib.KDA_ERR_UNSUPPORTED
    assert call(workspace=None) == _lib.KDA_ERR_WORKSPACE
    assert lib.kda_adapter_linear_add(None, p, None) == bad

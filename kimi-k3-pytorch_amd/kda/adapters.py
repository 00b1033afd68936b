"""Low-rank adapters of many requests beside a layer's shared projections.

A serving batch shares the weights of a projection, and each request may bring
a low-rank adapter of its own: row m of the batch is

    y_m = W x_m + bias + scaling_a B_a (A_a x_m),   a = its request's adapter,

``[out, rank]`` times ``[rank, in]`` beside the ``[out, in]`` weight.  The
adapters that a server keeps loaded are held stacked (``AdapterStack``), a batch
names one per request (a negative id: none).  ``adapter_linear`` is the
projection with them; ``layer.kda_attention_forward`` takes the stacks of its
projections as ``KDALayerAdapters``.  For serving: there is no derivative, and
tensors that need a gradient or carry a forward-mode tangent are refused.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _lib, _prep

_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
MAX_RANK = 256
# Rows and elements of x or y in one native call: a launch has fewer than 2^32
# threads (2^28 rows), and the library's f32 product takes 2 GiB at most.
PIECE_ROWS, PIECE_ELEMENTS = 1 << 27, 1 << 29


@dataclass(frozen=True)
class AdapterStack:
    """N adapters of one projection: ``a [N, rank, in]``, ``b [N, out, rank]`` and
    the f32 factors ``scaling [N]`` (None: 1).  Adapters of a smaller rank are
    padded with zeros."""

    a: torch.Tensor
    b: torch.Tensor
    scaling: torch.Tensor | None = None

    def __post_init__(self) -> None:
        if self.a.ndim != 3 or self.b.ndim != 3 or 0 in self.a.shape or 0 in self.b.shape:
            raise ValueError("adapters must have shapes a [N,rank,in] and b [N,out,rank]")
        if self.a.shape[0] != self.b.shape[0] or self.a.shape[1] != self.b.shape[2]:
            raise ValueError(f"a {tuple(self.a.shape)} and b {tuple(self.b.shape)} disagree on N or rank")
        if self.a.shape[1] > MAX_RANK:
            raise ValueError(f"adapters of rank up to {MAX_RANK}, got {self.a.shape[1]}")
        if self.a.dtype != self.b.dtype or self.a.dtype not in _DTYPES:
            raise TypeError(f"adapters must share one dtype of float32, float16 or bfloat16, "
                            f"got {self.a.dtype} and {self.b.dtype}")
        if self.a.device != self.b.device:
            raise ValueError("a and b must be on the same device")
        if self.scaling is not None:
            if self.scaling.shape != self.a.shape[:1] or self.scaling.dtype != torch.float32:
                raise ValueError(f"scaling must be float32 of shape {tuple(self.a.shape[:1])}")
            if self.scaling.device != self.a.device:
                raise ValueError("scaling and the adapters must be on the same device")


def _check(x, weight, bias, stack, adapter_ids) -> int:
    """Argument checks; the rows of x per id."""
    if x.ndim < 2 or x.shape[-1] == 0:
        raise ValueError(f"x must have shape [B,...,in], got {tuple(x.shape)}")
    if x.dtype not in _DTYPES:
        raise TypeError(f"unsupported dtype {x.dtype}")
    if weight.ndim != 2 or weight.shape[1] != x.shape[-1] or weight.shape[0] == 0:
        raise ValueError(f"weight must have shape [out,{x.shape[-1]}], got {tuple(weight.shape)}")
    out = weight.shape[0]
    if bias is not None and bias.shape != (out,):
        raise ValueError(f"bias must have shape [{out}], got {tuple(bias.shape)}")
    n, rank, d_in = stack.a.shape
    if d_in != x.shape[-1] or stack.b.shape[1] != out:
        raise ValueError(f"adapters {tuple(stack.a.shape)}, {tuple(stack.b.shape)} do not fit a weight "
                         f"{tuple(weight.shape)}")
    for name, t in (("weight", weight), ("bias", bias), ("the adapters", stack.a)):
        if t is not None and t.dtype != x.dtype:
            raise TypeError(f"{name} must have dtype {x.dtype}, got {t.dtype}")
    if adapter_ids.dtype not in (torch.int32, torch.int64):
        raise TypeError("adapter_ids must be int32 or int64")
    lead = x.shape[:-1]
    if adapter_ids.ndim < 1 or adapter_ids.shape != lead[: adapter_ids.ndim]:
        raise ValueError(f"adapter_ids must have the leading shape of x, {tuple(lead)} or a part of it from the left, "
                         f"got {tuple(adapter_ids.shape)}")
    for name, t in (("weight", weight), ("bias", bias), ("the adapters", stack.a), ("adapter_ids", adapter_ids)):
        if t is not None and t.device != x.device:
            raise ValueError(f"{name} must be on {x.device}, got {t.device}")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in
                                       (x, weight, bias, stack.a, stack.b, stack.scaling)):
        raise RuntimeError("adapter_linear has no backward; call it under torch.no_grad() or on detached tensors")
    _prep.refuse_tangents("adapter_linear", x, weight, bias, stack.a, stack.b, stack.scaling)
    _lib.require_gpu(x)
    return lead[adapter_ids.ndim:].numel()


def _autocast(x, weight, bias, stack):
    """The tensors of a projection in autocast's type (scaling stays f32)."""
    dtype = torch.get_autocast_dtype("cuda")

    def cast(t):
        return t.to(dtype) if t is not None and t.is_cuda and t.dtype in _DTYPES else t

    return cast(x), cast(weight), cast(bias), AdapterStack(cast(stack.a), cast(stack.b), stack.scaling)


def row_pieces(rows: int, span: int, most: int):
    """``(first row, rows, first id)`` of pieces of at most ``most`` rows, each of
    which can be taken by itself with ``span`` rows an id: it begins with an id's first
    row, or lies inside one id's rows."""
    first = 0
    while first < rows:
        if span <= most:
            n = most // span * span
        else:
            n = min(most, span - first % span)
        n = min(n, rows - first)
        yield first, n, first // span
        first += n


def adapter_linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None,
    stack: AdapterStack,
    adapter_ids: torch.Tensor,
) -> torch.Tensor:
    """``x @ weight.T + bias`` plus each row's adapter.

    ``x [B,...,in]``; ``adapter_ids`` (int32 or int64, on the GPU) names the adapter of
    each request, ``[B]``, or of each token, ``[B,T]`` (packed documents):
    ``stack.a[id]`` and ``stack.b[id]``; a negative id has none.  The call does not
    wait for the GPU, so an id past the stack cannot raise: its rows are NaN.
    All sums are in f32 and rounded once.  Under autocast the tensors are taken in its
    type, as torch's linear takes them."""
    if torch.is_autocast_enabled("cuda"):
        x, weight, bias, stack = _autocast(x, weight, bias, stack)
    span = _check(x, weight, bias, stack, adapter_ids)
    d_in, (d_out, rows) = x.shape[-1], (weight.shape[0], x.shape[:-1].numel())
    y = torch.empty(*x.shape[:-1], d_out, dtype=x.dtype, device=x.device)
    if rows == 0:
        return y
    xc, a, b, ids = x.contiguous(), stack.a.contiguous(), stack.b.contiguous(), adapter_ids.contiguous()
    bias = None if bias is None else bias.contiguous()
    scaling = None if stack.scaling is None else stack.scaling.contiguous()
    most = max(1, min(PIECE_ROWS, PIECE_ELEMENTS // max(d_in, d_out)))
    with _prep.on_device(x.device):
        if rows <= most:
            _rows(xc, weight, bias, a, b, scaling, ids, span, y, rows)
        else:
            xc, flat, ids = xc.view(rows, d_in), y.view(rows, d_out), ids.flatten()
            for first, n, first_id in row_pieces(rows, span, most):
                _rows(xc[first:first + n], weight, bias, a, b, scaling, ids[first_id:], span, flat[first:first + n], n)
    return y


def _rows(x, weight, bias, a, b, scaling, ids, span, y, rows) -> None:
    """``y [...,out]`` of ``rows`` rows ``x [...,in]``, on checked, contiguous tensors."""
    lib, (d_out, d_in) = _lib.load(), weight.shape
    args = _lib.AdapterArgs(x.data_ptr(), None, a.data_ptr(), b.data_ptr(), _lib.ptr(bias), _lib.ptr(scaling),
                            ids.data_ptr(), y.data_ptr(), None, 0, rows, span, d_in, d_out, a.shape[1], a.shape[0],
                            _lib.dtype_code(x.dtype), 1 if ids.dtype == torch.int64 else 0)
    ref = ctypes.addressof(args)
    if weight.is_contiguous():
        args.weight = weight.data_ptr()
        if not lib.kda_adapter_linear_takes_weight(ref):
            args.weight = None
    args.workspace_bytes = lib.kda_adapter_linear_workspace_bytes(ref)
    workspace = _prep.workspace(args.workspace_bytes, x.device, "adapter_linear")
    args.workspace = _lib.ptr(workspace)
    if args.weight is not None:
        _lib.check(lib.kda_adapter_linear(ref, _prep.stream(x.device)))
        return
    # many rows: the library's product, in f32 so that the sum is rounded once and an adapter's
    # part past f16's range can meet a product that brings it back.  (8195 rows 2048 -> 2048
    # rank 16: 115 us; a 16-bit sum that the product was added to took 96 us.)
    product = torch.empty(rows, d_out, dtype=torch.float32, device=x.device)
    if x.dtype == torch.float32:
        torch.mm(x.view(rows, d_in), weight.t(), out=product)
    else:
        torch.mm(x.view(rows, d_in), weight.t(), out_dtype=torch.float32, out=product)
    _lib.check(lib.kda_adapter_linear_add(ref, product.data_ptr(), _prep.stream(x.device)))


@dataclass
class KDALayerAdapters:
    """The adapters of a KDA layer's projections (None: the projection has none);
    one id per request picks the same entry of every stack."""

    q_proj: AdapterStack | None = None
    k_proj: AdapterStack | None = None
    v_proj: AdapterStack | None = None
    gate_proj: AdapterStack | None = None
    output_proj: AdapterStack | None = None


_LAYER = ("q_proj", "k_proj", "v_proj", "gate_proj", "output_proj")
STEP_ROWS = 32  # rows whose projections the kernels form themselves


def layer_step_args(w, x: torch.Tensor, stacks: KDALayerAdapters, adapter_ids: torch.Tensor):
    """``kda_layer_adapters`` of a decode step on ``x [B,1,d_model]``, or None where the
    call needs the single projections (more rows, other layouts); raises what
    ``adapter_linear`` raises."""
    rank, count = [0] * 5, [0] * 5
    a, b, scaling = [None] * 5, [None] * 5, [None] * 5
    native = x.shape[0] <= STEP_ROWS and adapter_ids.is_contiguous()
    for j, name in enumerate(_LAYER):
        stack = getattr(stacks, name)
        if stack is None:
            continue
        _check(x, getattr(w, name), getattr(w, name + "_bias" if j in (0, 1, 2) else name[:-5] + "_bias"), stack,
               adapter_ids)
        a[j], b[j] = stack.a.data_ptr(), stack.b.data_ptr()
        if not (stack.a.is_contiguous() and stack.b.is_contiguous()) or (a[j] | b[j]) & 15:
            native = False
        if stack.scaling is not None:
            scaling[j] = stack.scaling.data_ptr()
            native = native and stack.scaling.is_contiguous()
        count[j], rank[j] = stack.a.shape[0], stack.a.shape[1]
    if not native:
        return None
    P, L = ctypes.c_void_p * 5, ctypes.c_int64 * 5
    return _lib.LayerAdapters(P(*a), P(*b), P(*scaling), L(*rank), L(*count), adapter_ids.data_ptr(),
                              1 if adapter_ids.dtype == torch.int64 else 0)


__all__ = ["AdapterStack", "KDALayerAdapters", "adapter_linear"]

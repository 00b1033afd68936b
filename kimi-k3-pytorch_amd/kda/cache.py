"""Cache plumbing for serving: reorder and clone whole decode caches on the GPU.

A serving loop keeps one ``KDAState`` per KDA layer (recurrent state
``[B,H,K,V]``, three ShortConv histories ``[B,K_conv-1,width]`` and int64
``sequence_offset [B]``, src/kda/state.py:12-39).  Beam search reorders the
batch of every layer with the same indices (``HybridBackboneCache.reorder``,
src/hybrid_backbone/cache.py:118-126, one ``index_select`` per tensor per
layer in ``KDAState.reorder``, src/kda/state.py:50-67), and speculative or
branching decoders clone it (src/kda/state.py:41-48).  Here every tensor of
every layer is gathered by ``kda_cache_gather`` (csrc/kda_cache.hip): one
launch per 64 tensors, each selected row read once and written once.

``reorder_states(states, indices)`` and ``clone_states(states)`` take a
sequence of ``KDAState``; ``gather_rows`` is the tensor-level form.  GPU
tensors only: without the HIP library these raise ``RuntimeError``.

Sequences at rest (idle sessions, preempted requests, shared prompts) keep
their states in 8 bits: ``pack_states`` writes the caches of every layer into
slots of a pool (``packed_pool``), ``unpack_states`` reads slots back
(``kda_state_move``, csrc/kda_state_pack.hip: storing launches once per 64 tensors,
reading back as soon as LAUNCH_BYTES of states or 60 tensors are ready), and
``recurrent_kda`` and ``chunkwise_kda`` start straight from a ``PackedState``.
"""

from __future__ import annotations

import ctypes
from array import array
from collections.abc import Sequence

import torch

from . import _lib, _prep
from .state import KDAState, PackedKDAState, PackedState, ShortConvState


def _rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.contiguous()


def gather_rows(tensors: Sequence[torch.Tensor], indices: torch.Tensor | None) -> list[torch.Tensor]:
    """``[t.index_select(0, indices) for t in tensors]`` in one native pass.

    ``indices=None`` copies every tensor (a clone).  All tensors share the
    batch size of dimension 0 and live on one GPU; ``indices`` is a rank-1
    ``torch.long`` tensor on that GPU.  An index outside ``[0, batch)`` raises
    ``IndexError``, as ``index_select`` does.  Like ``index_select`` and
    ``clone`` (src/kda/state.py:41-67) the result is differentiable: the
    gradient of a source row is the sum of the gradients of the rows gathered
    from it.
    """
    tensors = [_rows(t) for t in tensors]
    if not tensors:
        return []
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        return list(_GatherRows.apply(indices, *tensors))
    return _gather(tensors, indices)


def _gather(tensors: list[torch.Tensor], indices: torch.Tensor | None) -> list[torch.Tensor]:
    outs, status = _launch_gather(tensors, indices)
    _check_indices(status, tensors[0].shape[0])
    return outs


# Tensors of the first launch.  The host takes about 2 us per tensor to make the
# outputs, 90 us for the 40 tensors of eight layers, and the call ends with a wait
# for the index check: the GPU starts on the first few (a layer's state among
# them, 40 us of copying at 64 sequences) while the rest are made.
FIRST_LAUNCH = 5


def _launch_gather(tensors: list[torch.Tensor],
                   indices: torch.Tensor | None) -> tuple[list[torch.Tensor], torch.Tensor | None]:
    """The gather's outputs and the status its kernels set for an index out of
    range (None for a copy), to be checked before the outputs are used."""
    device = tensors[0].device
    for t in tensors:
        if not t.is_cuda:
            _lib.require_gpu(t)
        if t.device != device:
            raise ValueError("all cache tensors must be on one device")
        if t.ndim == 0:
            raise ValueError("cache tensors must have a batch dimension")
    n_src = tensors[0].shape[0]
    if any(t.shape[0] != n_src for t in tensors):
        raise ValueError("all cache tensors must share the batch size")
    if indices is not None:
        if indices.ndim != 1 or indices.dtype != torch.long:
            raise ValueError("indices must be a rank-1 torch.long tensor")
        if indices.device != device:
            raise ValueError("indices and state must be on the same device")
        indices = _rows(indices)
    n_out = n_src if indices is None else indices.shape[0]
    if n_src == 0 and n_out > 0:
        raise IndexError("index out of range for an empty cache batch")
    if n_out == 0:
        return [t.new_empty((0, *t.shape[1:])) for t in tensors], None
    lib = _lib.load()
    status = None if indices is None else torch.zeros(1, dtype=torch.int32, device=device)
    stream, outs = _prep.stream(device), []
    for group in (tensors[:FIRST_LAUNCH], tensors[FIRST_LAUNCH:]):
        n = len(group)
        if n == 0:
            break
        new = [t.new_empty((n_out, *t.shape[1:])) for t in group]
        src = (ctypes.c_void_p * n)(*[t.data_ptr() for t in group])
        dst = (ctypes.c_void_p * n)(*[o.data_ptr() for o in new])
        row_bytes = (ctypes.c_int64 * n)(*[t.numel() // n_src * t.element_size() if n_src else 0 for t in group])
        _lib.check(lib.kda_cache_gather(src, dst, row_bytes, n, _lib.ptr(indices), n_src, n_out, _lib.ptr(status),
                                        stream))
        outs += new
    return outs, status


def _check_indices(status: torch.Tensor | None, n_src: int) -> None:
    if status is not None and int(status.item()) != 0:
        raise IndexError(f"index out of range for a cache batch of {n_src}")


class _GatherRows(torch.autograd.Function):
    """The native gather under autograd.  Backward: a clone passes gradients
    through; a reorder adds each output row's gradient into the source row it
    was read from (rows picked several times accumulate)."""

    @staticmethod
    def forward(ctx, indices, *tensors):
        ctx.indices = indices
        ctx.shapes = [t.shape for t in tensors]
        return tuple(_gather(list(tensors), indices))

    @staticmethod
    def backward(ctx, *grads):
        idx = ctx.indices
        out = []
        for shape, gr in zip(ctx.shapes, grads):
            if gr is None or idx is None:
                out.append(gr)
            else:
                out.append(torch.zeros(shape, dtype=gr.dtype, device=gr.device).index_add_(0, idx, gr))
        return (None, *out)


def _flatten(state: KDAState) -> list[torch.Tensor]:
    return [
        state.recurrent_state,
        state.q_conv_state.buffer,
        state.k_conv_state.buffer,
        state.v_conv_state.buffer,
        state.sequence_offset,
    ]


def _rebuild(parts: list[torch.Tensor]) -> KDAState:
    return KDAState(
        recurrent_state=parts[0],
        q_conv_state=ShortConvState(parts[1]),
        k_conv_state=ShortConvState(parts[2]),
        v_conv_state=ShortConvState(parts[3]),
        sequence_offset=parts[4],
    )


def reorder_states(states: Sequence[KDAState], indices: torch.Tensor) -> list[KDAState]:
    """Every layer's ``KDAState.reorder(indices)`` (src/kda/state.py:50-67) in one pass."""
    if indices.ndim != 1 or indices.dtype != torch.long:
        raise ValueError("indices must be a rank-1 torch.long tensor")
    flat = [t for s in states for t in _flatten(s)]
    if flat and indices.device != flat[0].device:
        raise ValueError("indices and state must be on the same device")
    if not flat or (torch.is_grad_enabled() and any(t.requires_grad for t in flat)):
        out, status = gather_rows(flat, indices), None
    else:
        out, status = _launch_gather([_rows(t) for t in flat], indices)
    new = [_rebuild(out[5 * i : 5 * i + 5]) for i in range(len(states))]  # while the GPU copies
    if status is not None:
        _check_indices(status, flat[0].shape[0])
    return new


def clone_states(states: Sequence[KDAState]) -> list[KDAState]:
    """Every layer's ``KDAState.clone()`` (src/kda/state.py:41-48) in one pass."""
    flat = [t for s in states for t in _flatten(s)]
    out = gather_rows(flat, None)
    return [_rebuild(out[5 * i : 5 * i + 5]) for i in range(len(states))]


_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _moves(tensors: list[tuple[int, int, int | None, int, int, int]]) -> ctypes.Array:
    """``kda_state_tensor`` records (src, dst, scales, rows, width, kind) as one array of words."""
    words = array("q", [word or 0 for record in tensors for word in record])
    return (ctypes.c_int64 * len(words)).from_buffer(words)


def _status(device: torch.device, index: torch.Tensor | None) -> torch.Tensor | None:
    """What the kernels set for a slot out of range: None without slots, or into a
    graph, where no one can read it."""
    if index is None or torch.cuda.is_current_stream_capturing():
        return None
    return torch.zeros(1, dtype=torch.int32, device=device)


def _move(tensors, code: int, src_index, n_src: int, dst_index, n_dst: int, n: int, status, stream: int) -> None:
    if n and tensors:
        _lib.check(_lib.load().kda_state_move(_moves(tensors), len(tensors), code, _lib.ptr(src_index), n_src,
                                              _lib.ptr(dst_index), n_dst, n, _lib.ptr(status), stream))


# Bytes of f32 states after which reading back launches what it has, so that the GPU
# starts while the host makes the outputs of the layers behind (8 layers of 64 MiB: 181 us
# a call, 229 in one launch; smaller layers and 48 of them the same either way).
LAUNCH_BYTES = 100 << 20


def _check_slots(status: torch.Tensor | None, slots: int) -> None:
    if status is not None and int(status.item()) != 0:
        raise IndexError(f"slot out of range for a pool of {slots}")


def _slots_arg(slots: torch.Tensor | None, device: torch.device) -> torch.Tensor | None:
    if slots is None:
        return None
    if slots.ndim != 1 or slots.dtype != torch.long:
        raise ValueError("slots must be a rank-1 torch.long tensor")
    if slots.device != device:
        raise ValueError("slots and state must be on the same device")
    return slots.contiguous()


def _bytes(src: torch.Tensor, dst: torch.Tensor) -> tuple:
    entries = src.shape[0]
    return (src.data_ptr(), dst.data_ptr(), 0, 1, src.nbytes // entries if entries else 0,
            _lib.MOVE_BYTES)


def _one_device(tensors: Sequence[torch.Tensor]) -> torch.device:
    device = tensors[0].device
    if device.type != "cuda":
        _lib.require_gpu(tensors[0])
    for t in tensors:
        if t.device != device:
            raise ValueError("all cache tensors must be on one device")
    return device


def pack_recurrent(state: torch.Tensor) -> PackedState:
    """Recurrent states ``[B,H,K,V]`` (f32, f16 or bf16) in 8 bits.  Every row
    ``(b,h,k)`` of V values has its own scale, its largest magnitude times 1/127,
    and holds the nearest whole multiples of it (halves to even).  A row whose
    largest magnitude is under 2^-100 reads back as zeros, one with a value
    that is not finite as NaN.  No gradient: raises for a state that needs one."""
    _check_packable(state)
    if torch.is_grad_enabled() and state.requires_grad:
        raise RuntimeError("packing has no backward; pack a detached state or call it under torch.no_grad()")
    _prep.refuse_tangents("pack_recurrent", state)
    _one_device([state])
    out = _empty_packed(state, state.shape[0])
    n = state.shape[0]
    with _prep.on_device(state.device):
        st = state.contiguous()
        _move([_pack(st, out)], _lib.dtype_code(st.dtype), None, n, None, n, n, None, _prep.stream(st.device))
    return out


def unpack_recurrent(packed: PackedState, slots: torch.Tensor | None = None,
                     dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """``values * scales`` of all entries, or of ``slots`` (a slot may be named
    more than once), as ``[B,H,K,V]`` of ``dtype``.  A slot out of range raises
    ``IndexError``; in a captured graph, which no one can ask, it reads as NaN."""
    _prep.refuse_tangents("unpack_recurrent", packed.scales)
    device = _one_device([packed.values])
    _check_float(dtype)
    slots = _slots_arg(slots, device)
    entries, rest = packed.values.shape[0], packed.values.shape[1:]
    n = entries if slots is None else slots.shape[0]
    _check_entries(n, entries)
    out = torch.empty(n, *rest, dtype=dtype, device=device)
    with _prep.on_device(device):
        status = _status(device, slots)
        _move([_unpack(packed, out)], _lib.dtype_code(dtype), slots, entries, None, n, n, status, _prep.stream(device))
        _check_slots(status, entries)
    return out


def read_slots(packed: PackedState, slots: torch.Tensor | None) -> torch.Tensor:
    """``unpack_recurrent`` to f32 for checked slots, without waiting for the GPU:
    NaN for a slot out of range."""
    entries = packed.values.shape[0]
    n = entries if slots is None else slots.shape[0]
    out = torch.empty(n, *packed.values.shape[1:], dtype=torch.float32, device=_one_device([packed.values]))
    with _prep.on_device(out.device):
        _move([_unpack(packed, out)], _lib.dtype_code(torch.float32), slots, entries, None, n, n, None,
              _prep.stream(out.device))
    return out


def packed_pool(states: Sequence[KDAState], slots: int) -> list[PackedKDAState]:
    """An empty pool of ``slots`` slots per layer (zero states), for the caches of
    these layers and any batch size."""
    pool = []
    for s in states:
        conv = lambda c: ShortConvState(c.buffer.new_zeros(slots, *c.buffer.shape[1:]))  # noqa: E731
        shape = (slots, *s.recurrent_state.shape[1:])
        packed = PackedState(s.recurrent_state.new_zeros(shape, dtype=torch.int8),
                             s.recurrent_state.new_zeros(shape[:3], dtype=torch.float32))
        pool.append(PackedKDAState(packed, conv(s.q_conv_state), conv(s.k_conv_state), conv(s.v_conv_state),
                                   s.sequence_offset.new_zeros(slots)))
    return pool


def pack_states(states: Sequence[KDAState], *, out: Sequence[PackedKDAState] | None = None,
                slots: torch.Tensor | None = None) -> list[PackedKDAState]:
    """Every layer's decode caches with their recurrent states in 8 bits
    (``pack_recurrent``), all tensors in one native pass.

    Without ``out`` the result is new tensors of the caches' batch.  With a pool
    in ``out`` (one ``PackedKDAState`` a layer) batch row i goes to slot
    ``slots[i]`` (a rank-1 ``torch.long`` tensor; None: slot i, for a pool of the
    batch's size) and the other slots stay as they are; a slot named twice takes
    the last row.  No tensor of the pool may overlap another one or the caches.
    A slot out of range raises ``IndexError`` (its row is written
    nowhere; in a captured graph, which no one can ask, only that).  No
    gradient: raises for states that need one."""
    states = list(states)
    if out is None and slots is not None:
        raise ValueError("slots need a pool in `out`")
    if out is not None and len(out) != len(states):
        raise ValueError(f"the pool has {len(out)} layers, the caches {len(states)}")
    if not states:
        return []
    layers = [_flatten(s) for s in states]
    if _prep.forward_mode():
        _prep.refuse_tangents("pack_states", *(t for layer in layers for t in layer))
    shapes = [t.shape for t in layers[0]]
    dtypes = [t.dtype for t in layers[0]]
    _check_packable(layers[0][0])
    device, batch = layers[0][0].device, shapes[0][0]
    if device.type != "cuda":
        _lib.require_gpu(layers[0][0])
    grad = torch.is_grad_enabled()
    for layer in layers:
        if layer[0].dtype != dtypes[0]:
            raise TypeError("the recurrent states of all layers must share one dtype")
        for t in layer:
            if t.device != device:
                raise ValueError("all cache tensors must be on one device")
            if t.shape[0] != batch:
                raise ValueError("all cache tensors must share the batch size")
            if grad and t.requires_grad:
                raise RuntimeError("pack_states has no backward; call it on detached states or under torch.no_grad()")
    slots = _slots_arg(slots, device)
    if slots is not None and slots.shape[0] != batch:
        raise ValueError(f"slots must name a slot for each of {batch} batch rows, got {slots.shape[0]}")
    if out is None:
        out = []
        for s in states:
            conv = lambda c: ShortConvState(torch.empty_like(c.buffer, memory_format=torch.contiguous_format))  # noqa: E731
            out.append(PackedKDAState(_empty_packed(s.recurrent_state, batch), conv(s.q_conv_state),
                                      conv(s.k_conv_state), conv(s.v_conv_state),
                                      torch.empty_like(s.sequence_offset, memory_format=torch.contiguous_format)))
    out = list(out)
    pools = [_packed_parts(p) for p in out]
    pool_shapes = [t.shape for t in pools[0]]
    entries = pool_shapes[0][0]
    if slots is None and entries != batch:
        raise ValueError(f"a batch of {batch} needs slots for a pool of {entries}")
    _check_entries(batch, entries)
    for i, (src, dst) in enumerate(zip(layers, pools)):  # every layer, before any is written
        for k, (a, b) in enumerate(zip(src, dst)):
            if i == 0 or a.shape != shapes[k] or b.shape != pool_shapes[k] or a.dtype != dtypes[k]:
                expected = torch.int8 if k == 0 else a.dtype
                if b.shape != (entries, *a.shape[1:]) or b.dtype != expected:
                    raise ValueError(f"pool tensors must have shape {(entries, *a.shape[1:])} and dtype {expected}, "
                                     f"got {tuple(b.shape)} and {b.dtype}")
            elif b.dtype != pools[0][k].dtype:
                raise ValueError(f"pool tensors must have dtype {pools[0][k].dtype}, got {b.dtype}")
            if b.device != device:
                raise ValueError("pool and states must be on the same device")
            if not b.is_contiguous():
                raise ValueError("pool tensors must be contiguous")
    with _prep.on_device(device):
        code, stream, status = _lib.dtype_code(dtypes[0]), _prep.stream(device), _status(device, slots)
        moves, keep = [], []
        for i, (src, dst) in enumerate(zip(layers, pools)):
            src = [_rows(t) for t in src]
            keep.append(src)
            moves.append(_pack(src[0], out[i].recurrent))
            moves += [_bytes(a, b) for a, b in zip(src[1:], dst[1:])]
        # one call for all layers: what overlaps among them is refused before anything is written
        _move(moves, code, None, batch, slots, entries, batch, status, stream)
        _check_slots(status, entries)
    return out


def unpack_states(packed: Sequence[PackedKDAState], slots: torch.Tensor | None = None,
                  dtype: torch.dtype = torch.float32) -> list[KDAState]:
    """The decode caches held in ``slots`` (all slots in order when None) of every
    layer, the recurrent states as ``dtype``, in one native pass; the other
    tensors bit for bit.  A slot may be named more than once; one out of range
    raises ``IndexError`` (in a captured graph, which no one can ask, its states
    are NaN)."""
    packed = list(packed)
    if not packed:
        return []
    _check_float(dtype)
    parts = [_packed_parts(p) for p in packed]
    if _prep.forward_mode():
        _prep.refuse_tangents("unpack_states", *(p.recurrent.scales for p in packed), *(t for part in parts for t in part))
    device = _one_device([t for part in parts for t in part])
    slots = _slots_arg(slots, device)
    entries = parts[0][0].shape[0]
    if any(t.shape[0] != entries for part in parts for t in part):
        raise ValueError("all tensors of a pool must share the number of slots")
    n = entries if slots is None else slots.shape[0]
    _check_entries(n, entries)
    with _prep.on_device(device):
        code, stream, status = _lib.dtype_code(dtype), _prep.stream(device), _status(device, slots)
        moves, keep, size, states = [], [], 0, []
        waiting: list[list[torch.Tensor]] = []  # outputs whose objects are made while the GPU copies
        for i, (p, part) in enumerate(zip(packed, parts)):
            rest = [_rows(t) for t in part[1:]]
            keep.append(rest)
            new = [torch.empty(n, *part[0].shape[1:], dtype=dtype, device=device)]
            new += [t.new_empty(n, *t.shape[1:]) for t in rest]
            moves.append(_unpack(p.recurrent, new[0]))
            moves += [_bytes(a, b) for a, b in zip(rest, new[1:])]
            waiting.append(new)
            size += new[0].numel() * 4
            if size >= LAUNCH_BYTES or len(moves) >= 60 or i + 1 == len(packed):
                _move(moves, code, slots, entries, None, n, n, status, stream)
                states += [_rebuild(x) for x in waiting]
                moves, size, waiting = [], 0, []
        _check_slots(status, entries)
    return states


def _check_float(dtype: torch.dtype) -> None:
    if dtype not in _FLOATS:
        raise TypeError(f"recurrent states are read as float32, float16 or bfloat16, not {dtype}")


def _check_packable(state: torch.Tensor) -> None:
    if state.ndim != 4:
        raise ValueError(f"recurrent states must have shape [B,H,K,V], got {tuple(state.shape)}")
    if state.dtype not in _FLOATS:
        raise TypeError(f"recurrent states of float32, float16 or bfloat16 are packed, not {state.dtype}")


def _check_entries(n: int, entries: int) -> None:
    if n and not entries:
        raise IndexError("slot out of range for an empty pool")


def _empty_packed(state: torch.Tensor, entries: int) -> PackedState:
    shape = (entries, *state.shape[1:])
    return PackedState(torch.empty(shape, dtype=torch.int8, device=state.device),
                       torch.empty(shape[:3], dtype=torch.float32, device=state.device))


def _pack(src: torch.Tensor, dst: PackedState) -> tuple:
    _, heads, key_dim, value_dim = dst.values.shape
    return (src.data_ptr(), dst.values.data_ptr(), dst.scales.data_ptr(), heads * key_dim, value_dim,
            _lib.MOVE_PACK)


def _unpack(src: PackedState, dst: torch.Tensor) -> tuple:
    _, heads, key_dim, value_dim = src.values.shape
    return (src.values.data_ptr(), dst.data_ptr(), src.scales.data_ptr(), heads * key_dim, value_dim,
            _lib.MOVE_UNPACK)


def _packed_parts(p: PackedKDAState) -> list[torch.Tensor]:
    return [p.recurrent.values, p.q_conv_state.buffer, p.k_conv_state.buffer, p.v_conv_state.buffer, p.sequence_offset]

"""Argument checks of the 8-bit state cache (no GPU: every error is raised before a launch)."""

from __future__ import annotations

import ctypes

import pytest
import torch

import kda
from kda import _lib, cache


def _packed(n=3, heads=2, key_dim=4, value_dim=8):
    return kda.PackedState(torch.zeros(n, heads, key_dim, value_dim, dtype=torch.int8), torch.zeros(n, heads, key_dim))


def _state(batch=3, dtype=torch.float32):
    conv = lambda: kda.ShortConvState(torch.zeros(batch, 3, 8))  # noqa: E731
    return kda.KDAState(torch.zeros(batch, 2, 4, 8, dtype=dtype), conv(), conv(), conv(),
                        torch.zeros(batch, dtype=torch.long))


def test_packed_types():
    with pytest.raises(ValueError):
        kda.PackedState(torch.zeros(2, 2, 4, 8), torch.zeros(2, 2, 4))
    with pytest.raises(ValueError):
        kda.PackedState(torch.zeros(2, 2, 4, 8, dtype=torch.int8), torch.zeros(2, 2, 8))
    with pytest.raises(ValueError):
        kda.PackedState(torch.zeros(2, 2, 8, 4, dtype=torch.int8).transpose(2, 3), torch.zeros(2, 2, 4))
    p, s = _packed(), _state()
    with pytest.raises(ValueError):
        kda.PackedKDAState(p, s.q_conv_state, s.k_conv_state, s.v_conv_state, torch.zeros(4, dtype=torch.long))
    with pytest.raises(TypeError):
        kda.PackedKDAState(p, s.q_conv_state, s.k_conv_state, s.v_conv_state, torch.zeros(3))
    with pytest.raises(ValueError):
        kda.PackedKDAState(p, kda.ShortConvState(torch.zeros(2, 3, 8)), s.k_conv_state, s.v_conv_state,
                           torch.zeros(3, dtype=torch.long))


def test_what_a_kernel_reads_cannot_be_exchanged():
    p = _packed()
    with pytest.raises(AttributeError):
        p.scales = torch.zeros(1)
    pool = cache.packed_pool([_state()], 2)[0]
    with pytest.raises(AttributeError):
        pool.recurrent = p
    stack = kda.adapters.AdapterStack(torch.zeros(2, 4, 8), torch.zeros(2, 6, 4))
    with pytest.raises(AttributeError):
        stack.b = torch.zeros(1, 6, 4)


def test_pack_and_unpack_checks():
    with pytest.raises(ValueError):
        cache.pack_recurrent(torch.zeros(2, 4, 8))
    with pytest.raises(TypeError):
        cache.pack_recurrent(torch.zeros(1, 2, 4, 8, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="backward"):
        cache.pack_recurrent(torch.zeros(1, 2, 4, 8, requires_grad=True))
    with pytest.raises(RuntimeError, match="GPU"):
        cache.pack_recurrent(torch.zeros(1, 2, 4, 8))
    with pytest.raises(RuntimeError, match="GPU"):
        cache.unpack_recurrent(_packed())
    with pytest.raises(RuntimeError, match="GPU"):
        cache.pack_states([_state()])
    with pytest.raises(ValueError):
        cache.pack_states([_state()], slots=torch.zeros(3, dtype=torch.long))
    with pytest.raises(ValueError):
        cache.pack_states([_state()], out=[])
    with pytest.raises(TypeError):
        cache.unpack_states(cache.packed_pool([_state()], 2), dtype=torch.float64)
    assert cache.pack_states([]) == [] and cache.unpack_states([]) == []
    pool = cache.packed_pool([_state()], 5)
    assert pool[0].recurrent.values.shape == (5, 2, 4, 8) and pool[0].sequence_offset.shape == (5,)


def test_a_tangent_is_refused_not_lost():
    fw, state = torch.autograd.forward_ad, _state()
    conv, p = state.q_conv_state, _packed()
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        recurrent = kda.KDAState(dual(state.recurrent_state), conv, conv, conv, state.sequence_offset)
        history = kda.KDAState(state.recurrent_state, conv, kda.ShortConvState(dual(conv.buffer)), conv,
                               state.sequence_offset)
        scales = kda.PackedState(p.values, dual(p.scales))
        pool = lambda packed, c: [kda.PackedKDAState(packed, c, conv, conv, state.sequence_offset)]  # noqa: E731
        q = torch.zeros(3, 1, 2, 4)
        args = [q, q, torch.zeros(3, 1, 2, 8), q, torch.zeros(3, 1, 2)]
        calls = [lambda: cache.pack_recurrent(recurrent.recurrent_state), lambda: cache.unpack_recurrent(scales),
                 lambda: cache.pack_states([state, recurrent]), lambda: cache.pack_states([history]),
                 lambda: cache.unpack_states(pool(scales, conv)),
                 lambda: cache.unpack_states(pool(p, kda.ShortConvState(dual(conv.buffer))))]
        for op in (kda.recurrent_kda, kda.chunkwise_kda):
            calls.append(lambda op=op: op(*args, scales))
            calls += [lambda op=op, i=i: op(*args[:i], dual(args[i]), *args[i + 1:], p) for i in range(5)]
        for call in calls:
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
        for call in (lambda: cache.pack_states([state]), lambda: cache.unpack_states(pool(p, conv)),
                     lambda: kda.recurrent_kda(*args, p)):
            with pytest.raises(RuntimeError, match="GPU"):  # a level alone changes nothing
                call()


@pytest.mark.parametrize("call", [kda.recurrent_kda, kda.chunkwise_kda])
def test_packed_initial_state_checks(call):
    q = torch.zeros(3, 1, 2, 4)
    args = (q, q, torch.zeros(3, 1, 2, 8), q, torch.zeros(3, 1, 2))
    with pytest.raises(ValueError, match="PackedState"):
        call(*args, None, state_slots=torch.zeros(3, dtype=torch.long))
    with pytest.raises(ValueError, match="shape"):
        call(*args, _packed(value_dim=4))
    with pytest.raises(ValueError, match="state_slots"):
        call(*args, _packed(n=4))
    with pytest.raises(ValueError, match="state_slots"):
        call(*args, _packed(), state_slots=torch.zeros(2, dtype=torch.long))
    with pytest.raises(ValueError, match="state_slots"):
        call(*args, _packed(), state_slots=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(IndexError):
        call(*args, _packed(n=0), state_slots=torch.zeros(3, dtype=torch.long))
    with pytest.raises(RuntimeError, match="GPU"):
        call(*args, _packed())


def test_packed_state_is_not_updated_in_place():
    q = torch.zeros(3, 1, 2, 4)
    with pytest.raises(ValueError, match="update_state_in_place"):
        kda.recurrent_kda(q, q, torch.zeros(3, 1, 2, 8), q, torch.zeros(3, 1, 2), _packed(),
                          update_state_in_place=True)


def test_move_entry_point_rejects_bad_arguments():
    lib, bad = _lib.load(), _lib.KDA_ERR_INVALID_ARGUMENT
    a, b, c = 1 << 20, 2 << 20, 3 << 20  # stand-in addresses, never dereferenced

    def move(src=a, dst=b, scales=c, rows=4, width=8, kind=_lib.MOVE_PACK, dtype=0, n_src=3, n_dst=3, n=3, count=1,
             index=None):
        t = cache._moves([(src or 0, dst or 0, scales, rows, width, kind)])
        return lib.kda_state_move(ctypes.addressof(t) if count else None, count, dtype, index, n_src, None, n_dst, n,
                                  None, None)

    for kw in (dict(src=None), dict(dst=None), dict(scales=None), dict(kind=5), dict(rows=-1), dict(width=-1),
               dict(width=1 << 32), dict(dtype=3), dict(n=4), dict(n_src=2), dict(n_dst=2), dict(n_src=0, index=a),
               dict(n=-1), dict(count=-1), dict(src=a + 2), dict(scales=c + 1), dict(dst=a), dict(scales=a + 32),
               dict(dst=a + 200), dict(kind=_lib.MOVE_UNPACK, dst=b + 2), dict(kind=_lib.MOVE_BYTES, dst=a + 8),
               dict(rows=1 << 40, width=1 << 30)):
        assert move(**kw) == bad, kw
    assert move(n=0) == _lib.KDA_OK and move(count=0) == _lib.KDA_OK
    # two tensors that write one place
    t = cache._moves([(a, b, None, 1, 8, 0), (c, b + 8, None, 1, 8, 0)])
    assert lib.kda_state_move(ctypes.addressof(t), 2, 0, None, 3, None, 3, 3, None, None) == bad

    def step(values=a, scales=a, slots=None, n_slots=3, dtype=2, q=a):
        return lib.kda_recurrent_fwd_packed(q, a, a, a, a, dtype, values, scales, slots, n_slots, a, a, None, 1, None,
                                            3, 3, 2, 128, 128, None)

    for kw in (dict(values=None), dict(scales=None), dict(n_slots=2), dict(n_slots=0, slots=a), dict(dtype=3),
               dict(q=None)):
        assert step(**kw) == bad, kw


def test_overlaps_are_refused_among_many_tensors():
    # whatever their order and distance, and one inside another; stand-in addresses, never dereferenced
    lib, bad = _lib.load(), _lib.KDA_ERR_INVALID_ARGUMENT
    a, b, c = 1 << 20, 2 << 20, 3 << 20
    for first, last in ((0, 199), (199, 0), (7, 130)):
        records = [((i + 1) << 20, (i + 501) << 20, None, 1, 8, 0) for i in range(200)]
        records[last] = (records[last][0], records[first][1] + 16, None, 1, 8, 0)  # writes into another's destination
        t = cache._moves(records)
        assert lib.kda_state_move(ctypes.addressof(t), 200, 0, None, 3, None, 3, 3, None, None) == bad
        records[last] = ((last + 1) << 20, (first + 1) << 20, None, 1, 4, 0)  # or into another's source
        t = cache._moves(records)
        assert lib.kda_state_move(ctypes.addressof(t), 200, 0, None, 3, None, 3, 3, None, None) == bad
    t = cache._moves([(a, b, None, 1, 1 << 16, 0), (c, 4 << 20, None, 1, 8, 0), (b + 300, 5 << 20, None, 1, 1, 0)])
    assert lib.kda_state_move(ctypes.addressof(t), 3, 0, None, 3, None, 3, 3, None, None) == bad


def test_tiles_of_an_entry_are_counted_past_32_bits():
    # an entry of nearly 2 GiB of bytes; nine of them are more tiles than a launch holds
    t = cache._moves([(1 << 40, 1 << 44, None, 1, (1 << 31) - 1, _lib.MOVE_BYTES)])
    assert _lib.load().kda_state_move(ctypes.addressof(t), 1, 0, None, 9, None, 9, 9, None, None) == \
        _lib.KDA_ERR_UNSUPPORTED

"""GPU parity of the 8-bit state cache: pack, pool, unpack and the recurrence from it.

Packing is exact by definition (the nearest whole multiple of an f32 scale), so
values and scales are compared bit for bit with the oracle; reading back is one
f32 product, rounded once to the type asked for.  A call from 8-bit states is
compared with the same call from the states read back, bit for bit where both
run the same kernel, and with the f64 oracle at the recurrence's tolerance.
"""

from __future__ import annotations

import pytest
import torch

import kda
from kda import cache
from kda.layer import KDALayerWeights, kda_attention_forward
from oracle import kda_oracle as ora
from tests._inputs import layer_weights, rel_err, workload

pytestmark = pytest.mark.gpu
DEV = "cuda"
SHAPES = [(1, 1, 1, 1), (3, 2, 5, 7), (2, 4, 128, 128), (2, 3, 64, 48), (1, 2, 96, 96), (2, 1, 40, 50), (1, 2, 16, 4),
          (1, 1, 8, 256), (1, 2, 8, 260), (1, 1, 3, 1030), (5, 2, 33, 64)]


def _state(*shape, dtype=torch.float32, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rows = torch.exp(3 * torch.randn(*shape[:-1], 1, generator=gen))
    return (torch.randn(*shape, generator=gen) * rows * 0.02).to(dtype)


def _caches(layers, batch, heads, key_dim, value_dim, dtype=torch.float32, conv_dtype=torch.bfloat16, taps=4, seed=0):
    gen = torch.Generator().manual_seed(seed)
    out = []
    for i in range(layers):
        conv = lambda w: kda.ShortConvState(torch.randn(batch, taps - 1, w, generator=gen).to(conv_dtype).to(DEV))  # noqa: E731
        out.append(kda.KDAState(_state(batch, heads, key_dim, value_dim, dtype=dtype, seed=seed + i).to(DEV),
                                conv(heads * key_dim), conv(heads * key_dim), conv(heads * value_dim),
                                torch.randint(0, 1 << 40, (batch,), generator=gen).to(DEV)))
    return out


def _parts(s):
    return [s.q_conv_state.buffer, s.k_conv_state.buffer, s.v_conv_state.buffer, s.sequence_offset]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_pack_and_unpack_are_exact(shape, dtype):
    state = _state(*shape, dtype=dtype)
    values, scales = ora.pack_rows(state)
    got = cache.pack_recurrent(state.to(DEV))
    assert torch.equal(got.values.cpu(), values) and torch.equal(got.scales.cpu(), scales)
    for to in (torch.float32, torch.bfloat16, torch.float16):
        back = cache.unpack_recurrent(got, dtype=to)
        assert torch.equal(back.cpu(), (values.float() * scales[..., None]).to(to))
    # half a step of the row's scale, and the f32 rounding of the product read back
    err = (cache.unpack_recurrent(got).cpu().double() - state.double()).abs()
    assert bool((err <= scales[..., None].double() * (0.5 + 128 * 2.0 ** -24)).all())


def test_quotients_at_ties_and_extremes():
    # rows whose largest magnitude is 127 s for a scale s of many bits, and whose
    # other values are at and next to (n + 1/2) s
    rows = []
    for seed in range(40):
        gen = torch.Generator().manual_seed(seed)
        s = torch.exp(20 * torch.randn(1, generator=gen)).float()
        n = torch.arange(-63, 63, dtype=torch.float32)
        mid = ((n + 0.5).double() * s.double()).float()
        top = torch.tensor([float((127 * s.double()).float())])
        bits = torch.randint(-1, 2, mid.shape, generator=gen, dtype=torch.int32)
        near = (mid.view(torch.int32) + bits).view(torch.float32)
        rows.append(torch.cat([near, top, -top]))
    state = torch.stack(rows).reshape(2, 4, 5, 128)
    values, scales = ora.pack_rows(state)
    for shape in ((2, 4, 5, 128), (40, 1, 1, 128)):
        got = cache.pack_recurrent(state.reshape(shape).to(DEV))
        assert torch.equal(got.values.cpu().reshape(values.shape), values)
        assert torch.equal(got.scales.cpu().reshape(scales.shape), scales)
    wide = torch.cat([state.reshape(4, 2, 5, 128), torch.zeros(4, 2, 5, 2)], -1)[..., :129].contiguous()  # value by value
    got = cache.pack_recurrent(wide.to(DEV))
    assert torch.equal(got.values.cpu()[..., :128].reshape(values.shape), values)
    # exact ties: scale 1
    tie = torch.zeros(1, 1, 1, 8)
    tie[0, 0, 0] = torch.tensor([127, 0.5, 1.5, 2.5, -0.5, -1.5, 126.5, 0.25])
    assert cache.pack_recurrent(tie.to(DEV)).values.cpu().flatten().tolist() == [127, 0, 2, 2, 0, -2, 126, 0]


@pytest.mark.parametrize("width", [128, 50, 7])
def test_rows_of_zeros_tiny_and_non_finite_values(width):
    state = _state(1, 1, 8, width)
    state[0, 0, 0] = 0
    state[0, 0, 1] = 1e-40  # subnormal
    state[0, 0, 2] = 2.0 ** -100
    state[0, 0, 3, width // 2] = float("inf")
    state[0, 0, 4, 0] = float("nan")
    state[0, 0, 5, -1] = float("-inf")
    state[0, 0, 6] = 3e38
    values, scales = ora.pack_rows(state)
    got = cache.pack_recurrent(state.to(DEV))
    assert torch.equal(got.values.cpu(), values)
    assert torch.equal(got.scales.cpu().nan_to_num(-1.0), scales.nan_to_num(-1.0))
    back = cache.unpack_recurrent(got).cpu()
    assert torch.count_nonzero(back[0, 0, :2]) == 0 and bool(back[0, 0, 3:6].isnan().all())
    assert bool(back[0, 0, 6:].isfinite().all()) and bool((back[0, 0, 2] == 2.0 ** -100).all())


@pytest.mark.parametrize("layers,batch,heads,key_dim,value_dim", [(1, 1, 2, 128, 128), (3, 5, 2, 64, 48), (20, 3, 1, 8, 7)])
def test_pool_slots_are_written_and_read(layers, batch, heads, key_dim, value_dim):
    # 20 layers are 80 tensors: two launches
    states = _caches(layers, batch, heads, key_dim, value_dim)
    pool = cache.packed_pool(states, 2 * batch + 1)
    before = _caches(layers, 2 * batch + 1, heads, key_dim, value_dim, seed=50)
    cache.pack_states(before, out=pool)
    old = [[t.clone() for t in (p.recurrent.values, p.recurrent.scales, *_parts(p))] for p in pool]
    slots = torch.randperm(2 * batch + 1, generator=torch.Generator().manual_seed(1))[:batch].to(DEV)
    assert cache.pack_states(states, out=pool, slots=slots)[0] is pool[0]
    fresh = cache.pack_states(states)
    rest = torch.ones(2 * batch + 1, dtype=torch.bool, device=DEV)
    rest[slots] = False
    for p, f, o in zip(pool, fresh, old):
        for now, new, was in zip((p.recurrent.values, p.recurrent.scales, *_parts(p)),
                                 (f.recurrent.values, f.recurrent.scales, *_parts(f)), o):
            assert torch.equal(now[slots], new) and torch.equal(now[rest], was[rest])
    # read back: some slots more than once
    names = slots.repeat(2)[: batch + 1]
    for got, p in zip(cache.unpack_states(pool, names), pool):
        assert torch.equal(got.recurrent_state, p.recurrent.values[names].float() * p.recurrent.scales[names][..., None])
        assert all(torch.equal(a, b[names]) for a, b in zip(_parts(got), _parts(p)))
    for got, f, s in zip(cache.unpack_states(fresh), fresh, states):
        assert torch.equal(got.recurrent_state, f.recurrent.values.float() * f.recurrent.scales[..., None])
        assert all(torch.equal(a, b) for a, b in zip(_parts(got), _parts(s)))


def test_a_slot_named_twice_takes_the_last_row():
    states = _caches(2, 600, 1, 8, 8)  # more rows than a workgroup has threads
    pool = cache.packed_pool(states, 7)
    slots = (torch.arange(600) * 5 % 7).to(DEV)
    cache.pack_states(states, out=pool, slots=slots)
    fresh = cache.pack_states(states)
    last = torch.tensor([max(i for i in range(600) if i * 5 % 7 == s) for s in range(7)], device=DEV)
    for p, f in zip(pool, fresh):
        assert torch.equal(p.recurrent.values, f.recurrent.values[last])
        assert all(torch.equal(a, b[last]) for a, b in zip(_parts(p), _parts(f)))


def test_slots_out_of_range_raise_and_write_nothing():
    states = _caches(2, 3, 2, 16, 8)
    pool = cache.packed_pool(states, 4)
    for bad in (4, -1, 1 << 40):
        before = [p.recurrent.values.clone() for p in pool]
        with pytest.raises(IndexError):
            cache.pack_states(states, out=pool, slots=torch.tensor([bad, bad, bad], device=DEV))
        assert all(torch.equal(p.recurrent.values, b) for p, b in zip(pool, before))
        with pytest.raises(IndexError):
            cache.unpack_states(pool, torch.tensor([0, bad], device=DEV))
        with pytest.raises(IndexError):
            cache.unpack_recurrent(pool[0].recurrent, torch.tensor([bad], device=DEV))
    empty = torch.zeros(0, dtype=torch.long, device=DEV)
    assert cache.unpack_states(pool, empty)[0].recurrent_state.shape == (0, 2, 16, 8)
    none = _caches(1, 0, 2, 16, 8)
    assert cache.pack_states(none)[0].recurrent.values.shape == (0, 2, 16, 8)
    with pytest.raises(IndexError):
        cache.unpack_states(cache.pack_states(none), torch.tensor([0], device=DEV))


def test_pool_tensors_that_do_not_fit_are_refused():
    states = _caches(2, 3, 2, 16, 8)
    pool = cache.packed_pool(states, 4)
    slots = torch.tensor([0, 1, 2], device=DEV)
    pool[1].v_conv_state.buffer = pool[1].v_conv_state.buffer[:3]
    with pytest.raises(ValueError):
        cache.unpack_states(pool, slots)
    with pytest.raises(ValueError):
        cache.pack_states(states, out=pool, slots=slots)
    for other in (_caches(2, 3, 2, 16, 4), _caches(2, 3, 1, 16, 8), _caches(2, 3, 2, 16, 8, conv_dtype=torch.float16)):
        with pytest.raises(ValueError):
            cache.pack_states(other, out=cache.packed_pool(states, 4), slots=slots)
    mixed = [_caches(1, 3, 2, 16, 8)[0], _caches(1, 3, 2, 16, 8, dtype=torch.bfloat16)[0]]
    with pytest.raises(TypeError):
        cache.pack_states(mixed)
    with pytest.raises(ValueError):
        cache.pack_states([_caches(1, 3, 2, 16, 8)[0], _caches(1, 2, 2, 16, 8)[0]])
    leaf = _caches(1, 3, 2, 16, 8)[0]
    leaf.q_conv_state.buffer.requires_grad_()
    with pytest.raises(RuntimeError):
        cache.pack_states([leaf])
    with torch.no_grad():
        cache.pack_states([leaf])


@pytest.mark.parametrize("layers,heads", [(2, 3300), (14, 2)])
def test_pool_tensors_named_twice_are_refused_before_anything_is_written(layers, heads):
    # 108 MiB of states a layer, and more layers than a launch holds: the call is no single launch
    states = _caches(layers, 2, heads, 64, 64)
    pool = cache.packed_pool(states, 3)
    twice = [*pool[:-1], pool[0]]
    slots = torch.tensor([2, 0], device=DEV)
    with pytest.raises(RuntimeError, match="overlap"):
        cache.pack_states(states, out=twice, slots=slots)
    offsets = [kda.PackedKDAState(p.recurrent, p.q_conv_state, p.k_conv_state, p.v_conv_state, pool[0].sequence_offset)
               for p in pool]
    with pytest.raises(RuntimeError, match="overlap"):
        cache.pack_states(states, out=offsets, slots=slots)
    with pytest.raises(RuntimeError, match="overlap"):  # a cache that lies in the pool
        within = kda.ShortConvState(pool[-1].q_conv_state.buffer[:2])
        cache.pack_states([kda.KDAState(s.recurrent_state, within, s.k_conv_state, s.v_conv_state, s.sequence_offset)
                           for s in states], out=pool, slots=slots)
    for p in pool:
        assert not bool(p.recurrent.values.any()) and not bool(p.recurrent.scales.any())
        assert not any(bool(t.any()) for t in _parts(p))
    cache.pack_states(states, out=pool, slots=slots)
    for s, back in zip(states, cache.unpack_states(pool, slots)):
        assert all(torch.equal(a, b) for a, b in zip(_parts(s), _parts(back)))


def test_layers_of_different_sizes_in_one_call():
    states = [_caches(1, 3, 2, 16, 8, seed=1)[0], _caches(1, 3, 1, 64, 128, seed=2)[0], _caches(1, 3, 3, 7, 5, seed=3)[0]]
    pool = cache.packed_pool(states, 5)
    slots = torch.tensor([4, 0, 2], device=DEV)
    cache.pack_states(states, out=pool, slots=slots)
    for s, p, back in zip(states, pool, cache.unpack_states(pool, slots)):
        want = cache.pack_recurrent(s.recurrent_state)
        assert torch.equal(p.recurrent.values[slots], want.values)
        assert torch.equal(back.recurrent_state, cache.unpack_recurrent(want))
        assert all(torch.equal(a, b) for a, b in zip(_parts(back), _parts(s)))


def test_layouts_of_the_float_side():
    state = _state(3, 4, 24, 20).to(DEV)
    want = cache.pack_recurrent(state)
    flipped = state.transpose(2, 3).contiguous().transpose(2, 3)
    off = torch.zeros(state.numel() + 1, device=DEV)[1:].copy_(state.flatten()).view(state.shape)
    for t in (flipped, off, torch.cat([state, state])[:3]):
        got = cache.pack_recurrent(t)
        assert torch.equal(got.values, want.values) and torch.equal(got.scales, want.scales)
    # values that start off a four-byte address
    shifted = torch.zeros(want.values.numel() + 1, dtype=torch.int8, device=DEV)[1:]
    shifted.copy_(want.values.flatten())
    odd = kda.PackedState(shifted.view(want.values.shape), want.scales)
    assert torch.equal(cache.unpack_recurrent(odd), cache.unpack_recurrent(want))
    q, k, v, g, beta, _ = workload(3, 1, 4, 24, 20, seed=3)
    args = [t.to(DEV) for t in (q, k, v, g, beta)]
    a, b = kda.recurrent_kda(*args, odd, True), kda.recurrent_kda(*args, want, True)
    assert torch.equal(a.hidden_states, b.hidden_states) and torch.equal(a.final_state, b.final_state)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,key_dim,value_dim", [(4, 128, 128), (2, 64, 64), (3, 40, 50), (1, 200, 16), (2, 128, 256)])
def test_decode_from_the_pool(heads, key_dim, value_dim, dtype):
    batch, slots = 5, 9
    pool = cache.pack_recurrent(_state(slots, heads, key_dim, value_dim).to(DEV))
    names = torch.tensor([8, 0, 3, 3, 5], device=DEV)
    inputs = workload(batch, 1, heads, key_dim, value_dim, seed=4, dtype=dtype)[:5]
    args = [t.to(DEV) for t in inputs]
    got = kda.recurrent_kda(*args, pool, True, state_slots=names)
    read = cache.unpack_recurrent(pool, names)
    want = kda.recurrent_kda(*args, read, True)
    assert got.hidden_states.dtype == dtype and got.final_state.dtype == torch.float32
    assert torch.equal(got.hidden_states, want.hidden_states) and torch.equal(got.final_state, want.final_state)
    ro, rs, _ = ora.recurrent(*(t.double() for t in inputs), read.cpu().double())
    tol = {torch.float32: 1e-5}.get(dtype, 1e-2)
    assert rel_err(got.hidden_states, ro) < tol and rel_err(got.final_state, rs) < 1e-5
    assert kda.recurrent_kda(*args, pool, state_slots=names).final_state is None


def test_sequences_masks_documents_and_prefill_from_the_pool():
    H, K, V = 2, 128, 128
    pool = cache.pack_recurrent(_state(6, H, K, V).to(DEV))
    names = torch.tensor([5, 1, 2], device=DEV)
    read = cache.unpack_recurrent(pool, names)
    args = [t.to(DEV) for t in workload(3, 70, H, K, V, seed=5)[:5]]
    mask = (torch.arange(70)[None] < torch.tensor([70, 1, 33])[:, None]).to(DEV)
    for call in (kda.recurrent_kda, kda.chunkwise_kda):
        for m in (None, mask):
            got, want = call(*args, pool, True, m, state_slots=names), call(*args, read, True, m)
            assert torch.equal(got.hidden_states, want.hidden_states)
            assert torch.equal(got.final_state, want.final_state)
        docs = [t.to(DEV) for t in workload(1, 90, H, K, V, seed=6)[:5]]
        got = call(*docs, pool, True, cu_seqlens=[0, 1, 50, 90], state_slots=names)
        want = call(*docs, read, True, cu_seqlens=[0, 1, 50, 90])
        assert torch.equal(got.hidden_states, want.hidden_states) and torch.equal(got.final_state, want.final_state)
    # without an f32 state, in f64, with per-token states and under autograd the states are read first
    got = kda.recurrent_kda(*args, pool, True, accumulate_state_in_fp32=False, state_slots=names)
    want = kda.recurrent_kda(*args, read, True, accumulate_state_in_fp32=False)
    assert got.final_state.dtype == torch.bfloat16 and torch.equal(got.final_state, want.final_state)
    wide = [t.double() for t in args]
    assert torch.equal(kda.recurrent_kda(*wide, pool, True, state_slots=names).final_state,
                       kda.recurrent_kda(*wide, read.double(), True).final_state)
    got = kda.recurrent_kda(*(t[:, :2] for t in args), pool, return_states_per_token=True, state_slots=names)
    want = kda.recurrent_kda(*(t[:, :2] for t in args), read, return_states_per_token=True)
    assert all(torch.equal(a, b) for a, b in zip(got.states_per_token, want.states_per_token))
    leaf = args[2].clone().requires_grad_()
    grads = [torch.autograd.grad(kda.chunkwise_kda(args[0], args[1], leaf, *args[3:], s, state_slots=n)
                                 .hidden_states.float().sum(), leaf)[0] for s, n in ((pool, names), (read, None))]
    assert torch.equal(*grads)


def test_a_missing_slot_gives_its_own_sequence_nan():
    pool = cache.pack_recurrent(_state(4, 2, 128, 128).to(DEV))
    names = torch.tensor([0, 4, 2, -1], device=DEV)
    args = [t.to(DEV) for t in workload(4, 1, 2, 128, 128, seed=7)[:5]]
    for call in (kda.recurrent_kda, kda.chunkwise_kda):
        out = call(*args, pool, True, state_slots=names)
        good = call(*(t[::2] for t in args), pool, True, state_slots=names[::2])
        for a, b in ((out.hidden_states, good.hidden_states), (out.final_state, good.final_state)):
            assert torch.equal(a[::2], b) and bool(a[1::2].isnan().all())


def test_a_layer_continues_from_caches_at_rest():
    # prompt, rest, three tokens; against the same with the states read back by hand
    weights = layer_weights(256, 2, 128, 128, dtype=torch.bfloat16)
    w = KDALayerWeights(**{n: t.to(DEV) if isinstance(t, torch.Tensor) else t for n, t in weights.items()})
    gen = torch.Generator().manual_seed(9)
    x = torch.randn(3, 20, 256, generator=gen).to(torch.bfloat16).to(DEV)
    state = kda_attention_forward(w, x[:, :17], None, None, "chunkwise", True).state
    packed = cache.pack_states([state])[0]
    by_hand = cache.unpack_states([packed])[0]
    for mode, part in (("chunkwise", x[:, 17:]), ("decode", x[:, 17:18])):
        got = kda_attention_forward(w, part, None, packed, mode, True)
        want = kda_attention_forward(w, part, None, by_hand, mode, True)
        assert torch.equal(got.hidden_states, want.hidden_states)
        assert torch.equal(got.state.recurrent_state, want.state.recurrent_state)
        assert torch.equal(got.state.sequence_offset, want.state.sequence_offset)
    with pytest.raises(ValueError):
        kda_attention_forward(w, x[:, 17:18], None, packed, "decode", update_state_in_place=True)


def test_captured_calls_replay():
    states = _caches(2, 4, 2, 128, 128)
    pool = cache.packed_pool(states, 6)
    slots = torch.tensor([5, 2, 0, 3], device=DEV)
    args = [t.to(DEV) for t in workload(4, 1, 2, 128, 128, seed=8)[:5]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.pack_states(states, out=pool, slots=slots)
        cache.unpack_states(pool, slots)
        kda.recurrent_kda(*args, pool[0].recurrent, True, state_slots=slots)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.pack_states(states, out=pool, slots=slots)
        back = cache.unpack_states(pool, slots)
        step = kda.recurrent_kda(*args, pool[0].recurrent, True, state_slots=slots)
    for seed in range(3):
        new = _state(4, 2, 128, 128, seed=30 + seed).to(DEV)
        states[0].recurrent_state.copy_(new)
        slots.copy_(torch.tensor([seed, 5, 4, 3]))
        for p in pool:
            p.recurrent.values.zero_()
        graph.replay()
        torch.cuda.synchronize()
        packed = cache.pack_recurrent(new)
        assert torch.equal(pool[0].recurrent.values[slots], packed.values)
        assert torch.equal(back[0].recurrent_state, cache.unpack_recurrent(packed))
        assert torch.equal(step.final_state, kda.recurrent_kda(*args, packed, True).final_state)
    # in a graph a slot that is not there reads as NaN, and is written nowhere
    slots.copy_(torch.tensor([1, 6, -1, 2]))
    graph.replay()
    torch.cuda.synchronize()
    assert bool(back[0].recurrent_state[1:3].isnan().all()) and bool(back[0].recurrent_state[::3].isfinite().all())


def test_offsets_past_two_to_the_31():
    # 2.3e9 values: entry, row and byte offsets of the last slots pass 32 bits
    H, K, V = 32, 128, 128
    slots = 4400
    pool = kda.PackedState(torch.zeros(slots, H, K, V, dtype=torch.int8, device=DEV),
                           torch.zeros(slots, H, K, device=DEV))
    state = _state(2, H, K, V).to(DEV)
    conv = kda.ShortConvState(torch.zeros(2, 3, 8, device=DEV))
    pconv = kda.ShortConvState(torch.zeros(slots, 3, 8, device=DEV))
    names = torch.tensor([slots - 1, 7], device=DEV)
    out = kda.PackedKDAState(pool, pconv, pconv_copy(pconv), pconv_copy(pconv),
                             torch.zeros(slots, dtype=torch.long, device=DEV))
    s = kda.KDAState(state, conv, conv, conv, torch.tensor([3, 4], device=DEV))
    cache.pack_states([s], out=[out], slots=names)
    want = cache.pack_recurrent(state)
    assert torch.equal(pool.values[names], want.values)
    assert torch.equal(cache.unpack_recurrent(pool, names), cache.unpack_recurrent(want))
    args = [t.to(DEV) for t in workload(2, 1, H, K, V, seed=10)[:5]]
    assert torch.equal(kda.recurrent_kda(*args, pool, True, state_slots=names).final_state,
                       kda.recurrent_kda(*args, want, True).final_state)


def pconv_copy(c):
    return kda.ShortConvState(c.buffer.clone())

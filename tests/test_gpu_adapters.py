"""GPU parity of adapters.adapter_linear against the f64 oracle, and of a layer with adapters.

Bound of an element: half a step of the result, half a step of the adapter's
part (rounded to the dtype before the product is added; f32 tensors: within the
next), and one 2^-24 of the terms' magnitudes for each rounding in a chain: at
most `in` in the products over x, `rank` in the product over s, and a few for
scaling, bias and joins.
"""

from __future__ import annotations

import ctypes

import pytest
import torch

import kda
from kda import _lib
from kda import adapters, cache, fused
from kda.layer import KDALayerWeights, kda_attention_forward
from oracle import kda_oracle as ora
from tests._bounds import assert_within, rounded
from tests._inputs import layer_weights

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
# batch, tokens, in, out, rank, adapters
SIZES = [(1, 1, 1, 1, 1, 1), (1, 1, 64, 48, 16, 2), (3, 1, 7, 5, 3, 2), (17, 1, 128, 256, 16, 5), (64, 1, 2048, 512, 8, 64),
         (65, 1, 192, 100, 64, 3), (200, 1, 320, 64, 32, 40), (5, 5, 1001, 77, 12, 4), (2, 33, 130, 63, 4, 3),
         (3, 100, 256, 128, 16, 2), (2, 300, 96, 520, 100, 4), (1, 700, 72, 40, 256, 1), (40, 16, 64, 64, 17, 9),
         (300, 2, 64, 64, 16, 300), (1, 16, 4096, 16, 16, 1)]


def _inputs(batch, tokens, d_in, d_out, rank, n, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rnd = lambda *s, std=1.0: (torch.randn(*s, generator=gen, dtype=torch.float64) * std).to(dtype)  # noqa: E731
    ids = torch.randint(-1, n, (batch,), generator=gen)
    return (rnd(batch, tokens, d_in), rnd(d_out, d_in, std=d_in ** -0.5), rnd(d_out, std=0.1),
            rnd(n, rank, d_in, std=d_in ** -0.5), rnd(n, d_out, rank, std=rank ** -0.5),
            0.5 + torch.rand(n, generator=gen), ids)


def _check(x, w, bias, a, b, scaling, ids, got, what="y"):
    dtype, d_in, rank = x.dtype, x.shape[-1], a.shape[1]
    flat = x.reshape(-1, d_in)
    row_ids = ids.flatten().repeat_interleave(flat.shape[0] // ids.numel())
    y, delta, (wide, low, up) = ora.adapter_linear(flat, w, bias, a, b, scaling, row_ids)
    units = (d_in + 8) * (wide + low) + (rank + 8) * up
    bound = rounded(y, dtype) + rounded(delta, dtype) * (1 + 2.0 ** -7) + 2.0 ** -24 * units * (1 + 2.0 ** -7)
    assert_within(got.reshape(y.shape), y, bound, what)


def _dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def _call(x, w, bias, a, b, scaling, ids):
    x, w, bias, a, b, scaling, ids = _dev(x, w, bias, a, b, scaling, ids)
    return adapters.adapter_linear(x, w, bias, adapters.AdapterStack(a, b, scaling), ids)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("plain", [False, True])
def test_adapter_linear_matches_oracle(size, dtype, plain):
    x, w, bias, a, b, scaling, ids = _inputs(*size, dtype)
    if plain:  # no bias, no factors, 32-bit ids
        bias, scaling, ids = None, None, ids.int()
    got = _call(x, w, bias, a, b, scaling, ids)
    assert got.dtype == dtype and got.shape == (*x.shape[:-1], w.shape[0])
    _check(x, w, bias, a, b, scaling, ids, got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [(8, 1, 128, 96, 16, 3), (40, 1, 128, 96, 16, 3), (200, 1, 320, 64, 32, 40),
                                  (24, 5, 1001, 77, 12, 9), (3, 100, 256, 128, 16, 2), (2, 300, 96, 520, 100, 4),
                                  (1, 2100, 72, 40, 20, 1)])
def test_the_sum_is_rounded_once(size, dtype):
    # half a step of the result, the f32 roundings, and for bf16 what its two parts of s leave
    x, w, bias, a, b, scaling, ids = _inputs(*size, dtype)
    got = _call(x, w, bias, a, b, scaling, ids)
    d_in, rank = x.shape[-1], a.shape[1]
    y, _, (wide, low, up) = ora.adapter_linear(x.reshape(-1, d_in), w, bias, a, b, scaling,
                                               ids.repeat_interleave(x.shape[1]))
    units = (d_in + 8) * (wide + low) + (rank + 8) * up
    f32 = 2.0 ** -24 * units + (2.0 ** -17 * up if dtype == torch.bfloat16 else 0.0)
    assert_within(got.reshape(y.shape), y, rounded(y, dtype) + f32 * (1 + 2.0 ** -7), "y")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,tokens", [(9, 1), (70, 1), (3, 60)])
def test_the_entry_point_without_a_product(batch, tokens, dtype):
    # the C entry with neither weight nor product: bias + c B A x alone
    x, w, bias, a, b, scaling, ids = _inputs(batch, tokens, 128, 72, 12, 4, dtype)
    xd, bd, ad, bbd, sd, idd = _dev(x, bias, a, b, scaling, ids)
    rows, y = batch * tokens, torch.full((batch * tokens, 72), 7.0, dtype=dtype, device=DEV)
    lib = _lib.load()
    args = _lib.AdapterArgs(xd.data_ptr(), None, ad.data_ptr(), bbd.data_ptr(), bd.data_ptr(), sd.data_ptr(),
                            idd.data_ptr(), y.data_ptr(), None, 0, rows, tokens, 128, 72, 12, 4, _lib.dtype_code(dtype), 1)
    ref = ctypes.addressof(args)
    args.workspace_bytes = lib.kda_adapter_linear_workspace_bytes(ref)
    workspace = torch.empty(max(1, args.workspace_bytes), dtype=torch.uint8, device=DEV)
    args.workspace = workspace.data_ptr()
    _lib.check(lib.kda_adapter_linear(ref, _lib.stream_of(y.device)))
    _, delta, (_, low, up) = ora.adapter_linear(x.reshape(rows, -1), w, bias, a, b, scaling, ids.repeat_interleave(tokens))
    f32 = 2.0 ** -24 * ((128 + 8) * low + (12 + 8) * up) + (2.0 ** -17 * up if dtype == torch.bfloat16 else 0.0)
    assert_within(y, delta, rounded(delta, dtype) + f32 * (1 + 2.0 ** -7), "y")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,tokens", [(4, 1), (40, 1), (4, 40), (1, 2100)])
def test_a_part_past_the_range_meets_a_product_that_brings_it_back(batch, tokens, dtype):
    # c B A x = 102400 (past f16's 65504), W x = -102400: all exact in f32, the bias is left
    x = torch.ones(batch, tokens, 64, dtype=dtype)
    w = torch.full((72, 64), -1600.0, dtype=dtype)
    a, b = torch.ones(1, 1, 64, dtype=dtype), torch.full((1, 72, 1), 800.0, dtype=dtype)
    bias = (torch.arange(72) / 8).to(dtype)
    got = _call(x, w, bias, a, b, torch.tensor([2.0]), torch.zeros(batch, dtype=torch.long))
    assert torch.equal(got.cpu(), bias.expand(batch, tokens, 72))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,tokens", [(1, 1), (20, 1), (3, 5), (2, 100), (1, 600)])
def test_all_rows_with_one_adapter_and_with_none(batch, tokens, dtype):
    x, w, bias, a, b, scaling, ids = _inputs(batch, tokens, 256, 96, 16, 4, dtype)
    for fill in (-1, 0, 3, -(1 << 20)):
        ids.fill_(fill)
        _check(x, w, bias, a, b, scaling, ids, _call(x, w, bias, a, b, scaling, ids), str(fill))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,order", [(90, "runs"), (90, "mixed"), (700, "runs"), (700, "mixed")])
def test_an_id_per_token(rows, order, dtype):
    # packed documents with an adapter each, and tokens in any order
    x, w, bias, a, b, scaling, _ = _inputs(1, rows, 128, 80, 16, 7, dtype)
    gen = torch.Generator().manual_seed(3)
    ids = torch.randint(-1, 7, (1, rows), generator=gen)
    if order == "runs":
        ids = torch.arange(rows)[None] * 9 // rows - 1  # the first run has none
        ids[ids > 6] = 2
    _check(x, w, bias, a, b, scaling, ids, _call(x, w, bias, a, b, scaling, ids))
    flat = _call(x[0], w, bias, a, b, scaling, ids[0])
    assert torch.equal(flat, _call(x, w, bias, a, b, scaling, ids)[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,tokens", [(12, 1), (12, 40), (150, 1)])
def test_rows_are_independent(batch, tokens, dtype):
    # an id past the stack is NaN in its own rows; another row's adapter or input that is not finite stays there
    x, w, bias, a, b, scaling, ids = _inputs(batch, tokens, 192, 70, 16, 5, dtype)
    ids = torch.arange(batch) % 4
    want = _call(x, w, bias, a, b, scaling, ids)
    bad = ids.clone()
    bad[3], bad[7] = 5, 1 << 30
    a2, b2 = a.clone(), b.clone()
    a2[4], b2[4] = float("inf"), float("nan")
    bad[5] = 4
    x2 = x.clone()
    x2[9] = float("nan")
    got = _call(x2, w, bias, a2, b2, scaling, bad)
    good = torch.ones(batch, dtype=torch.bool)
    good[[3, 5, 7, 9]] = False
    assert torch.equal(got[good], want[good])
    assert bool(got[~good].isnan().all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,tokens", [(6, 1), (60, 1), (6, 40)])
def test_infinities_stay_infinities(batch, tokens, dtype):
    # one infinite input, rank 1: every product of its row is an infinity of some sign
    x, w, bias, a, b, scaling, _ = _inputs(batch, tokens, 64, 64, 1, 3, dtype)
    ids = torch.arange(batch) % 3
    x[2, 0, 5] = float("inf")
    x[4, 0, 7] = float("-inf")
    got = _call(x, w, bias, a, b, scaling, ids).cpu().reshape(-1, 64)
    y, _, _ = ora.adapter_linear(x.reshape(-1, 64), w, bias, a, b, scaling, ids.repeat_interleave(tokens))
    assert bool(y.isinf().any())
    assert torch.equal(got.isnan(), y.isnan()) and torch.equal(got.isinf(), y.isinf())
    assert torch.equal(got[y.isinf()].sign().double(), y[y.isinf()].sign())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rank", [1, 40])
@pytest.mark.parametrize("batch,tokens", [(6, 1), (60, 1), (6, 40)])
def test_infinities_of_an_adapter_stay_infinities(batch, tokens, rank, dtype):
    # one infinite element of adapter 1's b and one of adapter 2's a: a single infinite term in a sum each
    x, w, bias, a, b, scaling, _ = _inputs(batch, tokens, 64, 64, rank, 3, dtype)
    ids = torch.arange(batch) % 3
    b[1, 7, rank - 1] = float("inf")
    a[2, rank - 1, 3] = float("-inf")
    got = _call(x, w, bias, a, b, scaling, ids).cpu().reshape(-1, 64)
    rows = ids.repeat_interleave(tokens)
    y, _, _ = ora.adapter_linear(x.reshape(-1, 64), w, bias, a, b, scaling, rows)
    assert bool(y[rows == 1][:, 7].isinf().all()) and bool(y[rows == 2].isinf().all())
    assert torch.equal(got.isnan(), y.isnan()) and torch.equal(got.isinf(), y.isinf())
    assert torch.equal(got[y.isinf()].sign().double(), y[y.isinf()].sign())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,tokens,most", [(7, 30, 64), (3, 100, 48), (90, 1, 40), (50, 16, 600)])
def test_more_rows_than_a_call_takes_are_served_in_pieces(batch, tokens, most, dtype, monkeypatch):
    # the limits of a real call are 2^27 rows: here a few, pieces of whole ids and inside one
    x, w, bias, a, b, scaling, ids = _inputs(batch, tokens, 128, 72, 16, 5, dtype)
    monkeypatch.setattr(adapters, "PIECE_ROWS", most)
    _check(x, w, bias, a, b, scaling, ids, _call(x, w, bias, a, b, scaling, ids))
    monkeypatch.setattr(adapters, "PIECE_ELEMENTS", 100)  # less than a row: one at a time
    if batch * tokens < 100:
        _check(x, w, bias, a, b, scaling, ids, _call(x, w, bias, a, b, scaling, ids))


@pytest.mark.parametrize("batch,tokens", [(4, 1), (50, 1), (3, 60)])
@pytest.mark.parametrize("to", [torch.bfloat16, torch.float16])
def test_autocast_takes_the_tensors_in_its_type(batch, tokens, to):
    x, w, bias, a, b, scaling, ids = _dev(*_inputs(batch, tokens, 64, 72, 8, 3, torch.float32))
    cast = lambda *ts: [t.to(to) for t in ts]  # noqa: E731
    xc, wc, bc, ac, bbc = cast(x, w, bias, a, b)
    want = adapters.adapter_linear(xc, wc, bc, adapters.AdapterStack(ac, bbc, scaling), ids)
    stack = adapters.AdapterStack(a, b, scaling)
    with torch.autocast("cuda", dtype=to):
        assert torch.nn.functional.linear(x, w, bias).dtype == to
        assert torch.equal(adapters.adapter_linear(x, w, bias, stack, ids), want)
        assert torch.equal(adapters.adapter_linear(xc, w, bc, stack, ids), want)
        with pytest.raises(RuntimeError, match="backward"):
            adapters.adapter_linear(x, w.clone().requires_grad_(), bias, stack, ids)
        with torch.autocast("cuda", enabled=False):
            full = adapters.adapter_linear(x, w, bias, stack, ids)
            assert full.dtype == torch.float32
            with pytest.raises(TypeError):
                adapters.adapter_linear(xc, w, bias, stack, ids)
    assert torch.equal(full, adapters.adapter_linear(x, w, bias, stack, ids))


@pytest.mark.parametrize("mode,tokens", [("chunkwise", 40), ("decode", 1)])
def test_a_layer_with_f32_projections_under_autocast(mode, tokens):
    d_model, H, K = 256, 2, 128
    weights = layer_weights(d_model, H, K, K, dtype=torch.bfloat16, biases=True, std=0.06)
    weights = {n: t.to(DEV) if isinstance(t, torch.Tensor) else t for n, t in weights.items()}
    names = ("q_proj", "k_proj", "v_proj", "gate_proj", "output_proj")
    gen = torch.Generator().manual_seed(8)
    rnd = lambda *s, std: (torch.randn(*s, generator=gen) * std).to(torch.bfloat16).to(DEV)  # noqa: E731
    stacks = {n: adapters.AdapterStack(rnd(3, 8, d_model, std=0.06), rnd(3, d_model, 8, std=0.1)) for n in names}
    wide = {n: adapters.AdapterStack(s.a.float(), s.b.float()) for n, s in stacks.items()}
    x, ids = rnd(4, tokens, d_model, std=1.0), torch.tensor([2, -1, 0, 1], device=DEV)
    lora = kda.adapters.KDALayerAdapters
    mask = torch.ones(4, tokens, dtype=torch.bool, device=DEV)  # the composed stages
    with torch.no_grad():
        want = kda_attention_forward(KDALayerWeights(**weights), x, mask, None, mode, adapters=lora(**stacks), adapter_ids=ids)
        w32 = KDALayerWeights(**{**weights, **{n: weights[n].float() for n in names}})
        with torch.autocast("cuda", dtype=torch.bfloat16):
            got = kda_attention_forward(w32, x.float(), mask, None, mode, adapters=lora(**wide), adapter_ids=ids)
    assert got.hidden_states.dtype == torch.bfloat16 and torch.equal(got.hidden_states, want.hidden_states)


@pytest.mark.parametrize("span", [8, 1 << 20])
def test_a_batch_past_one_piece(span):
    # 2^21 rows of 256 columns are a piece's 2^29 elements; rows on both sides of each border, and the last
    rows, d_in, d_out = (1 << 21) + 40, 64, 256
    rows = -(-rows // span) * span
    gen = torch.Generator(device=DEV).manual_seed(1)
    rnd = lambda *s, std=1.0: (torch.randn(*s, generator=gen, device=DEV) * std).to(torch.bfloat16)  # noqa: E731
    x, w, a, b = rnd(rows // span, span, d_in), rnd(d_out, d_in, std=0.1), rnd(5, 8, d_in, std=0.1), rnd(5, d_out, 8, std=0.3)
    ids = torch.randint(-1, 5, (rows // span,), generator=gen, device=DEV)
    y = adapters.adapter_linear(x, w, None, adapters.AdapterStack(a, b), ids).view(rows, d_out)
    pick = sorted({r for edge in (0, 1 << 20, 1 << 21, rows) for r in range(max(0, edge - 40), min(rows, edge + 40))})
    at = torch.tensor(pick, device=DEV)
    _check(x.view(rows, d_in)[at].cpu(), w.cpu(), None, a.cpu(), b.cpu(), None, ids[at // span].cpu(), y[at])


def test_layouts():
    x, w, bias, a, b, scaling, ids = _dev(*_inputs(6, 3, 96, 40, 8, 4, torch.bfloat16))
    stack = adapters.AdapterStack(a, b, scaling)
    want = adapters.adapter_linear(x, w, bias, stack, ids)
    wide = torch.zeros(6, 3, 200, dtype=x.dtype, device=DEV)
    wide[..., 51:147] = x
    odd = torch.zeros(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].copy_(x.flatten()).view(x.shape)
    flipped = adapters.AdapterStack(a.transpose(1, 2).contiguous().transpose(1, 2),
                                    torch.zeros(b.numel() + 1, dtype=b.dtype, device=DEV)[1:].copy_(b.flatten()).view(b.shape),
                                    torch.stack([scaling, scaling], 1)[:, 0])
    for xx, ww in ((wide[..., 51:147], w), (odd, w.t().contiguous().t()), (x, w)):
        got = adapters.adapter_linear(xx, ww, bias, flipped, torch.stack([ids, ids], 1)[:, 0])
        assert float((got.float() - want.float()).abs().max()) <= 2.0 ** -6 * float(want.float().abs().max())
    assert adapters.adapter_linear(x[:0], w, bias, stack, ids[:0]).shape == (0, 3, 40)
    assert adapters.adapter_linear(x[:, :0], w, bias, stack, ids).shape == (6, 0, 40)


def test_calls_repeat_bit_for_bit_on_two_streams():
    x, w, bias, a, b, scaling, ids = _dev(*_inputs(40, 1, 512, 256, 16, 9, torch.bfloat16))
    stack = adapters.AdapterStack(a, b, scaling)
    want = adapters.adapter_linear(x, w, bias, stack, ids)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(adapters.adapter_linear(x, w, bias, stack, ids))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("batch,tokens", [(24, 1), (3, 150)])
def test_captured_calls_replay_with_other_ids(batch, tokens):
    x, w, bias, a, b, scaling, ids = _dev(*_inputs(batch, tokens, 512, 256, 16, 9, torch.bfloat16))
    stack = adapters.AdapterStack(a, b, scaling)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        adapters.adapter_linear(x, w, bias, stack, ids)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = adapters.adapter_linear(x, w, bias, stack, ids)
    for seed in range(3):
        nx, *_, nids = _dev(*_inputs(batch, tokens, 512, 256, 16, 9, torch.bfloat16, seed=40 + seed))
        x.copy_(nx), ids.copy_(nids)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, adapters.adapter_linear(x, w, bias, stack, ids))


def _merged(weights, name, stack, n):
    """The weights with adapter n folded into one projection, in f64."""
    return weights[name].double() + float(stack.scaling[n]) * (stack.b[n].double() @ stack.a[n].double())


@pytest.mark.parametrize("mode,tokens", [("chunkwise", 70), ("decode", 1), ("recurrent", 3)])
def test_a_layer_with_adapters_is_the_layer_of_the_merged_weights(mode, tokens):
    d_model, H, K = 256, 2, 128
    weights = layer_weights(d_model, H, K, K, dtype=torch.float32, biases=True)
    w = KDALayerWeights(**{n: t.to(DEV) if isinstance(t, torch.Tensor) else t for n, t in weights.items()})
    gen = torch.Generator().manual_seed(2)
    names = ("q_proj", "k_proj", "v_proj", "gate_proj", "output_proj")
    stacks = {n: adapters.AdapterStack((torch.randn(3, 8, d_model, generator=gen) / 16).to(DEV),
                                       (torch.randn(3, d_model, 8, generator=gen) * 0.1).to(DEV),
                                       torch.rand(3, generator=gen).to(DEV)) for n in names}
    x = torch.randn(4, tokens, d_model, generator=gen)
    ids = torch.tensor([2, -1, 0, 2])
    got = kda_attention_forward(w, x.to(DEV), None, None, mode, True, adapters=kda.adapters.KDALayerAdapters(**stacks),
                                adapter_ids=ids.to(DEV))
    for i, n in enumerate(ids.tolist()):
        merged = {k: t.double() if isinstance(t, torch.Tensor) and k != "a_log" else t for k, t in weights.items()}
        if n >= 0:
            merged.update({k: _merged(weights, k, adapters.AdapterStack(s.a.cpu(), s.b.cpu(), s.scaling.cpu()), n)
                           for k, s in stacks.items()})
        out, state = ora.kda_layer(merged, x[i:i + 1].double(), None, None, mode, True)
        # f32 through the whole layer: the layer's own tolerance
        assert float((got.hidden_states[i].cpu().double() - out[0]).abs().max()) < 1e-4 * float(out.abs().max())
        assert float((got.state.recurrent_state[i].cpu().double() - state[0][0]).abs().max()) < \
            1e-4 * float(state[0].abs().max())
    # a projection without a stack keeps its plain product
    some = kda.adapters.KDALayerAdapters(q_proj=stacks["q_proj"])
    none = kda_attention_forward(w, x.to(DEV), None, None, mode, True, adapters=some,
                                 adapter_ids=torch.full((4,), -1, device=DEV))
    base = kda_attention_forward(w, x.to(DEV), None, None, mode, True)
    assert float((none.hidden_states - base.hidden_states).abs().max()) < 1e-4 * float(base.hidden_states.abs().max())


def test_a_served_request_end_to_end():
    # residual norm, a layer with adapters, its caches at rest in a pool, and on from there; bf16
    d_model, H, K = 256, 2, 128
    weights = layer_weights(d_model, H, K, K, dtype=torch.bfloat16)
    w = KDALayerWeights(**{n: t.to(DEV) if isinstance(t, torch.Tensor) else t for n, t in weights.items()})
    gen = torch.Generator().manual_seed(4)
    rnd = lambda *s, std=1.0: (torch.randn(*s, generator=gen) * std).to(torch.bfloat16).to(DEV)  # noqa: E731
    stack = adapters.AdapterStack(rnd(3, 16, d_model, std=0.06), rnd(3, d_model, 16, std=0.1))
    lora = kda.adapters.KDALayerAdapters(q_proj=stack, output_proj=stack)
    ids, norm_w = torch.tensor([1, -1, 2], device=DEV), rnd(d_model, std=0.1) + 1
    prompt, hidden = rnd(3, 50, d_model), rnd(3, 50, d_model)

    def block(x, r, state, mode):
        y, h = fused.add_rmsnorm(x, r, norm_w)
        out = kda_attention_forward(w, y, None, state, mode, True, adapters=lora, adapter_ids=ids)
        return out.hidden_states, h, out.state

    with torch.no_grad():
        out, h, state = block(prompt, hidden, None, "chunkwise")
        pool = cache.packed_pool([state], 8)
        slots = torch.tensor([6, 0, 3], device=DEV)
        cache.pack_states([state], out=pool, slots=slots)
        kept, rest = state, cache.unpack_states(pool, slots)[0]
        for step in range(4):
            x, r = rnd(3, 1, d_model), rnd(3, 1, d_model)
            a, _, kept = block(x, r, kept, "decode")
            b, _, rest = block(x, r, rest, "decode")
            q, scales, _ = fused.add_rmsnorm_quant(a, r, norm_w)
            y, _ = fused.add_rmsnorm(a, r, norm_w)
            # an 8-bit row is half an e4m3 step off at most
            assert bool(((q.float() * scales - y.float()).abs() <= y.float().abs() * 2.0 ** -3 + scales * 2.0 ** -9).all())
            assert bool(a.isfinite().all()) and bool(b.isfinite().all())
            # the states differ by the 8-bit rounding alone: a row is off by half its scale, and decays
            assert float((kept.recurrent_state - rest.recurrent_state).abs().max()) <= \
                float(pool[0].recurrent.scales[slots].max()) * K ** 0.5
            assert torch.equal(kept.sequence_offset, rest.sequence_offset)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("batch", [1, 5, 17, 32, 40])
@pytest.mark.parametrize("which", [("q_proj", "k_proj", "v_proj", "gate_proj", "output_proj"), ("v_proj",),
                                   ("k_proj", "output_proj"), ()])
def test_a_decode_step_with_adapters_is_the_composed_stages(batch, dtype, which):
    # up to 32 sequences run the native step, whose projections are the same kernels
    # as adapter_linear's; the stages around them round at the same places
    d_model, H, K = 256, 2, 128
    weights = layer_weights(d_model, H, K, K, dtype=dtype, biases=True, std=0.06)
    w = KDALayerWeights(**{n: t.to(DEV) if isinstance(t, torch.Tensor) else t for n, t in weights.items()})
    gen = torch.Generator().manual_seed(5)
    rnd = lambda *s, std=1.0: (torch.randn(*s, generator=gen) * std).to(dtype).to(DEV)  # noqa: E731
    stacks = {n: adapters.AdapterStack(rnd(4, 8 + 4 * i, d_model, std=0.06), rnd(4, d_model, 8 + 4 * i, std=0.1),
                                       torch.rand(4, generator=gen).to(DEV) if i % 2 else None)
              for i, n in enumerate(which)}
    lora = kda.adapters.KDALayerAdapters(**stacks)
    ids = torch.randint(-1, 4, (batch,), generator=gen).to(DEV)
    state = kda_attention_forward(w, rnd(batch, 9, d_model), None, None, "chunkwise", True).state
    x = rnd(batch, 1, d_model)
    mask = torch.ones(batch, 1, dtype=torch.bool, device=DEV)  # a mask keeps the composed stages
    want = kda_attention_forward(w, x, mask, state, "decode", adapters=lora, adapter_ids=ids)
    kept = state.recurrent_state.clone()
    got = kda_attention_forward(w, x, None, state, "decode", adapters=lora, adapter_ids=ids)
    assert torch.equal(state.recurrent_state, kept)
    tol = 4 * torch.finfo(dtype).eps  # a few roundings that may fall to the other side
    for a, b in ((got.hidden_states, want.hidden_states), (got.state.recurrent_state, want.state.recurrent_state),
                 (got.state.v_conv_state.buffer, want.state.v_conv_state.buffer)):
        assert float((a.double() - b.double()).abs().max()) <= tol * float(b.double().abs().max())
    assert torch.equal(got.state.sequence_offset, want.state.sequence_offset)
    again = kda_attention_forward(w, x, None, state, "decode", update_state_in_place=True, adapters=lora,
                                  adapter_ids=ids.int())
    assert again.state.recurrent_state is state.recurrent_state
    assert torch.equal(again.hidden_states, got.hidden_states)
    if which:
        bad = ids.clone()
        bad[0] = 99
        out = kda_attention_forward(w, x, None, want.state, "decode", adapters=lora, adapter_ids=bad).hidden_states
        assert bool(out[0].isnan().any()) and bool(out[1:].isfinite().all())


def test_a_captured_decode_step_with_adapters_replays_with_other_ids():
    d_model, H, K = 256, 2, 128
    weights = layer_weights(d_model, H, K, K, dtype=torch.bfloat16, std=0.06)
    w = KDALayerWeights(**{n: t.to(DEV) if isinstance(t, torch.Tensor) else t for n, t in weights.items()})
    gen = torch.Generator().manual_seed(6)
    rnd = lambda *s, std=1.0: (torch.randn(*s, generator=gen) * std).to(torch.bfloat16).to(DEV)  # noqa: E731
    stack = adapters.AdapterStack(rnd(4, 16, d_model, std=0.06), rnd(4, d_model, 16, std=0.1))
    lora = kda.adapters.KDALayerAdapters(q_proj=stack, output_proj=stack)
    ids = torch.tensor([1, 0, 3], device=DEV)
    state = kda_attention_forward(w, rnd(3, 9, d_model), None, None, "chunkwise", True).state
    x = rnd(3, 1, d_model)
    step = lambda: kda_attention_forward(w, x, None, state, "decode", adapters=lora, adapter_ids=ids)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for new in ([2, 2, 2], [-1, 3, 0], [0, -1, -1]):
        ids.copy_(torch.tensor(new))
        x.copy_(rnd(3, 1, d_model))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert torch.equal(out.hidden_states, want.hidden_states)
        assert torch.equal(out.state.recurrent_state, want.state.recurrent_state)

"""GPU parity of fused.add_rmsnorm, its backward and its 8-bit form against the f64 oracle.

Bounds (tests/_bounds.py).  A row's mean square sums D products over 256 (or
more) threads, ceil(D / 256) in a chain and ten joining steps; its rounding
enters y at half its size, with one for the mean, two for eps and the
reciprocal root (1 ulp), and two products: n = D / 512 + 16 units cover it.
The backward's row mean is a sum of that many terms of either sign, off by
twice that of the sum of their magnitudes.  A weight gradient is a sum over
the rows in chains of at most rows / 64 + 64 terms, each of four roundings.
"""

from __future__ import annotations

import pytest
import torch

from kda import fused
from oracle import kda_oracle as ora
from tests._bounds import assert_within, rounded, unit

pytestmark = pytest.mark.gpu
DEV = "cuda"
ALL = [torch.float32, torch.bfloat16, torch.float16, torch.float64]
SIZES = [(1, 1), (3, 7), (2, 64), (5, 100), (130, 128), (9, 512), (3, 1001), (70, 2048), (2, 4100), (33, 7168),
         (2, 9001), (1, 40000)]


def _rand(*shape, dtype, seed, scale=1.0, mean=0.0):
    gen = torch.Generator().manual_seed(seed)
    return (mean + torch.randn(*shape, generator=gen, dtype=torch.float64) * scale).to(dtype)


def _inputs(rows, width, dtype, seed=0):
    return (_rand(rows, width, dtype=dtype, seed=seed), _rand(rows, width, dtype=dtype, seed=seed + 1, scale=2.0),
            _rand(width, dtype=dtype, seed=seed + 2, scale=0.1, mean=1.0))


def _units(width, dtype):
    return (width / 512 + 16) * unit(dtype)


def _dev(t):
    return None if t is None else t.to(DEV)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("rows,width", SIZES)
@pytest.mark.parametrize("with_residual,with_weight", [(True, True), (False, True), (True, False)])
def test_add_rmsnorm_matches_oracle(rows, width, dtype, with_residual, with_weight):
    x, r, w = _inputs(rows, width, dtype)
    r, w = (r if with_residual else None), (w if with_weight else None)
    ref, ref_h = ora.add_rmsnorm(x, r, w)
    xd = _dev(x)
    y, h = fused.add_rmsnorm(xd, _dev(r), _dev(w))
    assert y.dtype == dtype and (h is xd if r is None else torch.equal(h.cpu(), ref_h))
    assert_within(y, ref, rounded(ref, dtype) + ref.abs() * _units(width, dtype), "y")


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("rows,width", SIZES + [(700, 256), (2500, 72)])
@pytest.mark.parametrize("with_residual,with_dh", [(True, True), (True, False), (False, True)])
def test_add_rmsnorm_gradients(rows, width, dtype, with_residual, with_dh):
    x, r, w = _inputs(rows, width, dtype)
    r = r if with_residual else None
    dy, dh = _rand(rows, width, dtype=dtype, seed=5), _rand(rows, width, dtype=dtype, seed=6)
    leaves = [t.to(DEV).requires_grad_() for t in (x, r, w) if t is not None]
    xd, rd, wd = leaves if r is not None else (leaves[0], None, leaves[1])
    y, h = fused.add_rmsnorm(xd, rd, wd)
    outs, grads = ((y, h), (_dev(dy), _dev(dh))) if with_dh and r is not None else ((y,), (_dev(dy),))
    got = torch.autograd.grad(outs, leaves, grads)
    _, hs = ora.add_rmsnorm(x, r, w)
    up = dh if len(outs) == 2 else None
    dx, dw = ora.add_rmsnorm_backward(hs, w, dy, up)
    hd, wdy = hs.double(), dy.double() * w.double()
    s = 1 / torch.sqrt(hd.square().mean(-1, keepdim=True) + 1e-6)
    terms = s * wdy.abs() + hd.abs() * s ** 3 * (wdy * hd).abs().mean(-1, keepdim=True)
    if up is not None:
        terms = terms + up.double().abs()
    bound = rounded(dx, dtype) + 3 * _units(width, dtype) * terms
    for t in got[:-1]:
        assert_within(t, dx, bound, "dx")
    sums = (dy.double() * hd * s).abs().sum(0)
    assert_within(got[-1], dw, rounded(dw, dtype) + (rows / 64 + 68 + width / 512 + 16) * unit(dtype) * sums, "dw")


def test_add_rmsnorm_gradients_against_differences():
    x, r, w = _inputs(3, 37, torch.float64)
    leaves = [t.to(DEV).requires_grad_() for t in (x, r, w)]
    assert torch.autograd.gradcheck(lambda *t: fused.add_rmsnorm(*t), leaves)
    assert torch.autograd.gradcheck(lambda a, b: fused.add_rmsnorm(a, None, b)[0], [leaves[0], leaves[2]])
    assert torch.autograd.gradcheck(lambda a, b: fused.add_rmsnorm(a, b, None), leaves[:2])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,width", [(3, 7), (40, 512), (9, 1001), (5, 7168), (1500, 264), (2, 40000)])
def test_a_weight_in_f32_beside_16_bit_tensors(rows, width, dtype):
    x, r, _ = _inputs(rows, width, dtype)
    w = _rand(width, dtype=torch.float32, seed=9, scale=0.1, mean=1.0)
    dy = _rand(rows, width, dtype=dtype, seed=5)
    leaves = [t.to(DEV).requires_grad_() for t in (x, r, w)]
    y, h = fused.add_rmsnorm(*leaves)
    got = torch.autograd.grad(y, leaves, dy.to(DEV))
    ref, hs = ora.add_rmsnorm(x, r, w)
    assert y.dtype == dtype and got[2].dtype == torch.float32
    assert_within(y, ref, rounded(ref, dtype) + ref.abs() * _units(width, dtype), "y")
    dx, dw = ora.add_rmsnorm_backward(hs, w, dy, None)
    hd, wdy = hs.double(), dy.double() * w.double()
    s = 1 / torch.sqrt(hd.square().mean(-1, keepdim=True) + 1e-6)
    terms = s * wdy.abs() + hd.abs() * s ** 3 * (wdy * hd).abs().mean(-1, keepdim=True)
    for t in got[:2]:
        assert_within(t, dx, rounded(dx, dtype) + 3 * _units(width, dtype) * terms, "dx")
    sums = (dy.double() * hd * s).abs().sum(0)
    assert_within(got[2], dw, (rows / 64 + 68 + width / 512 + 16) * 2.0 ** -24 * sums, "dw")
    with torch.no_grad():
        q, scales, _ = fused.add_rmsnorm_quant(*leaves)
    quotients, ref_scales = ora.e4m3_groups(ref, width)
    assert_within(scales, ref_scales, ref_scales * (_units(width, dtype) + 2.0 ** -23), "scales")
    assert float((q.float().cpu() - quotients).abs().max()) <= 448 * 2.0 ** -4 * 1.1


def test_gradients_of_inputs_that_are_used_twice_and_partly():
    # the sum is its own residual, and only one of the outputs is used
    x = _rand(4, 96, dtype=torch.float64, seed=3).to(DEV).requires_grad_()
    assert torch.autograd.gradcheck(lambda t: fused.add_rmsnorm(t, t)[0], [x])
    y, h = fused.add_rmsnorm(x, x.detach())
    (g,) = torch.autograd.grad(h, x, torch.ones_like(h))
    assert torch.equal(g, torch.ones_like(x))
    x.grad = None
    r = _rand(4, 96, dtype=torch.float64, seed=4).to(DEV).requires_grad_()
    y, h = fused.add_rmsnorm(x, r)
    (y.sum() + h.sum()).backward()
    gx = x.grad.clone()
    r.grad.zero_()  # the two gradients are tensors of their own
    assert torch.equal(x.grad, gx) and bool(gx.abs().sum() > 0)
    y, _ = fused.add_rmsnorm(x, r)
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_weight_gradient_is_the_same_every_time():
    x, r, w = (t.to(DEV).requires_grad_() for t in _inputs(3000, 520, torch.bfloat16))
    dy = _rand(3000, 520, dtype=torch.bfloat16, seed=8).to(DEV)
    first = None
    for _ in range(4):
        y, _ = fused.add_rmsnorm(x, r, w)
        got = torch.autograd.grad(y, (x, w), dy)
        first = got if first is None else first
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_layouts_and_leading_dimensions():
    dtype = torch.bfloat16
    x, r, w = _inputs(24, 200, dtype)
    ref, _ = fused.add_rmsnorm(*(t.to(DEV) for t in (x, r, w)))
    wide = torch.zeros(24, 301, dtype=dtype, device=DEV)
    wide[:, 33:233] = x.to(DEV)
    y, h = fused.add_rmsnorm(wide[:, 33:233], r.to(DEV).t().contiguous().t(), w.to(DEV))
    assert torch.equal(y, ref) and y.shape == (24, 200)
    # a base address that is off every vector
    flat = torch.zeros(24 * 200 + 1, dtype=dtype, device=DEV)[1:].copy_(x.to(DEV).flatten()).view(2, 3, 4, 200)
    y, h = fused.add_rmsnorm(flat, r.to(DEV).view(2, 3, 4, 200), w.to(DEV))
    assert torch.equal(y.view(24, 200), ref) and y.shape == (2, 3, 4, 200)
    y, h = fused.add_rmsnorm(x[0].to(DEV), None, w.to(DEV))
    assert y.shape == (200,)
    for empty in (torch.zeros(0, 64, device=DEV), torch.zeros(3, 0, 64, device=DEV)):
        y, h = fused.add_rmsnorm(empty, empty)
        assert y.shape == empty.shape and h.shape == empty.shape
        q, scales, _ = fused.add_rmsnorm_quant(empty, group_size=32)
        assert q.shape == empty.shape and scales.shape == (*empty.shape[:-1], 2)
    e = torch.zeros(0, 64, device=DEV, requires_grad=True)
    we = torch.ones(64, device=DEV, requires_grad=True)
    fused.add_rmsnorm(e, None, we)[0].sum().backward()
    assert torch.count_nonzero(we.grad) == 0 and e.grad.shape == e.shape


@pytest.mark.parametrize("width", [64, 1001, 2048])
def test_rows_of_zeros_and_non_finite_values(width):
    x, r, w = _inputs(6, width, torch.float32)
    x[0], r[0] = 0, 0
    x[1, 3], x[2, 5], x[3, 0] = float("inf"), float("-inf"), float("nan")
    ref, _ = ora.add_rmsnorm(x, r, w)
    y, _ = fused.add_rmsnorm(x.to(DEV), r.to(DEV), w.to(DEV))
    assert_within(y, ref, rounded(ref, torch.float32) + ref.abs() * _units(width, torch.float32), "y")
    q, scales, _ = fused.add_rmsnorm_quant(x.to(DEV), r.to(DEV), w.to(DEV))
    q, scales = q.float().cpu(), scales.cpu()
    assert torch.count_nonzero(q[0]) == 0 and float(scales[0]) == 0
    assert bool(scales[1:4].isnan().all()) and bool(scales[4:].isfinite().all()) and bool(q[4:].isfinite().all())
    if width % 32 == 0:  # a group without a NaN keeps its values
        _, scales, _ = fused.add_rmsnorm_quant(x.to(DEV), r.to(DEV), w.to(DEV), group_size=32)
        assert bool(scales[1:4, 0].isnan().all()) and torch.count_nonzero(scales[1:3, 1:].cpu()) == 0


QUANT_SIZES = [(1, 1, None), (3, 7, None), (2, 64, None), (2, 64, 64), (1, 32, 32), (3, 1001, None), (5, 352, 32),
               (70, 2048, None), (70, 2048, 128), (9, 2048, 256), (2, 4160, 64), (33, 7168, None), (33, 7168, 128),
               (2, 9001, None), (1, 40000, None), (1, 40000, 64)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,width,group", QUANT_SIZES)
@pytest.mark.parametrize("with_residual", [True, False])
def test_add_rmsnorm_quant_matches_oracle(rows, width, group, dtype, with_residual):
    x, r, w = _inputs(rows, width, dtype)
    r = r if with_residual else None
    y, ref_h = ora.add_rmsnorm(x, r, w)
    quotients, ref_scales = ora.e4m3_groups(y, group or width)
    xd = _dev(x)
    q, scales, h = fused.add_rmsnorm_quant(xd, _dev(r), _dev(w), group_size=group)
    assert q.dtype == torch.float8_e4m3fn and scales.dtype == torch.float32
    assert h is xd if r is None else torch.equal(h.cpu(), ref_h)
    units = _units(width, dtype) + 2 * unit(dtype)
    assert_within(scales, ref_scales, ref_scales * units, "scales")
    # half an e4m3 step: 2^-4 of the value, 2^-10 below the smallest normal one
    step = torch.maximum(quotients.abs() * 2.0 ** -4, torch.full_like(quotients, 2.0 ** -10))
    assert_within(q.float(), quotients, step * (1 + 2.0 ** -4) * (1 + units) + quotients.abs() * 2 * units, "q")
    # the largest value of a group is the type's largest
    assert torch.equal(q.float().cpu().unflatten(-1, (-1, group or width)).abs().amax(-1),
                       torch.full(ref_scales.shape, 448.0))


def test_tiny_groups_read_back_as_zeros():
    x = torch.ones(2, 64, device=DEV)
    w = torch.full((64,), 1e-31, device=DEV)  # under 2^-100
    w[32:] = 1e-29  # over it
    q, scales, _ = fused.add_rmsnorm_quant(x, None, w, group_size=32)
    assert torch.count_nonzero(q[:, :32].float()) == 0 and torch.count_nonzero(scales[:, 0]) == 0
    assert bool((q[:, 32:].float() == 448).all())


def test_captured_calls_replay_and_streams_are_followed():
    x, r, w = (t.to(DEV) for t in _inputs(300, 2048, torch.bfloat16))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fused.add_rmsnorm(x, r, w), fused.add_rmsnorm_quant(x, r, w, group_size=128)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h = fused.add_rmsnorm(x, r, w)
        q, scales, hq = fused.add_rmsnorm_quant(h, y, w, group_size=128)
    for seed in range(3):
        nx, nr, _ = _inputs(300, 2048, torch.bfloat16, seed=20 + seed)
        x.copy_(nx), r.copy_(nr)
        graph.replay()
        torch.cuda.synchronize()
        ey, eh = fused.add_rmsnorm(x, r, w)
        eq, es, ehq = fused.add_rmsnorm_quant(eh, ey, w, group_size=128)
        for a, b in ((y, ey), (h, eh), (q.float(), eq.float()), (scales, es), (hq, ehq)):
            assert torch.equal(a, b)


# A launch has fewer than 2^32 threads: 64 or 256 of them a row here.
@pytest.mark.parametrize("dtype,rows,width", [(torch.bfloat16, (1 << 25) + 5, 2), (torch.float64, (1 << 23) + 3, 1)])
def test_more_rows_than_a_launch_holds(dtype, rows, width):
    gen = torch.Generator(DEV).manual_seed(3)
    x, r, dy = (torch.randn(rows, width, generator=gen, device=DEV, dtype=torch.float32).to(dtype) for _ in range(3))
    w = _dev(_rand(width, dtype=dtype, seed=4, scale=0.1, mean=1.0)).requires_grad_()
    x.requires_grad_()
    y, h = fused.add_rmsnorm(x, r, w)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    cut = rows - 1000
    x2, r2, dy2 = (t.detach()[cut:].clone() for t in (x, r, dy))
    w2 = w.detach().clone().requires_grad_()
    x2.requires_grad_()
    y2, h2 = fused.add_rmsnorm(x2, r2, w2)
    dx2, = torch.autograd.grad(y2, [x2], dy2)
    assert torch.equal(y[cut:], y2) and torch.equal(h[cut:], h2) and torch.equal(dx[cut:], dx2)
    ref, _ = ora.add_rmsnorm(x2.detach().cpu(), r2.cpu(), w2.detach().cpu())
    assert_within(y2.detach().cpu(), ref, rounded(ref, dtype) + ref.abs() * _units(width, dtype), "y of the last rows")
    if dtype == torch.float64:  # the reference sums in f64 too: twice the bound of a sum over the rows
        h = h.detach()
        terms = dy * h * (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
        assert_within(dw.cpu(), terms.sum(0).cpu(), 2 * (rows / 64 + 68) * unit(dtype) * terms.abs().sum(0).cpu(), "dw")


def test_more_rows_than_a_launch_holds_in_8_bits():
    rows, width = (1 << 25) + 5, 4
    gen = torch.Generator(DEV).manual_seed(5)
    x = torch.randn(rows, width, generator=gen, device=DEV, dtype=torch.float32).to(torch.bfloat16)
    q, scales, _ = fused.add_rmsnorm_quant(x)
    cut = rows - 1000
    q2, scales2, _ = fused.add_rmsnorm_quant(x[cut:].clone())
    assert torch.equal(q[cut:].view(torch.uint8), q2.view(torch.uint8)) and torch.equal(scales[cut:], scales2)


@pytest.mark.parametrize("x_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width,group", [(256, 32), (1024, None), (4096, 128), (16896, 256), (20480, None), (33024, 64)])
def test_quotients_next_to_ties_are_those_of_the_division(width, group, x_dtype):
    # rows of +-1 have a mean square of 1 and, with an eps under half a step, a norm of exactly 1, so y
    # is +-weight: each group's largest magnitude m, and values within two f32 steps of where m's
    # quotients lie in the middle of two e4m3 values.  The definition in f32, bit for bit.
    gen = torch.Generator().manual_seed(width)
    n = group or width
    groups = width // n
    e4m3 = torch.arange(0x01, 0x7f, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    ties = (e4m3[1:] + e4m3[:-1]) / 2
    m = (1 + torch.rand(groups, 1, generator=gen)) * torch.exp2(torch.randint(-20, 20, (groups, 1), generator=gen).float())
    scale = m / 448
    pick = ties[torch.randint(0, ties.numel(), (groups, n), generator=gen)]
    near = (pick.double() * scale.double()).float()
    steps = torch.randint(-2, 3, (groups, n), generator=gen)
    near = (near.view(torch.int32) + steps.int()).view(torch.float32).minimum(m)
    near[:, n // 3] = m[:, 0]
    w = near.flatten()
    signs = torch.randint(0, 2, (3, width), generator=gen).float() * 2 - 1
    want = (w.view(groups, n) / scale * signs.view(3, groups, n)).to(torch.float8_e4m3fn).view(3, width)
    q, scales, _ = fused.add_rmsnorm_quant(signs.to(x_dtype).to(DEV), None, w.to(DEV), 2.0 ** -40, group_size=group)
    assert torch.equal(scales.cpu(), scale.view(1, groups).expand(3, groups))
    assert torch.equal(q.cpu().view(torch.uint8), want.view(torch.uint8))

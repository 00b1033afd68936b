"""Error bounds shared by the operator tests: tolerances that count roundings.

A value rounded once to a type is off by at most half a step, ``eps / 2`` of
its magnitude (or half the smallest subnormal step); an f32 computation of n
roundings in a chain adds n * 2^-24 of the magnitude of its terms, an f64
one n * 2^-53.
"""

from __future__ import annotations

import torch


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def unit(dtype: torch.dtype) -> float:
    """Half a step of the arithmetic type of tensors of `dtype`."""
    return 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24


def assert_within(actual: torch.Tensor, expected: torch.Tensor, bound: torch.Tensor, what: str) -> None:
    """|actual - expected| <= bound elementwise, NaN where NaN is expected."""
    a, e = actual.detach().double().cpu(), expected.double()
    assert a.shape == e.shape, f"{what}: shape {tuple(a.shape)}, expected {tuple(e.shape)}"
    nan = e.isnan()
    assert torch.equal(a.isnan(), nan), f"{what}: NaN in other places"
    same = (a == e) | nan
    over = ((a - e).abs() - bound).masked_fill(same, 0.0)
    if over.numel():
        worst = int(over.argmax())
        assert float(over.max()) <= 0, (f"{what}: {float(a.flatten()[worst])} against {float(e.flatten()[worst])}, "
                                        f"{float(over.max())} over the bound")


def rounded(expected: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The bound of one rounding of `expected` to `dtype`."""
    info = torch.finfo(dtype)
    return expected.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2

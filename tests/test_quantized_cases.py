"""The tests' definition of a cache in 4 bits (CPU)."""

import numpy as np
import pytest
import torch

from tests.quantized_cases import quantize, values


def test_ties_go_to_the_even_code():
    x = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.5, 7.0, -0.25, -0.75, -5.0] + [0.0] * 20, dtype=torch.bfloat16)
    codes, exponents = quantize(x)
    assert exponents.tolist() == [127] and codes[:12].tolist() == [0, 2, 2, 4, 4, 6, 6, 7, 7, 8, 10, 14]


@pytest.mark.parametrize("top,e", [(7.0, 0), (7.0625, 1), (3.5, -1), (3.515625, 0), (1.0, -2), (2.0**-133, -127), (2.0**-125, -127), (3.38e38, 126)])
def test_the_smallest_exponent(top, e):
    x = torch.zeros(32, dtype=torch.bfloat16)
    x[7] = top
    assert quantize(x)[1].tolist() == [e + 127]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_what_is_held_is_near_and_of_the_type(dtype):
    g = torch.Generator().manual_seed(0)
    big = torch.finfo(dtype).max
    x = torch.cat([torch.randn(60, 64, generator=g) * torch.logspace(-6, 3, 60)[:, None], (torch.rand(20, 64, generator=g) * 2 - 1) * big]).to(dtype)
    codes, exponents = quantize(x)
    held, scale = values(codes, exponents), 2.0 ** (np.repeat(exponents.astype(float), 32, axis=-1) - 127)
    assert torch.equal(held.to(dtype).double(), held)
    off, size = (held - x.double()).abs().numpy() / scale, x.double().abs().numpy() / scale
    step = np.where(size <= 2, 0.25, np.where(size <= 4, 0.5, 1.0))
    assert (off[:60] <= step[:60]).all() and (off * scale <= 0.25 * size.max(1, keepdims=True) * scale + 1e-30).all()
    none = x[:1].clone()
    none[0, 3], none[0, 40] = float("inf"), float("nan")
    assert torch.isnan(values(*quantize(none))).all()

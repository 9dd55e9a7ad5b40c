"""GELU's far negative side, where the output is h times a small probability: to the outputs' own rounding.

Tolerance (set before the first run). One product of 1 keeps h exact. The probability's fit is good to 2^-15.4 of itself,
and its exponential's argument, up to 104, is rounded three times in float32: 2^-16. So 2^-14 of the value beside the
rounding of the type (2^-8, 2^-11; 2^-25 for a subnormal float16)."""
import math

import pytest
import torch

from conftest import sub

pytestmark = pytest.mark.gpu

fd = sub("enhancers.fused_dense")


@pytest.mark.parametrize("dtype,unit,least", [(torch.bfloat16, 2.0 ** -8, 0.0), (torch.float16, 2.0 ** -11, 2.0 ** -25)])
def test_gelu_tail(native, dtype, unit, least):
    h = -torch.linspace(0.5, 12.0 if dtype == torch.bfloat16 else 6.0, 4001, device="cuda").to(dtype)
    ones = torch.ones(8, 1, device="cuda", dtype=dtype)
    y = fd.dense(h[:, None], ones, act="gelu").double()
    d = h.double()[:, None]
    want = 0.5 * d * torch.special.erfc(-d / math.sqrt(2))
    assert bool(((y - want).abs() <= (unit + 2.0 ** -14) * want.abs() + least).all()), \
        float((((y - want).abs() - least) / want.abs()).max())

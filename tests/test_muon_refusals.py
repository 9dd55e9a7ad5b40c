"""What an orthogonalised update refuses before anything has changed (CPU only: no kernel is launched)."""
import ctypes
import math

import pytest
import torch

from conftest import sub

native, fm = sub("_native"), sub("enhancers.fused_muon")


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("place", [(0,), (1,), (2,), (1, 2), (0, 1, 2)])
def test_coefficients_that_are_no_numbers(bad, place):
    # a NaN is lost in a maximum, so it has to be asked for: a step with one would make every parameter NaN
    abc = [bad if i in place else c for i, c in enumerate(fm.COEFFICIENTS)]
    held = (ctypes.c_double * 3)(*abc)
    assert native.lib().wf_orthogonalize(None, 0, 8, 9, 1, 5, held, 1e-7, None, 0, None) == native.EINVAL
    assert "coefficients" in native.last_error()
    assert native.lib().wf_muon(None, 0, 8, 9, 1, 0.9, 1, 1.0, 0.1, 5, held, 1e-7, None, 0, None) == native.EINVAL
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="coefficients"):
        fm.orthogonalize(x, coefficients=abc)
    with pytest.raises(ValueError, match="coefficients"):
        fm.muon_step([], [], [], coefficients=abc)
    with pytest.raises(ValueError, match="coefficients"):
        fm.Muon([torch.nn.Parameter(x)], coefficients=abc)


@pytest.mark.parametrize("good", [fm.COEFFICIENTS, (1.5, -0.5, 0.0), (2.0, -1.5, 0.5), (1.0, 0.0, 0.0), (-1.0, 0.0, -0.0)])
def test_bounded_coefficients_are_taken(good):
    held = (ctypes.c_double * 3)(*good)
    for steps in (1, 5, 32):
        assert native.lib().wf_orthogonalize(None, 0, 8, 9, 1, steps, held, 1e-7, None, 0, None) == native.OK, good

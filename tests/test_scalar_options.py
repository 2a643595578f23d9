"""Numbers among the kernels' options that fp32 does not hold are refused as others are, whatever their type (CPU only)."""

from __future__ import annotations

import math
import warnings

import pytest

from tensor_amd.kernels import builtin

OPTIONS = [("rms_norm", "eps"), ("rms_norm_fp8", "eps"), ("paged_attention", "scale")]


@pytest.mark.parametrize("kernel,option", OPTIONS)
@pytest.mark.parametrize("value", [10 ** 400, -10 ** 400, 10 ** 39, 1e39, -1e39, 3.5e38, math.inf, -math.inf, math.nan, 0, 0.0, -1,
                                   True, "1.0"], ids=lambda v: str(v)[:12])
def test_refused(kernel, option, value):
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        with pytest.raises(ValueError, match=option):
            builtin.manifest(kernel, **{option: value})


@pytest.mark.parametrize("kernel,option", OPTIONS)
@pytest.mark.parametrize("value", [1, 10 ** 38, 3.4e38, 1.5, 2.0 ** -100])
def test_taken(kernel, option, value):
    assert builtin.manifest(kernel, **{option: value})

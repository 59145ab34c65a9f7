"""Numbers that the dense operators refuse since what is formed of them would not fit: through the C ABI on a CUDA runtime that runs nothing."""
import pytest

import pim_dl_asplos_b200 as P
from test_dense_refusals import _attention, _call, lib, needs_objects  # noqa: F401


@needs_objects
@pytest.mark.parametrize("scale", [3e38, -2.4e38])
def test_a_scale_that_is_infinite_times_log2_e(lib, scale):  # noqa: F811
    p = _attention(lib.at)
    p.scale = scale
    rc, log = _call(lib, "lutamm_attention", p)
    assert rc == P.EINVAL and not log and b"scale" in _error(lib)


@needs_objects
@pytest.mark.parametrize("scale", [2.3e38, -2.3e38, 0.0, 1e-45])
def test_the_largest_and_smallest_scales_are_taken(lib, scale):  # noqa: F811
    p = _attention(lib.at)
    p.scale = scale
    assert _call(lib, "lutamm_attention", p)[0] == P.OK


def _error(lib):  # noqa: F811
    return lib.lutamm_last_error(lib.ctx)

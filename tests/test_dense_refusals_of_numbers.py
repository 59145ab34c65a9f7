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


@needs_objects
def test_an_output_that_covers_more_than_addresses_count(lib):  # noqa: F811
    """2^25 steps of 2^39 elements are 2^64: they must not count as none, and the axes with them as lying apart."""
    p = _attention(lib.at)
    p.batch, p.queries, p.heads, p.kv_heads = (1 << 25) + 1, 1 << 14, 1, 1
    step = 1 << 39
    p.out.head_stride, p.out.token_stride, p.out.batch_stride = 0, step, step
    p.q.token_stride = p.q.batch_stride = p.k.batch_stride = p.v.batch_stride = 0
    rc, log = _call(lib, "lutamm_attention", p)
    assert rc == P.EINVAL and not log

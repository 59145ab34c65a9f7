"""GPU checks of attention where its inputs differ in size by far more than half the bits tell apart."""
import math

import pytest
import torch

import dense_oracle as O

pytestmark = pytest.mark.gpu
ROWS = [1, 3, 6, 20, 100, 200]   # one, few and many rows: every kernel and form


def _inputs(seed, Q, K, D, H=1):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(1, n, H, D, generator=gen) for n in (Q, K, K)]


def _run(ctx, q, k, v, first=None, lengths=None, **kw):
    out = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
    i32 = lambda t: None if t is None else torch.tensor(t, dtype=torch.int32).cuda()   # noqa: E731
    ctx.attention(q.cuda(), k.cuda(), v.cuda(), out, first=i32(first), lengths=i32(lengths), **kw)
    return out.cpu()


def _fill_tensor_memory(ctx, value=1e37):
    """Leaves large numbers all over tensor memory."""
    t = torch.full((1, 64, 300, 128), value, dtype=torch.bfloat16, device="cuda")
    ctx.attention(torch.zeros_like(t), torch.zeros_like(t), t, torch.empty_like(t))


@pytest.mark.parametrize("Q", ROWS)
@pytest.mark.parametrize("D", [8, 40, 64, 80, 112])
def test_what_other_kernels_left_in_tensor_memory(ctx, Q, D):
    """Values that fall from tile to tile while scores rise, after kernels that left zeros and large numbers there: equal calls give equal bits."""
    q, k, v = _inputs(D, Q, 256, D)
    q[..., 0] = 4.0
    for tile in range(4):
        k[0, 64 * tile:64 * tile + 64, 0, 0] = 20.0 * (tile - 2) * math.sqrt(D) / 4
        v[0, 64 * tile:64 * tile + 64] *= 2.0 ** (-30 * (tile % 2))
    outs = []
    for value in (0.0, 1e37, 1e-3):
        _fill_tensor_memory(ctx, value)
        outs.append(_run(ctx, q, k, v))
    assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.parametrize("Q", ROWS)
def test_a_tile_of_large_values_that_half_of_the_rows_do_not_see(ctx, Q):
    """Values of 1e-27 in one tile, of 1e30 in the next: rows that see the first alone have theirs."""
    q, k, v = _inputs(7, Q, 128, 64)
    v[0, :64] *= 1e-27
    v[0, 64:] *= 1e30
    first = 63 - Q // 2
    got, want = _run(ctx, q, k, v, first=[first], window=(63, 0)), O.attention(q, k, v, None, (63, 0), 0, None, [first])
    rows = max(0, min(Q, 64 - first))
    # fp32 all the way: 64 products and sums of a score and its exponential, 64 of the result
    O.close(got[:, :rows], want[:, :rows], torch.float32, floor=256 * 2.0 ** -24 * float(v[0, :64].abs().amax()))
    assert got.isfinite().all()

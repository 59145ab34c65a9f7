"""GPU checks of attention where its inputs differ in size by far more than half the bits tell apart: outliers in a column, keys that some rows of a tile do
not see, values that change from tile to tile, results
near the type's largest number, infinities.  Bounds of each element by itself: attention_bound.py."""
import math

import pytest
import torch

import attention_bound as A
import dense_oracle as O

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
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


@pytest.mark.parametrize("Q", ROWS)
@pytest.mark.parametrize("D", [8, 64, 80, 128])
@pytest.mark.parametrize("outlier", [1e4, 1e6, 1e9])
def test_a_large_column_leaves_the_others_their_digits(ctx, Q, D, outlier):
    q, k, v = _inputs(D + Q, Q, 260, D)
    v[..., 3] *= outlier
    k[..., 5] *= outlier
    q[..., 5] = 0
    A.check(_run(ctx, q, k, v), *A.attention(q, k, v))
    q, k, v = _inputs(D + Q, Q, 260, D)
    q[..., 5] *= outlier
    k[..., 5] /= outlier
    A.check(_run(ctx, q, k, v), *A.attention(q, k, v))


@pytest.mark.parametrize("Q", ROWS)
@pytest.mark.parametrize("D", [40, 64, 128])
@pytest.mark.parametrize("large", [1e4, 1e9, 1e30])
def test_a_large_key_that_other_rows_see(ctx, Q, D, large):
    """Rows in front of it do not see it, and have what they would have without it; the ones behind do."""
    K = Q + 70
    q, k, v = _inputs(D, Q, K, D)
    at = 70 + Q // 2
    v[0, at] *= large
    k[0, at] *= large
    window = (64, 0)
    got, (want, bound) = _run(ctx, q, k, v, first=[70], window=window), A.attention(q, k, v, window=window, first=[70])
    before = Q // 2
    A.check(got[:, :before], want[:, :before], bound[:, :before])
    k[0, at] /= large
    got, (want, bound) = _run(ctx, q, k, v, first=[70], window=window), A.attention(q, k, v, window=window, first=[70])
    A.check(got, want, bound)


@pytest.mark.parametrize("Q", ROWS)
@pytest.mark.parametrize("D", [8, 40, 64, 80, 112])
@pytest.mark.parametrize("drop", [10, 20, 30, 40])
def test_values_that_fall_while_scores_rise(ctx, Q, D, drop):
    """Large values of small weight in one tile, small values of large weight in the next; tensor memory holds large numbers from before."""
    q, k, v = _inputs(D + drop, Q, 256, D)
    q[..., 0] = 4.0
    for tile in range(4):
        k[0, 64 * tile:64 * tile + 64, 0, 0] = 20.0 * (tile - 2) * math.sqrt(D) / 4
        v[0, 64 * tile:64 * tile + 64] *= 2.0 ** (-drop * (tile % 2))
    want, bound = A.attention(q, k, v)
    first = None
    for _ in range(3):
        _fill_tensor_memory(ctx)
        got = _run(ctx, q, k, v)
        A.check(got, want, bound)
        assert first is None or torch.equal(got, first)
        first = got


@pytest.mark.parametrize("Q", ROWS)
@pytest.mark.parametrize("small,large", [(1e-27, 1e30), (1e-25, 1e37), (1e30, 1e-27), (1e37, 1e-25)])
def test_values_of_two_ends_of_the_range(ctx, Q, small, large):
    """One tile of values, then one of another size that half of the rows do not see."""
    q, k, v = _inputs(7, Q, 128, 64)
    v[0, :64] *= small
    v[0, 64:] *= large
    first = [63 - Q // 2]
    A.check(_run(ctx, q, k, v, first=first, window=(63, 0)), *A.attention(q, k, v, window=(63, 0), first=first))


@pytest.mark.parametrize("Q,K,H,G,D", [(1, 300, 2, 2, 64), (4, 200, 2, 1, 128), (17, 500, 3, 3, 80), (64, 64, 2, 2, 64), (128, 128, 3, 3, 64), (197, 197, 2, 2, 64), (300, 300, 1, 1, 64),
                                       (100, 400, 4, 2, 128), (200, 200, 1, 1, 32), (130, 1000, 1, 1, 64), (9, 4000, 2, 2, 64)])
@pytest.mark.parametrize("window,sinks", [((-1, -1), 0), ((50, 50), 3)])
def test_the_error_of_random_numbers(ctx, Q, K, H, G, D, window, sinks):
    gen = torch.Generator().manual_seed(Q + K)
    q, k, v = torch.randn(2, Q, H, D, generator=gen), torch.randn(2, K, G, D, generator=gen), torch.randn(2, K, G, D, generator=gen)
    first = [K - Q, (K - Q) // 2]
    assert A.rms(_run(ctx, q, k, v, first=first, window=window, sinks=sinks), O.attention(q, k, v, None, window, sinks, None, first)) <= A.RMS
    v = v.abs()   # of one sign: what is lost towards zero adds up
    assert A.rms(_run(ctx, q, k, v, first=first, window=window, sinks=sinks), O.attention(q, k, v, None, window, sinks, None, first)) <= A.RMS


@pytest.mark.parametrize("Q", ROWS)
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("D,K", [(64, 130), (128, 700)])
def test_values_near_the_types_largest(ctx, Q, dtype, D, K):
    t = TYPES[dtype]
    q, k, v = _inputs(3, Q, K, D)
    q, k, v = (q / 4).to(t), k.to(t), (1e36 * (1 + v.abs() / 4)).to(t)
    got, (want, bound) = _run(ctx, q, k, v), A.attention(q, k, v)
    # (16-bit weights are rounded once)
    A.check(got, want, bound + (0 if t == torch.float32 else torch.finfo(t).eps / 2 * want.abs()), dtype=t)
    biggest = torch.full_like(v, 3.3e38)
    got = _run(ctx, q, k, biggest)
    A.check(got, biggest[:, :1].double().expand(got.shape), (24 + K / 4) * A.U * biggest[:, :1].double() * (1 if t == torch.float32 else 2.0 ** 16), dtype=t)


@pytest.mark.parametrize("Q", ROWS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 80])
def test_values_that_are_not_finite(ctx, Q, dtype, D):
    """An infinity or NaN in a value shows in the rows that see its key, in its column, and nowhere else."""
    t, K = TYPES[dtype], Q + 130
    q, k, v = (x.to(t) for x in _inputs(Q + D, Q, K, D))
    q = q / 2
    window, first = (100, 0), [K - Q]
    clean = v.clone()
    inf = float("inf")
    spots = [(K - 1, 0, inf), (K - 1 - Q // 2, 1, inf), (K - 1 - Q // 2, 2, -inf), (K - 2, D - 1, float("nan")), (K - Q // 2 - 3, 3, inf), (K - Q // 2 - 5, 3, -inf), (K - Q - 90, 4, -inf),
             (0, 5, inf)]
    for key, col, value in spots:
        v[0, key, 0, col] = value
    got = _run(ctx, q, k, v, first=first, window=window)
    seen = O.visible(Q, K, K, first[0], window, 0).double()
    finite = v[0, :, 0].isfinite()
    expected = O.attention(q, k, torch.where(v.isfinite(), v, torch.zeros((), dtype=t)), None, window, 0, None, first)
    plus, minus, nan = (seen @ m.double() > 0 for m in (v[0, :, 0] == inf, v[0, :, 0] == -inf, v[0, :, 0].isnan()))
    assert plus.any() and (seen @ (~finite).double() > 0).any() and not finite.all()
    for i in range(Q):
        for c in range(D):
            x = float(got[0, i, 0, c])
            if nan[i, c] or (plus[i, c] and minus[i, c]):
                assert math.isnan(x), (i, c, x)
            elif plus[i, c]:
                assert x == inf, (i, c, x)
            elif minus[i, c]:
                assert x == -inf, (i, c, x)
    plain = ~(plus | minus | nan)[None, :, None]
    floor = 0.0 if t == torch.float32 else 2 * torch.finfo(t).eps * float(clean.double().abs().amax())
    O.close(torch.where(plain, got, torch.zeros((), dtype=t)), torch.where(plain, expected, 0.0), t, floor=floor + 2 ** -18)


@pytest.mark.parametrize("Q", ROWS)
@pytest.mark.parametrize("dtype", TYPES)
def test_a_whole_tile_of_infinities(ctx, Q, dtype):
    t = TYPES[dtype]
    q, k, v = (x.to(t) for x in _inputs(Q, Q, 200, 64))
    v[0, 64:128] = float("inf")
    assert (_run(ctx, q / 4, k, v) == float("inf")).all()
    v[0, 70] = float("nan")
    assert _run(ctx, q / 4, k, v).isnan().all()


@pytest.mark.parametrize("Q", ROWS)
@pytest.mark.parametrize("dtype", TYPES)
def test_keys_and_queries_that_are_not_finite(ctx, Q, dtype):
    """A score of minus infinity is a key without weight; one of plus infinity, or NaN, is NaN in its row; others have what they had."""
    t, K = TYPES[dtype], Q + 130
    q, k, v = (x.to(t) for x in _inputs(Q + 1, Q, K, 64))
    inf = float("inf")
    q[..., 0] = q[..., 0].abs() + 0.5
    q[..., 1] = -q[..., 1].abs() - 0.5
    if Q > 2:
        q[0, Q // 3, 0, 0] = inf       # a row of its own: scores of plus or minus infinity
        q[0, Q // 2, 0, 7] = float("nan")
    k[0, K - Q - 70, 0, 0] = -inf
    k[0, K - 1, 0, 1] = inf            # the last row alone sees it
    k[0, K - 1 - Q // 4, 0, 0] = inf
    for window in ((-1, 0), (90, 0)):
        got = _run(ctx, q, k, v, first=[K - Q], window=window)
        seen = O.visible(Q, K, K, K - Q, window, 0)
        for i in range(Q):
            at = seen[i].nonzero()[:, 0]
            s = (k[0, at, 0].double() @ q[0, i, 0].double()) / 8
            w = torch.softmax(s, 0)
            want = torch.full((64,), float("nan")) if w.isnan().any() else w @ v[0, at, 0].double()
            assert torch.equal(got[0, i, 0].isnan(), want.isnan()), (window, i)
            if not want.isnan().any():
                O.close(got[0, i, 0], want, t, floor=2 ** -18 + (0.0 if t == torch.float32 else 2 * torch.finfo(t).eps * float(v.double().abs().amax())))


# ------------------------------------------------------------------------------------------------ CTAs of 256 rows
def _run_many(ctx, q, k, v, **kw):
    """One head's inputs as those of 150 heads, which gives every SM a CTA of 256 rows: the first one's results, which are the others', too."""
    got = _run(ctx, *(t.cuda().expand(-1, -1, 150, -1) for t in (q, k, v)), **kw)
    assert all(torch.equal(got[:, :, h].view(torch.int32), got[:, :, 0].view(torch.int32)) for h in range(1, 150))
    return got[:, :, :1]


@pytest.mark.parametrize("S,length,window,sinks", [(129, 129, (40, 10), 70), (197, 190, (64, 64), 1), (300, 300, (5, 0), 0), (512, 300, (128, 128), 1), (700, 700, (64, 0), 130),
                                                   (700, 3, (700, 700), 0), (700, 650, (0, 0), 0), (520, 520, (1, 200), 4), (257, 0, (3, 3), 0)])
@pytest.mark.parametrize("D", [8, 40, 64])
def test_two_tiles_of_rows(ctx, S, length, window, sinks, D):
    q, k, v = _inputs(S + D, S, S, D)
    want, bound = A.attention(q, k, v, window=window, sinks=sinks, lengths=[length])
    got = _run_many(ctx, q, k, v, lengths=[length], window=window, sinks=sinks)
    A.check(got, want, bound)
    if length:
        assert A.rms(got, want) <= A.RMS
    v[..., 3] *= 1e6
    want, bound = A.attention(q, k, v, window=window, sinks=sinks, lengths=[length])
    A.check(_run_many(ctx, q, k, v, lengths=[length], window=window, sinks=sinks), want, bound)


@pytest.mark.parametrize("large", [1e4, 1e9, 1e30])
def test_two_tiles_of_rows_and_a_large_key(ctx, large):
    q, k, v = _inputs(5, 300, 300, 64)
    v[0, 140] *= large
    A.check(_run_many(ctx, q, k, v, window=(30, 10)), *A.attention(q, k, v, window=(30, 10)))
    k[0, 140] *= large
    want, bound = A.attention(q, k, v, window=(30, 10))
    got = _run_many(ctx, q, k, v, window=(30, 10))
    for rows in (slice(0, 130), slice(171, 300)):
        A.check(got[:, rows], want[:, rows], bound[:, rows])


def test_two_tiles_of_rows_and_infinities(ctx):
    inf, nan = float("inf"), float("nan")
    q, k, v = _inputs(6, 300, 300, 64)
    q /= 2
    spots = {(0, 0): inf, (127, 1): -inf, (140, 2): nan, (140, 3): inf, (299, 4): inf, (200, 5): -inf}
    clean = v.clone()
    for (key, col), value in spots.items():
        v[0, key, 0, col], clean[0, key, 0, col] = value, 0
    got = _run_many(ctx, q, k, v, window=(30, 10))
    want, bound = A.attention(q, k, clean, window=(30, 10))
    seen = O.visible(300, 300, 300, 0, (30, 10), 0)
    for (key, col), value in spots.items():
        at = seen[:, key]
        assert (got[0, at, 0, col].isnan() if math.isnan(value) else got[0, at, 0, col] == value).all()
        got[0, at, 0, col] = want[0, at, 0, col].float()
    A.check(got, want, bound)
    k[0, 150, 0, 7] = -inf     # queries of one sign there: a key without weight for them, NaN for the others
    q[0, 100, 0, 9] = nan
    got = _run_many(ctx, q, k, clean, window=(30, 10))
    nans = seen[:, 150] & (q[0, :, 0, 7] < 0)
    nans[100] = True
    assert torch.equal(got[0, :, 0].isnan().all(1), nans) and torch.equal(got[0, :, 0].isnan().any(1), nans)
    k[0, 150, 0, 7] = 0
    hidden = torch.where((seen[:, 150] & (q[0, :, 0, 7] > 0))[:, None], 1, 0)[:, 0].bool()
    want, bound = A.attention(q, k, clean, window=(30, 10))
    A.check(got[:, ~(nans | hidden)], want[:, ~(nans | hidden)], bound[:, ~(nans | hidden)])
@pytest.mark.parametrize("Q", ROWS)
@pytest.mark.parametrize("D", [64, 128])
def test_scores_far_below_zero(ctx, Q, D):
    """A key whose score passes fp32's range downwards has no weight; large queries on small keys are like others."""
    q, k, v = _inputs(Q + D, Q, 150, D)
    for size in (1e9, 1e25):
        x, y = q.abs() * size, k / size
        y[0, 77] = -1e30 * (1 + k[0, 77].abs())
        want, bound = A.attention(x, torch.cat([y[:, :77], y[:, 78:]], 1), torch.cat([v[:, :77], v[:, 78:]], 1))
        A.check(_run(ctx, x, y, v), want, bound)


# ------------------------------------------------------------------------------------------------ large scores
@pytest.mark.parametrize("Q", ROWS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [1e3, 1e5, 1e8, 1e12])
@pytest.mark.parametrize("sign", [1, -1])
def test_the_largest_of_large_scores(ctx, Q, dtype, size, sign):
    """Scores so far apart that one key has all the weight: its value is the result, whatever the scores' size and sign."""
    t, K, D = TYPES[dtype], 200, 64
    size = min(size, 1e4) if t == torch.float16 else size
    q, k, v = _inputs(Q + 5, Q, K, D)
    q, k = (q * size).to(t), (k * size).to(t)
    if sign < 0:     # all scores below zero
        q, k = q.abs(), -k.abs()
    v = v.to(t)
    s = q[0, :, 0].double() @ k[0, :, 0].double().T / 8
    first, second = s.topk(2, 1).values.unbind(1)
    a = q[0, :, 0].double().abs() @ k[0, :, 0].double().abs().T / 8
    clear = first - second > torch.clamp(a.amax(1) * 2.0 ** -16, min=120)    # beyond what sums of 64 products in fp32 leave
    assert clear.sum() * 2 > Q or Q < 4
    got = _run(ctx, q, k, v)[0, :, 0]
    assert got.isfinite().all()
    # out = (p v) / p with one weight p, between 1/2 and 1: fp32's parts of p v are added up with four units lost at most, and rounded, as are 1 / p and its product
    # (8 units; 16 are allowed); 16-bit types round p once, and the result, half a step each
    O.close(got[clear], v[0, s.argmax(1)[clear], 0], t, steps=16.0 if t == torch.float32 else 2.0)


# ------------------------------------------------------------------------------------------------ 16-bit types
@pytest.mark.parametrize("Q,K,H,G,D", [(1, 300, 2, 2, 64), (4, 200, 2, 1, 128), (17, 500, 3, 3, 80), (64, 64, 2, 2, 64), (197, 197, 2, 2, 64), (100, 400, 4, 2, 128), (9, 1000, 2, 2, 64)])
@pytest.mark.parametrize("window,sinks", [((-1, -1), 0), ((50, 50), 3)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_half_the_bits_are_rounded_once(ctx, Q, K, H, G, D, window, sinks, dtype):
    """The result's own rounding, half a step, and of weights what their second part leaves: the square of half a step, at most a step of
    2^-24 where fp16's ends."""
    t = TYPES[dtype]
    gen = torch.Generator().manual_seed(Q + K)
    q, k, v = (torch.randn(1, n, h, D, generator=gen).to(t) for n, h in ((Q, H), (K, G), (K, G)))
    want, bound = A.attention(q, k, v, window=window, sinks=sinks, first=[K - Q])
    size = A.attention(q, k, v.abs(), window=window, sinks=sinks, first=[K - Q])[0]     # sum of w |v|
    half = torch.finfo(t).eps / 2
    A.check(_run(ctx, q, k, v, first=[K - Q], window=window, sinks=sinks), want, bound + (half * half + (2.0 ** -24 if t == torch.float16 else 0)) * size, dtype=t)


@pytest.mark.parametrize("Q", [20, 64])
@pytest.mark.parametrize("dtype", TYPES)
def test_sums_over_hundreds_of_thousands_of_keys(ctx, Q, dtype):
    """Equal weights, values of one sign: what is lost towards zero at each step would add up."""
    t, K = TYPES[dtype], 400000
    gen = torch.Generator().manual_seed(Q)
    v = (1 + torch.rand(1, K, 1, 64, generator=gen)).to(t).cuda()
    q, k = torch.zeros(1, Q, 150, 64, dtype=t, device="cuda"), torch.zeros(1, 1, 1, 64, dtype=t, device="cuda")
    out = torch.empty_like(q)
    ctx.attention(q, k.expand(-1, K, 150, -1), v.expand(-1, -1, 150, -1), out)
    want = v.double().mean(1, keepdim=True).cpu()
    # sums of some thousand tiles, each rounded to nearest, of tiles or some dozens of them, which lose up to two units at each of eight steps a tile
    O.close(out, want.expand(out.shape), t, floor=(512 + math.sqrt(K / 64)) * 2.0 ** -24 * 2)

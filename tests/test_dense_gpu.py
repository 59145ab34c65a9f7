"""GPU checks of the layer's dense operators - layer norm with its gradients, rotary positions, attention with a window - against
their definitions in 64 bits (dense_oracle.py), at the sizes, strides and masks where they can go wrong.

Tolerances: half a step of the output's type for its one rounding, and what fp32 arithmetic on the way may leave, counted in units u = 2^-24
per operation (the bounds stand at each check)."""
import itertools
import math

import pytest
import torch

import dense_oracle as O
import pim_dl_asplos_b200 as P

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rows(rows, width, dtype, stride, shift, gen, scale=1.0, offset=0.0):
    """A [rows, width] view at `shift` elements into a buffer whose rows are `stride` apart, on the GPU, and the buffer."""
    flat = torch.randn(rows * stride + shift, generator=gen) * scale + offset
    flat = flat.to(dtype).cuda()
    return flat[shift:shift + rows * stride].view(rows, stride)[:, :width], flat


# ------------------------------------------------------------------------------------------------ layer norm
SHAPES = [(1, 1, 1, 0), (3, 7, 7, 0), (5, 8, 8, 0), (4, 128, 128, 0), (9, 130, 131, 1), (130, 768, 768, 0), (33, 768, 2304, 768), (17, 769, 769, 0),
          (7, 1024, 1024, 0), (6, 1023, 1024, 1), (5, 1999, 1999, 0), (4, 2560, 2560, 0), (3, 5120, 5121, 0), (2, 8192, 8192, 0), (2, 8200, 8200, 0),
          (2, 9001, 9001, 0), (1, 20000, 20000, 0), (700, 64, 64, 0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,stride,shift", SHAPES)
def test_layer_norm(ctx, rows, width, stride, shift, dtype):
    t, gen = TYPES[dtype], _gen(rows * 7 + width)
    x, _ = _rows(rows, width, t, stride, shift, gen, 2.0, 0.5)
    r, _ = _rows(rows, width, t, stride + 3, 0, gen)
    w, b = torch.randn(width, generator=gen).cuda(), torch.randn(width, generator=gen).cuda()
    for res, wt, bs in ((None, w, b), (r, w, b), (r, None, None), (None, w, None)):
        buf = torch.full((rows, stride), 7.0, dtype=t, device="cuda")
        out, stats = buf[:, :width], torch.full((rows, 2), float("nan"), device="cuda")
        ctx.layer_norm(x, wt, bs, out, eps=1e-5, residual=res, stats=stats)
        want, mean, rstd = O.layer_norm(x.cpu(), None if wt is None else wt.cpu(), None if bs is None else bs.cpu(), 1e-5, None if res is None else res.cpu())
        # a sum runs through at most 40 elements of a thread (three passes of 512 x 8 for the longest), 5 exchanges and 16 warps
        n = 96
        xs = x.double().cpu()
        spread = (xs.abs().amax() + 1) * rstd.amax() * (1 if wt is None else wt.abs().amax().item()) + 3
        O.close(out, want, t, floor=float(n * U * spread))
        O.close(stats[:, 0], mean, torch.float32, floor=n * U * float(xs.abs().amax()))
        O.close(stats[:, 1], rstd, torch.float32, floor=2 * n * U * float(rstd.amax() * (1 + xs.abs().amax() * rstd.amax())))
        if stride > width:
            assert (buf[:, width:] == 7).all()


def test_layer_norm_in_place_constant_rows_and_nan(ctx):
    x = torch.randn(40, 768, generator=_gen(1)).cuda()
    x[3] = 2.5                                  # variance 0
    x[5, 7] = float("nan")
    x[6, 0] = float("inf")
    r = torch.randn(40, 768, generator=_gen(2)).cuda()
    fine = [i for i in range(40) if i not in (5, 6)]
    want = O.layer_norm(x.cpu(), None, None, 1e-6, r.cpu())[0]
    out = torch.empty_like(x)
    ctx.layer_norm(x, None, None, out, residual=r)
    assert out[5].isnan().all() and out[6].isnan().all()
    O.close(out[fine], want[fine], torch.float32, floor=96 * U * 10)
    y, z = x.clone(), r.clone()
    ctx.layer_norm(y, None, None, y, residual=r)
    ctx.layer_norm(x, None, None, z, residual=z)
    assert torch.equal(y[fine], out[fine]) and torch.equal(z[fine], out[fine])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,stride,shift", SHAPES + [(5000, 256, 256, 0), (3001, 1024, 1024, 0)])
def test_layer_norm_backward(ctx, rows, width, stride, shift, dtype):
    t, gen = TYPES[dtype], _gen(rows * 5 + width)
    x, _ = _rows(rows, width, t, stride, shift, gen, 2.0, 0.5)
    dy, _ = _rows(rows, width, t, stride + 1, 1, gen)
    w = torch.randn(width, generator=gen).cuda()
    stats = torch.stack(O.layer_norm(x.cpu(), None, None, 1e-5)[1:], 1).float().cuda()
    for wt, wanted in ((w, (1, 1, 1)), (None, (1, 1, 1)), (w, (1, 0, 0)), (w, (0, 1, 0)), (w, (0, 0, 1))):
        buf = torch.full((rows, stride), 7.0, dtype=t, device="cuda")
        dx = buf[:, :width] if wanted[0] else None
        dw, db = (torch.full((width,), float("nan"), device="cuda") if f else None for f in wanted[1:])
        ctx.layer_norm_backward(dy, x, wt, stats, dx, dw, db)
        want = O.layer_norm_backward(dy.cpu(), x.cpu(), None if wt is None else wt.cpu(), stats.cpu())
        d, st = dy.double().cpu(), stats.double().cpu()
        xh = (x.double().cpu() - st[:, :1]) * st[:, 1:]
        big = float(st[:, 1].amax() * d.abs().amax() * (1 if wt is None else wt.abs().amax().item()) * (1 + xh.abs().amax()) ** 2)
        off = float((x.double().cpu().abs() * st[:, 1:]).amax() + 1)   # x - mean loses this much of u
        if dx is not None:
            O.close(dx, want[0], t, floor=96 * U * big * off)
        # sums over rows: each term and each addition rounds once, the longest chain is at most the number of rows and 40
        chain = min(rows, 4000) + 40
        if dw is not None:
            O.close(dw, want[1], torch.float32, floor=float((chain + off) * U * (d * xh).abs().sum(0).amax()) + 1e-30)
        if db is not None:
            O.close(db, want[2], torch.float32, floor=float(chain * U * d.abs().sum(0).amax()) + 1e-30)
        if stride > width and dx is not None:
            assert (buf[:, width:] == 7).all()


@pytest.mark.parametrize("width", [33, 768, 1999, 8192, 8200, 9001])
def test_layer_norm_backward_in_place(ctx, width):
    """dx over x or over dout: the bits of dx elsewhere, dweight's and dbias's too."""
    gen, rows = _gen(width), 37
    x, dy = torch.randn(rows, width, generator=gen).cuda(), torch.randn(rows, width, generator=gen).cuda()
    w, stats = torch.randn(width, generator=gen).cuda(), torch.empty(rows, 2, device="cuda")
    ctx.layer_norm(x, w, None, torch.empty_like(x), stats=stats)
    def grads(dy, x, dx):
        dw, db = torch.empty(width, device="cuda"), torch.empty(width, device="cuda")
        ctx.layer_norm_backward(dy, x, w, stats, dx, dw, db)
        return dx, dw, db
    want = grads(dy, x, torch.empty_like(x))
    over_x, over_dy = x.clone(), dy.clone()
    for got in (grads(dy, over_x, over_x), grads(over_dy, x, over_dy)):
        assert all(torch.equal(g, r) for g, r in zip(got, want))


def test_layer_norm_backward_against_differences(ctx):
    """dx, dw and db of a weighted sum of outputs against central differences of the forward formula in 64 bits."""
    gen = _gen(3)
    x, w, b, dy = (torch.randn(*s, generator=gen).double() for s in ((3, 24), (24,), (24,), (3, 24)))
    stats = torch.empty(3, 2, device="cuda")
    out = torch.empty(3, 24, device="cuda")
    ctx.layer_norm(x.float().cuda(), w.float().cuda(), b.float().cuda(), out, eps=1e-5, stats=stats)
    dx, dw, db = torch.empty(3, 24, device="cuda"), torch.empty(24, device="cuda"), torch.empty(24, device="cuda")
    ctx.layer_norm_backward(dy.float().cuda(), x.float().cuda(), w.float().cuda(), stats, dx, dw, db)
    x, w, b, dy = (t.float().double() for t in (x, w, b, dy))
    h = 1e-5

    def loss():
        return float((O.layer_norm(x, w, b, 1e-5)[0] * dy).sum())

    for t, g in ((x, dx), (w, dw), (b, db)):
        flat, grad = t.view(-1), g.cpu().double().view(-1)
        for i in range(0, flat.numel(), 5):
            keep = float(flat[i])
            flat[i] = keep + h
            up = loss()
            flat[i] = keep - h
            down = loss()
            flat[i] = keep
            # differences in 64 bits are off by h^2 times the third derivative (below 10^3 here) and 2^-52 / h of the loss
            assert abs((up - down) / (2 * h) - float(grad[i])) < 1e-6 + 200 * U * 30


def test_layer_norm_without_rows_and_repeated(ctx):
    e = torch.empty(0, 16, device="cuda")
    w = torch.ones(16, device="cuda")
    ctx.layer_norm(e, w, w, e, stats=torch.empty(0, 2, device="cuda"))
    dw, db = torch.full((16,), 5.0, device="cuda"), torch.full((16,), 5.0, device="cuda")
    ctx.layer_norm_backward(e, e, w, torch.empty(0, 2, device="cuda"), e, dw, db)
    assert (dw == 0).all() and (db == 0).all()
    x, dy = torch.randn(3000, 768, generator=_gen(4)).cuda(), torch.randn(3000, 768, generator=_gen(5)).cuda()
    stats, out = torch.empty(3000, 2, device="cuda"), torch.empty_like(x)
    w = torch.randn(768, generator=_gen(6)).cuda()
    ctx.layer_norm(x, w, w, out, stats=stats)
    first = None
    for workspace in (None, None, torch.empty(ctx.layer_norm_backward_workspace(3000, 768), dtype=torch.uint8, device="cuda")):
        got = [torch.empty_like(x), torch.empty(768, device="cuda"), torch.empty(768, device="cuda")]
        ctx.layer_norm_backward(dy, x, w, stats, *got, workspace=workspace)
        assert first is None or all(torch.equal(a, b) for a, b in zip(first, got))
        first = got


# ------------------------------------------------------------------------------------------------ rotary positions
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved,inverse", list(itertools.product([False, True], [False, True])))
@pytest.mark.parametrize("B,S,H,extra,dim,sections", [(1, 1, 1, 0, 2, (1,)), (2, 5, 3, 0, 64, (16, 16)), (3, 197, 24, 12, 64, (16, 16)), (1, 33, 4, 0, 128, (16, 24, 24)),
                                                      (2, 9, 5, 0, 80, (20, 20)), (1, 7, 2, 1, 48, (8, 0, 8, 4)), (2, 3, 3, 0, 33, (5, 6)), (1, 300, 2, 0, 8, (4,)), (1, 4, 1, 0, 4096, (2048,))])
def test_rotary(ctx, B, S, H, extra, dim, sections, interleaved, inverse, dtype):
    t, gen = TYPES[dtype], _gen(S * 3 + dim)
    whole = torch.randn(B, S, H + extra, dim, generator=gen).to(t).cuda()
    x = whole[:, :, :H]
    pairs = sum(sections)
    freq = (10000.0 ** -(torch.arange(pairs) / pairs)).float().cuda()
    for far, per_sequence in ((64, False), (2 ** 31 - 1, True)):
        pos = torch.randint(-far, far, (B, S, len(sections)), generator=gen, dtype=torch.int32).cuda()
        if not per_sequence:
            pos = pos[0]
        out = torch.full((B, S, H, dim), float("nan"), dtype=t, device="cuda")
        ctx.rotary(x, pos, freq, sections, out, interleaved=interleaved, inverse=inverse)
        p64 = pos.cpu() if per_sequence else pos.cpu().expand(B, -1, -1)
        want = O.rotary(x.cpu(), p64, freq.cpu(), sections, interleaved, inverse)
        # cos and sin within 3 u (2 ulp at most 1, and the rest's product), two products and a sum; far angles: 2^31 turns of 2^-53 each
        O.close(out, want, t, floor=float((8 * U + (3e-6 if per_sequence else 0)) * 2 * x.abs().amax().double().cpu()))
        assert torch.equal(out[..., 2 * pairs:], x[..., 2 * pairs:])
        y = whole.clone()
        ctx.rotary(y[:, :, :H], pos, freq, sections, y[:, :, :H], interleaved=interleaved, inverse=inverse)
        assert torch.equal(y[:, :, :H], out) and torch.equal(y[:, :, H:], whole[:, :, H:])
    # heads first in memory, and an unaligned start
    flat = torch.zeros(B * S * H * dim + 1, dtype=t, device="cuda")
    z = flat[1:].view(B, H, S, dim).transpose(1, 2)
    ctx.rotary(x, pos, freq, sections, z, interleaved=interleaved, inverse=inverse)
    assert torch.equal(z, out)


def test_rotary_back_is_its_inverse_and_its_gradient(ctx):
    gen = _gen(8)
    x, g = torch.randn(2, 11, 3, 64, generator=gen).cuda(), torch.randn(2, 11, 3, 64, generator=gen).cuda()
    pos = torch.randint(0, 1000, (11, 2), generator=gen, dtype=torch.int32).cuda()
    freq = (100.0 ** -(torch.arange(32) / 32)).cuda()
    y, back, gx = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    ctx.rotary(x, pos, freq, (16, 16), y)
    ctx.rotary(y, pos, freq, (16, 16), back, inverse=True)
    O.close(back, x, torch.float32, floor=16 * U * 2 * float(x.abs().amax()))
    ctx.rotary(g, pos, freq, (16, 16), gx, inverse=True)
    leaf = x.cpu().double().requires_grad_()
    (O.rotary(leaf, pos.cpu().expand(2, -1, -1), freq.cpu(), (16, 16)) * g.cpu().double()).sum().backward()
    O.close(gx, leaf.grad, torch.float32, floor=8 * U * 2 * float(g.abs().amax()))


# ------------------------------------------------------------------------------------------------ attention
def _attention_floor(q, k, v, t, scale):
    """Of a score: a rounding for each of the head's products and sums, of the split into two f16 numbers and of the dropped product of
    their rests (four together); of a weight: twice that, exp2's 2 units in 2^-22, a rounding of the type it is multiplied in
    and one for each key summed; of a result: these times the largest value."""
    d, n = q.shape[-1], k.shape[1]
    s = float(scale * (q.double().abs().amax() * k.double().abs().amax()) * d) if n else 0.0
    typical = s / math.sqrt(d)   # of random signs; the products of one score do not all have the largest size
    weight = 2 * (d + 8) * U * typical + 2 ** -20 + (min(n, 4096) + 32) * U
    if t != torch.float32:
        weight += torch.finfo(t).eps
    return weight * (float(v.double().abs().amax()) if n else 0.0) + 1e-30


def _check_attention(ctx, B, Q, K, H, G, D, t, window=(-1, -1), sinks=0, lengths=None, first=None, scale=None, seed=0, layout="plain"):
    gen = _gen(seed + B + Q * 3 + K * 5 + D)
    if layout == "fused":
        qkv = torch.randn(B, K, 3, H, D, generator=gen).to(t).cuda()
        q, k, v = qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2]
    elif layout == "heads first":
        q = torch.randn(B, H, Q, D, generator=gen).to(t).cuda().transpose(1, 2)
        k, v = (torch.randn(B, G, K, D, generator=gen).to(t).cuda().transpose(1, 2) for _ in range(2))
    elif layout == "odd":   # nothing starts on 16 bytes
        q = torch.randn(B * Q * H * (D + 1) + 1, generator=gen).to(t).cuda()[1:].view(B, Q, H, D + 1)[..., :D]
        k, v = (torch.randn(B * K * G * (D + 3) + 3, generator=gen).to(t).cuda()[3:].view(B, K, G, D + 3)[..., :D] for _ in range(2))
    else:
        q = torch.randn(B, Q, H, D, generator=gen).to(t).cuda()
        k, v = (torch.randn(B, K, G, D, generator=gen).to(t).cuda() for _ in range(2))
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32).cuda()
    at = None if first is None else torch.tensor(first, dtype=torch.int32).cuda()
    out = torch.full((B, Q, H, D + 2), 7.0, dtype=t, device="cuda")
    ctx.attention(q, k, v, out[..., :D], scale=scale, window=window, sinks=sinks, lengths=ln, first=at)
    want = O.attention(q.cpu(), k.cpu(), v.cpu(), scale, window, sinks, lengths, first)
    O.close(out[..., :D], want, t, floor=_attention_floor(q, k, v, t, 1 / math.sqrt(D) if scale is None else scale))
    assert (out[..., D:] == 7).all()
    packed = torch.empty(B, Q, H, D, dtype=t, device="cuda")
    ctx.attention(q, k, v, packed, scale=scale, window=window, sinks=sinks, lengths=ln, first=at)
    again = torch.empty_like(packed)
    ctx.attention(q, k, v, again, scale=scale, window=window, sinks=sinks, lengths=ln, first=at)
    assert torch.equal(packed, again)
    O.close(packed, want, t, floor=_attention_floor(q, k, v, t, 1 / math.sqrt(D) if scale is None else scale))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K,lengths,window,sinks", [
    (1, None, (-1, -1), 0), (2, [2, 1, 0], (-1, 0), 0), (63, [63, 1, 40], (-1, -1), 0), (64, None, (10, 0), 3), (65, [65, 64, 63], (0, 0), 0), (200, [200, 3, 0], (7, 0), 2),
    (1000, [1000, 500, 129], (100, 0), 64), (4097, [4097, 4000, 17], (2047, 0), 8), (5000, [6000, -3, 5000], (-1, -1), 0), (333, None, (0, 0), 400)])
@pytest.mark.parametrize("Q,H,G,D", [(1, 1, 1, 64), (1, 12, 12, 64), (1, 4, 1, 128), (1, 16, 2, 32), (3, 2, 2, 80), (2, 6, 2, 8), (5, 3, 1, 64), (4, 8, 1, 128), (3, 11, 1, 72)])
def test_attention_of_few_rows(ctx, Q, H, G, D, K, lengths, window, sinks, dtype):
    B = 3
    first = [max(0, min(n, K)) - Q for n in (lengths or [K] * B)]
    _check_attention(ctx, B, Q, K, H, G, D, TYPES[dtype], window, sinks, lengths, first)


@pytest.mark.parametrize("layout", ["heads first", "odd"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Q,D", [(1, 64), (2, 40), (70, 64), (200, 128), (70, 8)])
def test_attention_of_other_layouts(ctx, Q, D, dtype, layout):
    _check_attention(ctx, 2, Q, 130, 4, 2, D, TYPES[dtype], (50, 20), 5, [130, 77], [130 - Q, 77 - Q], layout=layout)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S,lengths,window,sinks", [
    (1, None, (-1, -1), 0), (2, [2, 0], (0, 0), 0), (17, [17, 5], (3, 3), 1), (64, None, (-1, 0), 0), (65, None, (-1, -1), 0), (127, [127, 3], (5, 0), 0), (128, None, (-1, -1), 0),
    (129, [129, 128], (40, 10), 70), (197, None, (-1, -1), 0), (197, [197, 100], (64, 64), 1), (300, [300, 0], (-1, 30), 0), (512, [512, 300], (128, 128), 1), (700, None, (64, 0), 130),
    (700, [3, 699], (700, 700), 0), (1100, None, (10, -1), 4)])
@pytest.mark.parametrize("H,G,D", [(3, 3, 64), (4, 2, 128), (2, 2, 80), (2, 1, 32), (1, 1, 8)])
def test_attention_of_whole_sequences(ctx, H, G, D, S, lengths, window, sinks, dtype):
    _check_attention(ctx, 2, S, S, H, G, D, TYPES[dtype], window, sinks, lengths, layout="fused" if H == G else "plain")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Q,K,H,G,D,window,sinks", [(16, 4097, 12, 12, 80, (2047, 0), 8), (9, 3000, 8, 1, 64, (-1, 0), 0), (100, 5000, 4, 2, 128, (777, 0), 3), (257, 1500, 2, 2, 64, (-1, -1), 0),
                                                    (40, 40, 2, 2, 64, (3, 3), 1), (130, 20000, 1, 1, 64, (-1, 0), 0)])
def test_attention_of_a_chunk_behind_a_cache(ctx, Q, K, H, G, D, window, sinks, dtype):
    _check_attention(ctx, 2, Q, K, H, G, D, TYPES[dtype], window, sinks, [K, K // 2 + 7], [K - Q, K // 2 + 7 - Q])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Q", [1, 5, 23, 64, 200])
def test_attention_far_from_its_keys(ctx, Q, dtype):
    """Positions in front of and behind all keys, up to the ends of int32: rows that see nothing give zeros."""
    for first, window, sinks in (([-5, 2 ** 31 - 1], (3, 3), 0), ([-(2 ** 31), 90], (2 ** 31 - 1, 2 ** 31 - 1), 0), ([50, 60], (0, 0), 7), ([2 ** 31 - 1, 200], (10, 0), 2)):
        _check_attention(ctx, 2, Q, 100, 2, 2, 64, TYPES[dtype], window, sinks, [100, 80], first)
    _check_attention(ctx, 2, Q, 0, 2, 2, 64, TYPES[dtype])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Q,K", [(1, 300), (4, 90), (20, 90), (20, 2500), (90, 90), (260, 260)])
def test_attention_does_not_touch_what_no_query_sees(ctx, Q, K, dtype):
    """NaN and infinities behind the lengths and outside all windows; scores of any scale; a scale of zero."""
    t, gen = TYPES[dtype], _gen(Q + K)
    q, k, v = (torch.randn(2, n, 2, 64, generator=gen).to(t) for n in (Q, K, K))
    lengths, window, sinks = [K - 9, K // 2], (20, 0), 3
    first = [n - Q for n in lengths]
    for b in range(2):
        hidden = ~O.visible(Q, K, lengths[b], first[b], window, sinks).any(0)
        assert hidden.any()
        for bad, every in ((float("nan"), 2), (float("inf"), 3)):
            rows = hidden.nonzero()[::every, 0]
            k[b, rows], v[b, rows] = bad, -bad
    for scale in (None, 0.0, 3.0, -0.5):
        out = torch.empty(2, Q, 2, 64, dtype=t, device="cuda")
        ctx.attention(q.cuda(), k.cuda(), v.cuda(), out, scale=scale, window=window, sinks=sinks, lengths=torch.tensor(lengths, dtype=torch.int32).cuda(),
                      first=torch.tensor(first, dtype=torch.int32).cuda())
        kz, vz = k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0)
        want = O.attention(q, kz, vz, scale, window, sinks, lengths, first)
        O.close(out, want, t, floor=_attention_floor(q, kz, vz, t, abs(0.125 if scale is None else scale)))


@pytest.mark.parametrize("Q", [1, 8, 20, 150])
@pytest.mark.parametrize("magnitude", [1e-20, 1e-6, 1e-3, 300.0, 1e5, 1e15])
def test_attention_fp32_of_any_magnitude(ctx, Q, magnitude):
    """Values, and keys with the scale against them, far outside the range of half the bits; one key far above the others."""
    gen = _gen(11)
    q, k, v = (torch.randn(2, n, 2, 64, generator=gen) for n in (Q, 210, 210))
    out = torch.empty(2, Q, 2, 64, device="cuda")
    for qs, ks, vs, scale in ((1, magnitude, 1, 0.125 / magnitude), (magnitude, 1, 1, 0.125 / magnitude), (1, 1, magnitude, 0.125)):
        a, b, c = q * qs, k * ks, v * vs
        if vs != 1:
            c[:, 150] *= 1e3      # another tile's largest value
        ctx.attention(a.cuda(), b.cuda(), c.cuda(), out, scale=scale)
        O.close(out, O.attention(a, b, c, scale), torch.float32, floor=_attention_floor(a, b, c, torch.float32, scale))


def test_attention_of_offsets_beyond_32_bits(ctx):
    """A cache of more than 2^32 bytes: the last sequence's keys lie behind them."""
    S, D, B = 40000, 128, 450
    cache = torch.zeros(B, S, 1, D, dtype=torch.float16, device="cuda")       # 4.6 GB
    gen = _gen(12)
    tail = torch.randn(2, 300, 1, D, generator=gen).to(torch.float16)
    cache[B - 1, S - 300:] = tail[0].cuda()
    for Q in (1, 60):
        q = torch.randn(1, Q, 1, D, generator=gen).to(torch.float16)
        out = torch.empty(B, Q, 1, D, dtype=torch.float16, device="cuda")
        ctx.attention(q.cuda().expand(B, -1, -1, -1), cache, cache, out, window=(200, 0), first=torch.full((B,), S - Q, dtype=torch.int32, device="cuda"))
        want = O.attention(q, tail[:1], tail[:1], None, (200, 0), 0, None, [300 - Q])
        O.close(out[B - 1:], want, torch.float16, floor=_attention_floor(q, tail[:1], tail[:1], torch.float16, D ** -0.5))
        assert (out[:B - 1] == 0).all()

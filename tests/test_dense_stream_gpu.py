"""The dense operators on CUDA's default stream, where torch makes and reads tensors unless told otherwise: its handle is 1."""
import pytest
import torch

import pim_dl_asplos_b200 as P

pytestmark = pytest.mark.gpu


def test_the_default_stream_by_its_handle(ctx):
    gen = torch.Generator().manual_seed(1)
    a, w = torch.randn(4000, 1024, generator=gen).cuda(), torch.randn(1024, generator=gen).cuda()
    stats, want, back = torch.empty(4000, 2, device="cuda"), torch.empty_like(a), torch.empty_like(a)
    dw, dw_want = torch.empty(1024, device="cuda"), torch.empty(1024, device="cuda")
    triple = a * 3
    torch.cuda.synchronize()
    ctx.layer_norm(triple, w, None, want, stats=stats)
    ctx.layer_norm_backward(triple, triple, w, stats, back, dw_want)
    heads = want.view(50, 80, 16, 64)
    seen = torch.empty(50, 80, 16, 64, device="cuda")
    ctx.attention(heads, heads, heads, seen, window=(9, 0))
    ctx.sync()
    try:
        ctx.set_stream(1)
        for _ in range(5):
            x, out, dx, att = torch.zeros_like(a), torch.zeros_like(a), torch.zeros_like(a), torch.zeros_like(seen)
            for _ in range(20):
                x.add_(a)
            x.copy_(triple)
            ctx.layer_norm(x, w, None, out, stats=stats, flags=P.FLAG_ASYNC)
            ctx.layer_norm_backward(x, x, w, stats, dx, dw, flags=P.FLAG_ASYNC)
            h = out.view(50, 80, 16, 64)
            ctx.attention(h, h, h, att, window=(9, 0), flags=P.FLAG_ASYNC)
            x.zero_()                          # behind the calls that read it
            got = [t.clone() for t in (out, dx, dw, att)]
            for t in (out, dx, att):
                t.zero_()
            assert all(torch.equal(g, t) for g, t in zip(got, (want, back, dw_want, seen)))
    finally:
        ctx.set_stream(None)

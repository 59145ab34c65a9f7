"""The dense operators as an encoder layer runs them: one behind the other on the layer's stream, recorded and replayed, on other streams."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import dense_oracle as O
import oracle
import pim_dl_asplos_b200 as P
from pim_dl_asplos_b200 import layer as L

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def stream(ctx):
    s = torch.cuda.Stream()
    ctx.set_stream(s.cuda_stream)
    yield s
    s.synchronize()
    ctx.set_stream(None)


def _weights(D, F, separate, seed):
    cb = {"qkv": D // 2, "o": D // 2, "ffn1": D // 2, "ffn2": F // 2}
    w = L.random_layer_weights(D, F, cb, {k: 16 for k in cb}, seed=seed, separate_qkv=separate)
    rng = np.random.default_rng(seed)
    for k in ("ln1", "ln2"):
        w[k] = (rng.standard_normal(D).astype(np.float32), rng.standard_normal(D).astype(np.float32))
    return w


@pytest.mark.parametrize("separate", [False, True])
@pytest.mark.parametrize("S,B,H,D,turned,padded", [(16, 4, 4, 64, False, False), (197, 3, 2, 128, True, False), (130, 2, 4, 64, True, True), (1, 2, 2, 32, False, False)])
def test_layer_on_the_librarys_dense_operators(ctx, stream, S, B, H, D, turned, padded, separate):
    """Every operator in the layer against its definition on the very input that the layer gave it; recorded forwards give the ordinary one's bits."""
    w = _weights(D, 2 * D, separate, 5)
    gen = torch.Generator().manual_seed(3)
    hd = D // H
    dense = L.Dense(window=(40, 40), sinks=1)
    if turned:
        dense.positions = torch.randint(0, 14, (S, 2), generator=gen, dtype=torch.int32).cuda()
        dense.sections = (hd // 4, hd // 4)
        dense.inv_freq = (100.0 ** -(torch.arange(hd // 2) / (hd // 2))).cuda()
    lengths = [S] * B
    if padded:
        lengths = [S, S // 3]
        dense.lengths = torch.tensor(lengths, dtype=torch.int32).cuda()
    lay = L.LutTransformerLayer(ctx, w, S, B, H, first_layer_id=300, dense=dense)
    x = torch.from_numpy(L.synth.make_input(S * B, D, seed=7)).cuda()
    torch.cuda.synchronize()
    seen, orig = {}, lay._amm

    def spy(name, t):
        out = orig(name, t)
        ctx.sync()
        seen[name] = (t.detach().cpu().clone(), out.detach().cpu().clone())
        return out

    lay._amm = spy
    with torch.cuda.stream(stream):
        first = lay._finish(*lay._body(x))
    stream.synchronize()
    lay._amm = orig
    for name in lay.linears:
        cen, lut, bias, scale, lb = w[name]
        want = oracle.amm(seen[name][0].numpy(), cen, lut, bias, scale, lb)[0]
        if name == "ffn1":
            np.testing.assert_allclose(seen[name][1].numpy(), oracle.gelu_tanh(want), rtol=1e-5, atol=1e-9)
        else:
            assert np.array_equal(seen[name][1].numpy().view(np.uint32), want.view(np.uint32)), name
    if separate:
        q, k, v = (seen[n][1].view(B, S, H, hd) for n in ("q", "k", "v"))
    else:
        q, k, v = seen["qkv"][1].view(B, S, 3, H, hd).unbind(2)
    if turned:
        q, k = (O.rotary(t, dense.positions.cpu().expand(B, -1, -1), dense.inv_freq.cpu(), dense.sections) for t in (q, k))
    att = O.attention(q, k, v, None, (40, 40), 1, lengths)
    # scores: a rounding for each of the head's products and sums and of the rotation, of the split and the dropped product (three units each)
    s = float(q.double().abs().amax() * k.double().abs().amax()) * hd ** 0.5
    floor = (2 * (hd + 16) * U * s + 2 ** -20 + (S + 32) * U) * float(v.double().abs().amax())
    O.close(seen["o"][0].view(B, S, H, hd), att, torch.float32, floor=floor)
    ln = {k: [torch.from_numpy(a) for a in w[k]] for k in ("ln1", "ln2")}

    def norm_floor(t, wb):   # 96 roundings of sums, as large as the spread lets them be
        _, _, rstd = O.layer_norm(t, None, None, 1e-6)
        return float(96 * U * ((t.abs().amax() + 1) * rstd.amax() * wb[0].abs().amax() + 8))

    O.close(seen["ffn1"][0], O.layer_norm(seen["o"][1], *ln["ln1"], 1e-6, x.cpu())[0], torch.float32, floor=norm_floor(seen["o"][1].double(), ln["ln1"]))
    O.close(first, O.layer_norm(seen["ffn2"][1], *ln["ln2"], 1e-6, seen["ffn1"][0])[0], torch.float32, floor=norm_floor(seen["ffn2"][1].double(), ln["ln2"]))
    with torch.cuda.stream(stream):
        outs = []
        for _ in range(6):   # ordinary, recorded, replayed
            before = ctx.launch_count
            outs.append(lay.forward(x))
            outs.append(ctx.launch_count - before)
        other = lay.forward(x.flip(0).contiguous())
        back = lay.forward(x)
    stream.synchronize()
    assert S * B > L.GRAPH_TOKENS or lay._graph is not None
    assert all(torch.equal(o, first) for o in outs[::2]) and torch.equal(back, first) and not torch.equal(other, first)
    # as many launches replayed as queued, but for the table layouts and buffers of first calls
    assert outs[5] == outs[9] == outs[11] >= len(lay.linears) + 3 + turned * (2 if separate else 1)
    for lid in lay.ids.values():
        ctx.unload_weights(lid)


def _case(gen):
    """Inputs and outputs of one call of each operator, the attention in both its forms."""
    r = lambda *s: torch.randn(*s, generator=gen).cuda()   # noqa: E731
    c = dict(x=r(300, 768), r=r(300, 768), w=r(768), b=r(768), q=r(2, 150, 2, 64), k=r(2, 150, 2, 64), v=r(2, 150, 2, 64), one=r(2, 1, 2, 64))
    c["half"] = [t.half() for t in (c["q"], c["k"], c["v"])]
    c["pos"], c["freq"] = torch.randint(0, 99, (150, 1), generator=gen, dtype=torch.int32).cuda(), r(32).abs()
    return c


def _run(ctx, c, out):
    a = P.FLAG_ASYNC
    ctx.layer_norm(c["x"], c["w"], c["b"], out["y"], residual=c["r"], stats=out["st"], flags=a)
    ctx.layer_norm_backward(c["r"], c["x"], c["w"], out["st"], out["dx"], out["dw"], out["db"], flags=a)
    ctx.rotary(c["q"], c["pos"], c["freq"], (32,), out["t"], flags=a)
    ctx.attention(out["t"], c["k"], c["v"], out["att"], window=(50, 0), sinks=2, flags=a)
    ctx.attention(c["one"], c["k"], c["v"], out["one"], flags=a)
    ctx.attention(*c["half"], out["half"], flags=a)


def _outputs():
    e = lambda *s: torch.zeros(*s, device="cuda")   # noqa: E731
    return dict(y=e(300, 768), st=e(300, 2), dx=e(300, 768), dw=e(768), db=e(768), t=e(2, 150, 2, 64), att=e(2, 150, 2, 64), one=e(2, 1, 2, 64),
                half=e(2, 150, 2, 64).half())


def test_recorded_and_replayed_with_other_inputs(ctx, stream):
    a, b = _case(torch.Generator().manual_seed(1)), _case(torch.Generator().manual_seed(2))
    eager = []
    for c in (a, b):
        out = _outputs()
        torch.cuda.synchronize()
        _run(ctx, c, out)
        ctx.sync()
        eager.append(out)
    out, graph = _outputs(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graph.capture_begin(capture_error_mode="thread_local")
        _run(ctx, a, out)
        graph.capture_end()
        for _ in range(2):
            graph.replay()
            stream.synchronize()
            assert all(torch.equal(out[k], eager[0][k]) for k in out)
        for name, t in a.items():
            for to, of in zip(t if name == "half" else [t], b[name] if name == "half" else [b[name]]):
                to.copy_(of)
        graph.replay()
        stream.synchronize()
    assert all(torch.equal(out[k], eager[1][k]) for k in out)


def test_a_recorded_layer_follows_its_operators(ctx, stream):
    """After three forwards the layer replays a recording: a window, sinks, lengths, positions or a whole Dense set since count as in a layer of its own."""
    S, B, H, D = 24, 2, 2, 64
    w = _weights(D, 2 * D, False, 9)
    gen = torch.Generator().manual_seed(4)

    def positions(most):
        return dict(positions=torch.randint(0, most, (S, 1), generator=gen, dtype=torch.int32).cuda(), sections=(16,),
                    inv_freq=(50.0 ** -(torch.arange(16) / 16)).cuda())
    turned, turned_else = positions(20), positions(900)
    short = dict(lengths=torch.tensor([S, 5], dtype=torch.int32).cuda())
    steps = [dict(window=(4, 4)), dict(window=(2, 9)), dict(window=(2, 9), sinks=2), dict(window=(2, 9), sinks=2, **short), dict(**turned), dict(**turned_else),
             dict(interleaved=True, **turned_else), dict(), None]
    x = torch.from_numpy(L.synth.make_input(S * B, D, seed=7)).cuda()
    torch.cuda.synchronize()

    def layer(dense):
        return L.LutTransformerLayer(ctx, w, S, B, H, first_layer_id=320, dense=dense)
    with torch.no_grad(), torch.cuda.stream(stream):
        want = [layer(None if s is None else L.Dense(**s)).forward(x).clone() for s in steps]
        for whole in (False, True):
            lay = layer(L.Dense())
            for s, y in zip(steps, want):
                if whole or s is None:
                    lay.dense = None if s is None else L.Dense(**s)
                else:
                    for name, value in L.Dense(**s).__dict__.items():
                        setattr(lay.dense, name, value)
                for _ in range(4):
                    assert torch.equal(lay.forward(x), y), s
                assert lay._graph is not None
        stream.synchronize()
    assert len({tuple(y.flatten()[:4].tolist()) for y in want[:-1]}) > 4


def test_autograd_is_refused(ctx, stream):
    S, B, H, D = 8, 1, 2, 64
    lay = L.LutTransformerLayer(ctx, _weights(D, 2 * D, False, 9), S, B, H, first_layer_id=330, dense=L.Dense())
    x = torch.from_numpy(L.synth.make_input(S * B, D, seed=7)).cuda()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        with pytest.raises(RuntimeError, match="autograd"):
            lay.forward(x.requires_grad_())
        with torch.no_grad():
            assert lay.forward(x).shape == x.shape
        with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError, match="autograd"):
            lay.forward(torch.autograd.forward_ad.make_dual(x.detach(), x.detach()))
        stream.synchronize()


def test_contexts_on_streams_of_their_own_at_once(ctx):
    """Two contexts, each with its stream, queue the same operators side by side many times: no scratch is shared between them."""
    other = P.LutAmmContext(0)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    cases = [_case(torch.Generator().manual_seed(k)) for k in (5, 6)]
    want = []
    for c in cases:
        out = _outputs()
        torch.cuda.synchronize()
        _run(ctx, c, out)
        ctx.sync()
        want.append(out)
    try:
        for c, s in zip((ctx, other), streams):
            c.set_stream(s.cuda_stream)
        outs = [_outputs(), _outputs()]
        torch.cuda.synchronize()
        for _ in range(40):
            for c, case, out in zip((ctx, other), cases, outs):
                _run(c, case, out)
        ctx.sync()
        other.sync()
        for out, w in zip(outs, want):
            assert all(torch.equal(out[k], w[k]) for k in out)
    finally:
        ctx.set_stream(None)
        other.close()


def test_inputs_of_another_stream_are_waited_for_by_their_event(ctx, stream):
    """The operators run on the context's stream: what another stream makes is theirs once that stream has been waited for."""
    maker = torch.cuda.Stream()
    x, out = torch.zeros(4000, 1024, device="cuda"), torch.zeros(4000, 1024, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(maker):
        for _ in range(20):
            x.add_(1.0)
        x.mul_(torch.arange(1024, device="cuda"))
        done = torch.cuda.Event()
        done.record(maker)
    stream.wait_event(done)
    ctx.layer_norm(x, None, None, out, flags=P.FLAG_ASYNC)
    ctx.sync()
    O.close(out[:2], O.layer_norm(x[:2].cpu(), None, None, 1e-6)[0], torch.float32, floor=96 * U * 8)


def test_host_memory_is_refused(ctx):
    x = torch.zeros(4, 8)
    with pytest.raises(P.LutAmmError) as e:
        ctx.layer_norm(x, None, None, torch.zeros(4, 8, device="cuda"))
    assert e.value.code == P.EINVAL and "device" in str(e.value)


@pytest.mark.parametrize("driver", ["run_layer.py", "run_model.py"])
def test_launchers_run_on_the_dense_kernels(driver):
    eng = os.path.join(ROOT, "pim-dl-asplos_b200", "inference_engine")
    r = subprocess.run([sys.executable, os.path.join(eng, driver), "--transformer_config_file", os.path.join(eng, "configs", "bert_base_layer.yaml"), "--dense_kernels", "--window", "32", "--sinks", "1"],
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "AVG inference time" in r.stdout, r.stdout[-1500:] + r.stderr[-1500:]

"""The dense operators' CPython functions hand the library the same parameter blocks as the ctypes way, and leave to it what they do not
take: on the CPU, with entry points that only keep what they are given."""
import ctypes
import types

import pytest
import torch

import pim_dl_asplos_b200 as P

BLOCKS = {"layer_norm": P.NormParams, "layer_norm_backward": P.NormGradParams, "rotary": P.RotaryParams, "attention": P.AttentionParams}


def _fields(block):
    """A block's values, blocks and arrays in it opened (what lies between fields is anything)."""
    if isinstance(block, ctypes.Structure):
        return {f[0]: _fields(getattr(block, f[0])) for f in block._fields_}
    return list(block) if isinstance(block, ctypes.Array) else block


class _Context(P.LutAmmContext):
    def __init__(self):
        self.seen, self.device = [], 0
        self._h = ctypes.c_void_p(0x1000)
        self._entries = {n: ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_uint32)(self._keep(n, b)) for n, b in BLOCKS.items()}
        self._dense_address = {n: ctypes.cast(f, ctypes.c_void_p).value for n, f in self._entries.items()}
        self._L = types.SimpleNamespace(lutamm_destroy=lambda h: None, lutamm_layer_norm_backward_workspace=lambda *a: 64, **{
            "lutamm_" + n: (lambda f: lambda h, p, flags: f(h, ctypes.cast(p, ctypes.c_void_p), flags))(f) for n, f in self._entries.items()})

    def _keep(self, name, block):
        return lambda h, p, flags: self.seen.append((name, h, _fields(block.from_address(p)), flags)) or P.OK


def _calls():
    x, w, st = torch.zeros(6, 8), torch.zeros(8), torch.zeros(6, 2)
    half = torch.zeros(6, 20, dtype=torch.float16)[:, 4:12]
    pos, freq = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(4)
    h3, h4 = torch.zeros(3, 2, 8), torch.zeros(2, 5, 3, 7, 8, dtype=torch.bfloat16)[:, :3, 0]
    pos4 = torch.zeros(2, 3, 2, dtype=torch.int32)
    qkv = torch.zeros(2, 5, 3, 4, 16)
    n = torch.zeros(2, dtype=torch.int32)
    cache = torch.zeros(2, 1, 9, 16).transpose(1, 2)
    yield "layer_norm", (x, w, w, torch.zeros(6, 8)), {}
    yield "layer_norm", (half, w, None, torch.zeros(6, 8, dtype=torch.float16)), dict(eps=1e-5, residual=half, stats=st, flags=1)
    yield "layer_norm", (x, None, w, x), dict(residual=x, eps=0)
    yield "layer_norm", (x[:, :1], w[:1], w[:1], x[:, :1]), {}
    yield "layer_norm", (torch.zeros(1, 8), w, w, torch.zeros(1, 8)), dict(stats=torch.zeros(1, 2))
    yield "layer_norm", (x[:0], w, w, x[:0]), {}
    yield "layer_norm_backward", (x, x, w, st, x, w, w), dict(flags=1)
    yield "layer_norm_backward", (half, half, None, st), dict(dweight=w)
    yield "layer_norm_backward", (x, x, w, st, x, w, w, torch.zeros(64, dtype=torch.uint8)), {}
    yield "rotary", (h3, pos, freq, (2, 2), h3), {}
    yield "rotary", (h3, pos, freq, [4, 0], torch.zeros(3, 2, 8)), dict(interleaved=True, inverse=1, flags=1)
    yield "rotary", (h4, pos4, freq, (1, 3), torch.zeros(2, 3, 7, 8, dtype=torch.bfloat16)), {}
    yield "rotary", (h4, pos, freq, (1, 3), torch.zeros(2, 7, 3, 8, dtype=torch.bfloat16).transpose(1, 2)), {}
    yield "rotary", (h3, pos.expand(3, 2), freq[:0], (0, 0), h3), {}
    yield "attention", (qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], torch.zeros(2, 5, 4, 16)), {}
    yield "attention", (qkv[:, :1, 0], cache, cache, torch.zeros(2, 1, 4, 16)), dict(scale=2, window=(7, 0), sinks=3, lengths=n, first=n, flags=1)
    yield "attention", (qkv[:, :, 0], cache[:, :0], cache[:, :0], torch.zeros(2, 5, 4, 16)), dict(window=[-1, 4])


@pytest.mark.skipif(P._fast is None, reason="not built for this interpreter")
@pytest.mark.parametrize("name,args,kw", list(_calls()))
def test_both_ways_say_the_same(monkeypatch, name, args, kw):
    ctx = _Context()
    getattr(ctx, name)(*args, **kw)
    monkeypatch.setattr(P, "_fast", None)
    getattr(ctx, name)(*args, **kw)
    assert len(ctx.seen) == 2 and ctx.seen[0] == ctx.seen[1]


@pytest.mark.skipif(P._fast is None, reason="not built for this interpreter")
def test_the_ordinary_call_takes_the_short_way(monkeypatch):
    ctx = _Context()
    monkeypatch.setattr(P, "_dtype_of", lambda t: pytest.fail("the long way"))
    for name, args, kw in list(_calls())[:3]:
        getattr(ctx, name)(*args, **kw)
    assert len(ctx.seen) == 3


@pytest.mark.parametrize("fast", [True, False])
def test_numbers_beyond_the_blocks_fields_are_refused(monkeypatch, fast):
    if not fast:
        monkeypatch.setattr(P, "_fast", None)
    ctx = _Context()
    q, k = torch.zeros(1, 2, 1, 8), torch.zeros(1, 3, 1, 8)
    for kw in (dict(sinks=-1), dict(sinks=1 << 32), dict(window=(1 << 31, 0)), dict(window=(0, -(1 << 31) - 1)), dict(window=((1 << 32) + 3, 0)), dict(window=(1, 2, 3))):
        with pytest.raises(ValueError):
            ctx.attention(q, k, k, q.clone(), **kw)
    x = torch.zeros(1, dtype=torch.float16)
    tall = x.expand((1 << 32) + 1).unsqueeze(1)
    with pytest.raises(ValueError):
        ctx.layer_norm(tall, None, None, tall)
    with pytest.raises(ValueError):
        ctx.layer_norm_backward(tall, tall, None, torch.zeros(2).expand(tall.shape[0], 2), dbias=torch.zeros(1))
    with pytest.raises(ValueError):
        ctx.layer_norm_backward_workspace(1 << 32, 1)
    h = torch.zeros(3, 2, 8)
    for sections in ((-1, 5), (1 << 32, 4)):
        with pytest.raises(ValueError):
            ctx.rotary(h, torch.zeros(3, 2, dtype=torch.int32), torch.zeros(4), sections, h)
    assert not ctx.seen


def test_blocks_have_the_headers_layout(tmp_path):
    """Sizes and offsets of the ctypes blocks are those a C compiler gives the header's."""
    import os
    import shutil
    import subprocess
    if not shutil.which("gcc"):
        pytest.skip("no C compiler")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = {"lutamm_norm_params": P.NormParams, "lutamm_norm_grad_params": P.NormGradParams, "lutamm_heads": P.Heads, "lutamm_rotary_params": P.RotaryParams,
             "lutamm_attention_params": P.AttentionParams}
    lines = [f'printf("%zu", sizeof({c}));' + "".join(f'printf(" %zu", offsetof({c}, {f[0]}));' for f in b._fields_) + 'printf("\\n");' for c, b in names.items()]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "lutamm.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0;\n}\n")
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), "-o", str(tmp_path / "layout"), str(src)], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.splitlines()
    for line, (c, b) in zip(out, names.items()):
        assert [int(v) for v in line.split()] == [ctypes.sizeof(b)] + [getattr(b, f[0]).offset for f in b._fields_], c

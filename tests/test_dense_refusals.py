"""What the layer's dense operators refuse, through the C ABI on a CUDA runtime that runs nothing (fake_cudart.cpp) and through the
binding: no GPU."""
import ctypes
import glob
import os
import shutil
import subprocess
import types

import pytest
import torch

import pim_dl_asplos_b200 as P

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "pim-dl-asplos_b200", "csrc")
OBJECTS = sorted(glob.glob(os.path.join(CSRC, "build", "*.o")))
INCLUDE = "/usr/local/cuda/include"
needs_objects = pytest.mark.skipif(not (OBJECTS and shutil.which("g++") and os.path.exists(os.path.join(INCLUDE, "cuda_runtime.h"))),
                                   reason="the library's objects or the toolkit's headers are not here")


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    path = str(tmp_path_factory.mktemp("fake") / "libfake.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-I", CSRC, "-I", INCLUDE, "-o", path,
                    os.path.join(HERE, "fake_cudart.cpp")] + OBJECTS + ["-ldl"], check=True, timeout=300)
    L = ctypes.CDLL(path)
    L.fake_log.restype = L.lutamm_last_error.restype = ctypes.c_char_p
    L.lutamm_layer_norm_backward_workspace.restype = ctypes.c_size_t
    L.ctx = ctypes.c_void_p()
    assert L.lutamm_create(ctypes.byref(L.ctx), 0) == P.OK
    L.memory = ctypes.create_string_buffer(1 << 16)
    L.at = (ctypes.addressof(L.memory) + 255) // 256 * 256
    return L


def _norm(at):
    return P.NormParams(0, 4, 64, 1e-6, at, 64, 0, 0, at + 4096, 64, at + 8192, at + 8192, at + 12288)


def _grad(at):
    return P.NormGradParams(0, 4, 64, at, 64, at + 2048, 64, at + 4096, 64, at + 8192, at + 9216, at + 10240, at + 12288, 0)


def _rotary(at):
    return P.RotaryParams(0, 2, 3, 2, 16, 2, (4, 4), 0, 0, P.Heads(at, 96, 32, 16), P.Heads(at + 4096, 96, 32, 16), at + 8192, 0, 2, at + 9216)


def _attention(at):
    h = P.Heads(at, 96, 32, 16)
    return P.AttentionParams(0, 2, 3, 3, 2, 2, 16, 0, -1, -1, 0.25, h, h, h, P.Heads(at + 4096, 96, 32, 16), 0, 0)


CALLS = {"lutamm_layer_norm": _norm, "lutamm_layer_norm_backward": _grad, "lutamm_rotary": _rotary, "lutamm_attention": _attention}


def _call(lib, name, p, flags=P.FLAG_ASYNC):
    lib.fake_log()
    rc = getattr(lib, name)(lib.ctx, ctypes.byref(p), ctypes.c_uint32(flags))
    return rc, lib.fake_log().decode().splitlines()


@needs_objects
@pytest.mark.parametrize("name", CALLS)
def test_the_plain_call_launches_and_counts(lib, name):
    lib.lutamm_launch_count.restype = ctypes.c_uint64
    before = lib.lutamm_launch_count(lib.ctx)
    rc, log = _call(lib, name, CALLS[name](lib.at))
    assert rc == P.OK and len(log) == lib.lutamm_launch_count(lib.ctx) - before >= 1


SET = {
    "lutamm_layer_norm": [dict(dtype=3), dict(width=0), dict(width=1 << 31), dict(rows=1 << 31), dict(eps=-1.0), dict(eps=float("nan")), dict(x=0), dict(out=0), dict(x_stride=-64),
                          dict(out_stride=63), dict(out_stride=0), dict(x_stride=1 << 41), dict(dtype=0, x="+2"), dict(weight="+2"), dict(stats="+1"), dict(out="x", out_stride=65)],
    "lutamm_layer_norm_backward": [dict(dtype=9), dict(width=0), dict(rows=1 << 31), dict(dout=0), dict(x=0), dict(stats=0), dict(dx=0, dweight=0, dbias=0), dict(dx_stride=1),
                                   dict(dout_stride=-1), dict(workspace="x+4"), dict(dweight="+2"), dict(dx="x", dx_stride=128)],
    "lutamm_rotary": [dict(dtype=3), dict(axes=0), dict(axes=5), dict(head_dim=0), dict(head_dim=5000), dict(heads=1 << 21), dict(sections=(5, 4)), dict(sections=(2 ** 32 - 1, 9)), dict(positions=0),
                      dict(inv_freq=0), dict(positions="+2"), dict(x=(0, 96, 32, 16)), dict(out=(4096, 96, 32, 15)), dict(out=(4096, 0, 32, 16)), dict(x=(None, 96, 32, -16)),
                      dict(out=(0, 96, 32, 17)), dict(batch=1 << 30, tokens=1 << 30), dict(position_token_stride=-2)],
    "lutamm_attention": [dict(dtype=4), dict(head_dim=0), dict(head_dim=12), dict(head_dim=136), dict(kv_heads=0), dict(heads=3), dict(keys=1 << 31), dict(keys=(1 << 31) - 255), dict(queries=1 << 31), dict(scale=float("inf")),
                         dict(scale=float("nan")), dict(q=(None, 96, 32, 16)), dict(k=(None, 96, 32, 16)), dict(v=(None, 96, 32, 16)), dict(out=(None, 96, 32, 16)), dict(out=(0, 96, 32, 16)),
                         dict(out=(4096, 96, 32, 8)), dict(out=(4096, 96, 0, 16)), dict(k=(0, 96, -32, 16)), dict(lengths="+2"), dict(first="+1"), dict(batch=2 ** 31, queries=2 ** 30)],
}


@needs_objects
@pytest.mark.parametrize("name,change", [(n, c) for n in SET for c in SET[n]])
def test_what_is_refused_launches_nothing(lib, name, change):
    p = CALLS[name](lib.at)
    for field, value in change.items():
        if isinstance(value, str):
            base = p.x if value.startswith("x") else lib.at + 8192
            value = base + int(value.lstrip("x+") or 0)
        elif isinstance(value, tuple) and field != "sections":
            value = P.Heads(*(0 if value[0] is None else lib.at + value[0],) + value[1:]) if not (name == "lutamm_rotary" and field == "x" and value[0] == 0) else P.Heads(0, *value[1:])
        if field == "sections":
            value = (ctypes.c_uint32 * 4)(*value)
        setattr(p, field, value)
    rc, log = _call(lib, name, p)
    assert rc == P.EINVAL and not log and lib.lutamm_last_error(lib.ctx)


@needs_objects
@pytest.mark.parametrize("name", CALLS)
def test_contexts_params_and_flags(lib, name):
    p = CALLS[name](lib.at)
    f = getattr(lib, name)
    assert f(None, ctypes.byref(p), ctypes.c_uint32(0)) == P.EINVAL
    assert f(lib.ctx, None, ctypes.c_uint32(0)) == P.EINVAL
    assert _call(lib, name, p, 2)[0] == P.EINVAL and _call(lib, name, p, P.FLAG_ASYNC | 8)[0] == P.EINVAL
    assert _call(lib, name, p, 0)[0] == P.OK


@needs_objects
def test_empty_calls_do_nothing(lib):
    for name, change in (("lutamm_layer_norm", dict(rows=0, x=0, out=0)), ("lutamm_rotary", dict(batch=0)), ("lutamm_rotary", dict(heads=0)), ("lutamm_attention", dict(queries=0)),
                         ("lutamm_attention", dict(batch=0))):
        p = CALLS[name](lib.at)
        for k, v in change.items():
            setattr(p, k, v)
        assert _call(lib, name, p) == (P.OK, [])


@needs_objects
@pytest.mark.parametrize("change", [dict(dx=0, dx_stride=0), dict(dweight=0), dict(dbias=0), dict(weight=0), dict(dweight=0, dbias=0)])
def test_gradients_that_are_not_asked_for(lib, change):
    p = _grad(lib.at)
    for k, v in change.items():
        setattr(p, k, v)
    rc, log = _call(lib, "lutamm_layer_norm_backward", p)
    assert rc == P.OK and len(log) == (1 if "dweight" in change and "dbias" in change else 2)


class _Binding(P.LutAmmContext):
    """A context that hands its calls to nobody."""

    def __init__(self):
        self._h, self.device = None, 0
        self._L = types.SimpleNamespace(lutamm_layer_norm_backward_workspace=lambda *a: 64, **{n: lambda *a: P.OK for n in CALLS})


def test_shapes_types_and_layouts_that_the_binding_refuses():
    ctx = _Binding()
    x, w = torch.zeros(4, 8), torch.zeros(8)
    ctx.layer_norm(x, w, w, torch.zeros(4, 8), residual=x, stats=torch.zeros(4, 2))
    for bad in (dict(out=torch.zeros(4, 9)), dict(out=torch.zeros(4, 8).half()), dict(weight=torch.zeros(9)), dict(weight=w.double()), dict(residual=torch.zeros(3, 8)),
                dict(stats=torch.zeros(2, 4)), dict(stats=torch.zeros(2, 4).T), dict(out=torch.zeros(8, 4).T), dict(x=torch.zeros(4, 8).double())):
        with pytest.raises(ValueError):
            ctx.layer_norm(**{**dict(x=x, weight=w, bias=w, out=torch.zeros(4, 8)), **bad})
    st = torch.zeros(4, 2)
    ctx.layer_norm_backward(x, x, w, st, x, w, w)
    for bad in (dict(dx=torch.zeros(4, 7)), dict(dweight=torch.zeros(7)), dict(dout=torch.zeros(5, 8)), dict(stats=torch.zeros(4)), dict(workspace=torch.zeros(63, dtype=torch.uint8)),
                dict(workspace=torch.zeros(64))):
        with pytest.raises(ValueError):
            ctx.layer_norm_backward(**{**dict(dout=x, x=x, weight=w, stats=st), **bad})
    h, pos, f = torch.zeros(3, 2, 8), torch.zeros(3, 1, dtype=torch.int32), torch.zeros(4)
    ctx.rotary(h, pos, f, (4,), h)
    for bad in (dict(positions=pos.long()), dict(positions=torch.zeros(3, 2, dtype=torch.int32)), dict(inv_freq=torch.zeros(3)), dict(sections=()), dict(sections=(1,) * 5), dict(sections=(5, -1)),
                dict(out=torch.zeros(3, 2, 9)), dict(x=torch.zeros(3, 8), out=torch.zeros(3, 8))):
        with pytest.raises(ValueError):
            ctx.rotary(**{**dict(x=h, positions=pos, inv_freq=f, sections=(4,), out=h), **bad})
    q, k = torch.zeros(2, 3, 4, 8), torch.zeros(2, 5, 2, 8)
    ctx.attention(q, k, k, torch.zeros_like(q), lengths=torch.zeros(2, dtype=torch.int32))
    for bad in (dict(v=torch.zeros(2, 5, 1, 8)), dict(k=torch.zeros(1, 5, 2, 8)), dict(out=torch.zeros(2, 3, 4, 16)), dict(lengths=torch.zeros(2, dtype=torch.int64)), dict(first=torch.zeros(3, dtype=torch.int32)),
                dict(k=k.half()), dict(q=torch.zeros(3, 4, 8))):
        with pytest.raises(ValueError):
            ctx.attention(**{**dict(q=q, k=k, v=k, out=torch.zeros_like(q)), **bad})

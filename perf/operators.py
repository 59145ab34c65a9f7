"""Performance cases of the dense operators around the LUT-AMM linears of an encoder layer.

  norm       layer norm of a projection with the residual behind it (LutAmmContext.layer_norm)
  norm_grad  its backward pass: gradients of the input, the weight and the bias (layer_norm_backward)
  rotary     rotary positions with several axes on query and key heads, forwards or as a gradient's inverse (rotary)
  attention  attention with a sliding window and first tokens that stay visible, for whole sequences, for chunks and
             for single tokens behind a cache (attention)

Widths, head counts and sequence lengths are those of the package's configurations (BERT-base, BERT-large, ViT, the
hidden-size sweep) or generic.  Where `own` is false the operators are computed from elementary torch operations in 32 bits."""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _norm(name, op, rows, width, dtype, residual=False):
    c = dict(op=op, rows=rows, width=width, dtype=dtype, residual=residual)
    return dict(c, name=name) if name else c


def _rotary(name, batch, seq, heads, extra, dim, axes, far, dtype, interleaved, inverse):
    """`extra`: heads of the same rows that are not turned (the values of a fused projection)."""
    c = dict(op="rotary", batch=batch, seq=seq, heads=heads, extra=extra, dim=dim, axes=axes, far=far, dtype=dtype,
             interleaved=interleaved, inverse=inverse)
    return dict(c, name=name) if name else c


def _attention(name, batch, queries, keys, heads, kv_heads, dim, left, right, sinks, dtype, ragged=False, at_end=False, fused=False):
    c = dict(op="attention", batch=batch, queries=queries, keys=keys, heads=heads, kv_heads=kv_heads, dim=dim, left=left,
             right=right, sinks=sinks, dtype=dtype, ragged=ragged, at_end=at_end, fused=fused)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one BERT-base sequence of 128 tokens behind the attention-output linear: latency alone
        _norm("norm_base_128", "norm", 128, 768, "fp32", residual=True),
        # configs/vit_base_model.yaml: 64 images of 197 tokens
        _norm("norm_vit_12608", "norm", 64 * 197, 768, "fp32", residual=True),
        # 64 full-length sequences of BERT-large, a step that trains the norms
        _norm("norm_grad_large_32768", "norm_grad", 64 * 512, 1024, "fp32"),
        # a width that no vector divides, in half the bits
        _norm("norm_grad_odd_1576", "norm_grad", 8 * 197, 1999, "bf16"),
        # the query and key heads of ViT's fused projection, rows and columns of patches as two axes
        _rotary("rotary_vit_64x197", 64, 197, 24, 12, 64, 2, 64, "fp32", False, False),
        # a video of time x height x width far into a stream: the gradient of its queries
        _rotary("rotary_video_grad_16384", 1, 16384, 16, 0, 128, 3, 1 << 20, "bf16", True, True),
        # one BERT-base sequence: online inference
        _attention("attention_base_1x128", 1, 128, 128, 12, 12, 64, -1, -1, 0, "fp32", fused=True),
        # configs/vit_base_model.yaml, the whole batch
        _attention("attention_vit_64x197", 64, 197, 197, 12, 12, 64, -1, -1, 0, "fp32", fused=True),
        # configs/bert_large_layer.yaml: padded sequences of up to 512 tokens, a local window around each and the class token
        _attention("attention_large_16x512", 16, 512, 512, 16, 16, 64, 128, 128, 1, "fp32", ragged=True, fused=True),
        # a long document through the same heads
        _attention("attention_long_8192", 1, 8192, 8192, 16, 16, 64, 512, 512, 4, "bf16", fused=True),
        # a chunk of new tokens behind sequences of thousands, with ViT-huge's head width
        _attention("attention_chunk_4x16", 4, 16, 4097, 12, 12, 80, 2047, 0, 8, "fp16", ragged=True, at_end=True),
        # single tokens behind long ragged caches, four query heads to a key head
        _attention("attention_token_8x32768", 8, 1, 32768, 16, 4, 128, 16383, 0, 4, "bf16", ragged=True, at_end=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges."""
    while True:
        op = rng.choice(["norm", "norm_grad", "rotary", "attention", "attention", "attention"])
        dtype = rng.choice(["fp32", "fp32", "bf16", "fp16"])
        if op in ("norm", "norm_grad"):
            c = _norm("", op, _log_uniform(rng, 1, 32768), _log_uniform(rng, 16, 8192), dtype, op == "norm" and rng.random() < 0.7)
            if c["rows"] * c["width"] <= 64 * 512 * 1024:
                return c
            continue
        batch = _log_uniform(rng, 1, 64)
        if op == "rotary":
            heads, extra = rng.choice([(12, 0), (24, 12), (32, 16), (16, 0)])
            c = _rotary("", batch, _log_uniform(rng, 1, 16384), heads, extra, rng.choice([32, 64, 80, 128]), rng.choice([1, 2, 3]),
                        _log_uniform(rng, 16, 1 << 20), dtype, rng.random() < 0.5, rng.random() < 0.5)
            if c["batch"] * c["seq"] * heads * c["dim"] <= 1 << 25:
                return c
            continue
        dim = rng.choice([32, 64, 64, 64, 80, 128])
        left = rng.choice([-1, _log_uniform(rng, 1, 4096)])
        right = rng.choice([-1, 0, 0, _log_uniform(rng, 1, 4096)])
        sinks = rng.choice([0, 1, 4, rng.randrange(1, 130)])
        if rng.random() < 0.6:   # whole sequences
            heads = rng.choice([4, 12, 16])
            seq = _log_uniform(rng, 1, 8192)
            c = _attention("", batch, seq, seq, heads, heads, dim, left, right, sinks, dtype, ragged=rng.random() < 0.5, fused=True)
        else:                    # new tokens behind a cache
            heads, kv_heads = rng.choice([(12, 12), (16, 4), (16, 16), (8, 1)])
            queries = rng.choice([1, 1, rng.randrange(2, 9), _log_uniform(rng, 9, 512)])
            keys = _log_uniform(rng, 2 * queries, 32768)
            c = _attention("", batch, queries, keys, heads, kv_heads, dim, left, right, sinks, dtype, ragged=rng.random() < 0.7, at_end=True)
        if (batch * heads * c["queries"] * c["keys"] <= 16 * 8192 * 8192 and batch * c["keys"] * c["kv_heads"] * dim <= 1 << 27):
            return c


def _lengths(c):
    """Keys of each sequence: all, or from all down to half of them."""
    return [c["keys"] - (b * (c["keys"] // 2)) // c["batch"] if c["ragged"] else c["keys"] for b in range(c["batch"])]


def _sections(c):
    """Rotated pairs of each axis."""
    pairs = c["dim"] // 2
    each = pairs // c["axes"]
    return [pairs - each * (c["axes"] - 1)] + [each] * (c["axes"] - 1)


class _State:
    def __init__(self, case):
        self.case = case
        self.type = _TYPES[case["dtype"]]


def prepare(case, seed):
    st = _State(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    if case["op"] in ("norm", "norm_grad"):
        rows, width = case["rows"], case["width"]
        # a projection's outputs: a spread and an offset of their own for each feature
        st.x = (normal(rows, width) * (0.5 + normal(width).abs()) + 0.3 * normal(width)).to(st.type)
        st.weight, st.bias = 1 + 0.1 * normal(width), 0.1 * normal(width)
        if case["op"] == "norm":
            st.residual = normal(rows, width).to(st.type) if case["residual"] else None
            st.out = torch.empty_like(st.x)
            st.stats = torch.empty(rows, 2, device="cuda")
        else:
            st.dout = normal(rows, width).to(st.type)
            x = st.x.double()
            var, mean = torch.var_mean(x, 1, correction=0)
            st.stats = torch.stack([mean, (var + 1e-6).rsqrt()], 1).float()   # what the forward pass has left
            st.dx = torch.empty_like(st.x)
            st.dweight, st.dbias = torch.empty(width, device="cuda"), torch.empty(width, device="cuda")
    elif case["op"] == "rotary":
        B, S, H, E, D = case["batch"], case["seq"], case["heads"], case["extra"], case["dim"]
        st.x = normal(B, S, H + E, D).to(st.type)[:, :, :H]
        st.positions = torch.randint(0, case["far"], (S, case["axes"]), device="cuda", generator=gen, dtype=torch.int32)
        st.sections = _sections(case)
        each = [torch.arange(n, device="cuda", dtype=torch.float64) / n for n in st.sections]
        st.inv_freq = (10000.0 ** -torch.cat(each)).float()
        st.out = torch.empty(B, S, H, D, device="cuda", dtype=st.type)
    else:
        B, Q, K, H, G, D = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
        if case["fused"]:        # [tokens][Q | K | V], as the fused projection writes them
            qkv = normal(B, K, 3, H, D).to(st.type)
            st.q, st.k, st.v = qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2]
        else:
            st.q = normal(B, Q, H, D).to(st.type)
            st.k, st.v = normal(B, K, G, D).to(st.type), normal(B, K, G, D).to(st.type)
        st.lengths = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)
        st.first = st.lengths - Q if case["at_end"] else None
        st.out = torch.empty(B, Q, H, D, device="cuda", dtype=st.type)
    return st


_ctx = None


def _context():
    """What a process keeps: one context on the GPU, on the stream that makes the inputs and reads the outputs."""
    global _ctx
    if _ctx is None:
        import pim_dl_asplos_b200 as P
        _ctx = P.LutAmmContext(0)
        # 0, torch's default stream, would be the context's own: 1 is CUDA's handle for it
        _ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    return _ctx


def _run_own(st):
    import pim_dl_asplos_b200 as P
    ctx, c = _context(), st.case
    if c["op"] == "norm":
        ctx.layer_norm(st.x, st.weight, st.bias, st.out, eps=1e-6, residual=st.residual, stats=st.stats, flags=P.FLAG_ASYNC)
        return st.out, st.stats
    if c["op"] == "norm_grad":
        ctx.layer_norm_backward(st.dout, st.x, st.weight, st.stats, st.dx, st.dweight, st.dbias, flags=P.FLAG_ASYNC)
        return st.dx, st.dweight, st.dbias
    if c["op"] == "rotary":
        ctx.rotary(st.x, st.positions, st.inv_freq, st.sections, st.out, interleaved=c["interleaved"], inverse=c["inverse"],
                   flags=P.FLAG_ASYNC)
        return st.out
    ctx.attention(st.q, st.k, st.v, st.out, window=(c["left"], c["right"]), sinks=c["sinks"], lengths=st.lengths, first=st.first,
                  flags=P.FLAG_ASYNC)
    return st.out


def _plain_norm(st):
    x = st.x.float()
    mean = x.mean(1, keepdim=True)
    centred = x - mean
    rstd = ((centred * centred).mean(1, keepdim=True) + 1e-6).rsqrt()
    y = centred * rstd * st.weight + st.bias
    if st.residual is not None:
        y = y + st.residual.float()
    return y.to(st.type), torch.cat([mean, rstd], 1)


def _plain_norm_grad(st):
    dy, mean, rstd = st.dout.float(), st.stats[:, :1], st.stats[:, 1:]
    xhat = (st.x.float() - mean) * rstd
    g = dy * st.weight
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return dx.to(st.type), (dy * xhat).sum(0), dy.sum(0)


def _axis_of_pair(st):
    return torch.repeat_interleave(torch.arange(len(st.sections), device="cuda"), torch.tensor(st.sections, device="cuda"))


def _plain_rotary(st):
    c = st.case
    angle = st.positions.double()[:, _axis_of_pair(st)] * st.inv_freq.double()      # [S, pairs]; far positions need 64 bits
    cos, sin = angle.cos().float()[None, :, None], angle.sin().float()[None, :, None]
    if c["inverse"]:
        sin = -sin
    x = st.x.float()
    if c["interleaved"]:
        a, b = x[..., 0::2], x[..., 1::2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x.chunk(2, -1)
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return y.to(st.type)


def _plain_attention(st):
    c = st.case
    B, Q, K, H, G, D = (c[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    q = st.q.float().transpose(1, 2).reshape(B, G, H // G, Q, D)
    k, v = (t.float().transpose(1, 2).unsqueeze(2) for t in (st.k, st.v))
    at = torch.arange(Q, device="cuda")[None, :, None] + (st.first[:, None, None] if st.first is not None else 0)
    key = torch.arange(K, device="cuda")[None, None, :]
    hidden = key >= st.lengths[:, None, None]
    if c["left"] >= 0:
        hidden = hidden | ((key < at - c["left"]) & (key >= c["sinks"]))
    if c["right"] >= 0:
        hidden = hidden | (key > at + c["right"])
    s = (q @ k.transpose(-1, -2)).mul_(1 / math.sqrt(D))
    s.masked_fill_(hidden.view(B, 1, 1, -1, K), -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = s.sum(-1, keepdim=True)
    y = (s @ v) / torch.where(total == 0, 1.0, total)
    return y.reshape(B, H, Q, D).transpose(1, 2).to(st.type).contiguous()


def run(state):
    if own:
        return _run_own(state)
    return {"norm": _plain_norm, "norm_grad": _plain_norm_grad, "rotary": _plain_rotary, "attention": _plain_attention}[state.case["op"]](state)


def exact(case, seed):
    """From the definitions, in 64 bits."""
    st = prepare(case, seed)
    if case["op"] == "norm":
        x = st.x.double()
        n = x.shape[1]
        mean = x.sum(1) / n
        var = ((x - mean[:, None]) ** 2).sum(1) / n
        rstd = 1 / torch.sqrt(var + 1e-6)
        y = torch.addcmul(st.bias.double(), (x - mean[:, None]) / torch.sqrt(var + 1e-6)[:, None], st.weight.double())
        return (y + st.residual.double() if case["residual"] else y), torch.stack([mean, rstd], 1)
    if case["op"] == "norm_grad":
        # y = w * xhat + b: with J the Jacobian of xhat at x, dx = J (w * dy)
        x, dy, w = st.x.double(), st.dout.double(), st.weight.double()
        mean, rstd = st.stats.double().unbind(1)
        xhat = torch.einsum("rd,r->rd", x - mean[:, None], rstd)
        n = x.shape[1]
        along_one, along_x = torch.einsum("rd,d->r", dy, w) / n, torch.einsum("rd,d,rd->r", dy, w, xhat) / n
        dx = torch.einsum("r,rd->rd", rstd, dy * w - along_one[:, None] - xhat * along_x[:, None])
        return dx, torch.einsum("rd,rd->d", dy, xhat), torch.einsum("rd->d", dy)
    if case["op"] == "rotary":
        x = st.x.double()
        pairs = case["dim"] // 2
        z = torch.complex(x[..., 0::2], x[..., 1::2]) if case["interleaved"] else torch.complex(x[..., :pairs], x[..., pairs:])
        parts = [st.positions[:, a:a + 1].double() * f.double() for a, f in enumerate(torch.split(st.inv_freq, st.sections))]
        angle = torch.cat(parts, 1) * (-1 if case["inverse"] else 1)
        z = z * torch.polar(torch.ones_like(angle), angle)[None, :, None]
        return torch.view_as_real(z).flatten(-2) if case["interleaved"] else torch.cat([z.real, z.imag], -1)
    # attention, one head of one sequence at a time
    B, Q, H, G, D = (case[k] for k in ("batch", "queries", "heads", "kv_heads", "dim"))
    if B * H * Q * case["keys"] > 16 * 8192 * 8192:
        return None
    out = torch.zeros(B, Q, H, D, device="cuda", dtype=torch.float64)
    for b, n in enumerate(_lengths(case)):
        at = torch.arange(Q, device="cuda") + (n - Q if case["at_end"] else 0)
        key = torch.arange(n, device="cuda")
        distance = key[None, :] - at[:, None]
        seen = torch.ones_like(distance, dtype=torch.bool)
        if case["left"] >= 0:
            seen &= (distance >= -case["left"]) | (key < case["sinks"])[None, :]
        if case["right"] >= 0:
            seen &= distance <= case["right"]
        for g in range(G):
            k, v = st.k[b, :n, g].double(), st.v[b, :n, g].double()
            heads = slice(g * (H // G), (g + 1) * (H // G))
            s = torch.einsum("qhd,kd->hqk", st.q[b, :, heads].double(), k) / math.sqrt(D)
            weight = torch.softmax(s.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
            out[b, :, heads] = torch.einsum("hqk,kd->qhd", weight, v)
    return out


def _visible(c):
    """(pairs of a query and a key it sees, keys that any query sees), over all sequences."""
    pairs = keys = 0
    for n in _lengths(c):
        at = torch.arange(c["queries"], dtype=torch.int64) + (n - c["queries"] if c["at_end"] else 0)
        lo = (at - c["left"]).clamp(min=0) if c["left"] >= 0 else torch.zeros_like(at)
        hi = (at + c["right"] + 1).clamp(0, n) if c["right"] >= 0 else torch.full_like(at, n)
        lo = torch.minimum(lo, hi)
        first = torch.minimum(torch.full_like(at, c["sinks"]), hi)
        pairs += int((hi - lo + torch.minimum(lo, first)).sum())
        lo, hi = int(lo.min()), int(hi.max())
        keys += hi - lo + min(lo, int(first.max()))
    return pairs, keys


def work(case):
    """Inputs read once, outputs written once; of keys and values those that some query sees."""
    size = _TYPES[case["dtype"]].itemsize
    if case["op"] == "norm":
        n = case["rows"] * case["width"]
        return {"bytes": n * size * (3 if case["residual"] else 2) + 8 * case["width"] + 8 * case["rows"], "flops": 8 * n}
    if case["op"] == "norm_grad":
        n = case["rows"] * case["width"]
        return {"bytes": 3 * n * size + 12 * case["width"] + 8 * case["rows"], "flops": 14 * n}
    if case["op"] == "rotary":
        n = case["batch"] * case["seq"] * case["heads"] * case["dim"]
        return {"bytes": 2 * n * size + 4 * case["seq"] * case["axes"], "flops": 3 * n}
    pairs, keys = _visible(case)
    q = case["batch"] * case["queries"] * case["heads"] * case["dim"]
    return {"bytes": size * (2 * q + 2 * keys * case["kv_heads"] * case["dim"]), "flops": 4 * pairs * case["heads"] * case["dim"]}

"""Attention in 64 bits with what fp32 arithmetic may leave of each element, and fp32 products as three bfloat16 parts make them:
test infrastructure.

Of a score s = scale q k, with a = scale sum |q_d k_d|: an operand is held to within a unit (u = 2^-24) by its parts, the products of parts that
are left out are another; the ceil(head_dim / 16) products of 16 columns are added up in tensor memory, which rounds towards zero, two
units each, and as much again inside of one of them.  The factor scale * log2 e, its product and the distance to the maximum round
once each, relative to s.  A weight is relatively as far off as its score is absolutely, and by exp2's own four units; out = sum w v / sum w
moves by sum w delta (v - out).  Products w v and their sums: four products of 16 keys a tile towards zero, the tiles' sums (or those of a lane, which
has a quarter of the keys at most) and the division: all relative to sum w |v|.  None of it knows of other columns, or of keys that a query does not see."""
import math

import torch

import dense_oracle as O

U = 2.0 ** -24
RMS = 24 * U   # root mean square of the error, relative to that of results of random numbers: exp2 4, a score of some units 10, a tile's products 8


def attention(q, k, v, scale=None, window=(-1, -1), sinks=0, lengths=None, first=None):
    """(out, bound) in float64, on the CPU; a key that a row does not see counts for nothing in either, whatever it holds."""
    B, Q, H, D = q.shape
    K, G = k.shape[1:3]
    out, bound = (torch.zeros(B, Q, H, D, dtype=torch.float64) for _ in range(2))
    scale = 1 / math.sqrt(D) if scale is None else scale
    of_products, of_sums = 4 * math.ceil(D / 16) + 8, 24 + K / 4
    for b in range(B):
        seen = O.visible(Q, K, K if lengths is None else lengths[b], 0 if first is None else first[b], window, sinks)
        for h in range(H):
            kk, vv = k[b, :, h // (H // G)].double(), v[b, :, h // (H // G)].double()
            for i in range(Q):
                at = seen[i].nonzero()[:, 0]
                if not len(at):
                    continue
                x, y, z = q[b, i, h].double(), kk[at], vv[at]
                s, a = (y @ x) * scale, (y.abs() @ x.abs()) * abs(scale)
                w = torch.softmax(s, 0)
                r = w @ z
                delta = U * (of_products * a + 4 * s.abs() + 8)
                out[b, i, h] = r
                bound[b, i, h] = (w * delta) @ (z - r).abs() + U * of_sums * (w @ z.abs())
    return out, bound


def check(got, want, bound, steps=1.0, dtype=torch.float32):
    """Each element within its bound, and the rounding of the result."""
    got = got.double().cpu()
    allowed = bound + steps * torch.finfo(dtype).eps / 2 * want.abs()
    off = (got - want).abs()
    bad = ~(off <= allowed)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst by {float((off / allowed.clamp(min=1e-300)).nan_to_num(math.inf).max()):.3g} times what is allowed"


def rms(got, want):
    want = want.double()
    return float((got.double().cpu() - want).square().mean().sqrt() / want.square().mean().sqrt())


# ---- a product of fp32 numbers as the tensor cores make it: three bfloat16 parts of each, six of their nine products
TERMS = [(0, 2), (2, 0), (1, 1), (0, 1), (1, 0), (0, 0)]


def parts(x):
    """x = a + b + c: the leading bits, and what is left to nearest."""
    a = (x.contiguous().view(torch.int32) & -65536).view(torch.float32)
    b = (x - a).bfloat16().float()
    return a, b, (x - a - b).bfloat16().float()


def product(x, y, terms=TERMS):
    px, py = parts(x), parts(y)
    return sum(px[i].double() @ py[j].double() for i, j in terms)


def emulated(q, k, v, scale, terms_qk=TERMS, terms_pv=TERMS, halved=None):
    """[rows, d] of one head, with single-precision scores and weights; `halved`: an operand that is only held in half the bits."""
    q, k, v = (t.half().float() if halved == n else t for n, t in zip("qkv", (q, k, v)))
    s = product(q, k.T.contiguous(), terms_qk).float().double() * float(torch.tensor(scale * math.log2(math.e)).float())
    p = torch.exp2((s - s.amax(1, keepdim=True).ceil()).float().double()).float()
    p = p.half().float() if halved == "p" else p
    return (product(p, v, terms_pv) / p.double().sum(1, keepdim=True)).float()

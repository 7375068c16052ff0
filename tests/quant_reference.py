"""A quantised cache in plain 64-bit torch on the CPU: pages made, read and
attended over from the definition in include/aegkv.h."""

import math

import torch

LARGEST = {"mxfp4": 6.0, "mxfp8": 448.0}
BITS = {"mxfp4": 4, "mxfp8": 8}


def magnitudes(fmt):
    if fmt == "mxfp4":
        m = [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    else:
        m = [f / 8 * 2.0 ** -6 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7)
             for e in range(16) for f in range(8)]
        m[127] = math.nan
    return torch.tensor(m, dtype=torch.float64)


def quantise(fmt, x):
    """(codes, scale bytes) of values [..., head_dim], codes one a byte."""
    g = x.double().unflatten(-1, (-1, 32))
    most = g.abs().amax(-1)
    bad = ~torch.isfinite(g).all(-1)
    most = torch.where(bad, torch.zeros_like(most), most)
    e = torch.full_like(most, -111)
    for power in range(-111, 128):      # the least power that holds the largest
        e = torch.where((most > LARGEST[fmt] * 2.0 ** (power - 1)) & (power > -111),
                        torch.full_like(e, power), e)
    y = torch.where(bad[..., None], torch.zeros_like(g), g) / torch.exp2(e)[..., None]
    table = magnitudes(fmt)
    table = table[~table.isnan()]
    away = (y.abs()[..., None] - table).abs()
    least = away.amin(-1, keepdim=True)
    near = away == least                # one code, or two on a tie: the even one
    index = torch.arange(table.numel())
    even = torch.where(near & (index % 2 == 0), index, -1).amax(-1)
    any_ = torch.where(near, index, -1).amax(-1)
    code = torch.where((near.sum(-1) > 1), even, any_)
    sign = torch.signbit(y) & ~bad[..., None]
    code = code + sign * (1 << (BITS[fmt] - 1))
    byte = torch.where(bad, torch.full_like(e, 255), e + 127)
    return code.flatten(-2).to(torch.uint8), byte.to(torch.uint8)


def values(fmt, codes, scales):
    """64-bit values of codes (one a byte) and scale bytes."""
    table = magnitudes(fmt)
    table = torch.cat((table, -table))
    x = table[codes.long()].unflatten(-1, (-1, 32))
    s = torch.exp2(scales.double() - 127)
    s = torch.where(scales == 255, torch.full_like(s, math.nan), s)
    return (x * s[..., None]).flatten(-2)


class Pages:
    """Pages of K or of V as bytes, with codes and scales reached by place."""

    def __init__(self, fmt, num_blocks, block_size, kv_heads, head_dim, raw=None):
        self.fmt, self.bs, self.heads, self.d = fmt, block_size, kv_heads, head_dim
        self.code = head_dim * BITS[fmt] // 8
        self.chunk = block_size * (self.code + head_dim // 32)
        self.raw = (torch.zeros(num_blocks, kv_heads * self.chunk, dtype=torch.uint8)
                    if raw is None else raw.cpu().clone().view(num_blocks, -1))

    def _views(self):
        c = self.raw.view(-1, self.heads, self.chunk)
        cut = self.bs * self.code
        return (c[..., :cut].unflatten(-1, (self.bs, self.code)),
                c[..., cut:].unflatten(-1, (self.d // 32, self.bs)))

    def put(self, block, inside, codes, scales):
        if self.fmt == "mxfp4":
            codes = codes[..., 0::2] | (codes[..., 1::2] << 4)
        c, s = self._views()
        c[block, :, inside] = codes
        s[block, :, :, inside] = scales

    def get(self, block, inside):
        """64-bit [tokens, kv_heads, head_dim]."""
        c, s = self._views()
        codes, scales = c[block, :, inside], s[block, :, :, inside]
        if self.fmt == "mxfp4":
            codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
        return values(self.fmt, codes, scales)


def places(table, block_size, positions):
    return torch.tensor([table[p // block_size] for p in positions], dtype=torch.long), \
        torch.tensor([p % block_size for p in positions], dtype=torch.long)


def visible(n, m, window, sinks):
    """[m, n]: which positions the last m of n positions see."""
    j = torch.arange(n)
    p = torch.arange(n - m, n)[:, None]
    see = j <= p
    if window:
        see &= (p - j < window) | (j < sinks)
    return see


def attend(k, v, q, see, scale):
    """(out, weight) of one sequence in 64 bits: k, v [n, kv_heads, d], q [m, heads,
    d]; weight is the sum of probability times |v|, and with the largest sum of
    |q k| what tolerances are made of. Hidden places are left out, not
    multiplied by 0."""
    m, heads, d = q.shape
    group = heads // k.shape[1]
    out = torch.zeros(m, heads, d, dtype=torch.float64)
    weight = torch.zeros_like(out)
    size = torch.zeros(m, heads, 1, dtype=torch.float64)
    for i in range(m):
        j = see[i].nonzero()[:, 0]
        kk, vv = k[j].double(), v[j].double()
        kk, vv = kk.repeat_interleave(group, 1), vv.repeat_interleave(group, 1)
        qq = q[i].double()
        s = (kk * qq).sum(-1) * scale                   # [n', heads]
        p = torch.softmax(s, 0)
        out[i] = (p[..., None] * vv).sum(0)
        weight[i] = (p[..., None] * vv.abs()).sum(0)
        size[i, :, 0] = ((kk * qq).abs().sum(-1) * scale).amax(0)
    return out, weight, size


def tolerance(out, weight, size, n, d, dtype):
    """How far a row may be off. u: half a step of the type. The result is
    rounded (u |out|), each probability is rounded to the type (u weight), and
    what 32 bits lose: a score's product of d terms and its scaling move it by at
    most (d + 4) 2^-24 size, the exponent's argument and exp2 itself by another
    4 * 2^-24 (size + 1), which moves probabilities by twice that at most (their
    sum moves too); sums over n terms by (n + 8) 2^-24 weight."""
    u = torch.finfo(dtype).eps / 2
    f = 2.0 ** -24
    return (u * out.abs() + u * weight
            + weight * (2 * f * ((d + 8) * size + 4) + (n + 8) * f) * 1.01 + 1e-30)

"""Operators over an ordinary paged cache in plain 64-bit torch on the CPU, from the
definitions in include/aegkv.h, and how far 32-bit arithmetic may be from them."""

import math

import torch

F = 2.0 ** -24          # half a step of float32


def rotated(x, positions, frequencies, amplitude, interleaved):
    """x [tokens, heads, head_dim] in 64 bits, its first 2 * len(frequencies) values
    turned; and by how much 32-bit arithmetic may miss that before the last rounding."""
    x = x.double()
    r = 2 * len(frequencies)
    angle = positions.double()[:, None] * torch.as_tensor(frequencies, dtype=torch.float64)
    c, s = angle.cos()[:, None] * amplitude, angle.sin()[:, None] * amplitude
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    p, q = a * c - b * s, b * c + a * s
    y, off = x.clone(), torch.zeros_like(x)
    # The angle's rounding to 32 bits (at most 1 in units of half a turn) moves it by pi
    # 2^-25, cosine and sine are off by up to 4 half steps, the amplitude and its
    # product by one each, products and their sum by three: under 2^-21 of |a| + |b|.
    # Where the angle is a millions-fold frequency, 64 bits (both sides) lose 2^-52 of it.
    turn = (angle.abs() * 2.0 ** -50)[:, None]
    miss = (a.abs() + b.abs()) * abs(amplitude) * (2.0 ** -21 + turn)
    if interleaved:
        y[..., 0:r:2], y[..., 1:r:2] = p, q
        off[..., 0:r:2], off[..., 1:r:2] = miss, miss
    else:
        y[..., :r // 2], y[..., r // 2:r] = p, q
        off[..., :r // 2], off[..., r // 2:r] = miss, miss
    return y, off


def rounded(y, off, dtype):
    """How far a value of `dtype` may be: half a step, and half of the least one."""
    info = torch.finfo(dtype)
    return off * (1 + info.eps) + y.abs() * info.eps / 2 * 1.0001 + info.tiny * info.eps


def gather(pages, table, positions, block_size):
    """[len(positions), kv_heads, head_dim] of 4-D pages, in 64 bits."""
    p = torch.as_tensor(positions, dtype=torch.long)
    t = torch.as_tensor(table, dtype=torch.long)
    return pages.cpu()[t[p // block_size], p % block_size].double()


def scores(q, k, scale):
    """([m, heads, n] scores of q [m, heads, d] and k [n, kv_heads, d], the same sums of
    absolute values). Hidden places may hold anything: they give what they give."""
    group = q.shape[1] // k.shape[1]
    kk = k.double().repeat_interleave(group, 1).permute(1, 2, 0)
    qq = q.double().permute(1, 0, 2)
    return ((qq @ kk).permute(1, 0, 2) * scale,
            (qq.abs() @ kk.abs()).permute(1, 0, 2) * scale)


def attend(q, k, v, see, scale, dtype):
    """(out, its tolerance, lse, its tolerance) of one sequence, q [m, heads, d]."""
    m, heads, d = q.shape
    group, n = heads // k.shape[1], k.shape[0]
    out, tol = torch.zeros(m, heads, d, dtype=torch.float64), torch.zeros(m, heads, d,
                                                                          dtype=torch.float64)
    lse, lse_tol = (torch.zeros(m, heads, dtype=torch.float64) for _ in range(2))
    u = torch.finfo(dtype).eps / 2
    for i in range(m):
        j = see[i].nonzero()[:, 0]
        x, size = scores(q[i:i + 1], k[j], scale)
        x, size = x[0], size[0].amax(-1)                    # [heads, n'], [heads]
        p = torch.softmax(x, -1)
        vv = v[j].double().repeat_interleave(group, 1).permute(1, 0, 2)   # [heads, n', d]
        out[i] = (p[:, None] @ vv)[:, 0]
        weight = (p[:, None] @ vv.abs())[:, 0]
        lse[i] = torch.logsumexp(x, -1)
        # The result is rounded, each probability is rounded to the type; a score's d
        # products and its scaling lose (d + 4) F size, the exponent 4 F (size + 1), which
        # moves probabilities by twice that (their sum moves too), sums (n + 8) F.
        lost = F * ((d + 8) * size + 4)
        tol[i] = (u * out[i].abs() + u * weight
                  + weight * (2 * lost + (n + 8) * F)[:, None] * 1.01 + 1e-30
                  + torch.finfo(dtype).tiny * torch.finfo(dtype).eps)
        lse_tol[i] = 1.01 * (lost + (n + 8) * F + 4 * F * lse[i].abs())
    return out, tol, lse, lse_tol


def weigh(q, k, see, lse, scale, kv_heads):
    """(what each place gathers [kv_heads, n], its tolerance) of one sequence."""
    m, heads, d = q.shape
    group = heads // kv_heads
    x, size = scores(q, k, scale)
    e = torch.exp(x - lse.double()[..., None])
    e = torch.where(see[:, None], e, 0.0)
    size = torch.where(see[:, None], size, 0.0)
    w = e.view(m, kv_heads, group, -1).sum((0, 2))
    # as above for the score and the exponent, in which lse takes part
    lost = F * ((d + 8) * size + 8 * lse.double().abs()[..., None] + 4)
    off = (e * lost).view(m, kv_heads, group, -1).sum((0, 2))
    return w, 1.01 * off + (m * group + 8) * F * w + 1e-37


def evicted(weights, n, keep, sinks, recent):
    """The places that stay, of weights [n] of one sequence and head."""
    if n <= keep:
        return list(range(n))
    inner = [-math.inf if math.isnan(w) else w for w in weights[sinks:n - recent].tolist()]
    # no number is the least of all, below -inf
    number = [not math.isnan(w) for w in weights[sinks:n - recent].tolist()]
    order = sorted(range(len(inner)), key=lambda j: (not number[j], -inner[j], j))
    chosen = sorted(sinks + j for j in order[:keep - sinks - recent])
    return list(range(sinks)) + chosen + list(range(n - recent, n))

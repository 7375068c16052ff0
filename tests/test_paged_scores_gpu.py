"""Attention over an ordinary paged cache where scores are large, by values that are
known exactly: every row's largest score is far ahead of its others."""

import random

import pytest
import torch

import paged_reference as ref
from aegaeon_amd import ops
from quant_reference import visible

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def counted_pages(order, table, num, bs, heads, d, dtype):
    """(K, V) on the CPU: with q = (1, 128, -shift), position j scores order[j] - shift,
    exactly; K's third value is 1."""
    g = torch.Generator().manual_seed(len(order))
    k = torch.zeros(num, bs, heads, d, dtype=dtype)
    v = torch.randn(num, bs, heads, d, generator=g).to(dtype)
    for j, x in enumerate(order):
        place = k[table[j // bs], j % bs]
        place[:, 0], place[:, 1], place[:, 2] = x % 128, x // 128, 1
    return k, v


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n,new,group,window,sinks", [
    (5, 1, 3, 0, 0), (300, 1, 4, 0, 0), (300, 20, 2, 0, 0), (300, 100, 3, 0, 0),
    (300, 1, 4, 40, 4), (300, 20, 2, 40, 4), (300, 100, 3, 40, 4),
    (9000, 1, 4, 0, 0), (9000, 20, 2, 0, 0), (9000, 90, 2, 0, 0)])
@pytest.mark.parametrize("scale", [2.0 ** 13, 2.0 ** 100])
def test_scores_far_from_zero(gpu, dtype, d, n, new, group, window, sinks, scale):
    """Scores of 10^4 to 10^34, positive, negative and of both signs, in rows that are one
    item's, and cut and joined: each row takes the V of its largest score, alone."""
    bs, heads = 16, 2
    num = -(-n // bs) + 2
    order = list(range(n))
    random.Random(n + d).shuffle(order)
    table = list(range(num))
    random.Random(d).shuffle(table)
    k, v = counted_pages(order, table, num, bs, heads, d, dtype)
    top = 512 if n < 512 else 16384
    shifts = (0, top, top // 2)
    q = torch.zeros(new, heads * group, d, dtype=dtype)
    for h in range(heads * group):
        sign = torch.where(torch.arange(new) % 2 == 0, 1.0, -1.0)
        q[:, h, 0], q[:, h, 1], q[:, h, 2] = sign, 128 * sign, -sign * shifts[h % 3]
    cache = ops.PagedCache(k.to(gpu), v.to(gpu))
    batch = ops.CacheBatch([table], [n], [new], num_blocks=num, block_size=bs, kv_heads=heads,
                           heads=heads * group, window=window, sinks=sinks, device=gpu)
    out, lse = ops.paged_attend(cache, batch, q.to(gpu), scale=scale, return_lse=True)
    out, lse = out.cpu().double(), lse.cpu().double()

    kk, vv = (ref.gather(p, table, range(n), bs) for p in (k, v))
    x = ref.scores(q, kk, 1.0)[0]                               # whole numbers
    x = torch.where(visible(n, new, window, sinks)[:, None], x, -torch.inf)
    most, at = x.max(-1)
    want = vv[at, torch.arange(heads * group)[None] // group]
    # The other probabilities are exp(-scale) at the most: 0. Where scores are held
    # against their largest itself, its probability is a power of two and nothing is
    # rounded. Elsewhere its exponent is off by what rounds a sum of 2^16, and it and the
    # result are rounded to the type.
    far = (most * scale).abs() * 1.44 > 65536 + 8
    tol = torch.where(far[..., None], 0.0, 2.02 * torch.finfo(dtype).eps / 2 * want.abs()
                      + torch.finfo(dtype).tiny)
    bad = ~((out - want).abs() <= tol)
    assert not bad.any(), (bad.nonzero()[0].tolist(), float(out[bad][0]), float(want[bad][0]))
    # The logarithm's scale, product, reference, sum and factor are rounded once each, the
    # factor itself too; the sum's logarithm (8 at the most) is off by 2^-18.
    want = most * scale
    bad = ~((lse - want).abs() <= 7 * ref.F * want.abs() + 2.0 ** -18)
    assert not bad.any(), (bad.nonzero()[0].tolist(), float(lse[bad][0]), float(want[bad][0]))

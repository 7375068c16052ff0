"""Calls over an ordinary paged cache: what they refuse, and how they are ordered."""

import pytest
import torch

from aegaeon_amd import ops

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator().manual_seed(seed)


def test_caches_and_weights_with_tangents_are_refused(gpu):
    """Forward-mode tangents of what a call changes would be dropped, and are refused as
    gradients are."""
    num, bs, heads, d = 6, 16, 2, 64
    pages = [torch.zeros(num, bs, heads, d, dtype=BF16, device=gpu) for _ in range(2)]
    cache = ops.PagedCache(*pages)
    batch = ops.CacheBatch([[1, 2]], [20], [2], num_blocks=num, block_size=bs, kv_heads=heads,
                           device=gpu)
    x = torch.randn(2, heads, d, generator=gen(0)).to(BF16).to(gpu)
    weights = torch.zeros(num, heads, bs, device=gpu)
    out, lse = ops.paged_attend(cache, batch, x, return_lse=True)

    def calls(c, w):
        return [lambda: ops.paged_write(c, batch, x, x), lambda: ops.paged_attend(c, batch, x),
                lambda: ops.paged_weigh(c, batch, x, lse, w),
                lambda: ops.paged_evict(c, batch, w, 5)]

    ad = torch.autograd.forward_ad
    with ad.dual_level():
        dual = ad.make_dual(pages[0], torch.ones_like(pages[0]))
        with pytest.raises(ValueError, match="tangent"):
            ops.PagedCache(dual, pages[1])
        carried = ops.PagedCache(*pages)
        carried.v_pages = dual          # as one that came to it after the cache was made
        for call in calls(carried, weights):
            with pytest.raises(ValueError, match="tangent"):
                call()
        for call in calls(cache, ad.make_dual(weights, torch.ones_like(weights)))[2:]:
            with pytest.raises(ValueError, match="tangent"):
                call()
        assert torch.equal(ops.paged_attend(cache, batch, x), out)     # (none of its own)
    torch.cuda.synchronize()
    assert not weights.any() and not any(p.any() for p in pages)

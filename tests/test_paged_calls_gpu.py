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


@pytest.mark.parametrize("new", [[1, 0], [70, 0], [1, 1], [70, 70]])
def test_weights_over_a_common_prefix_that_one_sequence_sees(gpu, new):
    """Sequences share blocks, but the queries of one at the most see them: the weights are
    those of blocks of their own, and `shared` says which batches are taken."""
    num, bs, heads, d = 24, 16, 2, 64
    pages = [torch.randn(num, bs, heads, d, generator=gen(i)).to(BF16).to(gpu) for i in range(2)]
    cache = ops.PagedCache(*pages)
    window = 20 if new[1] else 0
    n = 128
    first, second = list(range(8)), [0, 1, *range(10, 16)]
    room = dict(num_blocks=num, block_size=bs, kv_heads=heads, heads=4, window=window, device=gpu)
    batch = ops.CacheBatch([first, second], [n, n], new, **room)
    t = sum(new)
    assert not batch.shared     # (a window of 20 over the last 70 begins at position 39)
    q = torch.randn(t, 4, d, generator=gen(2)).to(BF16).to(gpu)
    out, lse = ops.paged_attend(cache, batch, q, return_lse=True)
    weights = torch.rand(num, heads, bs, generator=gen(3)).to(gpu)
    want, at = weights.clone(), 0
    ops.paged_weigh(cache, batch, q, lse, weights)
    for table, m in zip((first, second), new):
        if m:
            one = ops.CacheBatch([table], [n], [m], **room)
            ops.paged_weigh(cache, one, q[at:at + m], lse[at:at + m], want)
        at += m
    assert torch.equal(weights, want)
    both = ops.CacheBatch([first, second], [n, n], [n - 32, n - 32], **room)
    assert both.shared
    x = torch.zeros(2 * (n - 32), 4, d, dtype=BF16, device=gpu)
    with pytest.raises(ValueError, match="one block"):
        ops.paged_weigh(cache, both, x, torch.zeros(2 * (n - 32), 4, device=gpu), weights)
    both.update([first, [20, 21, *second[2:]]], [n, n], [n - 32, n - 32])
    assert not both.shared

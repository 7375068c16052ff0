"""Calls over an ordinary paged cache: what they refuse, and how they are ordered."""

import pytest
import torch

import paged_reference as ref
from aegaeon_amd import ops
from quant_reference import places, visible

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator().manual_seed(seed)


def near(got, want, tol, what=""):
    got = got.cpu().double()
    bad = ~((got - want).abs() <= tol) & ~(got == want)
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[0].tolist(),
                           float(got[bad][0]), float(want[bad][0]))


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


def test_rotation_on_another_stream(gpu):
    """What a call on another stream reads is ordered before it, and kept, by the caller."""
    d, tokens, heads = 128, 4000, 8
    rotary = ops.Rotary(d, device=gpu)
    q = torch.randn(tokens, heads, d, generator=gen(0)).to(BF16).to(gpu)
    want = ops.rotate(rotary, torch.arange(tokens, device=gpu) + 5, q)
    side = torch.cuda.Stream()
    for _ in range(3):
        positions = torch.arange(tokens, device=gpu) + 5
        side.wait_stream(torch.cuda.current_stream())
        got = ops.rotate(rotary, positions, q, stream=side)
        side.synchronize()
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 4, 90])
@pytest.mark.parametrize("sinks", [0, 3])
def test_weights_beside_keys_that_are_no_number(gpu, dtype, d, new, sinks):
    """NaN and infinities of K, and weights of NaN, inside the sequences where no query sees
    them: before a window, between it and the first tokens, and in blocks of released
    columns. Seen places' weights match 64 bits, all others keep their bits."""
    bs, heads, group, n, window, num = 16, 2, 2, 400, 40, 60
    scale = d ** -0.5
    g = gen(d + new)
    k, v = (torch.randn(num, bs, heads, d, generator=g).to(dtype) for _ in range(2))
    order = torch.randperm(num - 1, generator=g)[:52] + 1       # (released columns read block 0)
    tables = [order[:26].tolist(), order[26:].tolist()]
    first = n - new - window + 1                # the first place in the window of a query
    gone = range(sinks and 1, first // bs)      # columns of the second that are released
    held = torch.rand(num, heads, bs, generator=g)
    for place in range(n):
        if sinks <= place < first:
            at = tables[0][place // bs], place % bs
            k[at] = [float("nan"), float("inf"), -float("inf")][place % 3]
            held[at[0], :, at[1]] = float("nan")
    k[0], held[0] = float("nan"), float("nan")
    for c in gone:
        k[tables[1][c]] = float("nan")
    batch_tables = [tables[0], [-1 if c in gone else b for c, b in enumerate(tables[1])]]
    cache = ops.PagedCache(k.to(gpu), v.to(gpu))
    batch = ops.CacheBatch(batch_tables, [n, n], [new, new], num_blocks=num, block_size=bs,
                           kv_heads=heads, heads=heads * group, window=window, sinks=sinks,
                           device=gpu)
    q = torch.randn(2 * new, heads * group, d, generator=g).to(dtype)
    out, lse = ops.paged_attend(cache, batch, q.to(gpu), return_lse=True)
    assert not out.isnan().any() and not lse.isnan().any()
    weights = held.to(gpu)
    ops.paged_weigh(cache, batch, q.to(gpu), lse, weights)
    got, rest = weights.cpu(), torch.ones(num, bs, dtype=torch.bool)
    see = visible(n, new, window, sinks)
    any_ = see.any(0).nonzero()[:, 0]
    assert any_.tolist() == [*range(sinks), *range(first, n)]
    for s, table in enumerate(tables):
        mine = slice(s * new, (s + 1) * new)
        kk = ref.gather(k, table, any_, bs)
        want, tol = ref.weigh(q[mine], kk, see[:, any_], lse[mine].cpu(), scale, heads)
        block, inside = places(table, bs, any_.tolist())
        want = want + torch.where(any_ >= n - new, 0.0, held[block, :, inside].double().T)
        near(got[block, :, inside].T, want, tol + 2 * ref.F * want.abs(), s)
        rest[block, inside] = False
    same = rest[:, None].expand_as(got)
    assert torch.equal(got[same].view(torch.int32), held[same].view(torch.int32))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,group", [(4, 3), (20, 3), (90, 2)])
@pytest.mark.parametrize("odd", [float("nan"), float("inf")])
def test_weights_of_rows_before_a_key_that_is_no_number(gpu, dtype, d, new, group, odd):
    """A key that only a prompt's later rows see (their log-sum-exps are given as they were
    without it): every other place gathers what it did, from all rows."""
    bs, heads, n, num = 16, 2, 300, 24
    scale = d ** -0.5
    g = gen(d + new)
    k, v = (torch.randn(num, bs, heads, d, generator=g).to(dtype) for _ in range(2))
    table = torch.randperm(num, generator=g)[:19].tolist()
    pages = [k.to(gpu), v.to(gpu)]
    cache = ops.PagedCache(*pages)
    batch = ops.CacheBatch([table], [n], [new], num_blocks=num, block_size=bs, kv_heads=heads,
                           heads=heads * group, device=gpu)
    q = torch.randn(new, heads * group, d, generator=g).to(dtype)
    _, lse = ops.paged_attend(cache, batch, q.to(gpu), return_lse=True)
    late = n - 1 - new // 3
    pages[0][table[late // bs], late % bs] = odd
    weights = torch.zeros(num, heads, bs, device=gpu)
    ops.paged_weigh(cache, batch, q.to(gpu), lse, weights)
    see = visible(n, new, 0, 0)
    others = [j for j in range(n) if j != late]
    kk = ref.gather(k, table, others, bs)
    want, tol = ref.weigh(q, kk, see[:, others], lse.cpu(), scale, heads)
    block, inside = places(table, bs, others)
    near(weights.cpu()[block, :, inside].T, want, tol + 2 * ref.F * want.abs())
    assert not torch.isfinite(weights[table[late // bs], :, late % bs]).all()

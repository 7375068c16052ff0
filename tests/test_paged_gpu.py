"""Rotary positions and an ordinary paged cache on the GPU: tokens written,
attention, the weight that tokens gather and eviction, against 64-bit definitions
(paged_reference.py)."""

import math
import random

import pytest
import torch

import paged_reference as ref
from aegaeon_amd import ops
from quant_reference import places, visible

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator().manual_seed(seed)


def make_pages(num_blocks, bs, heads, d, dtype, layout="tokens", seed=0, scale=1.0):
    """(K, V) pages on the CPU as 4-D views, laid out by tokens, by heads, or with K
    and V alternating in one tensor."""
    g = gen(seed)
    def values(*shape):
        return (torch.randn(*shape, generator=g) * scale).to(dtype)
    if layout == "heads":
        return tuple(values(num_blocks, heads, bs, d).transpose(1, 2) for _ in range(2))
    if layout == "alternating":
        both = values(num_blocks, 2, bs, heads, d)
        return both[:, 0], both[:, 1]
    return tuple(values(num_blocks, bs, heads, d) for _ in range(2))


def on(gpu, pages):
    """The same pages on the device, in the same layout."""
    k, v = pages
    if k.untyped_storage().data_ptr() == v.untyped_storage().data_ptr():
        both = torch.stack((k, v), 1).to(gpu)
        return both[:, 0], both[:, 1]
    if k.stride(1) < k.stride(2):
        return tuple(p.transpose(1, 2).contiguous().to(gpu).transpose(1, 2) for p in pages)
    return tuple(p.to(gpu) for p in pages)


def tables_for(lens, bs, num_blocks, seed=0):
    ids = list(range(num_blocks))
    random.Random(seed).shuffle(ids)
    out = []
    for n in lens:
        c = -(-n // bs)
        out.append(ids[:c])
        ids = ids[c:]
    return out


def batch_for(gpu, tables, lens, new, cache, **kw):
    return ops.CacheBatch(tables, lens, new, num_blocks=cache.num_blocks,
                          block_size=cache.block_size, kv_heads=cache.kv_heads, device=gpu, **kw)


def near(got, want, tol, what=""):
    got = got.cpu().double()
    bad = ~((got - want).abs() <= tol) & ~(got.isnan() & want.isnan()) & ~(got == want)
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[0].tolist(),
                           float(got[bad][0]), float(want[bad][0]))


# ---- rotary positions -------------------------------------------------------------


@pytest.mark.parametrize("head_dim,dim", [(64, 64), (128, 128), (256, 256), (128, 64), (128, 96),
                                          (64, 48), (80, 32), (80, 80), (100, 36), (2, 2),
                                          (256, 6), (1024, 1024), (192, 128)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rotate(gpu, head_dim, dim, interleaved, dtype):
    tokens, heads, kv_heads = 37, 5, 2
    g = gen(head_dim + dim)
    q = torch.randn(tokens, heads, head_dim, generator=g).to(dtype)
    k = torch.randn(tokens, kv_heads, head_dim, generator=g).to(dtype)
    positions = torch.randint(0, 1 << 17, (tokens,), generator=g)
    positions[:6] = torch.tensor([0, 1, -1, 2 ** 31 + 5, -3_000_000, 10 ** 7])
    rotary = ops.Rotary(head_dim, dim=dim, interleaved=interleaved, scaling="linear", factor=3.0,
                        device=gpu)
    got = ops.rotate(rotary, positions.to(gpu), q.to(gpu), k.to(gpu))
    for x, y in zip((q, k), got):
        want, off = ref.rotated(x, positions, rotary.frequencies, 1.0, interleaved)
        near(y, want, ref.rounded(want, off, dtype))
        assert torch.equal(y.cpu()[..., dim:], x[..., dim:])


@pytest.mark.parametrize("scaling", ["none", "linear", "base", "ramp", "smooth"])
def test_rotate_scaled(gpu, scaling):
    rotary = ops.Rotary(128, dim=64, base=1e6, scaling=scaling, factor=4.0, length=8192,
                        device=gpu)
    x = torch.randn(300, 3, 128, generator=gen(1))
    positions = torch.arange(300) * 997
    got = ops.rotate(rotary, positions.to(torch.int32).to(gpu), x.to(gpu))
    want, off = ref.rotated(x, positions, rotary.frequencies, rotary.amplitude, False)
    near(got, want, ref.rounded(want, off, F32))


@pytest.mark.parametrize("tokens", [0, 1, 2, 16, 17, 500])
@pytest.mark.parametrize("heads", [1, 40])
def test_rotate_in_place_and_strided(gpu, tokens, heads):
    """Rows of a fused projection, turned where they lie, and back by negative positions."""
    d = 128
    fused = torch.randn(tokens, (heads + 2) * d, generator=gen(tokens)).to(BF16).to(gpu)
    before = fused.clone()
    q = fused[:, :heads * d].view(tokens, heads, d)
    k = fused[:, heads * d:(heads + 1) * d].view(tokens, 1, d)
    positions = torch.arange(tokens, device=gpu) + 11
    rotary = ops.Rotary(d, device=gpu)
    out = ops.rotate(rotary, positions, q, k, out=(q, k))
    assert out[0] is q and out[1] is k
    old_q = before[:, :heads * d].view(tokens, heads, d)
    want, off = ref.rotated(old_q.cpu(), positions.cpu(), rotary.frequencies, 1.0, False)
    near(q, want, ref.rounded(want, off, BF16))
    assert torch.equal(fused[:, (heads + 1) * d:], before[:, (heads + 1) * d:])
    odd = torch.empty(tokens, heads, d + 1, dtype=BF16, device=gpu)[..., 1:]   # no aligned word
    odd.copy_(old_q)
    again = torch.empty(tokens, heads, d + 3, dtype=BF16, device=gpu)[..., :d]
    ops.rotate(rotary, positions, odd, out=again)
    assert torch.equal(again, q)
    back = ops.rotate(rotary, -positions, q)
    # two roundings of values of a length that the rotation keeps
    length = old_q.cpu().double().unflatten(-1, (2, -1)).norm(dim=-2, keepdim=True)
    tol = (2 * torch.finfo(BF16).eps * length).expand(-1, -1, 2, -1).flatten(-2) + 1e-4
    near(back, old_q.cpu().double(), tol)


# ---- writing -----------------------------------------------------------------------


@pytest.mark.parametrize("layout", ["tokens", "heads", "alternating"])
@pytest.mark.parametrize("d,bs", [(128, 16), (64, 32), (256, 16), (64, 128)])
@pytest.mark.parametrize("dtype,given", [(BF16, BF16), (F16, F16), (F16, F32), (BF16, F32),
                                         (F16, BF16)])
def test_write(gpu, layout, d, bs, dtype, given):
    heads, group = 3, 2
    lens = [1, 40, 17, 5 * bs + 3, 0, 16]
    new = [1, 1, 9, 2 * bs + 7, 0, 16]
    tables = tables_for(lens, bs, 24)
    pages = make_pages(24, bs, heads, d, dtype, layout)
    k_dev, v_dev = on(gpu, pages)
    cache = ops.PagedCache(k_dev, v_dev)
    assert cache.head_major == (layout == "heads")
    batch = batch_for(gpu, tables, lens, new, cache, heads=heads * group)
    t = sum(new)
    g = gen(3)
    k, v = (torch.randn(t + 2, heads, d, generator=g).to(given) for _ in range(2))
    q = torch.randn(t + 2, heads * group, d, generator=g).to(dtype)
    at = torch.cat([torch.arange(n - m, n) for n, m in zip(lens, new)])
    block = torch.cat([places(table, bs, range(n - m, n))[0]
                       for table, n, m in zip(tables, lens, new)])
    inside = at % bs

    def expect(k_new):
        want = [p.clone() for p in pages]
        want[0][block, inside] = k_new
        want[1][block, inside] = v[:t].float().to(dtype)
        return want

    # as they are: the same bits
    ops.paged_write(cache, batch, k.to(gpu), v.to(gpu))
    for got, want in zip((k_dev, v_dev), expect(k[:t].float().to(dtype))):
        assert torch.equal(got.cpu(), want)
    # rotated, at the places' positions and at others
    for positions, interleaved, dim in ((None, False, d), (at + 1000, True, d // 2)):
        rotary = ops.Rotary(d, dim=dim, interleaved=interleaved, scaling="ramp", factor=2.0,
                            length=4096, device=gpu)
        q_dev = q.to(gpu)
        out = torch.full_like(q_dev, 7.0)
        given_positions = None if positions is None else positions.to(gpu)
        assert ops.paged_write(cache, batch, k.to(gpu), v.to(gpu), rotary=rotary, q=q_dev,
                               positions=given_positions, out=out) is out
        p = at if positions is None else positions
        want, off = ref.rotated(k[:t], p, rotary.frequencies, rotary.amplitude, interleaved)
        near(k_dev.cpu()[block, inside], want, ref.rounded(want, off, dtype))
        others = torch.ones(24, bs, dtype=torch.bool)
        others[block, inside] = False
        assert torch.equal(k_dev.cpu()[others], pages[0][others])
        assert torch.equal(v_dev.cpu(), expect(0)[1])
        want, off = ref.rotated(q[:t], p, rotary.frequencies, rotary.amplitude, interleaved)
        near(out[:t], want, ref.rounded(want, off, dtype))
        assert (out[t:] == 7).all()
        # q in place gives the same
        ops.paged_write(cache, batch, k.to(gpu), v.to(gpu), rotary=rotary, q=q_dev,
                        positions=given_positions, out=q_dev)
        assert torch.equal(q_dev[:t], out[:t]) and torch.equal(q_dev[t:].cpu(), q[t:])


# ---- attention -----------------------------------------------------------------------

SHAPES = [(128, 16), (64, 32), (256, 16), (64, 128), (128, 64)]


def check_attend(got, lse, pages, tables, lens, new, q, bs, dtype, *, window=0, sinks=0,
                 scale=None):
    at, d = 0, q.shape[-1]
    scale = d ** -0.5 if scale is None else scale
    for table, n, m in zip(tables, lens, new):
        if m:
            see = visible(n, m, window, sinks)
            any_ = see.any(0).nonzero()[:, 0].tolist()
            k, v = (ref.gather(p, table, any_, bs) for p in pages)
            want, tol, sums, sums_tol = ref.attend(q[at:at + m].cpu(), k, v, see[:, any_], scale,
                                                   dtype)
            near(got[at:at + m], want, tol, ("out", n, m))
            if lse is not None:
                near(lse[at:at + m], sums, sums_tol, ("lse", n, m))
        at += m


@pytest.mark.parametrize("d,bs", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("layout", ["tokens", "heads", "alternating"])
@pytest.mark.parametrize("group,lens,new", [
    (1, [1, 2, 31, 32, 33, 100, 257], [1, 1, 1, 1, 1, 1, 1]),
    (4, [1, 15, 16, 17, 200, 0], [1, 2, 3, 4, 4, 0]),
    (7, [90, 300], [9, 1]),
    (3, [40, 400, 7], [13, 21, 7]),
    (2, [200, 130], [200, 65]),
    (5, [1, 150, 96], [1, 150, 40]),
])
def test_attention(gpu, d, bs, dtype, layout, group, lens, new):
    heads = 2
    tables = tables_for(lens, bs, 70)
    pages = make_pages(70, bs, heads, d, dtype, layout, seed=d + group)
    cache = ops.PagedCache(*on(gpu, pages))
    batch = batch_for(gpu, tables, lens, new, cache, heads=heads * group)
    q = torch.randn(sum(new), heads * group, d, generator=gen(9)).to(dtype)
    out, lse = ops.paged_attend(cache, batch, q.to(gpu), return_lse=True)
    check_attend(out, lse, pages, tables, lens, new, q, bs, dtype)
    assert torch.equal(ops.paged_attend(cache, batch, q.to(gpu)), out)


@pytest.mark.parametrize("d,bs", [(128, 16), (64, 32), (256, 16)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 0), (40, 4), (33, 40), (5000, 2),
                                          (100, 300)])
@pytest.mark.parametrize("new", [1, 9, 70])
def test_windows_and_first_tokens(gpu, d, bs, window, sinks, new):
    heads, group, dtype = 2, 3, BF16
    lens = [new, new + 20, new + 260]
    tables = tables_for(lens, bs, 60)
    pages = make_pages(60, bs, heads, d, dtype, seed=window)
    cache = ops.PagedCache(*on(gpu, pages))
    batch = batch_for(gpu, tables, lens, [new] * 3, cache, heads=heads * group, window=window,
                      sinks=sinks)
    q = torch.randn(3 * new, heads * group, d, generator=gen(2)).to(dtype)
    out, lse = ops.paged_attend(cache, batch, q.to(gpu), return_lse=True, scale=0.2)
    check_attend(out, lse, pages, tables, lens, [new] * 3, q, bs, dtype, window=window,
                 sinks=sinks, scale=0.2)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 12, 40, 90])
@pytest.mark.parametrize("window", [0, 30])
def test_what_is_not_seen_changes_nothing(gpu, dtype, d, new, window):
    """NaN and infinities behind the last token, in tokens after a query, and before its
    window: outputs and log-sum-exps of the rows that do not see them stay the same; rows
    that see an infinity in V get it."""
    bs, heads, group, n = 16, 2, 2, new + 75
    sinks = 3 if window else 0
    tables = tables_for([n, n], bs, 40)
    pages = make_pages(40, bs, heads, d, dtype, seed=d)
    k, v = pages
    for p in pages:     # behind the sequences' ends, and blocks of no sequence
        for table in tables:
            p[table[-1], n % bs:] = math.nan if p is k else math.inf
    if window:          # before the windows of all queries, behind the first tokens
        for p in pages:
            for j in range(sinks, n - new - window):
                p[tables[0][j // bs], j % bs] = math.nan
    q = torch.randn(2 * new, heads * group, d, generator=gen(4)).to(dtype)
    late = n - 1 - new // 3     # in the first sequence: seen by the last rows alone
    v[tables[0][late // bs], late % bs, 1, 5] = math.inf
    v[tables[0][late // bs], late % bs, 0, 9] = math.nan
    cache = ops.PagedCache(*on(gpu, pages))
    batch = batch_for(gpu, tables, [n, n], [new, new], cache, heads=heads * group, window=window,
                      sinks=sinks)
    out, lse = ops.paged_attend(cache, batch, q.to(gpu), return_lse=True)
    check_attend(out, lse, pages, tables, [n, n], [new, new], q, bs, dtype, window=window,
                 sinks=sinks)
    own = new - 1 - new // 3    # the row of that token itself
    assert out[own, 2 * group - 1, 5].isinf() and out[own, 0, 9].isnan()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("new", [1, 20, 90])
def test_scores_of_any_size(gpu, dtype, new):
    """Scores that grow along the sequence, of thousands, and of both signs."""
    bs, heads, d, n = 16, 1, 128, 300
    tables = tables_for([n], bs, 20)
    k, v = make_pages(20, bs, heads, d, dtype, seed=1)
    for j in range(n):
        k[tables[0][j // bs], j % bs] *= (j % 7) * (1.0 + j / 20)
    q = (torch.randn(new, 2, d, generator=gen(4)) * 8).to(dtype)
    cache = ops.PagedCache(*on(gpu, (k, v)))
    batch = batch_for(gpu, tables, [n], [new], cache, heads=2)
    for scale in (1e-4, d ** -0.5, 20.0, 1e4):
        out, lse = ops.paged_attend(cache, batch, q.to(gpu), scale=scale, return_lse=True)
        assert not out.isnan().any() and not lse.isnan().any()
        if scale <= d ** -0.5:      # beyond, tolerances say nothing
            check_attend(out, lse, (k, v), tables, [n], [new], q, bs, dtype, scale=scale)


def test_long_contexts_are_shared_out_and_joined(gpu):
    bs, heads, group, d, dtype = 16, 2, 7, 128, BF16
    lens, new = [9000, 3, 20011], [1, 1, 2]
    num = sum(-(-n // bs) for n in lens) + 3
    tables = tables_for(lens, bs, num)
    pages = make_pages(num, bs, heads, d, dtype, seed=5)
    cache = ops.PagedCache(*on(gpu, pages))
    batch = batch_for(gpu, tables, lens, new, cache, heads=heads * group)
    q = torch.randn(4, heads * group, d, generator=gen(4)).to(dtype)
    out, lse = ops.paged_attend(cache, batch, q.to(gpu), return_lse=True)
    check_attend(out, lse, pages, tables, lens, new, q, bs, dtype)


def test_blocks_behind_four_gibibytes(gpu):
    """Every call reaches the last blocks of a cache of over 4 GiB a tensor."""
    bs, heads, d, dtype, n = 128, 8, 256, BF16, 200
    num = (1 << 33) // (bs * heads * d * 2) + 5     # 8 GiB and some
    pages = [torch.zeros(num, bs, heads, d, dtype=dtype, device=gpu) for _ in range(2)]
    cache = ops.PagedCache(*pages)
    table = [num - 2, num - 1]
    batch = batch_for(gpu, [table], [n], [n], cache, heads=heads)
    k, v, q = (torch.randn(n, heads, d, generator=gen(i)).to(dtype) for i in range(3))
    ops.paged_write(cache, batch, k.to(gpu), v.to(gpu))
    small = [p[num - 2:].cpu() for p in pages]
    assert torch.equal(small[0].flatten(0, 1)[:n], k) and torch.equal(
        small[1].flatten(0, 1)[:n], v)
    out, lse = ops.paged_attend(cache, batch, q.to(gpu), return_lse=True)
    check_attend(out, lse, small, [[0, 1]], [n], [n], q, bs, dtype)
    weights = torch.zeros(num, heads, bs, device=gpu)
    ops.paged_weigh(cache, batch, q.to(gpu), lse, weights)
    total = weights[num - 2:].cpu().transpose(1, 2).flatten(0, 1)[:n].double().sum(0)
    near(total, torch.full((heads,), float(n), dtype=torch.float64), 1e-3)
    kept = ops.paged_evict(cache, batch, weights, 50, recent=10)
    got = pages[0][num - 2].cpu()
    for h in range(heads):
        assert torch.equal(got[:50, h], k[kept[0, h].cpu().long(), h])


def test_rows_behind_the_batch_are_kept_and_any_stride_is_taken(gpu):
    bs, heads, group, d, dtype = 16, 2, 3, 128, F16
    lens, new = [50, 200, 70], [1, 90, 12]
    tables = tables_for(lens, bs, 30)
    pages = make_pages(30, bs, heads, d, dtype, seed=5)
    cache = ops.PagedCache(*on(gpu, pages))
    batch = batch_for(gpu, tables, lens, new, cache, heads=heads * group)
    t = sum(new)
    q = torch.randn(t, heads * group, d, generator=gen(4)).to(dtype)
    want, sums = ops.paged_attend(cache, batch, q.to(gpu), return_lse=True)
    for pad in (1, 8):      # rows off 16 bytes, and on them
        wide = torch.full((t + 3, heads * group + 1, d + pad), 7.0, dtype=dtype, device=gpu)
        qq = wide.clone()[:, 1:, pad:]
        qq[:t] = q.to(gpu)
        out = wide[:, :-1, :d]
        lse = torch.full((t + 3, heads * group + 5), 7.0, device=gpu)[:, :heads * group]
        ops.paged_attend(cache, batch, qq, out=out, lse=lse)
        assert torch.equal(out[:t], want) and torch.equal(lse[:t], sums)
        assert (wide[t:] == 7).all() and (lse[t:] == 7).all()
        assert (wide[:, -1] == 7).all() and (wide[..., d:] == 7).all()
        w = [torch.zeros(30, heads, bs, device=gpu) for _ in range(2)]
        ops.paged_weigh(cache, batch, q.to(gpu), sums, w[0])
        ops.paged_weigh(cache, batch, qq, lse, w[1])
        assert torch.equal(*w)
        ops.paged_attend(cache, batch, qq, out=qq)
        assert torch.equal(qq[:t], want)


# ---- weights ---------------------------------------------------------------------------


@pytest.mark.parametrize("d,bs", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 3)])
@pytest.mark.parametrize("group,lens,new", [
    (1, [1, 2, 31, 300, 257], [1, 1, 1, 1, 1]),
    (4, [1, 16, 17, 600, 0, 256], [1, 2, 3, 4, 0, 9]),
    (16, [90, 300], [4, 5]),
    (2, [700, 130, 64], [200, 65, 64]),
    (5, [1, 555, 96], [1, 300, 40]),
])
def test_weights(gpu, d, bs, dtype, window, sinks, group, lens, new):
    heads = 2
    num = sum(-(-n // bs) for n in lens) + 3
    tables = tables_for(lens, bs, num)
    pages = make_pages(num, bs, heads, d, dtype, "heads" if d == 64 else "tokens", seed=3)
    cache = ops.PagedCache(*on(gpu, pages))
    batch = batch_for(gpu, tables, lens, new, cache, heads=heads * group, window=window,
                      sinks=sinks)
    q = torch.randn(sum(new), heads * group, d, generator=gen(7)).to(dtype)
    _, lse = ops.paged_attend(cache, batch, q.to(gpu), return_lse=True)
    before = torch.rand(num, heads, bs, generator=gen(8))
    at = 0
    for table, n, m in zip(tables, lens, new):      # new places hold anything
        for j in range(n - m, n):
            before[table[j // bs], :, j % bs] = math.nan
    weights = before.to(gpu)
    ops.paged_weigh(cache, batch, q.to(gpu), lse, weights)
    got, rest = weights.cpu(), torch.ones(num, bs, dtype=torch.bool)
    for table, n, m in zip(tables, lens, new):
        if not m:
            continue
        see = visible(n, m, window, sinks)
        any_ = see.any(0).nonzero()[:, 0]
        k = ref.gather(pages[0], table, any_, bs)
        want, tol = ref.weigh(q[at:at + m], k, see[:, any_], lse[at:at + m].cpu(), d ** -0.5,
                              heads)
        block, inside = places(table, bs, any_.tolist())
        old = torch.where(any_ >= n - m, 0.0, before[block, :, inside].double().T)
        want = want + old
        near(got[block, :, inside].T, want, tol + 2 * ref.F * want.abs(), (n, m))
        rest[block, inside] = False
        at += m
    same = rest[:, None].expand_as(got)
    assert torch.equal(got[same].nan_to_num(-1), before[same].nan_to_num(-1))


def test_weights_of_keys_that_are_no_number(gpu):
    """K that no query sees may hold anything, also beside seen places."""
    bs, heads, d, n, new = 16, 1, 128, 500, 200
    tables = tables_for([n], bs, 40)
    k, v = make_pages(40, bs, heads, d, BF16)
    k[tables[0][-1], n % bs:] = math.nan
    late = n - 15
    k[tables[0][late // bs], late % bs] = math.nan
    cache = ops.PagedCache(*on(gpu, (k, v)))
    for new in (1, 200):
        m = max(1, new - 30)    # queries before `late`
        batch = batch_for(gpu, tables, [late], [min(m, late)], cache, heads=2)
        q = torch.randn(m, 2, d, generator=gen(1)).to(BF16).to(gpu)
        out, lse = ops.paged_attend(cache, batch, q, return_lse=True)
        w = torch.zeros(40, heads, bs, device=gpu)
        ops.paged_weigh(cache, batch, q, lse, w)
        assert not out.isnan().any() and not w.isnan().any()
        near(w.sum(), torch.tensor(2.0 * m, dtype=torch.float64), 1e-3)


def test_weights_of_shared_blocks_are_refused(gpu):
    """Two sequences over common blocks would add to one place at once; a captured call that
    finds them after an update leaves the weights as they were."""
    bs, heads, d, num = 16, 2, 64, 12
    cache = ops.PagedCache(*(p.to(gpu) for p in make_pages(num, bs, heads, d, BF16)))
    weights = torch.ones(num, heads, bs, device=gpu)
    q = torch.randn(2, heads, d, generator=gen(0)).to(BF16).to(gpu)
    shared = batch_for(gpu, [[1, 2], [1, 3]], [20, 30], [1, 1], cache)
    out, lse = ops.paged_attend(cache, shared, q, return_lse=True)      # (fine)
    with pytest.raises(ValueError, match="one block"):
        ops.paged_weigh(cache, shared, q, lse, weights)
    room = dict(max_seqs=2, max_columns=8, max_tokens=2)
    batch = batch_for(gpu, [[1, 2], [4, 3]], [20, 30], [1, 1], cache, **room)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_weigh(cache, batch, q, lse, weights)
    batch.update([[1, 2], [1, 3]], [20, 30], [1, 1])
    graph.replay()
    torch.cuda.synchronize()
    assert (weights == 1).all()
    batch.update([[1, 2], [4, 3]], [20, 30], [1, 1])
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert not (weights[1, :, :16] == 1).any() and (weights[5:] == 1).all()
    # columns behind a sequence's end do not count
    batch.update([[1, 2, 3], [4, 3]], [20, 30], [1, 1])
    ops.paged_weigh(cache, batch, q, lse, weights)


@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 5)])
def test_captured_weights_follow_prompts_and_single_tokens(gpu, window, sinks):
    """One captured call, whose sequences' new tokens change from update to update: the same
    sums as calls with batches of their own."""
    bs, heads, group, d, num = 16, 2, 4, 64, 200
    cache = ops.PagedCache(*(p.to(gpu) for p in make_pages(num, bs, heads, d, F16)))
    lens = [1100, 900, 257]
    tables = tables_for(lens, bs, num)
    batch = batch_for(gpu, tables, lens, [70, 1, 1], cache, heads=heads * group, window=window,
                      sinks=sinks, max_seqs=3, max_columns=200, max_tokens=150)
    q = torch.randn(150, heads * group, d, generator=gen(0)).to(F16).to(gpu)
    lse = (torch.randn(150, heads * group, generator=gen(1)) + 5).to(gpu)
    weights = torch.zeros(num, heads, bs, device=gpu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_weigh(cache, batch, q, lse, weights)
    want = weights.clone()
    for new in ([70, 1, 1], [1, 1, 1], [1, 70, 70], [3, 0, 100], [70, 70, 1], [0, 0, 0], [1, 2, 17]):
        batch.update(tables, lens, new)
        graph.replay()
        eager = batch_for(gpu, tables, lens, new, cache, heads=heads * group, window=window,
                          sinks=sinks)
        n = sum(new)
        ops.paged_weigh(cache, eager, q[:n], lse[:n], want)
        torch.cuda.synchronize()
        assert torch.equal(weights, want), new
        assert not any(new) or float(want.sum()) > 0


# ---- eviction ----------------------------------------------------------------------------


@pytest.mark.parametrize("into", [False, True])
@pytest.mark.parametrize("d,bs,layout", [(128, 16, "tokens"), (64, 32, "heads"),
                                         (256, 16, "alternating"), (64, 128, "tokens")])
@pytest.mark.parametrize("keep,sinks,recent", [(1, 0, 0), (1, 0, 1), (1, 1, 0), (40, 4, 12),
                                               (40, 20, 20), (64, 0, 0), (257, 3, 100),
                                               (1500, 4, 30), (5000, 0, 0)])
def test_eviction(gpu, into, d, bs, layout, keep, sinks, recent):
    heads, lens = 3, [3, 0, keep, keep + 1, 700, 65, 2100]
    need = [-(-n // bs) for n in lens]
    spare = [-(-min(n, keep) // bs) for n in lens]
    num = sum(need) + sum(spare) + 3
    tables = tables_for([n * bs for n in need + spare], bs, num)
    pages = make_pages(num, bs, heads, d, BF16, layout)
    g = gen(keep)
    w = torch.randn(num, heads, bs, generator=g)
    w = torch.where(torch.rand(w.shape, generator=g) < 0.4, w.round(), w)   # equals
    w[torch.rand(w.shape, generator=g) < 0.05] = math.nan
    w[torch.rand(w.shape, generator=g) < 0.02] = math.inf
    w[torch.rand(w.shape, generator=g) < 0.02] = -math.inf
    w[torch.rand(w.shape, generator=g) < 0.02] = -0.0
    k_dev, v_dev = on(gpu, pages)
    cache = ops.PagedCache(k_dev, v_dev)
    batch = batch_for(gpu, tables[:len(lens)], lens, [min(1, n) for n in lens], cache)
    to_tables = tables[len(lens):] if into else tables[:len(lens)]
    target = batch_for(gpu, to_tables, [min(n, keep) for n in lens], [0] * len(lens),
                       cache) if into else None
    weights = w.to(gpu)
    kept = ops.paged_evict(cache, batch, weights, keep, sinks=sinks, recent=recent, into=target)
    assert kept.shape == (len(lens), heads, keep) and kept.dtype == torch.int32
    want = [pages[0].clone(), pages[1].clone(), w.clone()]
    for s, (table, to, n) in enumerate(zip(tables, to_tables, lens)):
        for h in range(heads):
            p = torch.arange(n)
            t = torch.tensor(table, dtype=torch.long)
            row = w[t[p // bs], h, p % bs] if n else w.new_zeros(0)
            chosen = ref.evicted(row, n, keep, sinks, recent)
            got = kept[s, h].cpu().tolist()
            assert got == chosen + [-1] * (keep - len(chosen)), (s, h)
            c = torch.tensor(chosen, dtype=torch.long)
            i = torch.arange(len(chosen))
            t2 = torch.tensor(to, dtype=torch.long)
            for x, y in zip(want[:2], pages):
                x[t2[i // bs], i % bs, h] = y[t[c // bs], c % bs, h]
            want[2][t2[i // bs], h, i % bs] = w[t[c // bs], h, c % bs]
    for got, x in zip((k_dev, v_dev, weights), want):
        assert torch.equal(got.cpu().nan_to_num(12345.0), x.nan_to_num(12345.0))


@pytest.mark.parametrize("n,keep", [(8191, 100), (8193, 8000), (33000, 4096), (70001, 20000)])
def test_eviction_from_long_sequences(gpu, n, keep):
    bs, heads, d = 16, 2, 64
    num = -(-n // bs)
    tables = tables_for([n], bs, num)
    pages = make_pages(num, bs, heads, d, F16)
    g = gen(n)
    w = torch.rand(num, heads, bs, generator=g).square()
    w = torch.where(torch.rand(w.shape, generator=g) < 0.9, (w * 8).round() / 8, w)
    k_dev, v_dev = on(gpu, pages)
    cache = ops.PagedCache(k_dev, v_dev)
    batch = batch_for(gpu, tables, [n], [1], cache)
    weights = w.to(gpu)
    kept = ops.paged_evict(cache, batch, weights, keep, sinks=4, recent=64).cpu()
    t, p = torch.tensor(tables[0]), torch.arange(n)
    i = torch.arange(keep)
    for h in range(heads):
        chosen = ref.evicted(w[t[p // bs], h, p % bs], n, keep, 4, 64)
        assert kept[0, h].tolist() == chosen
        c = torch.tensor(chosen)
        for got, x in zip((k_dev, v_dev), pages):
            assert torch.equal(got.cpu()[t[i // bs], i % bs, h], x[t[c // bs], c % bs, h])
        assert torch.equal(weights.cpu()[t[i // bs], h, i % bs], w[t[c // bs], h, c % bs])


# ---- together ------------------------------------------------------------------------------


def test_a_request_prefills_decodes_and_is_evicted_from(gpu):
    """A prompt in two chunks, decode steps, eviction when the cache is full, more
    steps at their true positions: each step's outputs and the weights against a
    64-bit simulation that keeps each head's tokens in lists."""
    bs, heads, group, d, dtype, keep, sinks, recent = 16, 2, 2, 64, BF16, 40, 2, 8
    num = 12
    pages = [torch.zeros(num, bs, heads, d, dtype=dtype, device=gpu) for _ in range(2)]
    weights = torch.full((num, heads, bs), math.nan, device=gpu)
    cache = ops.PagedCache(*pages)
    rotary = ops.Rotary(d, scaling="smooth", factor=8.0, length=64, device=gpu)
    table = [7, 2, 9, 4, 0, 11]
    more = dict(num_blocks=num, block_size=bs, kv_heads=heads, heads=heads * group)
    held, position = 0, 0
    k_sim = [torch.zeros(0, d, dtype=torch.float64) for _ in range(heads)]
    v_sim = [torch.zeros(0, d, dtype=torch.float64) for _ in range(heads)]
    w_sim = [torch.zeros(0, dtype=torch.float64) for _ in range(heads)]
    g = gen(0)
    for step, m in enumerate([35, 30] + [1] * 6 + [3, 1, 1]):
        if held + m > 72:
            batch = ops.CacheBatch([table], [held], [0], **more, device=gpu)
            kept = ops.paged_evict(cache, batch, weights, keep, sinks=sinks, recent=recent)
            for h in range(heads):
                # by the device's own weights: 32 bits may order near ones otherwise
                p, t = torch.arange(held), torch.tensor(table)
                c = kept[0, h].cpu().long()
                assert c[:sinks].tolist() == list(range(sinks))
                assert c[-recent:].tolist() == list(range(held - recent, held))
                assert (c[1:] > c[:-1]).all()
                k_sim[h], v_sim[h], w_sim[h] = k_sim[h][c], v_sim[h][c], w_sim[h][c]
                del p, t
            held = keep
        k, v = (torch.randn(m, heads, d, generator=g).to(dtype) for _ in range(2))
        q = torch.randn(m, heads * group, d, generator=g).to(dtype)
        held += m
        positions = torch.arange(position, position + m)
        position += m
        batch = ops.CacheBatch([table], [held], [m], **more, device=gpu)
        qr = ops.paged_write(cache, batch, k.to(gpu), v.to(gpu), rotary=rotary, q=q.to(gpu),
                             positions=positions.to(gpu))
        out, lse = ops.paged_attend(cache, batch, qr, return_lse=True)
        ops.paged_weigh(cache, batch, qr, lse, weights)
        want_q, off = ref.rotated(q, positions, rotary.frequencies, 1.0, False)
        near(qr, want_q, ref.rounded(want_q, off, dtype))
        kr = ref.gather(pages[0], table, range(held - m, held), bs)     # rounded as they are
        want_k, off = ref.rotated(k, positions, rotary.frequencies, 1.0, False)
        near(kr, want_k, ref.rounded(want_k, off, dtype))
        see = visible(held, m, 0, 0)
        for h in range(heads):
            k_sim[h] = torch.cat((k_sim[h], kr[:, h]))
            v_sim[h] = torch.cat((v_sim[h], v[:, h].double()))
            w_sim[h] = torch.cat((w_sim[h], torch.zeros(m, dtype=torch.float64)))
            mine = qr.cpu()[:, h * group:(h + 1) * group]
            want, tol, sums, sums_tol = ref.attend(mine, k_sim[h][:, None], v_sim[h][:, None], see,
                                                   d ** -0.5, dtype)
            near(out[:, h * group:(h + 1) * group], want, tol, step)
            near(lse[:, h * group:(h + 1) * group], sums, sums_tol, step)
            add, tol = ref.weigh(mine, k_sim[h][:, None], see, sums, d ** -0.5, 1)
            w_sim[h] = w_sim[h] + add[0]
            t, p = torch.tensor(table), torch.arange(held)
            near(weights.cpu()[t[p // bs], h, p % bs], w_sim[h], 1e-5 * (step + 1) + tol[0], step)
    assert position > held


def test_a_quantised_cache_takes_rotated_keys(gpu):
    """rotate, then quant_write and quant_attend: the path of a quantised cache."""
    bs, heads, d, n = 16, 2, 128, 40
    cache = ops.QuantCache(*(torch.zeros(4, ops.quant_page_bytes("mxfp8", bs, heads, d),
                                         dtype=torch.uint8, device=gpu) for _ in range(2)),
                           kv_heads=heads, head_dim=d, block_size=bs, fmt="mxfp8")
    batch = ops.CacheBatch([[2, 0, 3]], [n], [n], num_blocks=4, block_size=bs, kv_heads=heads,
                           heads=4, device=gpu)
    q = torch.randn(n, 4, d, generator=gen(0)).to(BF16).to(gpu)
    k, v = (torch.randn(n, heads, d, generator=gen(i)).to(BF16).to(gpu) for i in (1, 2))
    qr, kr = ops.rotate(ops.Rotary(d, device=gpu), torch.arange(n, device=gpu), q, k)
    ops.quant_write(cache, batch, kr, v)
    out = ops.quant_attend(cache, batch, qr)
    kq, vq = (x.cpu().double() for x in ops.quant_read(cache, batch, dtype=F32))
    want, tol, _, _ = ref.attend(qr.cpu(), kq, vq, visible(n, n, 0, 0), d ** -0.5, BF16)
    near(out, want, tol * 1.1)      # (its sum is of the rounded probabilities)


def test_a_cache_and_its_weights_are_swapped_out_and_in(gpu):
    """K, V and weights of a composite cache move together; attention and
    eviction go on in other blocks."""
    from aegaeon_amd.layout import (allocate_composite_cache, kv_tensor_specs,
                                    weight_tensor_specs)

    num, bs, heads, d, n = 9, 16, 2, 64, 60
    specs = kv_tensor_specs(1, num, bs, heads, d, 2) + weight_tensor_specs(1, num, bs, heads)
    comp = allocate_composite_cache(specs, num, gpu)
    k, v = (comp.segment_tensor(i).view(BF16).view(num, bs, heads, d) for i in range(2))
    weights = comp.segment_tensor(2).view(F32).view(num, heads, bs)
    cache = ops.PagedCache(k, v)
    args = dict(num_blocks=num, block_size=bs, kv_heads=heads, heads=4, device=gpu)
    before, after = [1, 5, 3, 8], [0, 2, 4, 6]
    batch = ops.CacheBatch([before], [n], [n], **args)
    x = [torch.randn(n, heads, d, generator=gen(i)).to(BF16).to(gpu) for i in range(2)]
    q = torch.randn(n, 4, d, generator=gen(3)).to(BF16).to(gpu)
    ops.paged_write(cache, batch, *x)
    out, lse = ops.paged_attend(cache, batch, q, return_lse=True)
    ops.paged_weigh(cache, batch, q, lse, weights)
    w = [weights[b].clone() for b in before]
    page = comp.page_size_bytes
    host = ops.PinnedHostPool(num * page)
    sizes = [s.page_size_bytes for s in comp.segments]
    offsets = [s.cpu_offset for s in comp.segments]
    layout = ops.SegmentLayout([comp.segment_tensor(i) for i in range(3)], sizes, offsets,
                               [1, 1, 1], num, [1], host.tensor, page, 0)
    ids = list(range(4))
    ones = [1] * 4
    layout.swap(before, ids, [0] * 4, [0] * 4, ones, False)
    torch.cuda.synchronize()
    for i in range(3):
        comp.segment_tensor(i).fill_(0)
    layout.swap(ids, after, [0] * 4, [0] * 4, ones, True)
    moved = ops.CacheBatch([after], [n], [n], **args)
    again, lse2 = ops.paged_attend(cache, moved, q, return_lse=True)
    assert torch.equal(again, out) and torch.equal(lse2, lse)
    for a, b in zip(after, w):
        assert torch.equal(weights[a], b)
    ops.paged_evict(cache, moved, weights, 20, recent=4)
    torch.cuda.synchronize()
    host.free()


# ---- graphs, streams, refusals ---------------------------------------------------------------


def test_captured_steps_follow_the_batch(gpu):
    """One decode step (write, attend, weigh) captured and replayed over updates, with
    eager work between the replays."""
    bs, heads, group, d, dtype, num = 16, 2, 4, 128, BF16, 60
    pages = [p.to(gpu) for p in make_pages(num, bs, heads, d, dtype)]
    cache = ops.PagedCache(*pages)
    weights = torch.zeros(num, heads, bs, device=gpu)
    rotary = ops.Rotary(d, device=gpu)
    tables = tables_for([300, 200, 100], bs, num)
    room = dict(max_seqs=4, max_columns=60, max_tokens=8)
    batch = batch_for(gpu, tables, [40, 30, 20], [1, 1, 1], cache, heads=heads * group, **room)
    k, v = (torch.zeros(8, heads, d, dtype=dtype, device=gpu) for _ in range(2))
    q = torch.zeros(8, heads * group, d, dtype=dtype, device=gpu)
    positions = torch.zeros(8, dtype=torch.int64, device=gpu)
    qr, out = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.zeros(8, heads * group, device=gpu)

    def step(b, *args):
        kk, vv, qq, pp, qo, oo, ll, c, w = args
        ops.paged_write(c, b, kk, vv, rotary=rotary, q=qq, positions=pp, out=qo)
        ops.paged_attend(c, b, qo, out=oo, lse=ll)
        ops.paged_weigh(c, b, qo, ll, w)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(batch, k, v, q, positions, qr, out, lse, cache, weights)
    other = [p.clone() for p in pages]
    other_cache, other_weights = ops.PagedCache(*other), weights.clone()
    g = gen(1)
    lens = [40, 30, 20]
    for turn in range(6):
        seqs = [0, 1, 2] if turn % 2 == 0 else [2, 0]
        for s in seqs:
            lens[s] += 1
        batch.update([tables[s] for s in seqs], [lens[s] for s in seqs], [1] * len(seqs))
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, generator=g).to(dtype))
        positions.copy_(torch.randint(0, 9999, (8,), generator=g))
        qr.fill_(3), out.fill_(3), lse.fill_(3)
        graph.replay()
        eager = batch_for(gpu, [tables[s] for s in seqs], [lens[s] for s in seqs],
                          [1] * len(seqs), cache, heads=heads * group)
        want = [torch.full_like(x, 3) for x in (qr, out, lse)]
        step(eager, k, v, q, positions, *want, other_cache, other_weights)
        torch.cuda.synchronize()
        for got, x in zip((qr, out, lse, *pages, weights), (*want, *other, other_weights)):
            if got.dtype == F32:
                assert torch.allclose(got, x, rtol=1e-5, atol=1e-6), turn
            else:
                assert (got.float() - x.float()).abs().max() <= 0.02, turn
        assert torch.equal(qr, want[0]) and torch.equal(pages[0], other[0])
        torch.randn(1000, 1000, device=gpu) @ torch.randn(1000, 1000, device=gpu)
    with pytest.raises(ValueError, match="room|replay"):
        short = torch.zeros(3, heads, d, dtype=dtype, device=gpu)
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.paged_write(cache, batch, short, short)
    with pytest.raises(ValueError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.paged_evict(cache, batch, weights, 10)


def test_other_streams(gpu):
    """Calls on a side stream, and an eviction into another stream's batch, are ordered
    behind the batches' uploads."""
    bs, heads, d, dtype, num = 16, 2, 64, F16, 40
    pages = [p.to(gpu) for p in make_pages(num, bs, heads, d, dtype)]
    cache = ops.PagedCache(*pages)
    tables = tables_for([200, 100], bs, num)
    weights = torch.rand(num, heads, bs, device=gpu)
    want_pages = [p.clone() for p in pages]
    want_weights = weights.clone()
    rotary = ops.Rotary(d, device=gpu)
    k, v, q = (torch.randn(6, heads, d, device=gpu).to(dtype) for _ in range(3))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()

    def all_of(c, w, stream, other):
        batch = batch_for(gpu, [tables[0]], [100], [6], c, stream=other)
        into = batch_for(gpu, [tables[1]], [30], [0], c)
        qr = ops.paged_write(c, batch, k, v, rotary=rotary, q=q, stream=stream)
        out, lse = ops.paged_attend(c, batch, qr, return_lse=True, stream=stream)
        ops.paged_weigh(c, batch, qr, lse, w, stream=stream)
        kept = ops.paged_evict(c, batch, w, 30, into=into, stream=stream)
        r = ops.rotate(rotary, torch.arange(6, device=gpu), q, stream=stream)
        torch.cuda.synchronize()
        return qr, out, lse, kept, r

    got = all_of(cache, weights, side, None)
    want = all_of(ops.PagedCache(*want_pages), want_weights, None, torch.cuda.Stream())
    for a, b in zip((*got, *pages, weights), (*want, *want_pages, want_weights)):
        assert torch.equal(a, b)


def test_the_general_path_gives_the_same(gpu, monkeypatch):
    """Plain calls are checked and made natively; the general path gives the same bits,
    and refuses what the native one leaves to it."""
    from aegaeon_amd import _lib

    bs, heads, d, dtype, num = 32, 2, 64, F16, 20
    outs, calls = [], []

    class Counted:
        def __getattr__(self, name):
            fn = getattr(native, name)

            def call(*args):
                done = fn(*args)
                calls.append((name, done is not None))
                return done
            return call

    native = _lib.hostargs()
    for readers in (Counted(), _lib._GeneralPath):
        monkeypatch.setattr(_lib, "_hostargs", readers)
        pages = [p.to(gpu) for p in make_pages(num, bs, heads, d, dtype)]
        cache = ops.PagedCache(*pages)
        batch = batch_for(gpu, tables_for([90, 33], bs, num), [90, 33], [3, 1], cache, heads=6)
        g = gen(3)
        k, v = (torch.randn(4, heads, d, generator=g).to(F32).to(gpu) for _ in range(2))
        q = torch.randn(4, 6, d, generator=g).to(dtype).to(gpu)
        rotary = ops.Rotary(d, dim=32, interleaved=True, device=gpu)
        positions = torch.tensor([5, 6, 7, 8], dtype=torch.int32, device=gpu)
        w = torch.ones(num, heads, bs, device=gpu)
        assert ops.paged_write(cache, batch, k, v) is None
        first = [p.clone() for p in pages]
        ops.paged_write(cache, batch, k, v, rotary=rotary)
        second = [p.clone() for p in pages]
        qr = ops.paged_write(cache, batch, k, v, rotary=rotary, positions=positions, q=q)
        out, lse = ops.paged_attend(cache, batch, qr, return_lse=True, scale=0.3)
        given = torch.zeros_like(lse)
        again = torch.zeros_like(out)
        a, b = ops.paged_attend(cache, batch, qr, out=again, lse=given, scale=0.3)
        assert a is again and b is given
        ops.paged_weigh(cache, batch, qr, lse, w, scale=0.3)
        qk = ops.rotate(rotary, positions, q, q[:, :2])
        alone = ops.rotate(rotary, positions, q, out=torch.zeros_like(q))
        outs.append((*first, *second, *pages, qr, out, lse, again, given, w, *qk, alone,
                     ops.paged_attend(cache, batch, q)))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert len(calls) == 9 and all(done for _, done in calls)


def test_calls_take_their_own_kind_of_cache(gpu):
    pages = [p.to(gpu) for p in make_pages(4, 16, 2, 64, BF16)]
    paged = ops.PagedCache(*pages)
    quant = ops.QuantCache(*(torch.zeros(4, ops.quant_page_bytes("mxfp8", 16, 2, 64),
                                         dtype=torch.uint8, device=gpu) for _ in range(2)),
                           kv_heads=2, head_dim=64, block_size=16, fmt="mxfp8")
    batch = batch_for(gpu, [[1]], [3], [3], paged)
    x = torch.zeros(3, 2, 64, dtype=BF16, device=gpu)
    with pytest.raises(ValueError, match="another kind of cache take a QuantCache"):
        ops.paged_attend(quant, batch, x)
    with pytest.raises(ValueError, match="another kind of cache take a PagedCache"):
        ops.quant_attend(paged, batch, x)


def test_refusals(gpu):
    bs, heads, d, dtype, num = 16, 2, 64, BF16, 10
    pages = [p.to(gpu) for p in make_pages(num, bs, heads, d, dtype)]
    cache = ops.PagedCache(*pages)
    batch = batch_for(gpu, [[1, 2], [3]], [20, 5], [2, 1], cache, heads=4)
    k = torch.zeros(3, heads, d, dtype=dtype, device=gpu)
    q = torch.zeros(3, 4, d, dtype=dtype, device=gpu)
    lse = torch.zeros(3, 4, device=gpu)
    weights = torch.zeros(num, heads, bs, device=gpu)
    rotary = ops.Rotary(d, device=gpu)
    before = [p.clone() for p in pages]

    def bad(match, fn, *args, **kw):
        with pytest.raises(ValueError, match=match):
            fn(*args, **kw)

    # caches
    bad("page must lie together", ops.PagedCache, pages[0][:, :, :1], pages[1][:, :, :1])
    bad("16, 32", ops.PagedCache, *(p.reshape(-1, 8, heads, d) for p in pages))
    bad("64, 128", ops.PagedCache, *(p.reshape(num, bs, 4, 32) for p in pages))
    bad("bfloat16 or float16", ops.PagedCache, *(p.float() for p in pages))
    bad("equally large", ops.PagedCache, pages[0], pages[1].half())
    bad("laid out", ops.PagedCache, pages[0],
        pages[1].transpose(1, 2).contiguous().transpose(1, 2))
    bad("gradient", ops.PagedCache, pages[0].clone().requires_grad_(), pages[1])
    bad("device", ops.PagedCache, pages[0].cpu(), pages[1].cpu())
    # writes
    bad("differ", ops.paged_write, cache, batch, k, k[:2])
    bad("holds 2", ops.paged_write, cache, batch, k[:2], k[:2])
    bad("\\[tokens, 2, 64\\]", ops.paged_write, cache, batch, q, q)
    bad("not supported", ops.paged_write, cache, batch, k.double(), k.double())
    bad("rotary", ops.paged_write, cache, batch, k, k, q=q)
    bad("rotary", ops.paged_write, cache, batch, k, k, positions=torch.zeros(3, device=gpu).int())
    bad("heads of 128", ops.paged_write, cache, batch, k, k, rotary=ops.Rotary(128, device=gpu))
    bad("int32 or int64", ops.paged_write, cache, batch, k, k, rotary=rotary,
        positions=torch.zeros(3, device=gpu))
    bad("positions of 3", ops.paged_write, cache, batch, k, k, rotary=rotary,
        positions=torch.zeros(2, device=gpu, dtype=torch.int32))
    bad("overlap", ops.paged_write, cache, batch, pages[0][0, :3], k)
    bad("overlap", ops.paged_write, cache, batch, k, k, rotary=rotary, q=q,
        out=pages[1].view(-1)[:3 * 4 * d].view(3, 4, d))
    bad("overlap", ops.paged_write, ops.PagedCache(pages[0], pages[0]), batch, k, k)
    bad("gradient", ops.paged_write, cache, batch, k.clone().requires_grad_(), k)
    # attention and weights
    bad("not supported", ops.paged_attend, cache, batch, q.half())
    bad("overlap", ops.paged_attend, cache, batch, q,
        out=pages[0].view(-1)[:3 * 4 * d].view(3, 4, d))
    buffer = torch.zeros(4 * 4 * d, dtype=dtype, device=gpu)
    bad("overlap", ops.paged_attend, cache, batch, buffer[:3 * 4 * d].view(3, 4, d),
        out=buffer[4 * d:].view(3, 4, d))
    bad("overlap", ops.paged_attend, cache, batch, q, out=buffer[:3 * 4 * d].view(3, 4, d),
        lse=buffer.view(torch.float32)[:12].view(3, 4))
    bad("rows of lse", ops.paged_attend, cache, batch, q, lse=lse[:2])
    bad("float32", ops.paged_attend, cache, batch, q, lse=lse.half())
    bad("positive", ops.paged_attend, cache, batch, q, scale=0.0)
    bad("\\[10, 2, 16\\]", ops.paged_weigh, cache, batch, q, lse, weights[:5])
    bad("float32", ops.paged_weigh, cache, batch, q, lse, weights.double())
    inside = pages[0].view(-1).view(torch.float32)[:num * heads * bs].view(num, heads, bs)
    bad("overlap", ops.paged_weigh, cache, batch, q, lse, inside)
    bad("overlap", ops.paged_evict, cache, batch, inside, 5)
    # evictions
    bad("to keep", ops.paged_evict, cache, batch, weights, 0)
    bad("to keep", ops.paged_evict, cache, batch, weights, 5, sinks=3, recent=3)
    bad("itself", ops.paged_evict, cache, batch, weights, 5, into=batch)
    shared = batch_for(gpu, [[1, 2], [1]], [20, 5], [1, 0], cache, heads=4)
    bad("block 1", ops.paged_evict, cache, shared, weights, 5)
    target = batch_for(gpu, [[2], [7]], [5, 5], [0, 0], cache, heads=4)
    bad("block 2", ops.paged_evict, cache, batch, weights, 5, into=target)
    target = batch_for(gpu, [[8], [7]], [4, 5], [0, 0], cache, heads=4)
    bad("into 4 places", ops.paged_evict, cache, batch, weights, 5, into=target)
    target = batch_for(gpu, [[8], [8]], [5, 5], [0, 0], cache, heads=4)
    bad("block 8", ops.paged_evict, cache, batch, weights, 5, into=target)
    bad("other sequences", ops.paged_evict, cache, batch, weights, 5,
        into=batch_for(gpu, [[8]], [5], [0], cache, heads=4))
    released = batch_for(gpu, [[-1, 2], [3]], [20, 5], [1, 1], cache, heads=4, window=2)
    bad("released", ops.paged_evict, cache, released, weights, 5)
    # rotation
    positions = torch.arange(3, device=gpu)
    bad("heads|head_dim|\\[tokens", ops.rotate, rotary, positions, q.view(3, 2, 128))
    bad("positions of 3", ops.rotate, rotary, positions[:2], q)
    bad("overlap", ops.rotate, rotary, positions, buffer[:3 * 4 * d].view(3, 4, d),
        out=buffer[4 * d:].view(3, 4, d))
    bad("overlap", ops.rotate, rotary, positions, q, k, out=(buffer[:3 * 4 * d].view(3, 4, d),
                                                            buffer[:3 * 2 * d].view(3, 2, d)))
    bad("tensors", ops.rotate, rotary, positions, q, k, out=buffer[:3 * 4 * d].view(3, 4, d))
    bad("tensors", ops.rotate, rotary, positions, q, q, out=torch.zeros_like(q).expand(2, 3, 4, d))
    bad("what it goes to", ops.rotate, rotary, positions, q, k.half())
    if torch.cuda.device_count() == 1:
        bad("on cpu", ops.rotate, rotary, positions.cpu(), q)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(pages, before)) and not weights.any()


def test_empty_batches(gpu):
    bs, heads, d, num = 16, 2, 128, 6
    pages = [p.to(gpu) for p in make_pages(num, bs, heads, d, F16)]
    before = [p.clone() for p in pages]
    cache = ops.PagedCache(*pages)
    weights = torch.ones(num, heads, bs, device=gpu)
    empty = torch.zeros(0, heads, d, dtype=F16, device=gpu)
    rotary = ops.Rotary(d, device=gpu)
    for tables, lens, new in (([], [], []), ([[], [3]], [0, 9], [0, 0])):
        batch = batch_for(gpu, tables, lens, new, cache)
        assert ops.paged_write(cache, batch, empty, empty, rotary=rotary, q=empty).shape[0] == 0
        out, lse = ops.paged_attend(cache, batch, empty, return_lse=True)
        assert out.shape == empty.shape and lse.shape == (0, heads)
        ops.paged_weigh(cache, batch, empty, lse, weights)
        kept = ops.paged_evict(cache, batch, weights, 4)
        assert kept.shape == (len(lens), heads, 4)
    assert (weights == 1).all()
    # the second sequence of 9 equal weights kept its first 4 places where they were
    assert kept[1].tolist() == [[0, 1, 2, 3]] * heads and (kept[0] == -1).all()
    assert all(torch.equal(a, b) for a, b in zip(pages, before))

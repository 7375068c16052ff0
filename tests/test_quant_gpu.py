"""Quantised caches on the GPU: written pages, tokens read back and attention
against the 64-bit definition (quant_reference.py)."""

import ctypes
import math
import random

import pytest
import torch

import quant_reference as ref
from aegaeon_amd import ops

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def make(gpu, fmt, num_blocks, bs, heads, d, seed=0, random_bytes=True):
    """(QuantCache, K pages, V pages as references) of random codes and of
    scales near 1."""
    gen = torch.Generator().manual_seed(seed)
    refs = []
    for _ in range(2):
        p = ref.Pages(fmt, num_blocks, bs, heads, d)
        if random_bytes:
            c, s = p._views()
            c.copy_(torch.randint(0, 256, c.shape, generator=gen, dtype=torch.uint8))
            if fmt == "mxfp8":
                c[(c & 127) > 118] -= 16        # no codes that are no number
            s.copy_(torch.randint(118 if fmt == "mxfp8" else 123, 121 if fmt == "mxfp8" else 127,
                                  s.shape, generator=gen, dtype=torch.uint8))
        refs.append(p)
    dev = [p.raw.to(gpu) for p in refs]
    return ops.QuantCache(*dev, kv_heads=heads, head_dim=d, block_size=bs, fmt=fmt), *refs


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


def check_attend(out, k, v, tables, lens, new, q, bs, dtype, *, window=0, sinks=0, scale=None):
    at = 0
    d = q.shape[-1]
    scale = d ** -0.5 if scale is None else scale
    for table, n, m in zip(tables, lens, new):
        if m:
            see = ref.visible(n, m, window, sinks)
            any_ = see.any(0).nonzero()[:, 0].tolist()
            at_places = ref.places(table, bs, any_)
            want, weight, size = ref.attend(k.get(*at_places), v.get(*at_places),
                                            q[at:at + m].cpu(), see[:, any_], scale)
            tol = ref.tolerance(want, weight, size, len(any_), d, dtype)
            got = out[at:at + m].cpu().double()
            bad = ~((got - want).abs() <= tol) & ~(got.isnan() & want.isnan())
            assert not bad.any(), (n, m, int(bad.sum()), float((got - want).abs().max()),
                                   bad.nonzero()[0].tolist())
        at += m


SHAPES = [("mxfp4", 128, 16), ("mxfp8", 128, 16), ("mxfp4", 64, 32), ("mxfp8", 64, 128),
          ("mxfp4", 256, 16), ("mxfp8", 256, 64)]


@pytest.mark.parametrize("fmt,d,bs", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_written_pages_are_the_definition_s_bytes(gpu, fmt, d, bs, dtype):
    heads, lens, new = 3, [1, 40, 17, 5 * bs + 3, 0, 16], [1, 1, 9, 2 * bs + 7, 0, 16]
    tables = tables_for(lens, bs, 24)
    cache, k_ref, v_ref = make(gpu, fmt, 24, bs, heads, d)
    t = sum(new)
    gen = torch.Generator().manual_seed(5)
    kv = []
    for shift in (0.0, 1.0):
        x = torch.randn(t, heads, d, generator=gen) * torch.exp2(
            torch.randint(-12, 12, (t, heads, d // 32, 1), generator=gen).float()).expand(
                -1, -1, -1, 32).reshape(t, heads, d) + shift
        kv.append(x.to(dtype))
    batch = batch_for(gpu, tables, lens, new, cache)
    ops.quant_write(cache, batch, kv[0].to(gpu), kv[1].to(gpu))
    at = 0
    for table, n, m in zip(tables, lens, new):
        block, inside = ref.places(table, bs, range(n - m, n))
        for p, x in ((k_ref, kv[0]), (v_ref, kv[1])):
            p.put(block, inside, *ref.quantise(fmt, x[at:at + m]))
        at += m
    assert torch.equal(cache.k_pages.cpu(), k_ref.raw)
    assert torch.equal(cache.v_pages.cpu(), v_ref.raw)


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_writing_odd_groups(gpu, fmt):
    """Groups of zeros, of the type's extremes, of ties and borders, with NaN and
    infinities."""
    rows = [torch.zeros(32), torch.full((32,), -0.0), torch.full((32,), 1e-40),
            torch.full((32,), 3e38), torch.full((32,), -1.5), torch.arange(32) / 4 - 4,
            torch.full((32,), ref.LARGEST[fmt]), torch.full((32,), ref.LARGEST[fmt] * 1.001)]
    rows += [ref.magnitudes(fmt)[:32].float().repeat(4)[:32]]
    m = ref.magnitudes(fmt)
    m = m[~m.isnan()]
    ties = torch.cat(((m[1:] + m[:-1]) / 2, m[-1:])).float()
    for part in ties.split(31):
        r = torch.full((32,), float(m[-1]))
        r[:part.numel()] = part
        rows += [r, -r, r * 2.0 ** -20]
    for bad in (math.nan, math.inf, -math.inf):
        r = torch.randn(32)
        r[7] = bad
        rows.append(r)
    while len(rows) % 4:
        rows.append(torch.ones(32) * 2.0 ** -115)
    x = torch.stack(rows).view(-1, 1, 128)
    t = x.size(0)
    cache, k_ref, v_ref = make(gpu, fmt, 4, 16, 1, 128, random_bytes=False)
    batch = batch_for(gpu, [[2, 0, 3]], [t], [t], cache)
    ops.quant_write(cache, batch, x.to(gpu), (-x).to(gpu))
    place = ref.places([2, 0, 3], 16, range(t))
    k_ref.put(*place, *ref.quantise(fmt, x))
    v_ref.put(*place, *ref.quantise(fmt, -x))
    assert torch.equal(cache.k_pages.cpu(), k_ref.raw)
    assert torch.equal(cache.v_pages.cpu(), v_ref.raw)


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_reading_every_code_under_every_scale(gpu, fmt, dtype):
    codes = 1 << ref.BITS[fmt]
    groups = 256 * max(1, codes // 32)
    t = groups // 4
    p = ref.Pages(fmt, t // 16, 16, 1, 128)
    c = torch.arange(t * 128) % codes
    s = torch.arange(t * 4) // max(1, codes // 32) % 256
    p.put(*ref.places(list(range(t // 16)), 16, range(t)),
          c.to(torch.uint8).view(t, 1, 128), s.to(torch.uint8).view(t, 1, 4))
    dev = p.raw.to(gpu)
    cache = ops.QuantCache(dev, dev.clone(), kv_heads=1, head_dim=128, block_size=16, fmt=fmt)
    batch = batch_for(gpu, [list(range(t // 16))], [t], [0], cache)
    k, v = ops.quant_read(cache, batch, dtype=dtype)
    want = p.get(*ref.places(list(range(t // 16)), 16, range(t))).to(F32).to(dtype)
    if fmt == "mxfp8":      # 2^-136 and below is no float32 of full precision: left to it
        assert torch.allclose(k.cpu(), want, rtol=0, atol=2.0 ** -126, equal_nan=True)
    else:
        assert torch.equal(k.cpu().nan_to_num(nan=7.5), want.nan_to_num(nan=7.5))
    assert torch.equal(k.nan_to_num(nan=7.5), v.nan_to_num(nan=7.5))


@pytest.mark.parametrize("fmt,d,bs", SHAPES)
@pytest.mark.parametrize("dtype,group,lens,new", [
    (BF16, 4, [1, 2, 16, 17, 33, 130, 1000], [1] * 7),
    (F16, 1, [31, 32, 64, 5], [1, 1, 1, 1]),
    (BF16, 7, [40, 700, 9], [2, 3, 4]),
    (F16, 3, [300, 129], [129, 64]),
    (BF16, 16, [50, 70, 0], [50, 3, 0]),
])
def test_attention(gpu, fmt, d, bs, dtype, group, lens, new):
    heads = 2
    blocks = sum(-(-n // bs) for n in lens) + 3
    tables = tables_for(lens, bs, blocks)
    cache, k, v = make(gpu, fmt, blocks, bs, heads, d, seed=len(lens))
    batch = batch_for(gpu, tables, lens, new, cache, heads=heads * group)
    q = torch.randn(sum(new), heads * group, d, generator=torch.Generator().manual_seed(9)).to(
        dtype).to(gpu)
    out = ops.quant_attend(cache, batch, q)
    check_attend(out, k, v, tables, lens, new, q, bs, dtype)


@pytest.mark.parametrize("fmt,d,bs", [SHAPES[0], SHAPES[3], SHAPES[4]])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 0), (40, 4), (33, 40), (5000, 2),
                                          (128, 200)])
@pytest.mark.parametrize("new", [1, 9, 70])
def test_windows_and_first_tokens(gpu, fmt, d, bs, window, sinks, new):
    lens = [new, 75, 300, 641]
    news = [min(new, n) for n in lens]
    blocks = sum(-(-n // bs) for n in lens) + 3
    tables = tables_for(lens, bs, blocks)
    cache, k, v = make(gpu, fmt, blocks, bs, 2, d, seed=3)
    held = [list(t) for t in tables]
    for t, n, m in zip(held, lens, news):        # columns that nothing sees are released
        see = ref.visible(n, m, window, sinks).any(0)
        for c in range(len(t)):
            if not see[c * bs:(c + 1) * bs].any():
                t[c] = -1
    batch = batch_for(gpu, held, lens, news, cache, heads=4, window=window, sinks=sinks)
    q = torch.randn(sum(news), 4, d, generator=torch.Generator().manual_seed(1)).to(BF16).to(gpu)
    out = ops.quant_attend(cache, batch, q)
    check_attend(out, k, v, tables, lens, news, q, bs, BF16, window=window, sinks=sinks)


def test_no_number_in_places_that_are_not_seen(gpu):
    """Stale bytes of every kind behind the sequence's end, outside the window
    and in blocks of others; NaN tokens poison only the rows that see them."""
    for fmt, d, window, sinks in (("mxfp4", 128, 0, 0), ("mxfp8", 64, 20, 3),
                                  ("mxfp4", 256, 33, 0), ("mxfp8", 128, 9, 17)):
        bs, lens, new = 16, [90, 37], [40, 1]
        blocks = 12
        tables = tables_for(lens, bs, blocks, seed=4)
        _, k, v = make(gpu, fmt, blocks, bs, 2, d, seed=8)
        for p in (k, v):        # whatever was there before
            junk = p.raw.clone().random_(0, 256, generator=torch.Generator().manual_seed(2))
            junk[:, ::5] = 255
            for table, n, m in zip(tables, lens, new):
                see = ref.visible(n, m, window, sinks).any(0).nonzero()[:, 0].tolist()
                block, inside = ref.places(table, bs, see)
                fresh = ref.Pages(fmt, blocks, bs, 2, d, raw=junk)
                c, s = p._views()
                cc, ss = c[block, :, inside], s[block, :, :, inside]
                if fmt == "mxfp4":
                    cc = torch.stack((cc & 15, cc >> 4), -1).flatten(-2)
                fresh.put(block, inside, cc, ss)
                junk = fresh.raw
            p.raw.copy_(junk)
        # tokens 70 and 85 of the first sequence hold a NaN in V's first group and
        # in its last one, token 88 one in K
        for t, p, group in ((70, v, 0), (85, v, d // 32 - 1), (88, k, 0)):
            block, inside = ref.places(tables[0], bs, [t])
            p._views()[1][block, 1, group, inside] = 255
        cache = ops.QuantCache(k.raw.to(gpu), v.raw.to(gpu), kv_heads=2, head_dim=d,
                               block_size=bs, fmt=fmt)
        batch = batch_for(gpu, tables, lens, new, cache, heads=6, window=window, sinks=sinks)
        q = torch.randn(sum(new), 6, d, generator=torch.Generator().manual_seed(1)).to(BF16).to(
            gpu)
        out = ops.quant_attend(cache, batch, q)
        check_attend(out, k, v, tables, lens, new, q, bs, BF16, window=window, sinks=sinks)
        got = out[:40].isnan().cpu()
        assert not got[:, :3].any() and not got[:20].any()      # head 0; rows before token 70
        assert got[38, 3:].all()                                # token 88 itself


def test_attention_keeps_rows_behind_the_batch_and_takes_any_stride(gpu):
    lens, new = [20, 200], [2, 3]
    tables = tables_for(lens, 16, 20)
    cache, k, v = make(gpu, "mxfp4", 20, 16, 2, 128, seed=1)
    batch = batch_for(gpu, tables, lens, new, cache, heads=8)
    gen = torch.Generator().manual_seed(3)
    for dtype in (BF16, F16):
        wide = torch.randn(9, 3 * 8 * 128 + 1, generator=gen).to(dtype).to(gpu)
        q = wide.as_strided((9, 8, 128), (3 * 8 * 128 + 1, 3 * 128, 1), 1)   # odd places
        out = torch.full((8, 9, 128), 7.0, dtype=dtype, device=gpu).transpose(0, 1)
        assert ops.quant_attend(cache, batch, q, out=out) is out
        assert (out[5:] == 7).all()
        check_attend(out, k, v, tables, lens, new, q, 16, dtype)
        same = q.contiguous()
        ops.quant_attend(cache, batch, same, out=same)          # in place
        assert torch.equal(same[:5], out[:5]) and torch.equal(same[5:], q[5:])


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_writing_and_reading_take_any_stride_and_keep_the_rest(gpu, fmt):
    bs, heads, d = 32, 3, 64
    lens, new = [50, 7, 33], [21, 1, 33]
    t = sum(new)
    tables = tables_for(lens, bs, 9)
    gen = torch.Generator().manual_seed(3)
    wide = torch.randn(t + 4, 2 * heads * d + 3, generator=gen)
    for dtype in (BF16, F32):
        cache, k_ref, v_ref = make(gpu, fmt, 9, bs, heads, d, seed=2)
        w = wide.to(dtype).to(gpu)
        k = w[:, 3:3 + heads * d].unflatten(1, (heads, d))
        v = w[:, 3 + heads * d:].unflatten(1, (heads, d))
        batch = batch_for(gpu, tables, lens, new, cache)
        ops.quant_write(cache, batch, k, v[:, :1].expand(-1, heads, -1))    # one V for all heads
        at = 0
        for table, n, m in zip(tables, lens, new):
            place = ref.places(table, bs, range(n - m, n))
            k_ref.put(*place, *ref.quantise(fmt, k[at:at + m].cpu()))
            v_ref.put(*place, *ref.quantise(fmt, v[at:at + m, :1].cpu().expand(-1, heads, -1)))
            at += m
        assert torch.equal(cache.k_pages.cpu(), k_ref.raw)
        assert torch.equal(cache.v_pages.cpu(), v_ref.raw)
        total = sum(lens)
        outs = [torch.full((total + 2, heads * d + 1), 5.0, dtype=dtype, device=gpu)
                for _ in range(2)]
        views = tuple(o[:, 1:].unflatten(1, (heads, d)) for o in outs)
        ops.quant_read(cache, batch, out=views)
        for o, p in zip(outs, (k_ref, v_ref)):
            want = torch.cat([p.get(*ref.places(table, bs, range(n)))
                              for table, n in zip(tables, lens)])
            assert torch.equal(o[:total, 1:].cpu(), want.to(dtype).flatten(1))
            assert (o[total:] == 5).all() and (o[:, 0] == 5).all()
        fresh = ops.quant_read(cache, batch, tokens="new", dtype=dtype)
        at, back = 0, 0
        for n, m in zip(lens, new):
            for got, whole in zip(fresh, views):
                assert torch.equal(got[at:at + m], whole[back + n - m:back + n])
            at, back = at + m, back + n


def test_empty_batches_and_sequences(gpu):
    cache, _, _ = make(gpu, "mxfp4", 4, 16, 2, 128)
    before = cache.k_pages.clone()
    for lens, new, tables in (([], [], []), ([0, 0], [0, 0], [[], [1]]), ([20], [0], [[0, 3]])):
        batch = batch_for(gpu, tables, lens, new, cache, heads=4)
        x = torch.zeros(0, 2, 128, dtype=BF16, device=gpu)
        ops.quant_write(cache, batch, x, x)
        assert ops.quant_attend(cache, batch, x.new_zeros(0, 4, 128)).shape == (0, 4, 128)
        assert ops.quant_attend(cache, batch, x.new_ones(3, 4, 128),
                                out=(o := x.new_ones(3, 4, 128))) is o and (o == 1).all()
        k, _ = ops.quant_read(cache, batch)
        assert k.size(0) == sum(lens)
        assert ops.quant_read(cache, batch, tokens="new")[0].size(0) == 0
    assert torch.equal(before, cache.k_pages)


def test_long_contexts_are_shared_out_and_joined(gpu):
    """Rows whose tiles go to many workgroups, and their sums of 40,000 terms."""
    lens, new = [40000, 9001], [1, 2]
    blocks = sum(-(-n // 128) for n in lens) + 1
    for dtype, fmt in ((BF16, "mxfp4"), (F16, "mxfp8")):
        tables = tables_for(lens, 128, blocks, seed=6)
        cache, k, v = make(gpu, fmt, blocks, 128, 1, 64, seed=5)
        batch = batch_for(gpu, tables, lens, new, cache, heads=7)
        q = torch.randn(3, 7, 64, generator=torch.Generator().manual_seed(2)).to(dtype).to(gpu)
        out = ops.quant_attend(cache, batch, q)
        check_attend(out, k, v, tables, lens, new, q, 128, dtype)
        assert all(torch.equal(ops.quant_attend(cache, batch, q), out) for _ in range(3))


def test_blocks_behind_four_gibibytes(gpu):
    """A cache whose last blocks lie past 2^32 bytes."""
    heads, bs, d = 8, 128, 128
    page = ops.quant_page_bytes("mxfp4", bs, heads, d)
    blocks = (1 << 32) // page + 5
    k = torch.empty(blocks, page, dtype=torch.uint8, device=gpu)
    v = torch.empty(blocks, page, dtype=torch.uint8, device=gpu)
    k[-4:] = 0
    v[-4:] = 0
    cache = ops.QuantCache(k, v, kv_heads=heads, head_dim=d, block_size=bs)
    lens, tables = [200, 100], [[blocks - 1, blocks - 3], [blocks - 2]]
    batch = batch_for(gpu, tables, lens, lens, cache, heads=8)
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(300, heads, d, generator=gen).to(BF16)
    ops.quant_write(cache, batch, x.to(gpu), -x.to(gpu))
    refs = [ref.Pages("mxfp4", 5, bs, heads, d) for _ in range(2)]
    near = [[4, 2], [3]]
    for p, y in zip(refs, (x, -x)):
        at = 0
        for t, n in zip(near, lens):
            p.put(*ref.places(t, bs, range(n)), *ref.quantise("mxfp4", y[at:at + n]))
            at += n
    assert torch.equal(k[-4:].cpu(), refs[0].raw[1:]) and torch.equal(v[-4:].cpu(), refs[1].raw[1:])
    q = torch.randn(300, heads, d, generator=gen).to(BF16).to(gpu)
    check_attend(ops.quant_attend(cache, batch, q), *refs, near, lens, lens, q, bs, BF16)
    got, _ = ops.quant_read(cache, batch)
    want = torch.cat([refs[0].get(*ref.places(t, bs, range(n))) for t, n in zip(near, lens)])
    assert torch.equal(got.cpu().double(), want)


def test_captured_calls_follow_the_batch(gpu):
    """A decode step captured once serves later steps: other lengths, other
    blocks, fewer sequences; eager work and another graph over the same
    batch lie between the replays."""
    heads, d, bs, blocks = 2, 128, 16, 200
    cache, k_ref, v_ref = make(gpu, "mxfp4", blocks, bs, heads, d, seed=7)
    steps = [([900, 33, 70], 1), ([901, 34, 71], 2), ([17, 1400], 3), ([5, 6, 7, 8], 4)]
    lens = steps[0][0]
    batch = batch_for(gpu, tables_for(lens, bs, blocks), lens, [1] * 3, cache, heads=8,
                      max_seqs=4, max_columns=180, max_tokens=4)
    gen = torch.Generator().manual_seed(1)
    kv = torch.zeros(2, 4, heads, d, dtype=BF16, device=gpu)
    q = torch.zeros(4, 8, d, dtype=BF16, device=gpu)
    out = torch.zeros_like(q)
    other = torch.zeros_like(q)
    new = (torch.zeros_like(kv[0]), torch.zeros_like(kv[0]))

    def step(to):
        ops.quant_write(cache, batch, kv[0], kv[1])
        ops.quant_attend(cache, batch, q, out=to)
        ops.quant_read(cache, batch, tokens="new", out=new)

    step(out)
    for table, length in zip(tables_for(lens, bs, blocks), lens):   # zeros were written
        place = ref.places(table, bs, [length - 1])
        for p in (k_ref, v_ref):
            p.put(*place, *ref.quantise("mxfp4", torch.zeros(1, heads, d)))
    torch.cuda.synchronize()
    graphs = []
    for to in (out, other):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(to)
        graphs.append(g)
    for lens, seed in steps:
        tables = tables_for(lens, bs, blocks, seed=seed)
        batch.update(tables, lens, [1] * len(lens))
        n = len(lens)
        x = torch.randn(2, 4, heads, d, generator=gen).to(BF16)
        kv.copy_(x)
        q.copy_(torch.randn(4, 8, d, generator=gen))
        out.fill_(3)
        other.fill_(3)
        for g in graphs:
            g.replay()
        for i, (table, length) in enumerate(zip(tables, lens)):
            place = ref.places(table, bs, [length - 1])
            k_ref.put(*place, *ref.quantise("mxfp4", x[0, i:i + 1]))
            v_ref.put(*place, *ref.quantise("mxfp4", x[1, i:i + 1]))
        assert torch.equal(cache.k_pages.cpu(), k_ref.raw)
        assert torch.equal(out, other) and (out[n:] == 3).all()
        check_attend(out, k_ref, v_ref, tables, lens, [1] * n, q, bs, BF16)
        eager = ops.quant_attend(cache, batch, q)
        assert torch.equal(eager[:n], out[:n])
        graphs[0].replay()
        torch.cuda.synchronize()
        assert torch.equal(eager[:n], out[:n])


def test_capture_has_to_hold_all_that_a_replay_may_reach(gpu):
    cache, _, _ = make(gpu, "mxfp4", 40, 16, 2, 128)
    batch = batch_for(gpu, [[0]], [3], [1], cache, max_seqs=4, max_columns=20, max_tokens=4)
    x = torch.zeros(2, 2, 128, dtype=BF16, device=gpu)
    ops.quant_write(cache, batch, x, x)             # eager: one token is enough
    out = torch.zeros_like(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for call in (lambda: ops.quant_write(cache, batch, x, x),
                     lambda: ops.quant_attend(cache, batch, x, out=out),
                     lambda: ops.quant_read(cache, batch, tokens="new", out=(x, out)),
                     lambda: ops.quant_read(cache, batch, out=(x, out))):
            with pytest.raises(ValueError, match="replay"):
                call()
        with pytest.raises(ValueError, match="outside the capture"):
            batch.update([[0]], [4], [1])
        out.fill_(1)
    with pytest.raises(ValueError, match="do not fit"):
        batch.update([[0, 1, 2]], [40], [20])
    wide = batch_for(gpu, [[0]], [3], [1], cache, max_columns=20, max_tokens=20)
    with pytest.raises(ValueError, match="room"):
        wide.update([[0, 1, 2]], [40], [20])        # 20 rows where up to 16 were planned for
    wide.update([[0, 1, 2]], [40], [16])
    with pytest.raises(ValueError, match="do not fit"):
        batch.update([[i] for i in range(5)], [1] * 5, [1] * 5)
    batch.update([[i] for i in range(4)], [1] * 4, [1] * 4)


def test_a_captured_read_of_released_columns_reads_nothing(gpu):
    cache, k, _ = make(gpu, "mxfp8", 12, 16, 2, 64)
    batch = batch_for(gpu, [[3, 4, 5]], [40], [1], cache, window=8, max_columns=4)
    out = tuple(torch.zeros(64, 2, 64, dtype=F16, device=gpu) for _ in range(2))
    ops.quant_read(cache, batch, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.quant_read(cache, batch, out=out)
    for table, whole in (([6, 7, 8], True), ([-1, -1, 8], False), ([1, 2, 3], True)):
        batch.update([table], [40], [1])
        out[0].fill_(9)
        g.replay()
        if whole:
            want = k.get(*ref.places(table, 16, range(40))).to(F16)
            assert torch.equal(out[0][:40].cpu(), want) and (out[0][40:] == 9).all()
        else:
            assert (out[0] == 9).all()


def test_dedicated_streams(gpu):
    lens = [300]
    tables = tables_for(lens, 16, 20)
    cache, k, v = make(gpu, "mxfp4", 20, 16, 2, 128, seed=1)
    q = torch.randn(1, 8, 128, generator=torch.Generator().manual_seed(3)).to(BF16).to(gpu)
    batch = batch_for(gpu, tables, lens, [1], cache, heads=8)
    own = ops.DedicatedStream(gpu)
    own.stream.wait_stream(torch.cuda.current_stream())
    out = ops.quant_attend(cache, batch, q, stream=own.stream)
    got, _ = ops.quant_read(cache, batch, dtype=F32, stream=own.stream)
    own.stream.synchronize()
    check_attend(out, k, v, tables, lens, [1], q, 16, BF16)
    assert torch.equal(got.cpu(), k.get(*ref.places(tables[0], 16, range(300))).float())
    own.close()
    batch.update(tables, lens, [1])             # behind calls on a stream that is gone
    assert torch.equal(ops.quant_attend(cache, batch, q), out)
    home = ops.DedicatedStream(gpu)
    home.stream.wait_stream(torch.cuda.current_stream())
    batch = batch_for(gpu, tables, lens, [1], cache, heads=8, stream=home.stream)
    home.close()
    assert torch.equal(ops.quant_attend(cache, batch, q), out)
    batch.update(tables, lens, [1])
    assert torch.equal(ops.quant_attend(cache, batch, q), out)
    del batch
    torch.cuda.synchronize()


def test_the_general_path_gives_the_same(gpu, monkeypatch):
    """Without the native argument readers."""
    from aegaeon_amd import _lib

    lens, new = [70, 33], [3, 1]
    tables = tables_for(lens, 32, 8)
    outs = []
    for general in (False, True):
        if general:
            monkeypatch.setattr(_lib, "_hostargs", _lib._GeneralPath)
        cache, _, _ = make(gpu, "mxfp8", 8, 32, 2, 64, seed=4)
        batch = batch_for(gpu, tables, lens, new, cache, heads=6)
        gen = torch.Generator().manual_seed(3)
        x, y = torch.randn(2, 4, 2, 64, generator=gen).to(F16).to(gpu)
        q = torch.randn(4, 6, 64, generator=gen).to(F16).to(gpu)
        ops.quant_write(cache, batch, x, y)
        outs.append((cache.k_pages, cache.v_pages, ops.quant_attend(cache, batch, q),
                     ops.quant_attend(cache, batch, q, scale=1), *ops.quant_read(cache, batch),
                     *ops.quant_read(cache, batch, tokens="new", dtype=F32)))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_streams_other_than_the_batch_s_own(gpu):
    """Calls on several streams over one batch, updates between them, and the
    batch dropped while they run."""
    lens = [700, 90]
    tables = tables_for(lens, 16, 60)
    cache, k, v = make(gpu, "mxfp4", 60, 16, 2, 128, seed=1)
    q = torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(3)).to(BF16).to(gpu)
    streams = [torch.cuda.Stream() for _ in range(3)]
    busy = torch.randn(4096, 4096, device=gpu)
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    (busy @ busy).sum()
    batch = batch_for(gpu, tables, lens, [1, 1], cache, heads=8, max_columns=60)
    outs = []
    for i, st in enumerate(streams):
        outs.append((lens, ops.quant_attend(cache, batch, q, stream=st)))
        with torch.cuda.stream(st):
            outs.append((lens, ops.quant_attend(cache, batch, q)))
        lens = [lens[0] - 100, lens[1] + 5]
        batch.update(tables_for([700, 200], 16, 60), lens, [1, 1], stream=streams[(i + 1) % 3])
        tables = tables_for([700, 200], 16, 60)
    last = [700, 90]
    del batch
    torch.empty(1 << 20, dtype=torch.uint8, device=gpu).fill_(255)
    torch.cuda.synchronize()
    for i, (n, out) in enumerate(outs):
        at = tables_for(last, 16, 60) if i < 2 else tables
        check_attend(out, k, v, at, n, [1, 1], q, 16, BF16)


def test_a_dropped_batch_s_memory_waits_for_the_stream_it_moved_to(gpu):
    """The stream that a batch was made on, whose allocations may take the plan's
    memory next, is behind the calls on the stream it was updated to."""
    lens = [300]
    tables = tables_for(lens, 16, 20)
    cache, k, v = make(gpu, "mxfp4", 20, 16, 2, 128, seed=1)
    q = torch.randn(1, 8, 128, generator=torch.Generator().manual_seed(3)).to(BF16).to(gpu)
    made, moved = torch.cuda.Stream(), torch.cuda.Stream()
    for calls_elsewhere in (False, True):
        torch.cuda.synchronize()
        batch = batch_for(gpu, tables, lens, [1], cache, heads=8, stream=made)
        batch.update(tables, lens, [1], stream=moved)
        with torch.cuda.stream(moved):
            if calls_elsewhere:
                outs = [ops.quant_attend(cache, batch, q, stream=torch.cuda.default_stream())]
            torch.cuda._sleep(1 << 29)      # a good fraction of a second
            out = ops.quant_attend(cache, batch, q)
        del batch
        behind = made.record_event()
        assert not behind.query()
        behind.synchronize()
        assert moved.query()
        check_attend(out, k, v, tables, lens, [1], q, 16, BF16)
        if calls_elsewhere:
            assert torch.equal(outs[0], out)


def test_an_update_that_fails_leaves_no_batch_by_halves(gpu, monkeypatch):
    """Calls go by the host's plan and kernels by the device's."""
    tables = tables_for([300, 40], 16, 30)
    cache, k, v = make(gpu, "mxfp4", 30, 16, 2, 128, seed=1)
    q = torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(3)).to(BF16).to(gpu)
    batch = batch_for(gpu, tables, [300, 40], [1, 1], cache, heads=8, max_tokens=20)
    before = ops.quant_attend(cache, batch, q)
    host = batch._host.copy()
    empty = torch.empty

    def no_pinned_memory(*args, **kw):
        if kw.get("pin_memory"):
            raise RuntimeError("none left")
        return empty(*args, **kw)

    with monkeypatch.context() as m:
        m.setattr(torch, "empty", no_pinned_memory)
        with pytest.raises(RuntimeError, match="none left"):
            batch.update(tables, [100, 20], [1, 1])
    assert (batch._host == host).all()
    assert torch.equal(ops.quant_attend(cache, batch, q), before)

    class NoCopy:
        data_ptr = batch._plan.data_ptr

        def copy_(self, *args, **kw):
            raise RuntimeError("no copy")

    plan, batch._plan = batch._plan, NoCopy()
    with pytest.raises(RuntimeError, match="no copy"):
        batch.update(tables, [100, 20], [1, 1])
    batch._plan = plan
    x = torch.zeros(2, 2, 128, dtype=BF16, device=gpu)
    for call in (lambda: ops.quant_attend(cache, batch, q), lambda: ops.quant_read(cache, batch),
                 lambda: ops.quant_write(cache, batch, x, x),
                 lambda: batch.update(tables, [300, 40], [1, 1])):
        with pytest.raises(ValueError, match="no plan"):
            call()


def test_an_update_during_a_capture_of_the_batch_s_stream_is_refused(gpu):
    """On any stream: it would wait for the captured calls, and so join them."""
    lens = [300]
    tables = tables_for(lens, 16, 20)
    cache, k, v = make(gpu, "mxfp4", 20, 16, 2, 128, seed=1)
    q = torch.randn(1, 8, 128, generator=torch.Generator().manual_seed(3)).to(BF16).to(gpu)
    home, other = torch.cuda.Stream(), torch.cuda.Stream()
    batch = batch_for(gpu, tables, lens, [1], cache, heads=8, max_columns=20, stream=home)
    want = ops.quant_attend(cache, batch, q)
    out = torch.zeros_like(want)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=home):
        ops.quant_attend(cache, batch, q, out=out)
        with torch.cuda.stream(other):
            with pytest.raises(ValueError, match="outside the capture"):
                batch.update(tables, lens, [1])
        with pytest.raises(ValueError, match="outside the capture"):
            batch.update(tables, lens, [1], stream=other)
        with torch.cuda.stream(other):
            with pytest.raises(ValueError, match="while a stream is captured"):
                batch_for(gpu, tables, lens, [1], cache, stream=home)
    for _ in range(3):
        out.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    batch.update(tables, [200], [1], stream=other)
    check_attend(ops.quant_attend(cache, batch, q), k, v, tables, [200], [1], q, 16, BF16)


def test_a_cache_is_written_attended_moved_and_attended_again(gpu):
    """One model step after another as a serving engine makes them: two layers
    over a composite cache, a prompt, decode steps, a swap to the host and back to other
    blocks beside a copy within HBM, and a decode step over what came back."""
    from aegaeon_amd.layout import allocate_composite_cache, quant_kv_tensor_specs

    layers, heads, d, bs, blocks = 2, 2, 128, 16, 24
    specs = quant_kv_tensor_specs(layers, blocks, bs, heads, d, "mxfp4")
    composite = allocate_composite_cache(specs, blocks, gpu)
    caches = [ops.QuantCache(composite.segment_tensor(2 * i), composite.segment_tensor(2 * i + 1),
                             kv_heads=heads, head_dim=d, block_size=bs) for i in range(layers)]
    gen = torch.Generator().manual_seed(4)
    table = [3, 9, 4, 11]
    length = 50
    k_refs = [ref.Pages("mxfp4", blocks, bs, heads, d) for _ in range(layers)]
    v_refs = [ref.Pages("mxfp4", blocks, bs, heads, d) for _ in range(layers)]

    def model_step(table, length, new):
        batch = batch_for(gpu, [table], [length], [new], caches[0], heads=8)
        q = torch.randn(new, 8, d, generator=gen).to(BF16).to(gpu)
        for cache, kr, vr in zip(caches, k_refs, v_refs):
            k, v = torch.randn(2, new, heads, d, generator=gen).to(BF16)
            ops.quant_write(cache, batch, k.to(gpu), v.to(gpu))
            place = ref.places(table, bs, range(length - new, length))
            kr.put(*place, *ref.quantise("mxfp4", k))
            vr.put(*place, *ref.quantise("mxfp4", v))
            out = ops.quant_attend(cache, batch, q)
            check_attend(out, kr, vr, [table], [length], [new], q, bs, BF16)

    model_step(table, length, length)
    for length in (51, 52):
        model_step(table, length, 1)
    page = specs[0].size // blocks
    pool = ops.PinnedHostPool(8 * composite.page_size_bytes)
    layout = ops.SegmentLayout(composite.backing, [page] * 4, [s.cpu_offset for s in
                                                               composite.segments],
                               [1] * 4, blocks, [1], pool.tensor, composite.page_size_bytes, 0)
    host, back, moved = [5, 0, 2, 7], [20, 1, 6, 15], [8, 22]
    layout.swap(table, host, [0] * 4, [0] * 4, [1] * 4, False)
    for t in composite.backing:
        t.view(blocks, page)[table] = -1
    layout.swap(host, back, [0] * 4, [0] * 4, [1] * 4, True)
    ops.copy_blocks([t.view(blocks, page) for t in composite.backing], back[:2], moved)
    for p in (*k_refs, *v_refs):
        p.raw[back] = p.raw[table]
        p.raw[moved] = p.raw[back[:2]]
    model_step(moved + back[2:], 53, 1)
    torch.cuda.synchronize()
    pool.free()


def test_partial_pages_of_kernel_blocks(gpu):
    """Manager pages of two kernel blocks: the batch names kernel blocks, the
    swap moves the live ones of a page."""
    from aegaeon_amd.cache_groups import CacheGroupRuntimeConfig

    group = CacheGroupRuntimeConfig("attention", 32, 16)
    pages, heads, d, length = 10, 2, 128, 75        # pages of 32: two whole, one by 11 tokens
    cache, k, v = make(gpu, "mxfp4", 2 * pages, 16, heads, d, seed=6)
    page = 2 * cache.page_bytes
    backing = [cache.k_pages.view(pages, page), cache.v_pages.view(pages, page)]
    pool = ops.PinnedHostPool(6 * 2 * page)
    layout = ops.SegmentLayout(backing, [page] * 2, [0, page], [1, 1], pages, [2], pool.tensor,
                               2 * page, 0)
    table, back = [7, 2, 5], [1, 9, 4]
    q = torch.randn(1, 6, d, generator=torch.Generator().manual_seed(1)).to(BF16).to(gpu)

    def attend(ids):
        batch = batch_for(gpu, [group.to_kernel_block_ids(ids)], [length], [1], cache, heads=6)
        return ops.quant_attend(cache, batch, q)

    before = attend(table)
    check_attend(before, k, v, [group.to_kernel_block_ids(table)], [length], [1], q, 16, BF16)
    extents = ([0] * 3, [0] * 3, [2, 2, 1])
    layout.swap(table, [3, 0, 4], *extents, False)
    for t in backing:
        t[table] = -1
    layout.swap([3, 0, 4], back, *extents, True)
    assert torch.equal(attend(back), before)
    torch.cuda.synchronize()
    pool.free()


def test_refusals_on_the_device(gpu):
    cache, _, _ = make(gpu, "mxfp4", 8, 16, 2, 128)
    batch = batch_for(gpu, [[0, 1]], [20], [2], cache, heads=4)
    ok = torch.zeros(2, 2, 128, dtype=BF16, device=gpu)
    q = torch.zeros(2, 4, 128, dtype=BF16, device=gpu)

    def bad(match, fn):
        with pytest.raises(ValueError, match=match):
            fn()

    bad("tokens", lambda: ops.quant_write(cache, batch, ok[:1], ok[:1]))
    bad("must be", lambda: ops.quant_write(cache, batch, ok[:, :1], ok[:, :1]))
    bad("differ", lambda: ops.quant_write(cache, batch, ok, ok.half()))
    bad("not supported", lambda: ops.quant_write(cache, batch, ok.double(), ok.double()))
    bad("contiguous", lambda: ops.quant_write(cache, batch, ok.transpose(1, 2).contiguous()
                                              .transpose(1, 2), ok))
    bad("gradient", lambda: ops.quant_write(cache, batch, ok.clone().requires_grad_(), ok))
    bad("on cpu", lambda: ops.quant_write(cache, batch, ok.cpu(), ok.cpu()))
    bad("not supported", lambda: ops.quant_attend(cache, batch, q.float()))
    bad("scale", lambda: ops.quant_attend(cache, batch, q, scale=0.0))
    bad("scale", lambda: ops.quant_attend(cache, batch, q, scale=math.nan))
    bad("rows of out", lambda: ops.quant_attend(cache, batch, q, out=q.new_zeros(3, 4, 128)))
    bad("overlap", lambda: ops.quant_attend(cache, batch, q, out=q[:, :1].expand(-1, 4, -1)))
    bad("overlap", lambda: ops.quant_read(cache, batch, tokens="new",
                                          out=(ok[:1].expand(2, -1, -1), ok)))
    bad("'all' or 'new'", lambda: ops.quant_read(cache, batch, tokens="some"))
    same = ops.QuantCache(cache.k_pages, cache.k_pages, kv_heads=2, head_dim=128, block_size=16)
    bad("overlap", lambda: ops.quant_write(same, batch, ok, ok))
    small = ops.QuantCache(cache.k_pages[:4].contiguous(), cache.v_pages[:4].contiguous(),
                           kv_heads=2, head_dim=128, block_size=16)
    bad("blocks", lambda: ops.quant_write(small, batch, ok, ok))
    holes = batch_for(gpu, [[-1, -1, 5]], [40], [1], cache, window=4)
    bad("released", lambda: ops.quant_read(cache, holes))
    assert ops.quant_read(cache, holes, tokens="new")[0].shape == (1, 2, 128)
    other = batch_for(gpu, [[0]], [3], [1], small)
    ops.quant_attend(cache, other, ok[:1])
    with pytest.raises(ValueError, match="pages"):
        ops.QuantCache(cache.k_pages[:, :-16].contiguous(), cache.v_pages, kv_heads=2,
                       head_dim=128, block_size=16)


def test_what_a_call_writes_shares_no_byte_with_its_other_arguments(gpu):
    """Shifted views and the like are refused; slices of one buffer that only
    interleave are not, and rows behind the batch's last token do not count."""
    lens, new = [40, 20], [2, 1]
    tables = tables_for(lens, 16, 8)
    cache, k, v = make(gpu, "mxfp4", 8, 16, 2, 128, seed=1)
    batch = batch_for(gpu, tables, lens, new, cache, heads=4)
    buf = torch.randn(7, 4, 256, generator=torch.Generator().manual_seed(3)).to(BF16).to(gpu)
    q = buf[:3, :, :128]
    kept = buf.clone()
    pages = cache.k_pages.view(-1)[:6 * 2 * 128 * 2 * 2].view(BF16).view(-1, 4, 128)

    def bad(match, fn):
        with pytest.raises(ValueError, match=match):
            fn()

    bad("out and q overlap", lambda: ops.quant_attend(cache, batch, q, out=buf[1:4, :, :128]))
    bad("out and q overlap", lambda: ops.quant_attend(cache, batch, q, out=buf[:3, :, 64:192]))
    bad("out and q overlap", lambda: ops.quant_attend(
        cache, batch, q, out=buf.view(-1)[:3 * 512].view(3, 4, 128)))
    bad("out and the K cache", lambda: ops.quant_attend(cache, batch, q, out=pages[:3]))
    bad("k and v overlap", lambda: ops.quant_read(cache, batch, tokens="new", out=(
        buf[:3, :2, :128], buf[:3, :2, :128])))
    bad("k and v overlap", lambda: ops.quant_read(cache, batch, tokens="new", out=(
        buf[:3, :2, :128], buf[:3, 1:3, :128])))
    bad("v and the K cache", lambda: ops.quant_read(cache, batch, tokens="new", out=(
        buf[:3, :2, :128], pages[:3, :2])))
    bad("k and the K cache", lambda: ops.quant_write(cache, batch, pages[:3, :2],
                                                     buf[:3, :2, :128]))
    bad("K cache and the V cache", lambda: ops.quant_write(
        ops.QuantCache(cache.k_pages, cache.k_pages, kv_heads=2, head_dim=128, block_size=16),
        batch, buf[:3, :2, :128], buf[:3, 2:, :128]))
    roomy = batch_for(gpu, tables, lens, new, cache, heads=4, max_seqs=64)
    inside = roomy._plan[:3 * 4 * 256].view(BF16).view(3, 4, 128)
    bad("out and the plan", lambda: ops.quant_attend(cache, roomy, q, out=inside))
    assert torch.equal(buf, kept) and torch.equal(cache.k_pages.cpu(), k.raw)
    # one buffer's halves, and its rows behind the batch's last
    want = ops.quant_attend(cache, batch, q)
    check_attend(want, k, v, tables, lens, new, q, 16, BF16)
    beside = buf[:3, :, 128:]
    assert torch.equal(ops.quant_attend(cache, batch, q, out=beside), want)
    assert torch.equal(q, kept[:3, :, :128])
    behind = buf[3:, :, :128]
    assert torch.equal(ops.quant_attend(cache, batch, buf[:4, :, :128], out=behind)[:3], want)
    got = ops.quant_read(cache, batch, tokens="new", out=(buf[:3, :2, :128], buf[:3, 2:, :128]))
    assert all(torch.equal(a, b) for a, b in zip(
        got, ops.quant_read(cache, batch, tokens="new")))


@pytest.mark.parametrize("fmt,d,bs", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("new", [1, 12, 60])
def test_no_numbers_that_a_write_stored(gpu, fmt, d, bs, dtype, new):
    """A NaN or an infinity in a token's K makes every row that sees it none, one in V
    the 32 values of its group: also in old tokens, whose tiles every row sees,
    and as quant_write stores them (codes of 0 under the byte 255)."""
    n, heads = 300, 3
    tables = tables_for([n], bs, 24)
    cache, k_ref, v_ref = make(gpu, fmt, 24, bs, heads, d, seed=2)
    gen = torch.Generator().manual_seed(5)
    k, v = (torch.randn(n, heads, d, generator=gen) for _ in range(2))
    k[37, 0, d - 1] = math.nan          # all of head 0's queries
    v[5, 1, 3] = math.inf               # the first group of head 1's
    v[n - 1, 2, d - 1] = -math.inf      # the last group of head 2's last query
    whole = batch_for(gpu, tables, [n], [n], cache)
    ops.quant_write(cache, whole, k.to(dtype).to(gpu), v.to(dtype).to(gpu))
    place = ref.places(tables[0], bs, range(n))
    k_ref.put(*place, *ref.quantise(fmt, k.to(dtype)))
    v_ref.put(*place, *ref.quantise(fmt, v.to(dtype)))
    batch = batch_for(gpu, tables, [n], [new], cache, heads=2 * heads)
    q = torch.randn(new, 2 * heads, d, generator=gen).to(dtype).to(gpu)
    out = ops.quant_attend(cache, batch, q)
    check_attend(out, k_ref, v_ref, tables, [n], [new], q, bs, dtype)
    none = out.isnan().cpu()
    want = torch.zeros_like(none)
    want[:, :2] = True
    want[:, 2:4, :32] = True
    want[-1, 4:, -32:] = True
    assert torch.equal(none, want)


def test_an_error_that_other_code_left_is_not_a_call_s_own(gpu):
    """HIP keeps a thread's last error until someone asks: a call over a quantised
    cache neither fails for it nor runs a second time (in place that would take
    results for queries)."""
    lens, new = [400, 90], [1, 30]
    tables = tables_for(lens, 16, 40)
    cache, k, v = make(gpu, "mxfp4", 40, 16, 2, 128, seed=1)
    batch = batch_for(gpu, tables, lens, new, cache, heads=8)
    gen = torch.Generator().manual_seed(3)
    q = torch.randn(31, 8, 128, generator=gen).to(BF16).to(gpu)
    x = torch.randn(31, 2, 128, generator=gen).to(BF16).to(gpu)
    hip = ctypes.CDLL("libamdhip64.so.7")

    def leave_an_error():
        assert hip.hipSetDevice(4096) != 0      # no such device: nothing else happens
        assert hip.hipPeekAtLastError() != 0

    for stream in (None, torch.cuda.current_stream()):
        want = ops.quant_attend(cache, batch, q)
        same = q.clone()
        torch.cuda.synchronize()
        leave_an_error()
        ops.quant_attend(cache, batch, same, out=same, stream=stream)
        assert torch.equal(same, want)
        leave_an_error()
        ops.quant_write(cache, batch, x, x, stream=stream)
        leave_an_error()
        ops.quant_read(cache, batch, stream=stream)
        ops.quant_write(cache, batch, x, x)
        assert hip.hipGetLastError() == 0


def test_a_call_that_fails_is_not_made_again(gpu):
    """The native path takes what it cannot read to the general one; a call that the
    library itself refused or could not finish is an error at once."""
    import struct

    from aegaeon_amd import _lib

    cache, _, _ = make(gpu, "mxfp4", 8, 16, 2, 128)
    batch = batch_for(gpu, [[0, 1]], [20], [2], cache, heads=4)
    x = torch.zeros(2, 2, 128, dtype=BF16, device=gpu)
    q = torch.zeros(2, 4, 128, dtype=BF16, device=gpu)
    calls = []

    @ctypes.CFUNCTYPE(ctypes.c_int)
    def fails():
        calls.append(1)
        return 98       # hipErrorInvalidDeviceFunction, as a launch would return it

    at = ctypes.cast(fails, ctypes.c_void_p).value
    was = cache._packed
    cache._packed = struct.pack("3q", at, at, at) + was[24:]
    for call in (lambda: ops.quant_write(cache, batch, x, x),
                 lambda: ops.quant_read(cache, batch),
                 lambda: ops.quant_read(cache, batch, tokens="new", out=(x, x.clone())),
                 lambda: ops.quant_attend(cache, batch, q)):
        calls.clear()
        with pytest.raises(_lib.AegkvError):
            call()
        assert len(calls) == 1
    cache._packed = was
    with pytest.raises(ValueError, match="tokens"):
        ops.quant_write(cache, batch, x[:1], x[:1])
    ops.quant_attend(cache, batch, q)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("new", [1, 20, 90])
def test_scores_of_any_size(gpu, dtype, new):
    """Scores as large as 32 bits hold, of either sign: their differences count.
    One value of a query times one of a key, so that every score is exact; the
    tokens with the largest one share the result."""
    d, n, heads = 64, 400, 2
    tables = tables_for([n], 16, 30)
    big = 2.0 ** 100 if dtype == BF16 else 2.0 ** 13
    for sign in (1, -1):
        k_ref = ref.Pages("mxfp8", 30, 16, heads, d)
        v_ref = ref.Pages("mxfp8", 30, 16, heads, d)
        gen = torch.Generator().manual_seed(5)
        k = torch.zeros(n, heads, d)
        k[:, :, 0] = sign * big * (1 + torch.randint(0, 8, (n, heads), generator=gen) / 8)
        v = torch.randn(n, heads, d, generator=gen)
        place = ref.places(tables[0], 16, range(n))
        k_ref.put(*place, *ref.quantise("mxfp8", k))
        v_ref.put(*place, *ref.quantise("mxfp8", v))
        assert torch.equal(k_ref.get(*place), k.double())       # no key was rounded
        cache = ops.QuantCache(k_ref.raw.to(gpu), v_ref.raw.to(gpu), kv_heads=heads, head_dim=d,
                               block_size=16, fmt="mxfp8")
        batch = batch_for(gpu, tables, [n], [new], cache, heads=4)
        for size in ((1, 2.0 ** 20) if dtype == BF16 else (1, 2.0 ** 15)):
            q = torch.zeros(new, 4, d)
            q[:, :, 0] = size
            q = q.to(dtype)
            out = ops.quant_attend(cache, batch, q.to(gpu), scale=1.0).cpu().double()
            see = ref.visible(n, new, 0, 0)
            want, weight, _ = ref.attend(k_ref.get(*place), v_ref.get(*place), q, see, 1.0)
            # scores are exact and differ by 2^9 and more, where they do: beside what
            # rounds probabilities and result, only sums of up to n terms in 32 bits
            u = torch.finfo(dtype).eps / 2
            tol = u * want.abs() + weight * (u + (n + 8) * 2.0 ** -24) * 1.01
            assert ((out - want).abs() <= tol).all(), (sign, size, float((out - want).abs().max()))


@pytest.mark.parametrize("fmt,d,bs", SHAPES)
@pytest.mark.parametrize("new", [1, 12, 60])
@pytest.mark.parametrize("group,window,sinks", [(1, 0, 0), (4, 0, 0), (4, 50, 5)])
def test_values_beyond_the_queries_type(gpu, fmt, d, bs, new, group, window, sinks):
    """V of up to 3e5 under float16 queries: rows that see it have the sum as 32 bits
    hold it, the others are as without it; a code that is no number (mxfp8) makes one
    value none, in the rows that see its token."""
    n, heads = 200, 2
    tables = tables_for([n], bs, 16)
    cache, k, v = make(gpu, fmt, 16, bs, heads, d, seed=4)
    c, s = v._views()
    byte = {"mxfp4": 127 + 15, "mxfp8": 127 + 9}[fmt]
    tokens = [3, 33, n - new, n - new // 2 - 1, n - 1]
    for i, t in enumerate(tokens):
        block, inside = ref.places(tables[0], bs, [t])
        s[block, i % heads, i % (d // 32), inside] = byte
    if fmt == "mxfp8":
        block, inside = ref.places(tables[0], bs, [n - 1])
        c[block, 1, inside, d - 3] = 0x7F
    cache = ops.QuantCache(k.raw.to(gpu), v.raw.to(gpu), kv_heads=heads, head_dim=d,
                           block_size=bs, fmt=fmt)
    batch = batch_for(gpu, tables, [n], [new], cache, heads=heads * group, window=window,
                      sinks=sinks)
    q = torch.randn(new, heads * group, d, generator=torch.Generator().manual_seed(1))
    q = q.to(F16).to(gpu)
    out = ops.quant_attend(cache, batch, q)
    see = ref.visible(n, new, window, sinks)
    any_ = see.any(0).nonzero()[:, 0].tolist()
    place = ref.places(tables[0], bs, any_)
    want, weight, size = ref.attend(k.get(*place), v.get(*place), q.cpu(), see[:, any_], d ** -0.5)
    tol = ref.tolerance(want, weight, size, len(any_), d, F16)
    got = out.cpu().double()
    near = (got - want).abs() <= tol
    # the result is a float16 itself: from 65520 on, half a step past the largest
    # one, a sum that is right rounds to infinity
    far = (got == want.sign() * math.inf) & (want.abs() + tol >= 65520)
    assert (near | far | (got.isnan() & want.isnan())).all()
    none = out.isnan().cpu()
    if fmt == "mxfp8":
        assert none[-1, group:, d - 3].all()
        none[-1, group:, d - 3] = False
    assert not none.any()


@pytest.mark.parametrize("fmt,d,bs", [SHAPES[0], SHAPES[1]])
def test_values_of_two_to_the_128_stay_with_the_rows_that_see_them(gpu, fmt, d, bs):
    """The one power of two that bfloat16 and float32 lack."""
    n, new = 100, 40
    tables = tables_for([n], bs, 16)
    cache, k, v = make(gpu, fmt, 16, bs, 2, d, seed=4)
    c, s = v._views()
    block, inside = ref.places(tables[0], bs, [n - 1])
    s[block, 1, 0, inside] = 254 if fmt == "mxfp4" else 248
    c[block, 1, inside, 0] = 0x66 if fmt == "mxfp4" else 0x78       # 4 * 2^127, 256 * 2^121
    cache = ops.QuantCache(k.raw.to(gpu), v.raw.to(gpu), kv_heads=2, head_dim=d, block_size=bs,
                           fmt=fmt)
    batch = batch_for(gpu, tables, [n], [new], cache)
    q = torch.randn(new, 2, d, generator=torch.Generator().manual_seed(1)).to(BF16).to(gpu)
    out = ops.quant_attend(cache, batch, q)
    assert not out[-1, 1, 0].isfinite()
    assert out[:-1].isfinite().all() and out[-1, 0].isfinite().all()
    check_attend(out[:-1], k, v, tables, [n - 1], [new - 1], q[:-1], bs, BF16)


def test_a_step_captured_at_its_largest_serves_smaller_ones(gpu):
    """The room is what the first batch holds itself; later steps have fewer
    sequences, longer ones and other places in their blocks."""
    heads, d, bs, blocks = 2, 128, 16, 420
    cache, k, v = make(gpu, "mxfp4", blocks, bs, heads, d, seed=7)
    lens = [128] * 16
    batch = batch_for(gpu, tables_for(lens, bs, blocks), lens, [1] * 16, cache, heads=8,
                      max_seqs=16, max_columns=128, max_tokens=16)
    gen = torch.Generator().manual_seed(1)
    q = torch.randn(16, 8, d, generator=gen).to(BF16).to(gpu)
    out = torch.zeros_like(q)
    ops.quant_attend(cache, batch, q, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.quant_attend(cache, batch, q, out=out)
    for seed, lens, new in ((1, [2048], [1]), (2, [1024, 17, 900], [1, 4, 2]), (3, [128] * 16,
                            [1] * 16), (4, [], []), (5, [31, 0, 1500], [3, 0, 1])):
        tables = tables_for(lens, bs, blocks, seed=seed)
        batch.update(tables, lens, new)
        out.fill_(3)
        g.replay()
        n = sum(new)
        check_attend(out, k, v, tables, lens, new, q, bs, BF16)
        assert (out[n:] == 3).all()
        assert torch.equal(ops.quant_attend(cache, batch, q)[:n], out[:n])


def test_tangents_are_refused(gpu, monkeypatch):
    """As gradients are: a derivative would be lost without a word."""
    from torch.autograd import forward_ad

    from aegaeon_amd import _lib

    cache, _, _ = make(gpu, "mxfp4", 8, 16, 2, 128)
    batch = batch_for(gpu, [[0, 1]], [20], [2], cache, heads=4)
    x = torch.zeros(2, 2, 128, dtype=BF16, device=gpu)
    q = torch.zeros(2, 4, 128, dtype=BF16, device=gpu)
    for general in (False, True):
        if general:
            monkeypatch.setattr(_lib, "_hostargs", _lib._GeneralPath)
        with forward_ad.dual_level():
            dx = forward_ad.make_dual(x, torch.ones_like(x))
            dq = forward_ad.make_dual(q, torch.ones_like(q))
            for call in (lambda: ops.quant_write(cache, batch, dx, x),
                         lambda: ops.quant_write(cache, batch, x, dx),
                         lambda: ops.quant_attend(cache, batch, dq),
                         lambda: ops.quant_attend(cache, batch, q, out=dq),
                         lambda: ops.quant_read(cache, batch, tokens="new", out=(x, dx))):
                with pytest.raises(ValueError, match="tangent"):
                    call()
            ops.quant_attend(cache, batch, q)
        ops.quant_write(cache, batch, x, x)


@pytest.mark.parametrize("fmt,byte", [("mxfp4", 127 + 16), ("mxfp8", 127 + 9)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_values_beyond_the_queries_type_in_rows_that_are_cut(gpu, fmt, byte, dtype):
    """In long contexts, whose parts are joined, for single tokens and for many rows."""
    d, bs, lens, new = 64, 16, [9000, 3000], [1, 150]
    blocks = sum(-(-n // bs) for n in lens) + 2
    tables = tables_for(lens, bs, blocks, seed=3)
    cache, k, v = make(gpu, fmt, blocks, bs, 1, d, seed=5)
    c, s = v._views()
    for table, n, m in zip(tables, lens, new):
        for i, t in enumerate((0, 31, n // 2, n - m, n - 1)):
            block, inside = ref.places(table, bs, [t])
            s[block, 0, i % 2, inside] = byte
        if fmt == "mxfp8":      # no numbers: one that all rows see, one that only the last does
            for t, at in ((n // 3, 5), (n - 1, 40)):
                block, inside = ref.places(table, bs, [t])
                c[block, 0, inside, at] = 0xFF
    cache = ops.QuantCache(k.raw.to(gpu), v.raw.to(gpu), kv_heads=1, head_dim=d, block_size=bs,
                           fmt=fmt)
    batch = batch_for(gpu, tables, lens, new, cache, heads=7)
    assert batch._workspace[d] > 0
    q = torch.randn(sum(new), 7, d, generator=torch.Generator().manual_seed(2)).to(dtype).to(gpu)
    out = ops.quant_attend(cache, batch, q)
    check_attend(out, k, v, tables, lens, new, q, bs, dtype)
    none = torch.zeros(sum(new), 7, d, dtype=torch.bool)
    if fmt == "mxfp8":
        none[:, :, 5] = True
        none[[0, -1], :, 40] = True
    assert torch.equal(out.isnan().cpu(), none)

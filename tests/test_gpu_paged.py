"""Paged attention, paged q/k/v post-processing, page copies and the cache that
uses them, against plain forms in 64 bits."""
import math

import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu

bf = torch.bfloat16


def rows(T, width, dev, seed=1, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, width, generator=g) * std).to(bf).to(dev)


def check_attention(batch, heads, dev, *, window=0, sinks=0, scale=None, max_q=None, missing=(), q=None, seed=1):
    from alveare_amd import attention_paged

    D = batch.D
    scale = 1.5 / math.sqrt(D) if scale is None else scale
    q = rows(batch.T, heads * D, dev, seed) if q is None else q
    want, tol = R.attention(q, batch, heads, window, sinks, scale, missing)
    for mq in ((0, max(max(batch.n), 1)) if max_q is None else (max_q,)):
        out = torch.full((batch.T, heads * D), 7.0, dtype=bf, device=dev)
        attention_paged(q, *batch.args(), heads=heads, window=window, sinks=sinks, scale=scale, max_q=mq, out=out)
        m = want.shape[0]
        got = out[:m].double().cpu().view_as(want)
        assert torch.isfinite(got).all(), f"max_q={mq}"
        bad = (got - want).abs() > tol
        assert not bad.any(), (f"max_q={mq}: {int(bad.sum())} of {bad.numel()} values off, worst "
                               f"{float(((got - want).abs() / tol).max()):.2f} tolerances, first {bad.nonzero()[0].tolist()}")
        assert (out[m:] == 7.0).all(), "rows past the last sequence changed"
    return q


LAYOUTS = [(16, 8, 256), (16, 1, 512), (4, 1, 256), (32, 8, 64), (6, 2, 128), (1, 1, 64), (5, 5, 128), (12, 4, 256),
           (17, 1, 64), (40, 1, 128)]


@pytest.mark.parametrize("heads,kv_heads,D", LAYOUTS)
@pytest.mark.parametrize("page", [16, 64])
def test_attention_decode(dev, heads, kv_heads, D, page):
    """One token each, lengths around tile and page ends, one and zero included."""
    total = [1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 0, 33]
    n = [min(1, t) for t in total]
    b = R.Batch(n, total, kv_heads=kv_heads, D=D, page=page, dev=dev, extra_rows=2)
    check_attention(b, heads, dev)


@pytest.mark.parametrize("heads,kv_heads,D", LAYOUTS)
def test_attention_ragged_chunks(dev, heads, kv_heads, D):
    """Chunks of many lengths, some sequences without a row, some without a past."""
    n = [5, 0, 37, 1, 64, 3, 70]
    past = [100, 40, 0, 77, 3, 0, 131]
    b = R.Batch(n, [a + c for a, c in zip(n, past)], kv_heads=kv_heads, D=D, page=32, dev=dev, extra_rows=5)
    check_attention(b, heads, dev)


@pytest.mark.parametrize("heads,kv_heads,D", [(16, 8, 256), (16, 1, 512), (32, 8, 64), (6, 2, 128)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 0), (64, 4), (65, 1), (100, 70), (1000, 3)])
def test_attention_window_and_sinks(dev, heads, kv_heads, D, window, sinks):
    n = [1, 40, 9, 1]
    past = [333, 150, 0, 2]
    b = R.Batch(n, [a + c for a, c in zip(n, past)], kv_heads=kv_heads, D=D, page=16, dev=dev)
    check_attention(b, heads, dev, window=window, sinks=sinks)


@pytest.mark.parametrize("heads,kv_heads,D", [(4, 2, 64), (4, 1, 256), (16, 1, 512)])
def test_attention_long_prompt_rows(dev, heads, kv_heads, D):
    """More rows than a tile, from position 0, with a window that leaves early tiles."""
    b = R.Batch([259, 131], [259, 200], kv_heads=kv_heads, D=D, page=64, dev=dev)
    check_attention(b, heads, dev)
    check_attention(b, heads, dev, window=50, sinks=2)


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("n", [1, 3, 80])
def test_attention_splits_of_a_long_axis(dev, D, n):
    """Few rows over a long cache: the axis is split and joined."""
    b = R.Batch([n], [2501], kv_heads=1, D=D, page=128, dev=dev)
    check_attention(b, 2, dev)


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("n", [1, 6, 90])
def test_attention_what_is_masked_reaches_no_row(dev, D, n):
    """NaN and infinities in later tokens of the chunk, behind the window, in the
    rest of the last page and in pages that are gone."""
    L = 260 + n
    b = R.Batch([n, n], [L, L], kv_heads=1, D=D, page=32, dev=dev)
    inf, nan = math.inf, math.nan
    window, sinks = 100, 2
    for p in range(sinks, L - n + 1 - window):  # behind every row's window
        b.put(0, p, k=nan if p % 2 else inf, v=inf if p % 3 else nan)
    check_attention(b, 2, dev, window=window, sinks=sinks)
    if n == 1:
        return
    # sequence 1: its last token's k and v poison that row alone
    b.put(1, L - 1, k=nan, v=inf)
    b.put(1, L - 2, v=-inf)
    q = rows(b.T, 2 * D, dev, 3)
    from alveare_amd import attention_paged

    want, tol = R.attention(q, b, 2, window, sinks, 0.1)
    for mq in (0, n):
        got = attention_paged(q, *b.args(), heads=2, window=window, sinks=sinks, scale=0.1, max_q=mq)
        got = got.double().cpu().view_as(want)
        ok = torch.ones(2 * n, dtype=torch.bool)
        ok[2 * n - 2:] = False
        assert torch.isfinite(got[ok]).all()
        assert ((got - want).abs() <= tol)[ok].all()
        assert (got[2 * n - 2] == -inf).all()      # the row that sees one -inf value
        assert torch.isnan(got[2 * n - 1]).all()   # the one whose score is NaN


@pytest.mark.parametrize("heads,kv_heads,D", [(8, 2, 64), (4, 2, 128), (16, 8, 256), (16, 1, 512)])
def test_attention_missing_pages(dev, heads, kv_heads, D):
    """Entries outside the pool hold nothing; a row whose pages are all gone gets zeros."""
    n, total = [3, 50, 2, 1], [70, 90, 30, 257]
    b = R.Batch(n, total, kv_heads=kv_heads, D=D, page=16, dev=dev)
    gone = [(0, 0), (0, 3), (1, 2), (1, 4), (2, 0), (2, 1), (3, 1), (3, 16)]
    for i, (s, p) in enumerate(gone):
        b.table[s, p] = (-1, b.pages, -2 ** 31, 2 ** 31 - 1)[i % 4]
    q = check_attention(b, heads, dev, missing=gone)
    from alveare_amd import attention_paged

    out = attention_paged(q, *b.args(), heads=heads, scale=0.1)
    assert (out[53:55] == 0).all()


def test_attention_extreme_scores(dev):
    """Scores far apart, all alike, and a scale of zero."""
    for D in (64, 256):
        b = R.Batch([1, 40], [500, 300], kv_heads=2, D=D, page=16, dev=dev)
        check_attention(b, 4, dev, scale=0.0)
        q = rows(b.T, 4 * D, dev, 5, std=0.05)
        check_attention(b, 4, dev, scale=20.0, q=q)
        check_attention(b, 4, dev, q=torch.zeros_like(q))


def test_attention_malformed_sequences(dev):
    """A length below its rows or above its table: zeros, and the others as they are."""
    from alveare_amd import attention_paged

    b = R.Batch([2, 3, 1, 2], [40, 50, 60, 70], kv_heads=2, D=64, page=16, dev=dev)
    q = rows(b.T, 4 * 64, dev)
    good = attention_paged(q, *b.args(), heads=4)
    b.kv_len[1] = 2
    b.kv_len[2] = 16 * b.table.shape[1] + 1
    for mq in (0, 3):
        out = attention_paged(q, *b.args(), heads=4, max_q=mq)
        assert (out[2:6] == 0).all()
        assert torch.equal(out[:2], good[:2]) or mq != 0
        assert torch.allclose(out[6:].float(), good[6:].float(), atol=0.05)
    # starts that go backwards or past the batch: nothing out of bounds, the well formed sequence as it was
    b.kv_len.copy_(torch.tensor([40, 50, 60, 70]))
    b.q_start.copy_(torch.tensor([0, 2, 1, 900, -5]))
    out = attention_paged(q, *b.args(), heads=4)
    assert torch.allclose(out[:1].float(), good[:1].float(), atol=0.05)


def test_attention_strides(dev):
    """q inside the packed qkv rows, interleaved K and V pages, a wider table, strided out."""
    from alveare_amd import attention_paged

    for D, n in ((64, [1, 1, 1]), (128, [3, 70, 2]), (256, [1, 33, 4])):
        b = R.Batch(n, [v + 60 for v in n], kv_heads=2, D=D, page=16, dev=dev)
        q = rows(b.T, 4 * D, dev)
        want = attention_paged(q, *b.args(), heads=4, scale=0.1, max_q=max(n))
        pool = torch.stack([b.kp, b.vp], 1).contiguous()
        wide = torch.full((len(n), b.table.shape[1] + 9), 77777, dtype=torch.int32, device=dev)
        wide[:, :b.table.shape[1]] = b.table
        qkv = torch.cat([q, rows(b.T, 2 * D, dev, 9)], 1)
        out = torch.zeros(b.T, 4 * D + 8, dtype=bf, device=dev)
        attention_paged(qkv[:, :4 * D], pool[:, 0], pool[:, 1], wide[:, :b.table.shape[1]], b.q_start, b.kv_len,
                        heads=4, scale=0.1, max_q=max(n), out=out[:, :4 * D])
        assert torch.equal(out[:, :4 * D], want)
        assert (out[:, 4 * D:] == 0).all()


def test_attention_offsets_past_32_bits(dev):
    """Pages whose byte and element offsets need more than 32 bits."""
    from alveare_amd import attention_paged

    D, page = 512, 1024
    pages = (1 << 32) // (D * page) + 3  # more than 2^32 values in each pool
    b = R.Batch([1, 20], [1500, 900], kv_heads=1, D=D, page=page, dev=dev)
    k, v = (torch.empty(pages, 1, page, D, dtype=bf, device=dev) for _ in range(2))
    table = torch.full_like(b.table, -1)
    used = [(i, j) for i in range(2) for j in range(b.table.shape[1]) if int(b.table[i, j]) >= 0]
    for x, (i, j) in enumerate(used):
        p = pages - 1 - x
        k[p], v[p], table[i, j] = b.kp[b.table[i, j]], b.vp[b.table[i, j]], p
    q = rows(b.T, 4 * D, dev)
    for mq in (1, 20):
        want = attention_paged(q, *b.args(), heads=4, scale=0.05, max_q=mq)
        assert torch.equal(attention_paged(q, k, v, table, b.q_start, b.kv_len, heads=4, scale=0.05, max_q=mq), want)


@pytest.mark.parametrize("n", [1, 48])
def test_attention_large_batch(dev, n):
    """More sequences than a wave looks at in one step; bits do not change from call to call."""
    B = 150
    total = [n + (i * 37) % 90 for i in range(B)]
    b = R.Batch([n] * B, total, kv_heads=2, D=64, page=16, dev=dev)
    q = check_attention(b, 2, dev, max_q=n)
    from alveare_amd import attention_paged

    a = [attention_paged(q, *b.args(), heads=2, scale=0.1, max_q=n) for _ in range(3)]
    assert torch.equal(a[0], a[1]) and torch.equal(a[0], a[2])


def test_attention_graphs_and_streams(dev):
    """Two captured graphs replayed at once on two streams, with lengths changed in
    between, against eager calls; a call on a stream that is not the current one."""
    from alveare_amd import attention_paged

    D, heads = 128, 8
    made = []
    for seed, n in ((1, 1), (2, 60)):
        b = R.Batch([n] * 4, [900 + n, 500 + n, n, 33 + n], kv_heads=2, D=D, page=32, dev=dev, seed=seed)
        q = rows(b.T, heads * D, dev, seed)
        out = torch.zeros_like(q)
        s = torch.cuda.Stream(dev)
        s.wait_stream(torch.cuda.current_stream(dev))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            attention_paged(q, *b.args(), heads=heads, scale=0.1, max_q=n, out=out)
        made.append((b, q, out, s, g, n))
    for turn in range(4):
        for b, q, out, s, g, n in made:
            q.copy_(rows(b.T, heads * D, dev, 10 + turn))
            b.kv_len.copy_(torch.tensor([900 + n - 7 * turn, 500 + n - turn, n, 33 + n - turn]))
        torch.cuda.synchronize()
        for b, q, out, s, g, n in made:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for b, q, out, s, g, n in made:
            want = attention_paged(q, *b.args(), heads=heads, scale=0.1, max_q=n)
            assert torch.equal(out, want), f"turn {turn}, n={n}"


def test_attention_like_the_one_token_op(dev):
    """The same work as layer.attention on a cache in one piece."""
    from alveare_amd import attention_paged, layer as L

    for heads, kv_heads, D, window in ((16, 8, 256, 1024), (16, 1, 512, 0), (32, 8, 64, 0)):
        n = 1500
        b = R.Batch([1], [n], kv_heads=kv_heads, D=D, page=64, dev=dev)
        q = rows(1, heads * D, dev)
        kc, vc = (torch.zeros(kv_heads, 2048, D, dtype=bf, device=dev) for _ in range(2))
        kc[:, :n], vc[:, :n] = b.k[0].transpose(0, 1).to(bf).to(dev), b.v[0].transpose(0, 1).to(bf).to(dev)
        one = L.attention(q.view(-1), kc, vc, torch.tensor([n - 1], dtype=torch.int32, device=dev), heads=heads,
                          window=window, scale=0.08)
        got = attention_paged(q, *b.args(), heads=heads, window=window, scale=0.08, max_q=1)
        _, tol = R.attention(q, b, heads, window, 0, 0.08)
        assert ((got.double().cpu().view_as(tol) - one.double().cpu().view_as(tol)).abs() <= 2 * tol).all()


# ---- q/k/v post-processing -------------------------------------------------------------

@pytest.mark.parametrize("heads,kv_heads,D,v_raw", [(16, 8, 256, False), (16, 1, 512, True), (4, 1, 256, False),
                                                    (32, 8, 64, False), (6, 2, 128, False), (1, 1, 64, True)])
@pytest.mark.parametrize("half_of", [2, 8])
def test_post_is_the_one_token_op(dev, heads, kv_heads, D, v_raw, half_of):
    """Every row has the bits that layer.qkv_post writes for it, and nothing else
    in the pages changes."""
    from alveare_amd import layer as L, qkv_post_paged

    n, total = [1, 0, 17, 3], [40, 9, 17, 66]
    b = R.Batch(n, total, kv_heads=kv_heads, D=D, page=16, dev=dev, extra_rows=3)
    k_off = heads * D
    v_off = -1 if v_raw else k_off + kv_heads * D
    width = k_off + (1 if v_raw else 2) * kv_heads * D
    qkv = rows(b.T, width, dev, 4, std=2.0)
    g = torch.Generator().manual_seed(2)
    q_w, k_w = ((1 + 0.2 * torch.randn(D, generator=g)).to(dev) for _ in range(2))
    half = D // half_of
    rope = rows(80, 2 * half, dev, 8)
    kp, vp = b.kp.clone(), b.vp.clone()
    q_out = torch.full((b.T, heads * D), 7.0, dtype=bf, device=dev)
    for norm in ((True, True, True), (True, False, False), (False, True, True)):
        kw = dict(heads=heads, k_off=k_off, v_off=v_off, q_w=q_w, k_w=k_w, norm_q=norm[0], norm_k=norm[1], norm_v=norm[2])
        qkv_post_paged(qkv, b.kp, b.vp, b.table, b.q_start, b.kv_len, rope=rope, q_out=q_out, **kw)
        kc, vc = (torch.zeros(kv_heads, 80, D, dtype=bf, device=dev) for _ in range(2))
        t = 0
        for s in range(len(n)):
            for i in range(n[s]):
                pos = total[s] - n[s] + i
                want = L.qkv_post(qkv[t].contiguous(), torch.tensor([pos], dtype=torch.int32, device=dev), kc, vc,
                                  kv_heads=kv_heads, D=D, rope=rope.view(-1), rope_stride=2 * half, sin_off=half,
                                  half=half, **kw)
                assert torch.equal(q_out[t], want), (s, i)
                pg, sl = int(b.table[s, pos // 16]), pos % 16
                assert torch.equal(b.kp[pg, :, sl], kc[:, pos]) and torch.equal(b.vp[pg, :, sl], vc[:, pos])
                kp[pg, :, sl], vp[pg, :, sl] = kc[:, pos], vc[:, pos]
                t += 1
        assert (q_out[t:] == 7.0).all()
        for a, c in ((b.kp, kp), (b.vp, vp)):
            assert torch.equal(a.view(torch.int16), c.view(torch.int16))


def test_post_against_the_formula(dev):
    """Strided rows, an unusual table layout, no norm weights; within the roundings."""
    from alveare_amd import qkv_post_paged

    heads, kv_heads, D, half = 4, 2, 128, 24
    n, total = [70, 2], [70, 33]
    b = R.Batch(n, total, kv_heads=kv_heads, D=D, page=32, dev=dev)
    k_off, v_off = heads * D + 8, heads * D + kv_heads * D + 16
    width = v_off + kv_heads * D
    wide = rows(b.T, width + 40, dev, 3, std=3.0)
    rope = rows(75, 90, dev, 6)
    q_out = torch.zeros(b.T, heads * D + 16, dtype=bf, device=dev)
    qkv_post_paged(wide[:, :width], b.kp, b.vp, b.table, b.q_start, b.kv_len, heads=heads, k_off=k_off, v_off=v_off,
                   rope=rope, cos_off=40, sin_off=3, half=half, eps=1e-5, q_out=q_out[:, :heads * D])
    t = 0
    for s in range(2):
        for i in range(n[s]):
            pos = total[s] - n[s] + i
            q, k, v = R.post(wide[t], b, pos, heads=heads, k_off=k_off, v_off=v_off, q_w=None, k_w=None,
                             norm=(1, 1, 1), eps=1e-5, rope=rope, half=half, cos_off=40, sin_off=3)
            pg, sl = int(b.table[s, pos // 32]), pos % 32
            for got, want in ((q_out[t, :heads * D].view(heads, D), q), (b.kp[pg, :, sl], k), (b.vp[pg, :, sl], v)):
                # the norm's rounding may fall to the other side of a tie (a whole step, 2 halves) of each of
                # the two products, then the result's own
                scale = want.abs() + want.abs().amax(-1, keepdim=True) * 2
                assert ((got.double().cpu() - want).abs() <= R.BF16 * (want.abs() + 2 * scale)).all()
            t += 1
    assert (q_out[:, heads * D:] == 0).all()


def test_post_positions_that_do_not_fit(dev):
    """Malformed sequences, missing pages and positions past the rope table: zeros
    for q where nothing can be computed, and no page changes."""
    from alveare_amd import qkv_post_paged

    heads, kv_heads, D = 2, 1, 64
    b = R.Batch([2, 2, 2, 2], [20, 30, 40, 50], kv_heads=kv_heads, D=D, page=16, dev=dev)
    qkv = rows(b.T, 4 * D, dev)
    kw = dict(heads=heads, k_off=2 * D, v_off=3 * D)
    good = qkv_post_paged(qkv, b.kp.clone(), b.vp.clone(), b.table, b.q_start, b.kv_len, **kw)
    b.kv_len[0] = 1
    b.kv_len[1] = 16 * b.table.shape[1] + 1
    b.table[2, 2] = b.pages
    rope = torch.zeros(49, D, dtype=bf, device=dev)
    rope[:, :D // 2] = 1  # cos 1, sin 0: no rotation
    k0, v0 = b.kp.clone(), b.vp.clone()
    out = qkv_post_paged(qkv, b.kp, b.vp, b.table, b.q_start, b.kv_len, rope=rope, **kw)
    assert (out[:4] == 0).all() and torch.equal(out[4:7], good[4:7]) and (out[7] == 0).all()
    pg = int(b.table[3, 3])
    k0[pg, :, 0], v0[pg, :, 0] = b.kp[pg, :, 0], b.vp[pg, :, 0]  # position 48, the one that fits
    assert torch.isfinite(b.kp[pg, :, 0].float()).all()
    assert torch.equal(k0.view(torch.int16), b.kp.view(torch.int16))
    assert torch.equal(v0.view(torch.int16), b.vp.view(torch.int16))


# ---- page copies ------------------------------------------------------------------------

@pytest.mark.parametrize("caches,pages,shape,pairs,dtype", [
    (1, 4, (1, 16, 64), 1, bf), (3, 50, (2, 16, 128), 20, bf), (130, 40, (1, 16, 64), 17, bf),
    (2, 900, (1, 16, 64), 400, bf), (2, 9, (5, 128, 256), 4, bf), (2, 7, (16,), 3, torch.uint8)])
def test_copy_pages(dev, caches, pages, shape, pairs, dtype):
    from alveare_amd import copy_pages

    g = torch.Generator().manual_seed(3)
    pool = torch.randint(0, 256, (caches, pages + 1, *shape), generator=g).to(dtype).to(dev)
    perm = torch.randperm(pages, generator=g).tolist()
    src, dst = perm[:pairs], perm[pairs:2 * pairs]
    if pairs > 2:
        src[1] = src[0]  # one page to two places
    want = pool.clone()
    want[:, dst] = pool[:, src]
    copy_pages([c[:pages] for c in pool], src, dst)
    assert torch.equal(pool, want)
    copy_pages(list(pool), [], [])
    assert torch.equal(pool, want)


def test_copy_pages_strided(dev):
    """Interleaved K and V: pages apart by more than their size."""
    from alveare_amd import copy_pages

    pool = torch.arange(10 * 2 * 16 * 64, device=dev).view(10, 2, 1, 16, 64).to(bf)
    want = pool.clone()
    want[[7, 1], 1] = pool[[0, 9], 1]
    copy_pages([pool[:, 1]], [0, 9], [7, 1])
    assert torch.equal(pool, want)


def test_copy_pages_refusals(dev):
    from alveare_amd import copy_pages

    pool = torch.zeros(4, 1, 16, 64, dtype=bf, device=dev)
    for src, dst in (([0], [4]), ([-1], [1]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([3], [3]), ([0], [1, 2]),
                     ([0], [2 ** 40])):
        with pytest.raises(ValueError):
            copy_pages([pool], src, dst)
    with pytest.raises(TypeError):
        copy_pages([pool], [0.5], [1])
    with pytest.raises(ValueError):
        copy_pages([pool], torch.tensor([0], device=dev), [1])
    with pytest.raises(ValueError):
        copy_pages([pool, pool[:3]], [0], [1])
    with pytest.raises(ValueError):
        copy_pages([pool.transpose(2, 3)], [0], [1])
    assert (pool == 0).all()


# ---- refusals -----------------------------------------------------------------------------

def test_attention_refusals(dev):
    from alveare_amd import attention_paged

    b = R.Batch([1, 2], [20, 30], kv_heads=2, D=64, page=16, dev=dev)
    q = rows(3, 4 * 64, dev)
    ok = dict(q=q, kpages=b.kp, vpages=b.vp, page_table=b.table, q_start=b.q_start, kv_len=b.kv_len, heads=4)
    for change in (dict(q=q.float()), dict(q=q[:, :128]), dict(q=q.view(-1)), dict(q=q.t()), dict(heads=3),
                   dict(kpages=b.kp.half()), dict(kpages=b.kp[:2]), dict(kpages=b.kp.transpose(1, 2)),
                   dict(page_table=b.table.long()), dict(page_table=b.table[:1]), dict(q_start=b.q_start[:2]),
                   dict(kv_len=b.kv_len.float()), dict(window=-1), dict(sinks=-1), dict(scale=float("nan")),
                   dict(scale=-1.0), dict(scale=math.inf), dict(max_q=-1), dict(out=torch.zeros(2, 256, dtype=bf, device=dev)),
                   dict(kpages=b.kp[:, :, :8], vpages=b.vp[:, :, :8]), dict(q=q.cpu()),
                   dict(kpages=b.kp[..., :32].contiguous(), vpages=b.vp[..., :32].contiguous(), heads=8)):
        with pytest.raises((TypeError, ValueError)):
            kw = {**ok, **change}
            attention_paged(kw.pop("q"), kw.pop("kpages"), kw.pop("vpages"), kw.pop("page_table"), kw.pop("q_start"),
                            kw.pop("kv_len"), **kw)
    assert attention_paged(q[:0], *b.args(), heads=4).shape == (0, 256)


# ---- the cache, and the operators in a row -----------------------------------------------

def test_cache_contents_follow_the_bookkeeping(dev):
    """Random reserves, forks, truncations, frees and compactions; every slot's
    positions hold what was inserted for it."""
    import random

    from alveare_amd import PagedCache, qkv_post_paged

    rng = random.Random(4)
    H, D = 2, 64
    c = PagedCache(layers=2, kv_heads=H, D=D, pages=40, page_size=16, slots=5, max_pages=12, device=dev)
    held = [[] for _ in range(5)]  # the number inserted at each position
    count = 0
    for step in range(150):
        act, s = rng.choice(["add", "add", "add", "fork", "cut", "free", "compact"]), rng.randrange(5)
        if act == "add":
            who = rng.sample(range(5), rng.randint(1, 3))
            n = [rng.randint(0, 20) for _ in who]
            try:
                c.reserve(who, n)
            except (MemoryError, ValueError):
                continue
            table, q_start, kv_len = c.batch(who, n)
            vals = torch.arange(count, count + sum(n), device=dev)
            count += sum(n)
            # exact in bf16: a low and a high part
            row = torch.zeros(sum(n), (1 + 2) * H * D, device=dev)
            row[:, ::2], row[:, 1::2] = (vals % 128)[:, None], (vals // 128)[:, None]
            for i in range(2):
                qkv_post_paged((row + 0).to(bf), c.k[i], c.v[i], table, q_start, kv_len, heads=H, k_off=H * D,
                               v_off=2 * H * D, norm_q=False, norm_k=False, norm_v=False)
            at = count - sum(n)
            for w, m in zip(who, n):
                held[w] += range(at, at + m)
                at += m
        elif act == "fork":
            to = rng.randrange(5)
            if to != s and not held[to]:
                c.fork(s, to)
                held[to] = list(held[s])
        elif act == "cut":
            m = rng.randint(0, len(held[s]))
            c.truncate(s, m)
            del held[s][m:]
        elif act == "free":
            c.free(s)
            held[s] = []
        else:
            c.compact()
        for w in range(5):
            t = c.table(w)
            assert c.length(w) == len(held[w]) and len(t) == -(-len(held[w]) // 16)
            for x in (c.k[0], c.v[1]):
                if held[w]:
                    got = x[t].transpose(1, 2).reshape(-1, H * D)[:len(held[w]), :2].long()
                    assert (got[:, 0] + 128 * got[:, 1]).tolist() == held[w], (step, act)


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("part", [0.0, 0.5, 0.999])
@pytest.mark.parametrize("n,total", [(5, 70), (150, 150), (150, 1500)])
def test_attention_an_infinity_in_one_column_of_v(dev, D, part, n, total):
    """The last token's v, which only its own row may see."""
    from alveare_amd import attention_paged

    heads, col = 2, int(part * D)
    b = R.Batch([n], [total], kv_heads=1, D=D, page=32, dev=dev)
    b.kp[int(b.table[0, (total - 1) // 32]), 0, (total - 1) % 32] = 0  # its weight is no zero
    b.k[0][total - 1] = 0
    q = rows(n, heads * D, dev, 5)
    want, tol = R.attention(q, b, heads, scale=0.05)
    b.vp[int(b.table[0, (total - 1) // 32]), 0, (total - 1) % 32, col] = math.inf
    for mq in (0, n):
        got = attention_paged(q, *b.args(), heads=heads, scale=0.05, max_q=mq).double().cpu().view_as(want)
        hit = torch.zeros_like(want, dtype=torch.bool)
        hit[-1, :, col] = True
        assert (got[hit] == math.inf).all()
        assert torch.isfinite(got[~hit]).all()
        assert ((got - want).abs() <= tol)[~hit].all()


@pytest.mark.parametrize("heads,kv_heads,D", [(8, 2, 64), (4, 1, 128), (4, 2, 256), (8, 1, 512)])
@pytest.mark.parametrize("n,past", [([200, 1, 1, 2, 1, 1], [0, 500, 33, 128, 0, 64]), ([1, 130, 150], [900, 20, 0]),
                                    ([70, 70, 70], [0, 10, 200])])
def test_attention_chunks_and_single_tokens(dev, heads, kv_heads, D, n, past):
    """Both kinds of sequences in one call, and every max_q: a wrong one costs time alone."""
    b = R.Batch(n, [a + c for a, c in zip(n, past)], kv_heads=kv_heads, D=D, page=32, dev=dev)
    q = rows(b.T, heads * D, dev, 6)
    want, tol = R.attention(q, b, heads, scale=0.1)
    from alveare_amd import attention_paged

    for mq in (0, 1, 17, max(n) // 2, max(n) - 1, max(n), 10 * max(n)):
        got = attention_paged(q, *b.args(), heads=heads, scale=0.1, max_q=mq).double().cpu().view_as(want)
        assert ((got - want).abs() <= tol).all(), f"max_q={mq}"


@pytest.mark.parametrize("D", [64, 512])
def test_attention_seventy_chunks(dev, D):
    """More sequences than lanes, of one tile each and more, with empty ones among them."""
    n = [(7 * i) % 53 for i in range(70)]
    past = [(11 * i) % 90 for i in range(70)]
    b = R.Batch(n, [a + c for a, c in zip(n, past)], kv_heads=1, D=D, page=16, dev=dev)
    check_attention(b, 4, dev)


@pytest.mark.parametrize("half", [1, 3, 12, 29])
@pytest.mark.parametrize("shift", [0, 1])
def test_post_odd_halves_and_rows_off_their_alignment(dev, half, shift):
    """As the one-token op, where no eight columns share a path or a 16-byte access."""
    from alveare_amd import layer as L, qkv_post_paged

    heads, kv_heads, D = 3, 1, 64
    n, total = [5, 1], [5, 20]
    b = R.Batch(n, total, kv_heads=kv_heads, D=D, page=16, dev=dev)
    width = (heads + 2) * D
    qkv = rows(b.T, width + 3, dev, 4)[:, shift:shift + width]
    rope = rows(20, 2 * half + 1, dev, 8)
    got = qkv_post_paged(qkv, b.kp, b.vp, b.table, b.q_start, b.kv_len, heads=heads, k_off=heads * D,
                         v_off=(heads + 1) * D, rope=rope, sin_off=half, half=half)
    kc, vc = (torch.zeros(kv_heads, 20, D, dtype=bf, device=dev) for _ in range(2))
    for t, (s, pos) in enumerate([(0, 0), (0, 1), (0, 2), (0, 3), (0, 4), (1, 19)]):
        want = L.qkv_post(qkv[t].clone(), torch.tensor([pos], dtype=torch.int32, device=dev), kc, vc, heads=heads,
                          kv_heads=kv_heads, D=D, k_off=heads * D, v_off=(heads + 1) * D,
                          rope=rope[:, :2 * half].contiguous().view(-1), rope_stride=2 * half, sin_off=half, half=half)
        pg, sl = int(b.table[s, pos // 16]), pos % 16
        assert torch.equal(got[t], want)
        assert torch.equal(b.kp[pg, :, sl], kc[:, pos]) and torch.equal(b.vp[pg, :, sl], vc[:, pos])


# ---- the operators together --------------------------------------------------------------

def test_prompts_forks_drafts_and_decode_steps(dev):
    """A small model served as these operators are meant to be used: prompts in
    chunks, two continuations of one prompt, drafts of which some are taken back,
    sampled decode steps, a sequence freed and the pool compacted. Each call is
    checked on the inputs it got, and the cache against what was inserted."""
    import types

    from alveare_amd import PagedCache, attention_paged, qkv_post_paged, sample

    heads, kv_heads, D, hidden, vocab, layers, page = 4, 2, 64, 96, 5000, 2, 16
    g = torch.Generator().manual_seed(9)
    mat = lambda *s: (torch.randn(*s, generator=g) / math.sqrt(s[0])).to(bf).to(dev)  # noqa: E731
    emb = mat(vocab, hidden) * 8
    w_qkv, w_o, w_head = ([mat(hidden, (heads + 2 * kv_heads) * D) for _ in range(layers)],
                          [mat(heads * D, hidden) for _ in range(layers)], mat(hidden, vocab) * 4)
    rope = rows(200, D, dev, 3)
    c = PagedCache(layers=layers, kv_heads=kv_heads, D=D, pages=40, page_size=page, slots=4, max_pages=12, device=dev)
    kept = [[([], []) for _ in range(layers)] for _ in range(4)]  # by slot and layer, each position's k and v

    def step(slots, tokens):
        """tokens: a list per slot. Returns the logits of each slot's last token."""
        n = [len(t) for t in tokens]
        c.reserve(slots, n)
        table, q_start, kv_len = c.batch(slots, n)
        x = emb[torch.tensor(sum(tokens, []), device=dev)]
        for i in range(layers):
            qkv = x @ w_qkv[i]
            q = qkv_post_paged(qkv, c.k[i], c.v[i], table, q_start, kv_len, heads=heads, k_off=heads * D,
                               v_off=(heads + kv_heads) * D, rope=rope)
            at = 0
            for s, m in zip(slots, n):
                for j in range(m):
                    pos = c.length(s) - m + j
                    _, k, v = R.post(qkv[at], types.SimpleNamespace(D=D, kv_heads=kv_heads), pos, heads=heads,
                                     k_off=heads * D, v_off=(heads + kv_heads) * D, q_w=None, k_w=None, norm=(1, 1, 1),
                                     eps=1e-6, rope=rope, half=D // 2, cos_off=0, sin_off=D // 2)
                    pg, sl = c.table(s)[pos // page], pos % page
                    for got, want, keep in ((c.k[i][pg, :, sl], k, kept[s][i][0]), (c.v[i][pg, :, sl], v, kept[s][i][1])):
                        got = got.double().cpu()
                        # (as in test_post_against_the_formula)
                        scale = want.abs() + want.abs().amax(-1, keepdim=True) * 2
                        assert ((got - want).abs() <= R.BF16 * (want.abs() + 2 * scale)).all()
                        keep.append(got)
                    at += 1
            out = attention_paged(q, c.k[i], c.v[i], table, q_start, kv_len, heads=heads, scale=0.125, max_q=max(n))
            b = types.SimpleNamespace(n=n, total=[c.length(s) for s in slots], page=page, kv_heads=kv_heads, D=D,
                                      k=[torch.stack(kept[s][i][0]) for s in slots],
                                      v=[torch.stack(kept[s][i][1]) for s in slots])
            want, tol = R.attention(q, b, heads, scale=0.125)
            assert ((out.double().cpu().view_as(want) - want).abs() <= tol).all()
            x = x + out @ w_o[i]
        last = torch.tensor([sum(n[:k + 1]) - 1 for k in range(len(n))], device=dev)
        return (x[last] @ w_head).float()

    def draw(logits):
        u = torch.rand(len(logits), generator=g).to(dev)
        token, prob = sample(logits, u, temperature=0.9, top_k=50, top_p=0.95, min_p=0.01)
        for k in range(len(logits)):
            assert R.sample(logits[k], float(u[k]), 0.9, 50, 0.95, 0.01)[0] == int(token[k])
        assert ((prob > 0) & (prob <= 1)).all()
        return token.tolist()

    prompts = [torch.randint(vocab, (m,), generator=g).tolist() for m in (75, 18, 3)]
    step([0, 1], [prompts[0][:40], prompts[1]])
    logits = step([0, 2], [prompts[0][40:], prompts[2]])
    c.fork(0, 3)  # a second continuation
    kept[3] = [([*k], [*v]) for k, v in kept[0]]
    tokens = draw(logits[[0, 1, 0]])
    for _ in range(3):
        tokens = draw(step([0, 2, 3], [[t] for t in tokens]))
    step([0, 1], [[tokens[0], 5, 6, 7], [9, 8]])  # drafts: two of the first's are taken back
    c.truncate(0, c.length(0) - 2)
    for k, v in kept[0]:
        del k[-2:], v[-2:]
    c.free(2)
    kept[2] = [([], []) for _ in range(layers)]
    assert c.compact() >= 0
    tokens = draw(step([3, 0, 1], [[4], [5], [6]]))
    draw(step([2, 3, 1, 0], [prompts[2] * 9, [tokens[0]], [], [tokens[1]]])[[0, 1, 3]])
    for s in range(4):
        t = c.table(s)
        for i in range(layers):
            for pool, keep in ((c.k[i], kept[s][i][0]), (c.v[i], kept[s][i][1])):
                got = pool[t].transpose(1, 2).reshape(-1, kv_heads, D)[:c.length(s)]
                assert torch.equal(got.double().cpu(), torch.stack(keep))


def test_a_captured_decode_step(dev):
    """Insert, attention and sampling of a batch in one graph, replayed while the
    sequences grow over pages, against the same calls made one by one."""
    from alveare_amd import PagedCache, attention_paged, qkv_post_paged, sample

    heads, kv_heads, D, vocab, B = 4, 2, 64, 6000, 3
    g = torch.Generator().manual_seed(1)
    emb, w = rows(vocab, (heads + 2 * kv_heads) * D, dev, 1), rows(heads * D, vocab, dev, 2, std=0.3)
    caches = [PagedCache(layers=1, kv_heads=kv_heads, D=D, pages=30, page_size=16, slots=B, max_pages=6, device=dev)
              for _ in range(2)]
    for c in caches:
        c.reserve(range(B), [14, 1, 40])
        c.pool.copy_(torch.randn(c.pool.shape, generator=torch.Generator().manual_seed(5)).to(bf))
        c.truncate(1, 0)
    table = torch.full((B, 6), -1, dtype=torch.int32, device=dev)
    q_start, kv_len = torch.arange(B + 1, dtype=torch.int32, device=dev), torch.zeros(B, dtype=torch.int32, device=dev)
    u = torch.zeros(B, device=dev)
    token = torch.tensor([3, 4, 5], dtype=torch.int32, device=dev)
    prob = torch.zeros(B, device=dev)

    def step(c, table, q_start, kv_len, token, prob):
        q = qkv_post_paged(emb[token.long()], c.k[0], c.v[0], table, q_start, kv_len, heads=heads, k_off=heads * D,
                           v_off=(heads + kv_heads) * D)
        out = attention_paged(q, c.k[0], c.v[0], table, q_start, kv_len, heads=heads, scale=0.125, max_q=1)
        sample((out @ w).float(), u, temperature=1.2, top_k=100, top_p=0.9, token=token, prob=prob)

    eager_token, eager_prob = token.clone(), prob.clone()
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        step(caches[0], table, q_start, kv_len, token.clone(), prob.clone())  # nothing fits: no page changes
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        step(caches[0], table, q_start, kv_len, token, prob)
    for _ in range(6):
        for c in caches:
            c.reserve(range(B), [1] * B)
        t, q, k = caches[0].batch(range(B), [1] * B)
        u.copy_(torch.rand(B, generator=g))
        table.copy_(t), kv_len.copy_(k)
        graph.replay()
        step(caches[1], *caches[1].batch(range(B), [1] * B), eager_token, eager_prob)
        torch.cuda.synchronize()
        assert torch.equal(token, eager_token) and torch.equal(prob, eager_prob)
        assert torch.equal(caches[0].pool, caches[1].pool)


def test_numbers_past_32_bits(dev):
    """A window or a max_q of any size counts as no limit; offsets are refused."""
    from alveare_amd import attention_paged, qkv_post_paged

    b = R.Batch([3, 40], [300, 40], kv_heads=1, D=64, page=16, dev=dev)
    q = rows(b.T, 128, dev)
    want = attention_paged(q, *b.args(), heads=2, scale=0.1)
    for big in (2 ** 31 - 1, 2 ** 32 + 1, 2 ** 40):
        assert torch.equal(attention_paged(q, *b.args(), heads=2, scale=0.1, window=big, sinks=big), want)
        R_max = attention_paged(q, *b.args(), heads=2, scale=0.1, max_q=big)
        assert torch.equal(R_max, attention_paged(q, *b.args(), heads=2, scale=0.1, max_q=2 ** 31 - 1))
    rope, qkv = rows(300, 64, dev), rows(b.T, 256, dev)
    for kw in (dict(cos_off=2 ** 32), dict(sin_off=2 ** 32), dict(half=2 ** 32 + 8), dict(cos_off=-8)):
        with pytest.raises(ValueError):
            qkv_post_paged(qkv, *b.args(), heads=2, k_off=128, v_off=192, rope=rope, **kw)


@pytest.mark.parametrize("heads,kv_heads,D,n,past", [(16, 1, 64, [560, 0, 300, 1], [0, 5, 40, 900]), (4, 1, 512, [450], [0]),
                                                     (8, 4, 128, [150, 290], [700, 0]), (6, 2, 256, [333], [31])])
def test_attention_tiles_in_parts_of_unequal_number(dev, heads, kv_heads, D, n, past):
    """Causal prompts whose late tiles are cut and whose early ones are not, more
    than a wave's lanes of them, with and without a window."""
    b = R.Batch(n, [a + c for a, c in zip(n, past)], kv_heads=kv_heads, D=D, page=64, dev=dev, extra_rows=2)
    check_attention(b, heads, dev)
    check_attention(b, heads, dev, window=170, sinks=40)


@pytest.mark.parametrize("D,most", [(64, 10), (64, 20), (128, 10), (128, 20), (256, 5), (256, 10)])
def test_attention_many_drafts(dev, D, most):
    """So many sequences that drafts of 16, 32 and 64 rows stream past K and V."""
    n = [1 + (5 * i) % most for i in range(132)]
    n[7] = 0
    past = [(29 * i) % 150 for i in range(132)]
    b = R.Batch(n, [a + c for a, c in zip(n, past)], kv_heads=2, D=D, page=16, dev=dev, extra_rows=1)
    check_attention(b, 6, dev)
    if D == 128:
        check_attention(b, 6, dev, window=60, sinks=5)
    # a value that is no number in the last token's v of one sequence
    from alveare_amd import attention_paged

    q = rows(b.T, 6 * D, dev, 3)
    want, tol = R.attention(q, b, 6, scale=0.1)
    s = 60
    b.put(s, b.total[s] - 1, v=math.nan)
    got = attention_paged(q, *b.args(), heads=6, scale=0.1, max_q=most)[:want.shape[0]].double().cpu().view_as(want)
    hit = torch.zeros(len(want), dtype=torch.bool)
    hit[sum(n[:s + 1]) - 1] = True
    assert torch.isnan(got[hit]).all() and ((got - want).abs() <= tol)[~hit].all()


def test_copy_pages_refuses_what_is_no_cache(dev):
    from alveare_amd import copy_pages

    c = torch.zeros(4, 2, 16, 64, dtype=bf, device=dev)
    for bad in ([c, 1], [c, None], [c, c.cpu()], [c, c[:2]], [c, c.float()], [c, c.transpose(1, 2)]):
        with pytest.raises(ValueError):
            copy_pages(bad, [0], [1])
    assert (c == 0).all()


def test_attention_more_tiles_than_max_q_tells_of(dev):
    """max_q = 1 for a sequence of 68000 rows of 128 heads: the merge's table has one entry, the call 68000
    tiles. Nothing behind the workspace is written, and the rows are right."""
    import ctypes

    from alveare_amd import lib

    T, heads, D, window = 68000, 128, 64, 16
    b = R.Batch([T], [T], kv_heads=1, D=D, page=1024, dev=dev)
    q = torch.randn(T, heads * D, generator=torch.Generator(dev).manual_seed(1), device=dev).to(bf)
    out = torch.full_like(q, 7.0)
    need = lib().alv_attention_paged_workspace(heads, 1, D, 1, T, 1)
    ws = torch.full((need + (4 << 20),), 0xA5, dtype=torch.uint8, device=dev)
    ptr = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    rc = lib().alv_attention_paged(ptr(q), heads * D, ptr(b.kp), ptr(b.vp), 1024 * D, 1024 * D, b.pages, 1024, ptr(b.table),
                                   b.table.shape[1], b.table.shape[1], ptr(b.q_start), ptr(b.kv_len), 1, T, 1, heads, 1, D,
                                   window, 0, 0.1, ptr(out), heads * D, ptr(ws), need,
                                   ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream))
    assert rc == 0
    assert (ws[need:] == 0xA5).all()
    for t in (0, 1, 15, 16, 17, 1023, 1024, 33333, T - 2, T - 1):
        lo = max(0, t + 1 - window)
        one = R.Batch([1], [t + 1 - lo], kv_heads=1, D=D, page=16, dev="cpu")
        one.k[0], one.v[0] = b.k[0][lo:t + 1], b.v[0][lo:t + 1]
        want, tol = R.attention(q[t:t + 1], one, heads, scale=0.1)
        assert ((out[t].double().cpu().view_as(want[0]) - want[0]).abs() <= tol[0]).all(), t


@pytest.mark.parametrize("D,pad", [(64, 1200), (64, 100), (128, 1200), (256, 6000), (512, 6000)])
def test_attention_mostly_padding(dev, D, pad):
    """Rows enough for many tiles, of which the sequences own a few: the tile kernel is launched and has none
    (pad = 100: few enough that it takes the batch alone)."""
    b = R.Batch([1, 2, 0, 1], [300, 2, 40, 1], kv_heads=8, D=D, page=16, dev=dev, extra_rows=pad)
    check_attention(b, 64 if D <= 128 else 8, dev, max_q=0)


@pytest.mark.parametrize("heads,kv_heads,D", [(32, 8, 64), (16, 8, 128), (16, 8, 256), (16, 1, 512)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (257, 5)])
def test_attention_whole_tiles_beside_single_tokens(dev, heads, kv_heads, D, window, sinks):
    """Tiles enough that none is split, of two chunks, and sequences of one and two rows in the same call."""
    from alveare_amd import attention_paged

    n, past = [1400, 1, 900, 2], [100, 611, 0, 64]
    total = [a + b for a, b in zip(n, past)]
    b = R.Batch(n, total, kv_heads=kv_heads, D=D, page=32, dev=dev)
    q = rows(b.T, heads * D, dev)
    scale = 1.5 / math.sqrt(D)
    for mq in (0, 1400):
        out = attention_paged(q, *b.args(), heads=heads, window=window, sinks=sinks, scale=scale, max_q=mq)
        at = 0
        for s, (m, L) in enumerate(zip(n, total)):
            for i in sorted({0, 1, 31, 32, 127, 128, 500, 899, m // 2, m - 1}):
                if i >= m:
                    continue
                one = R.Batch([1], [L - m + i + 1], kv_heads=kv_heads, D=D, page=16, dev="cpu")
                one.k[0], one.v[0] = b.k[s][:L - m + i + 1], b.v[s][:L - m + i + 1]
                want, tol = R.attention(q[at + i:at + i + 1], one, heads, window, sinks, scale)
                got = out[at + i].double().cpu().view_as(want[0])
                assert ((got - want[0]).abs() <= tol[0]).all(), (mq, s, i)
            at += m

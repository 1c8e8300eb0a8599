"""Attention of sequences that share their first pages, against plain forms in 64
bits, and the serving operators as one run over a cache whose slots were forked."""
import math

import pytest
import torch

import more_ref as M
import paged_ref as R

pytestmark = pytest.mark.gpu

bf = torch.bfloat16


def rows(T, width, dev, seed=1, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, width, generator=g) * std).to(bf).to(dev)


def check(b, heads, dev, *, window=0, sinks=0, scale=None, missing=(), q=None, seed=1):
    from alveare_amd import attention_shared_paged

    D = b.D
    scale = 1.5 / math.sqrt(D) if scale is None else scale
    q = rows(b.T, heads * D, dev, seed) if q is None else q
    want, tol = M.attention(q, b, heads, window, sinks, scale, missing)
    for mq in (0, max(max(b.n), 1)):
        out = torch.full((b.T, heads * D), 7.0, dtype=bf, device=dev)
        attention_shared_paged(q, *b.args(), *b.groups(), heads=heads, window=window, sinks=sinks, scale=scale, max_q=mq,
                               out=out, scales=b.scales)
        m = want.shape[0]
        got = out[:m].double().cpu().view_as(want)
        assert torch.isfinite(got).all(), f"max_q={mq}"
        bad = (got - want).abs() > tol
        assert not bad.any(), (f"max_q={mq}: {int(bad.sum())} of {bad.numel()} values off, worst "
                               f"{float(((got - want).abs() / tol).max()):.2f} tolerances, first {bad.nonzero()[0].tolist()}")
        assert (out[m:] == 7.0).all(), "rows past the last sequence changed"
    return q


def batch(n, own, groups, **kw):
    """Sequences of n new rows, `own` positions (the new ones included) behind what their group shares."""
    total, at = list(own), 0
    for count, s in groups:
        for b in range(at, at + count):
            total[b] += s
        at += count
    return M.Batch(n, total, groups=groups, **kw)


LAYOUTS = [(16, 8, 256), (16, 1, 512), (4, 1, 256), (32, 8, 64), (6, 2, 128), (1, 1, 64), (5, 5, 128), (40, 1, 128)]


@pytest.mark.parametrize("heads,kv_heads,D", LAYOUTS)
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("page", [16, 64])
def test_shared_decode(dev, heads, kv_heads, D, bits, page):
    """One token each: a group of many, one of one, one that shares nothing, sequences in none."""
    own = [1, 20, 7, 65, 3, 1, 40, 100, 9, 17, 1]
    b = batch([1] * 11, own, [(6, 192), (1, 64), (2, 0)], kv_heads=kv_heads, D=D, page=page, dev=dev, bits=bits,
              extra_rows=2)
    check(b, heads, dev)


@pytest.mark.parametrize("heads,kv_heads,D", LAYOUTS)
@pytest.mark.parametrize("bits", [16, 8])
def test_shared_ragged_chunks(dev, heads, kv_heads, D, bits):
    n = [5, 0, 37, 1, 64, 3]
    own = [105, 40, 37, 78, 67, 3]
    b = batch(n, own, [(3, 96), (3, 320)], kv_heads=kv_heads, D=D, page=32, dev=dev, bits=bits, extra_rows=5)
    check(b, heads, dev)


@pytest.mark.parametrize("heads,kv_heads,D", [(16, 8, 256), (16, 1, 512), (32, 8, 64), (6, 2, 128)])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 0), (64, 4), (65, 200), (100, 70), (300, 3), (1000, 3)])
def test_shared_window_and_sinks(dev, heads, kv_heads, D, bits, window, sinks):
    """Windows that end within what is shared, behind it, and that leave nothing of it but the first tokens;
    first tokens beyond it."""
    n = [1, 40, 9, 1, 1]
    own = [133, 50, 9, 2, 1]
    b = batch(n, own, [(3, 208), (2, 112)], kv_heads=kv_heads, D=D, page=16, dev=dev, bits=bits)
    check(b, heads, dev, window=window, sinks=sinks)


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("n", [1, 3, 30])
def test_shared_long(dev, D, bits, n):
    """A long shared axis, split and joined; few own positions."""
    b = batch([n] * 5, [n, n + 1, n + 40, n, n + 9], [(5, 2304)], kv_heads=1, D=D, page=128, dev=dev, bits=bits)
    check(b, 2, dev)


@pytest.mark.parametrize("D", [64, 256, 512])
@pytest.mark.parametrize("bits", [16, 8])
def test_shared_rows_within_it(dev, D, bits):
    """Sequences no longer than what their group shares, a shared length that ends within a page or beyond the
    first sequence, rows whose own positions are shared ones."""
    n, total = [3, 2, 1, 5], [70, 40, 64, 69]
    for s in (64, 79, 1000):
        b = M.Batch(n, total, groups=[(4, s)], kv_heads=2, D=D, page=16, dev=dev, bits=bits)
        assert b.shared == [64] * 4
        check(b, 4, dev)
        check(b, 4, dev, window=9, sinks=1)


@pytest.mark.parametrize("D", [64, 256, 512])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("n", [1, 6])
def test_shared_what_is_masked_reaches_no_row(dev, D, bits, n):
    """What is not finite behind the window, shared or not, and where only some of a tile's rows see it."""
    from alveare_amd import attention_shared_paged

    nan = math.nan
    b = batch([n] * 4, [n + 50, n + 2, n + 90, n], [(3, 256)], kv_heads=1, D=D, page=32, dev=dev, bits=bits)
    window, sinks = 100, 2
    for p in range(sinks, 256 + n + 2 - n + 1 - window):  # no row of the group sees it
        b.put(0, p, k=nan if p % 2 else None, v=nan if p % 3 else None)
    check(b, 2, dev, window=window, sinks=sinks)
    # position 200 is within sequence 1's window alone
    b.put(0, 160, v=nan)
    q = rows(b.T, 2 * D, dev, 3)
    want, tol = M.attention(q, b, 2, window, sinks, 0.1)
    got = attention_shared_paged(q, *b.args(), *b.groups(), heads=2, window=window, sinks=sinks, scale=0.1, max_q=n,
                                 scales=b.scales).double().cpu().view_as(want)
    poisoned = torch.isnan(want)
    assert poisoned.any() and not poisoned.all()
    assert torch.equal(torch.isnan(got), poisoned)
    assert ((got - want).abs() <= tol)[~poisoned].all()


@pytest.mark.parametrize("heads,kv_heads,D,B", [(8, 8, 64, 5), (32, 8, 64, 7), (16, 2, 64, 7), (32, 8, 64, 40), (6, 2, 128, 30),
                                                (16, 8, 256, 30), (16, 1, 512, 6), (2, 2, 512, 12), (2, 2, 512, 40)])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("window,sinks", [(5, 0), (60, 3), (150, 70)])
def test_shared_window_decode(dev, heads, kv_heads, D, B, bits, window, sinks):
    """One token each, few rows of a group and many: all of them streamed, groups in tiles beside streamed
    sequences, and all in tiles."""
    own = [1 + (i * 29) % 67 for i in range(B)]
    b = batch([1] * B, own, [(B - 2, 176), (1, 64)], kv_heads=kv_heads, D=D, page=16, dev=dev, bits=bits, extra_rows=1)
    check(b, heads, dev, window=window, sinks=sinks)


@pytest.mark.parametrize("window,sinks", [(0, 0), (1200, 9)])
def test_shared_one_long_tile_beside_short_ones(dev, window, sinks):
    """A group's long tile and sequences' shorter ones in as many parts as run at once."""
    b = batch([17] * 5, [900 + 77 * i for i in range(5)], [(5, 8192)], kv_heads=32, D=64, page=128, dev=dev, bits=16)
    check(b, 32, dev, window=window, sinks=sinks)


@pytest.mark.parametrize("D", [64, 256, 512])
@pytest.mark.parametrize("n", [1, 9])
def test_shared_same_bits_and_apart(dev, D, n):
    """The same bits from call to call; the same answer in groups of one, in none and by attention that shares nothing."""
    from alveare_amd import attention_paged, attention_shared_paged

    b = batch([n] * 4, [n + 700, n + 3, n + 64, n], [(4, 512)], kv_heads=2, D=D, page=64, dev=dev)
    q = rows(b.T, 8 * D, dev)
    kw = dict(heads=8, scale=0.1, max_q=n, scales=b.scales)
    a = [attention_shared_paged(q, *b.args(), *b.groups(), **kw) for _ in range(3)]
    assert torch.equal(a[0], a[1]) and torch.equal(a[0], a[2])
    for s in range(1, 4):
        b.table[s, :8] = b.table[0, :8]
    want, tol = M.attention(q, b, 8, 0, 0, 0.1)
    i32 = dict(dtype=torch.int32, device=dev)
    for got in (a[0], attention_paged(q, *b.args(), **kw),
                attention_shared_paged(q, *b.args(), torch.arange(5, **i32), torch.full((4,), 512, **i32), **kw),
                attention_shared_paged(q, *b.args(), torch.zeros(1, **i32), torch.zeros(0, **i32), **kw)):
        assert ((got.double().cpu().view_as(want) - want).abs() <= tol).all()


@pytest.mark.parametrize("heads,kv_heads,D", [(32, 8, 64), (6, 2, 128), (16, 8, 256), (16, 1, 512)])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("mq", [1, 2, 20, 100000])
def test_shared_any_hint(dev, heads, kv_heads, D, bits, mq):
    """max_q spreads the work; one that is wrong changes no row beyond its last bits, shared or not."""
    from alveare_amd import attention_paged, attention_shared_paged

    for n, own, groups in (([40, 1, 3, 0, 150], [60, 1, 90, 5, 170], [(4, 160), (1, 80)]), ([7], [40], [(1, 96)]),
                           ([1] * 30, [1 + 3 * i for i in range(30)], [(30, 96)])):
        b = batch(n, own, groups, kv_heads=kv_heads, D=D, page=16, dev=dev, bits=bits, extra_rows=2)
        q = rows(b.T, heads * D, dev)
        want, tol = M.attention(q, b, heads, 50, 3, 0.1)
        kw = dict(heads=heads, window=50, sinks=3, scale=0.1, max_q=mq, scales=b.scales)
        m = want.shape[0]
        got = attention_shared_paged(q, *b.args(), *b.groups(), out=torch.full_like(q, 7.0), **kw)
        assert ((got[:m].double().cpu().view_as(want) - want).abs() <= tol).all() and (got[m:] == 7.0).all()
        at = 0
        for count, s in groups:  # every sequence's own table names the shared pages too
            s = min(s, b.total[at]) // 16
            for c in range(at, at + count):
                b.table[c, :s] = b.table[at, :s]
            at += count
        got = attention_paged(q, *b.args(), out=torch.full_like(q, 7.0), **kw)
        assert ((got[:m].double().cpu().view_as(want) - want).abs() <= tol).all() and (got[m:] == 7.0).all()


@pytest.mark.parametrize("bits", [16, 8])
def test_shared_missing_pages(dev, bits):
    """Shared pages that are gone are gone for all; a row with none left gets zeros."""
    from alveare_amd import attention_shared_paged

    n = [1, 2, 1, 1]
    b = batch(n, [1, 2, 30, 1], [(3, 64), (1, 16)], kv_heads=2, D=64, page=16, dev=dev, bits=bits)
    b.table[0, 1], b.table[3, 0], b.table[3, 1] = -1, b.pages, -7
    gone = [(0, 1), (1, 1), (2, 1), (3, 0), (3, 1)]
    q = check(b, 4, dev, missing=gone)
    out = attention_shared_paged(q, *b.args(), *b.groups(), heads=4, scale=0.1, scales=b.scales)
    assert (out[4] == 0).all()


@pytest.mark.parametrize("bits", [16, 8])
def test_shared_malformed(dev, bits):
    """Sequences that do not fit give zeros; groups that are none share nothing; nothing goes out of bounds."""
    from alveare_amd import attention_paged, attention_shared_paged

    n, total = [2, 3, 1, 2], [70, 80, 90, 75]
    b = M.Batch(n, total, kv_heads=2, D=64, page=16, dev=dev, bits=bits)
    q = rows(b.T, 256, dev)
    kw = dict(heads=4, scale=0.2, scales=b.scales)
    plain = attention_paged(q, *b.args(), **kw).float()

    def run(start, length):
        i32 = dict(dtype=torch.int32, device=dev)
        return attention_shared_paged(q, *b.args(), torch.tensor(start, **i32), torch.tensor(length, **i32), **kw).float()

    for start, length in (([0], []), ([0, 4], [0]), ([0, 4], [-5]), ([0, 4], [15]), ([-2, 3], [64]), ([2, 9], [64]),
                          ([3, 1], [64]), ([1, 1, 1], [64, 64]), ([2 ** 31 - 1, -2 ** 31], [64])):
        assert torch.allclose(run(start, length), plain, atol=0.03), (start, length)
    b.kv_len[1], b.kv_len[2] = 2, 16 * b.table.shape[1] + 1
    out = run([0, 4], [64])
    assert (out[2:6] == 0).all() and torch.isfinite(out).all()
    assert torch.allclose(out[:2], plain[:2], atol=0.03)
    b.kv_len[0] = -3
    assert (run([0, 4], [64])[:2] == 0).all()
    b.q_start.copy_(torch.tensor([0, 2, 1, 900, -5]))
    run([0, 4], [64])
    torch.cuda.synchronize()


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("n", [1, 12])
def test_shared_large_batch(dev, bits, n):
    """More sequences, and more groups, than a wave looks at in one step; the same bits from call to call."""
    from alveare_amd import attention_shared_paged

    B = 150
    groups = [(1 + i % 3, 16 * (i % 4)) for i in range(72)]  # 144 sequences
    b = batch([n] * B, [n + (i * 37) % 50 for i in range(B)], groups, kv_heads=2, D=64, page=16, dev=dev, bits=bits)
    q = check(b, 2, dev)
    kw = dict(heads=2, scale=0.1, max_q=n, scales=b.scales)
    a = [attention_shared_paged(q, *b.args(), *b.groups(), **kw) for _ in range(3)]
    assert torch.equal(a[0], a[1]) and torch.equal(a[0], a[2])


@pytest.mark.parametrize("bits", [16, 8])
def test_shared_big_group(dev, bits):
    """One group of 200 sequences of one token."""
    b = batch([1] * 200, [1 + i % 7 for i in range(200)], [(200, 160)], kv_heads=2, D=64, page=16, dev=dev, bits=bits)
    check(b, 4, dev)
    check(b, 4, dev, window=40, sinks=1)


def test_shared_strides(dev):
    from alveare_amd import attention_shared_paged

    for D, n in ((64, [1, 1, 1]), (256, [1, 33, 4]), (512, [2, 40, 1])):
        b = batch(n, [v + 20 for v in n], [(3, 64)], kv_heads=2, D=D, page=16, dev=dev)
        q = rows(b.T, 4 * D, dev)
        kw = dict(heads=4, scale=0.1, max_q=max(n))
        want = attention_shared_paged(q, *b.args(), *b.groups(), scales=b.scales, **kw)
        pool = torch.stack([b.kp.view(torch.uint8), b.vp.view(torch.uint8)], 1).contiguous().view(M.E4M3)
        wide = torch.full((len(n), b.table.shape[1] + 9), 77777, dtype=torch.int32, device=dev)
        wide[:, :b.table.shape[1]] = b.table
        qkv = torch.cat([q, rows(b.T, 2 * D, dev, 9)], 1)
        out = torch.zeros(b.T, 4 * D + 8, dtype=bf, device=dev)
        attention_shared_paged(qkv[:, :4 * D], pool[:, 0], pool[:, 1], wide[:, :b.table.shape[1]], b.q_start, b.kv_len,
                               *b.groups(), out=out[:, :4 * D], scales=b.scales, **kw)
        assert torch.equal(out[:, :4 * D], want)
        assert (out[:, 4 * D:] == 0).all()


@pytest.mark.parametrize("bits", [16, 8])
def test_shared_graphs_and_streams(dev, bits):
    """Two captured graphs replayed at once on two streams; lengths, groups and what is shared change in between."""
    from alveare_amd import attention_shared_paged

    D, heads = 128, 8
    made = []
    for seed, n in ((1, 1), (2, 40)):
        b = batch([n] * 4, [90 + n, 50 + n, n, 33 + n], [(4, 320)], kv_heads=2, D=D, page=32, dev=dev, seed=seed, bits=bits)
        q = rows(b.T, heads * D, dev, seed)
        out = torch.zeros_like(q)
        start, length = torch.zeros(3, dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
        s = torch.cuda.Stream(dev)
        s.wait_stream(torch.cuda.current_stream(dev))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            attention_shared_paged(q, *b.args(), start, length, heads=heads, scale=0.1, max_q=n, out=out, scales=b.scales)
        for c in range(1, 4):  # every sequence's own table names the shared pages too
            b.table[c, :10] = b.table[0, :10]
        made.append((b, q, out, start, length, s, g, n))
    for turn, (gs, ln) in enumerate((([0, 4, 4], [320, 0]), ([0, 2, 4], [320, 64]), ([0, 0, 3], [0, 160]), ([0, 1, 1], [9, 9]))):
        for b, q, out, start, length, s, g, n in made:
            q.copy_(rows(b.T, heads * D, dev, 10 + turn))
            b.kv_len.copy_(torch.tensor([410 + n - 7 * turn, 370 + n - turn, 320 + n, 353 + n - turn]))
            start.copy_(torch.tensor(gs))
            length.copy_(torch.tensor(ln))
        torch.cuda.synchronize()
        for b, q, out, start, length, s, g, n in made:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for b, q, out, start, length, s, g, n in made:
            kw = dict(heads=heads, scale=0.1, max_q=n, scales=b.scales)
            want = attention_shared_paged(q, *b.args(), start, length, **kw)
            assert torch.equal(out, want), f"turn {turn}, n={n}"


def test_shared_refusals(dev):
    from alveare_amd import attention_shared_paged

    b = batch([1, 1], [20, 30], [(2, 16)], kv_heads=2, D=64, page=16, dev=dev)
    q = rows(2, 256, dev)
    gs, sl = b.groups()
    kw = dict(heads=4, scales=b.scales)
    with pytest.raises(ValueError):
        attention_shared_paged(q, *b.args(), gs[:1], sl, **kw)
    with pytest.raises(TypeError):
        attention_shared_paged(q, *b.args(), gs.long(), sl, **kw)
    with pytest.raises(TypeError):
        attention_shared_paged(q, *b.args(), gs, sl.cpu(), **kw)
    with pytest.raises(TypeError):
        attention_shared_paged(q, *b.args(), gs, sl, heads=4)
    assert attention_shared_paged(q[:0], *b.args(), gs, sl, **kw).shape == (0, 256)


@pytest.mark.parametrize("dtype", [bf, M.E4M3])
def test_forked_slots_through_the_cache(dev, dtype):
    """A prompt, forks of it, steps of all slots as a server makes them: post, shared attention, adjusted logits,
    sampling; captured and replayed against eager calls, and against attention that shares nothing."""
    import alveare_amd as aa

    heads, kv_heads, D, S = 8, 2, 64, 16
    cache = aa.PagedCache(layers=2, kv_heads=kv_heads, D=D, pages=64, page_size=S, slots=6, max_pages=12, device=dev,
                          dtype=dtype)
    g = torch.Generator().manual_seed(0)
    rope = torch.randn(12 * S, D, generator=g).to(bf).to(dev)
    proj = (torch.randn(heads * D, 500, generator=g) / 16).to(dev)
    kw = dict(heads=heads, k_off=heads * D, v_off=(heads + kv_heads) * D, rope=rope)

    def post(layer, x, args):
        return aa.qkv_post_paged(x, cache.k[layer], cache.v[layer], *args, scales=cache.scales[layer], **kw)

    # two prompts, the first one forked to four, the second to two
    for slot, length in ((0, 75), (4, 33)):
        cache.reserve([slot], length)
        args = cache.batch([slot], length)
        for layer in range(2):
            post(layer, rows(length, (heads + 2 * kv_heads) * D, dev, 20 + slot + layer), args)
    for dst in (1, 2, 3):
        cache.fork(0, dst)
    cache.fork(4, 5)
    slots = [0, 1, 2, 3, 4, 5]
    tokens = torch.full((6, 32), -1, dtype=torch.int32, device=dev)
    n_tok = torch.zeros(6, dtype=torch.int32, device=dev)
    words = torch.randint(-2 ** 31, 2 ** 31 - 1, (6, 16), generator=g).to(torch.int32).to(dev)
    graph = None
    x = [torch.empty(6, (heads + 2 * kv_heads) * D, dtype=bf, device=dev) for _ in range(2)]
    u = torch.zeros(6, device=dev)

    def step(args, groups, shared=True):
        out = None
        for layer in range(2):
            q = post(layer, x[layer], args)
            pools = cache.k[layer], cache.v[layer]
            if shared:
                out = aa.attention_shared_paged(q, *pools, *args, *groups, heads=heads, scale=0.125, max_q=1,
                                                scales=cache.scales[layer])
            else:
                out = aa.attention_paged(q, *pools, *args, heads=heads, scale=0.125, max_q=1, scales=cache.scales[layer])
        logits = out.float() @ proj
        l2 = aa.adjust_logits(logits, tokens=tokens, n_tokens=n_tok, repetition=1.3, frequency=0.2, presence=0.1,
                              allowed=words)
        token, prob = aa.sample(l2, u, temperature=0.8, top_k=20)
        return out, l2, token, prob

    held = None
    for turn in range(4):
        cache.reserve(slots, 1)
        args = cache.batch(slots, 1)
        groups = cache.shared(slots)
        if turn == 0:
            assert groups[0].tolist() == [0, 4, 6] and groups[1].tolist() == [64, 32]
        for layer in range(2):
            x[layer].copy_(rows(6, x[layer].shape[1], dev, 40 + 2 * turn + layer))
        u.copy_(torch.rand(6, generator=g))
        eager = step(args, groups)
        apart = step(args, groups, shared=False)[0]
        assert torch.allclose(eager[0].float(), apart.float(), atol=2 * R.BF16 * float(apart.abs().max()))
        if graph is None:
            held = args + tuple(groups)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                replayed = step(held[:3], held[3:])
        for t, v in zip(held, args + tuple(groups)):
            t.copy_(v)
        graph.replay()
        for a, c in zip(eager, replayed):
            assert torch.equal(a, c), turn
        tokens.scatter_(1, n_tok[:, None].long(), eager[2][:, None])
        n_tok += 1
    assert (n_tok == 4).all()
    # a compaction moves the powers with the codes
    cache.free(2)
    q = rows(3, heads * D, dev, 90)
    run = lambda: aa.attention_shared_paged(q, cache.k[1], cache.v[1], *cache.batch([0, 1, 3], 1),  # noqa: E731
                                            *cache.shared([0, 1, 3]), heads=heads, scale=0.1, scales=cache.scales[1])
    want = run()
    cache.compact()
    assert torch.equal(run(), want)

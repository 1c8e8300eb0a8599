"""8-bit pages: what is written to them against the definition, and attention over
them against plain forms in 64 bits."""
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


def check(batch, heads, dev, *, window=0, sinks=0, scale=None, missing=(), q=None, seed=1):
    from alveare_amd import attention_paged

    D = batch.D
    scale = 1.5 / math.sqrt(D) if scale is None else scale
    q = rows(batch.T, heads * D, dev, seed) if q is None else q
    want, tol = M.attention(q, batch, heads, window, sinks, scale, missing)
    for mq in (0, max(max(batch.n), 1)):
        out = torch.full((batch.T, heads * D), 7.0, dtype=bf, device=dev)
        attention_paged(q, *batch.args(), heads=heads, window=window, sinks=sinks, scale=scale, max_q=mq, out=out,
                        scales=batch.scales)
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


# ---- what is written -------------------------------------------------------------------

def post_both(x, b, dev, heads, kv_heads, D, **kw):
    """(k, v) bf16 rows as the bf16 pages hold them, and the codes and powers of 8-bit ones; the q of both."""
    from alveare_amd import qkv_post_paged

    q, K = heads * D, kv_heads * D
    kw = dict(heads=heads, k_off=q, v_off=q + K, **kw)
    k16, v16 = (torch.zeros(b.kp.shape, dtype=bf, device=dev) for _ in range(2))
    q16 = qkv_post_paged(x, k16, v16, b.table, b.q_start, b.kv_len, **kw)
    before = [t.view(torch.uint8).clone() for t in (b.kp, b.vp, b.scales)]
    q8 = qkv_post_paged(x, *b.args(), scales=b.scales, **kw)
    assert torch.equal(q16, q8)
    return k16, v16, before


def check_post(x, b, dev, heads, kv_heads, D, **kw):
    k16, v16, before = post_both(x, b, dev, heads, kv_heads, D, **kw)
    want = [t.cpu() for t in before]
    at = 0
    for s, (n, total) in enumerate(zip(b.n, b.total)):
        for i in range(n):
            p = total - n + i
            page, slot = int(b.table[s, p // b.page]), p % b.page
            for j, pool in enumerate((k16, v16)):
                c, e = M.encode(pool[page, :, slot])
                want[j][page, :, slot] = c
                want[2][page, :, slot, j] = e
        at += n
    for got, w, name in zip((b.kp, b.vp, b.scales), want, ("k", "v", "scales")):
        got = got.view(torch.uint8).cpu()
        if name != "scales":  # either NaN
            got, w = (torch.where(t == 255, 127, t) for t in (got, w))
        bad = (got != w).nonzero()
        assert len(bad) == 0, (name, len(bad), bad[0].tolist(), int(got[tuple(bad[0])]), int(w[tuple(bad[0])]))


@pytest.mark.parametrize("heads,kv_heads,D", LAYOUTS)
@pytest.mark.parametrize("norm_v,half", [(True, None), (False, 8)])
def test_post8(dev, heads, kv_heads, D, norm_v, half):
    n, total = [3, 0, 1, 20], [40, 9, 1, 20]
    b = M.Batch(n, total, kv_heads=kv_heads, D=D, page=16, dev=dev)
    x = rows(b.T, (heads + 2 * kv_heads) * D, dev, std=1.5)
    g = torch.Generator().manual_seed(4)
    rope = torch.randn(64, D, generator=g).to(bf).to(dev)
    w = 1 + 0.3 * torch.randn(D, generator=g).to(dev)
    check_post(x, b, dev, heads, kv_heads, D, q_w=w, k_w=w, norm_v=norm_v, rope=rope, half=half)


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_post8_ties_and_edges(dev, D):
    """Values as they are (no norm, no rotation): every magnitude of a bf16 mantissa at many scales, halves
    between codes, the largest at 448 and next to it, zeros, values that leave nothing, not finite ones."""
    from alveare_amd import qkv_post_paged

    T = 96
    x = torch.zeros(T, 3 * D)
    v = x[:, D:].view(T, 2, D)
    i = torch.arange(D)
    for t in range(40):  # steps of 1/64 up to 2 (a bf16 mantissa has 1/128)
        v[t] = (i % 128 + 128) / 128.0 * 2.0 ** ((i // 16) % 24 - 12.0) * 2.0 ** (t - 20)
    v[40], v[41, 0, :3], v[42, 0, 0] = 0.0, torch.tensor([448.0, 1.0, -0.0]), 450.0
    v[43, :, 5], v[44, :, 7] = 2.0 ** -133, 2.0 ** -120
    v[45], v[46] = 3.3895313892515355e38, -3.3895313892515355e38
    v[47, 0, 3], v[47, 1, 4], v[48] = math.inf, math.nan, -math.inf
    v[47, :, 9] = 5.0
    g = torch.Generator().manual_seed(3)
    v[49:] = torch.randn(T - 49, 2, D, generator=g) * torch.exp(20 * torch.randn(T - 49, 2, 1, generator=g))
    x = x.to(bf).to(dev)
    b = M.Batch([T], [T], kv_heads=1, D=D, page=32, dev=dev)
    check_post(x, b, dev, 1, 1, D, norm_q=False, norm_k=False, norm_v=False)
    # v the un-normalised k
    b2 = M.Batch([T], [T], kv_heads=1, D=D, page=32, dev=dev)
    qkv_post_paged(x[:, :2 * D].contiguous(), *b2.args(), heads=1, k_off=D, v_off=-1, norm_q=False, norm_k=False,
                   norm_v=False, scales=b2.scales)
    pages = b2.table[0, :3].long()
    assert torch.equal(b2.kp.view(torch.uint8)[pages], b2.vp.view(torch.uint8)[pages])
    assert torch.equal(b2.kp.view(torch.uint8)[pages], b.kp.view(torch.uint8)[b.table[0, :3].long()])


def test_post8_strides_padding_and_malformed(dev):
    """Interleaved pools, odd offsets and alignments, rows behind the last sequence, a missing page, a sequence
    that does not fit its table."""
    from alveare_amd import qkv_post_paged

    heads, kv_heads, D, S = 4, 2, 64, 16
    b = M.Batch([2, 5, 3], [30, 21, 18], kv_heads=kv_heads, D=D, page=S, dev=dev, extra_rows=4)
    x = rows(b.T, (heads + 2 * kv_heads) * D, dev)
    kw = dict(heads=heads, norm_v=False)
    a = [t.view(torch.uint8).clone() for t in (b.kp, b.vp, b.scales)]
    k, v, s = a[0].view(M.E4M3), a[1].view(M.E4M3), a[2].view(M.E8M0)
    b.table[1, 1] = b.pages  # position 16 .. 20 of sequence 1 are nowhere
    b.kv_len[2] = S * b.table.shape[1] + 1
    q = torch.full((b.T, heads * D), 3.0, dtype=bf, device=dev)
    before = [t.clone() for t in a]
    qkv_post_paged(x, k, v, b.table, b.q_start, b.kv_len, k_off=256, v_off=384, q_out=q, scales=s, **kw)
    assert (q[7:10] == 0).all() and (q[10:] == 3).all() and (q[:7] != 0).any()
    page = int(b.table[0, 1])
    changed = torch.zeros(b.pages, kv_heads, S, dtype=torch.bool, device=dev)
    changed[page, :, 28 - 16:30 - 16] = True
    for t, o in zip(a[:2], before[:2]):
        assert torch.equal((t != o).any(-1) & ~changed, torch.zeros_like(changed))
        assert (t != o).any(-1)[changed].all()
    # the same into pools whose k and v pages alternate, from rows that no wide access fits
    pool = torch.zeros(b.pages, 2, kv_heads, S, D, dtype=torch.uint8, device=dev)
    powers = torch.zeros(b.pages, 3, kv_heads, S, 2, dtype=torch.uint8, device=dev)
    odd = torch.zeros(b.T, 520, dtype=bf, device=dev)
    odd[:, 1:257], odd[:, 260:516] = x[:, :256], x[:, 256:]
    qkv_post_paged(odd[:, 1:], pool[:, 0].view(M.E4M3), pool[:, 1].view(M.E4M3), b.table, b.q_start, b.kv_len, k_off=259,
                   v_off=387, scales=powers[:, 1].view(M.E8M0), **kw)
    assert torch.equal(pool[page, 0][:, 12:14], a[0][page][:, 12:14])
    assert torch.equal(pool[page, 1][:, 12:14], a[1][page][:, 12:14])
    assert torch.equal(powers[page, 1][:, 12:14], a[2][page][:, 12:14])
    assert (powers[:, 0] == 0).all() and (powers[:, 2] == 0).all()


# ---- attention -------------------------------------------------------------------------

@pytest.mark.parametrize("heads,kv_heads,D", LAYOUTS)
@pytest.mark.parametrize("page", [16, 64])
def test_attention8_decode(dev, heads, kv_heads, D, page):
    total = [1, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 300, 0, 33]
    n = [min(1, t) for t in total]
    b = M.Batch(n, total, kv_heads=kv_heads, D=D, page=page, dev=dev, extra_rows=2)
    check(b, heads, dev)


@pytest.mark.parametrize("heads,kv_heads,D", LAYOUTS)
def test_attention8_ragged_chunks(dev, heads, kv_heads, D):
    n = [5, 0, 37, 1, 64, 3, 70]
    past = [100, 40, 0, 77, 3, 0, 131]
    b = M.Batch(n, [a + c for a, c in zip(n, past)], kv_heads=kv_heads, D=D, page=32, dev=dev, extra_rows=5)
    check(b, heads, dev)


@pytest.mark.parametrize("heads,kv_heads,D", [(16, 8, 256), (16, 1, 512), (32, 8, 64), (6, 2, 128)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 0), (64, 4), (65, 1), (100, 70), (1000, 3)])
def test_attention8_window_and_sinks(dev, heads, kv_heads, D, window, sinks):
    n = [1, 40, 9, 1]
    past = [333, 150, 0, 2]
    b = M.Batch(n, [a + c for a, c in zip(n, past)], kv_heads=kv_heads, D=D, page=16, dev=dev)
    check(b, heads, dev, window=window, sinks=sinks)


@pytest.mark.parametrize("heads,kv_heads,D", [(4, 2, 64), (4, 2, 128), (4, 1, 256), (16, 1, 512)])
def test_attention8_long_prompt_rows(dev, heads, kv_heads, D):
    b = M.Batch([259, 131], [259, 200], kv_heads=kv_heads, D=D, page=64, dev=dev)
    check(b, heads, dev)
    check(b, heads, dev, window=50, sinks=2)


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("n", [1, 3, 80])
def test_attention8_splits_of_a_long_axis(dev, D, n):
    b = M.Batch([n], [2501], kv_heads=1, D=D, page=128, dev=dev)
    check(b, 2, dev)


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("n", [1, 6, 90])
def test_attention8_what_is_masked_reaches_no_row(dev, D, n):
    """NaN codes in later tokens of the chunk, behind the window, in the rest of the last page (the batch's own)."""
    from alveare_amd import attention_paged

    L, nan = 260 + n, math.nan
    b = M.Batch([n, n], [L, L], kv_heads=1, D=D, page=32, dev=dev)
    window, sinks = 100, 2
    for p in range(sinks, L - n + 1 - window):
        b.put(0, p, k=nan if p % 2 else None, v=nan if p % 3 else None)
    check(b, 2, dev, window=window, sinks=sinks)
    if n == 1:
        return
    b.put(1, L - 1, k=nan, v=nan)
    b.put(1, L - 2, v=nan)
    q = rows(b.T, 2 * D, dev, 3)
    want, tol = M.attention(q, b, 2, window, sinks, 0.1)
    for mq in (0, n):
        got = attention_paged(q, *b.args(), heads=2, window=window, sinks=sinks, scale=0.1, max_q=mq, scales=b.scales)
        got = got.double().cpu().view_as(want)
        ok = torch.ones(2 * n, dtype=torch.bool)
        ok[2 * n - 2:] = False
        assert torch.isfinite(got[ok]).all()
        assert ((got - want).abs() <= tol)[ok].all()
        assert torch.isnan(got[2 * n - 2:]).all()


@pytest.mark.parametrize("heads,kv_heads,D", [(8, 2, 64), (4, 2, 128), (16, 8, 256), (16, 1, 512)])
def test_attention8_missing_pages(dev, heads, kv_heads, D):
    from alveare_amd import attention_paged

    n, total = [3, 50, 2, 1], [70, 90, 30, 257]
    b = M.Batch(n, total, kv_heads=kv_heads, D=D, page=16, dev=dev)
    gone = [(0, 0), (0, 3), (1, 2), (1, 4), (2, 0), (2, 1), (3, 1), (3, 16)]
    for i, (s, p) in enumerate(gone):
        b.table[s, p] = (-1, b.pages, -2 ** 31, 2 ** 31 - 1)[i % 4]
    q = check(b, heads, dev, missing=gone)
    out = attention_paged(q, *b.args(), heads=heads, scale=0.1, scales=b.scales)
    assert (out[53:55] == 0).all()


def test_attention8_powers_far_apart(dev):
    """Heads whose powers differ by 2^40, the smallest and largest powers, scores all alike."""
    for D in (64, 128, 256, 512):
        for n in (1, 40):
            b = M.Batch([n, n], [200, 150 + n], kv_heads=2, D=D, page=16, dev=dev)
            e = b.scales.view(torch.uint8)
            g = torch.Generator().manual_seed(D)
            for s in range(2):
                up = torch.randint(-20, 21, (b.total[s], 2), generator=g)
                up[5] = 60  # one value that outweighs the rest
                for p in range(b.total[s]):
                    page, slot = int(b.table[s, p // 16]), p % 16
                    e[page, :, slot, 1] = (e[page, :, slot, 1].cpu().long() + up[p]).to(torch.uint8).to(dev)
                b.v[s] = torch.ldexp(b.v[s], up[..., None].double())
            check(b, 4, dev)
            check(b, 4, dev, scale=0.0)
            # keys near 2^-126 and queries that make nothing of them
            e[..., 0] = 1
            b.k = [k * 2.0 ** -119 for k in b.k]
            check(b, 4, dev)


def test_attention8_malformed_sequences(dev):
    from alveare_amd import attention_paged

    b = M.Batch([2, 3, 1, 2], [40, 50, 60, 70], kv_heads=2, D=64, page=16, dev=dev)
    q = rows(b.T, 4 * 64, dev)
    kw = dict(heads=4, scale=0.2, scales=b.scales)
    good = attention_paged(q, *b.args(), **kw)
    b.kv_len[1] = 2
    b.kv_len[2] = 16 * b.table.shape[1] + 1
    for mq in (0, 3):
        out = attention_paged(q, *b.args(), max_q=mq, **kw)
        assert (out[2:6] == 0).all()
        assert torch.allclose(out[:2].float(), good[:2].float(), atol=0.05)
        assert torch.allclose(out[6:].float(), good[6:].float(), atol=0.05)
    b.kv_len.copy_(torch.tensor([40, 50, 60, 70]))
    b.q_start.copy_(torch.tensor([0, 2, 1, 900, -5]))
    out = attention_paged(q, *b.args(), **kw)
    assert torch.allclose(out[:1].float(), good[:1].float(), atol=0.05)


def test_attention8_strides(dev):
    """q inside the packed qkv rows, interleaved pools and powers, a wider table, strided out."""
    from alveare_amd import attention_paged

    for D, n in ((64, [1, 1, 1]), (128, [3, 70, 2]), (256, [1, 33, 4]), (512, [2, 40, 1])):
        b = M.Batch(n, [v + 60 for v in n], kv_heads=2, D=D, page=16, dev=dev)
        q = rows(b.T, 4 * D, dev)
        kw = dict(heads=4, scale=0.1, max_q=max(n))
        want = attention_paged(q, *b.args(), scales=b.scales, **kw)
        pool = torch.stack([b.kp.view(torch.uint8), b.vp.view(torch.uint8)], 1).contiguous().view(M.E4M3)
        powers = torch.stack([b.scales.view(torch.uint8)] * 3, 1).contiguous()
        powers[:, 0], powers[:, 2] = 99, 200
        wide = torch.full((len(n), b.table.shape[1] + 9), 77777, dtype=torch.int32, device=dev)
        wide[:, :b.table.shape[1]] = b.table
        qkv = torch.cat([q, rows(b.T, 2 * D, dev, 9)], 1)
        out = torch.zeros(b.T, 4 * D + 8, dtype=bf, device=dev)
        attention_paged(qkv[:, :4 * D], pool[:, 0], pool[:, 1], wide[:, :b.table.shape[1]], b.q_start, b.kv_len,
                        out=out[:, :4 * D], scales=powers.view(M.E8M0)[:, 1], **kw)
        assert torch.equal(out[:, :4 * D], want)
        assert (out[:, 4 * D:] == 0).all()


def test_attention8_offsets_past_32_bits(dev):
    """Pages whose byte offsets need more than 32 bits."""
    from alveare_amd import attention_paged, qkv_post_paged

    D, page = 512, 1024
    pages = (1 << 32) // (D * page) + 3
    b = M.Batch([1, 20], [1500, 900], kv_heads=1, D=D, page=page, dev=dev)
    k, v = (torch.empty(pages, 1, page, D, dtype=torch.uint8, device=dev).view(M.E4M3) for _ in range(2))
    s = torch.empty(pages, 1, page, 2, dtype=torch.uint8, device=dev).view(M.E8M0)
    table = torch.full_like(b.table, -1)
    used = [(i, j) for i in range(2) for j in range(b.table.shape[1]) if int(b.table[i, j]) >= 0]

    def fill():
        for x, (i, j) in enumerate(used):
            p, o = pages - 1 - x, int(b.table[i, j])
            table[i, j] = p
            for to, of in ((k, b.kp), (v, b.vp), (s, b.scales)):
                to.view(torch.uint8)[p] = of.view(torch.uint8)[o]

    fill()
    q = rows(b.T, 4 * D, dev)
    kw = dict(heads=4, scale=0.05)
    for mq in (1, 20):
        want = attention_paged(q, *b.args(), max_q=mq, scales=b.scales, **kw)
        assert torch.equal(attention_paged(q, k, v, table, b.q_start, b.kv_len, max_q=mq, scales=s, **kw), want)
    x = rows(b.T, 6 * D, dev)
    post = dict(heads=4, k_off=4 * D, v_off=5 * D)
    qkv_post_paged(x, *b.args(), scales=b.scales, **post)
    qkv_post_paged(x, k, v, table, b.q_start, b.kv_len, scales=s, **post)
    for i, j in used:
        for to, of in ((k, b.kp), (v, b.vp), (s, b.scales)):
            assert torch.equal(to.view(torch.uint8)[int(table[i, j])], of.view(torch.uint8)[int(b.table[i, j])])


@pytest.mark.parametrize("n", [1, 48])
def test_attention8_large_batch(dev, n):
    from alveare_amd import attention_paged

    B = 150
    total = [n + (i * 37) % 90 for i in range(B)]
    b = M.Batch([n] * B, total, kv_heads=2, D=64, page=16, dev=dev)
    q = check(b, 2, dev)
    a = [attention_paged(q, *b.args(), heads=2, scale=0.1, max_q=n, scales=b.scales) for _ in range(3)]
    assert torch.equal(a[0], a[1]) and torch.equal(a[0], a[2])


def test_attention8_graphs_and_streams(dev):
    """Two captured graphs replayed at once on two streams, lengths changed in between, against eager calls."""
    from alveare_amd import attention_paged

    D, heads = 128, 8
    made = []
    for seed, n in ((1, 1), (2, 60)):
        b = M.Batch([n] * 4, [900 + n, 500 + n, n, 33 + n], kv_heads=2, D=D, page=32, dev=dev, seed=seed)
        q = rows(b.T, heads * D, dev, seed)
        out = torch.zeros_like(q)
        s = torch.cuda.Stream(dev)
        s.wait_stream(torch.cuda.current_stream(dev))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            attention_paged(q, *b.args(), heads=heads, scale=0.1, max_q=n, out=out, scales=b.scales)
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
            want = attention_paged(q, *b.args(), heads=heads, scale=0.1, max_q=n, scales=b.scales)
            assert torch.equal(out, want), f"turn {turn}, n={n}"


def test_attention8_empty_and_refusals(dev):
    from alveare_amd import Q4ValueError, attention_paged, qkv_post_paged

    b = M.Batch([1, 2], [20, 30], kv_heads=2, D=64, page=16, dev=dev)
    q = rows(3, 256, dev)
    none = attention_paged(q[:0], *b.args(), heads=4, scales=b.scales)
    assert none.shape == (0, 256)
    kw = dict(heads=4, scales=b.scales)
    with pytest.raises(TypeError):  # 8-bit pages need scales, bf16 ones have none
        attention_paged(q, *b.args(), heads=4)
    with pytest.raises(TypeError):
        attention_paged(q, b.kp.float().to(bf), b.vp.float().to(bf), *b.args()[2:], **kw)
    with pytest.raises(TypeError):
        attention_paged(q, *b.args(), heads=4, scales=b.scales.view(torch.uint8))
    with pytest.raises(ValueError):
        attention_paged(q, *b.args(), heads=4, scales=b.scales[:-1])
    with pytest.raises(ValueError):
        attention_paged(q, *b.args(), heads=4, scales=b.scales.view(torch.uint8)[..., :1].expand(-1, -1, -1, 2).view(M.E8M0))
    with pytest.raises(Q4ValueError):
        attention_paged(q, *b.args(), **{**kw, "heads": 3})
    with pytest.raises(Q4ValueError):
        attention_paged(q, *b.args(), window=-1, **kw)
    x = rows(3, 512, dev)
    with pytest.raises(TypeError):
        qkv_post_paged(x, *b.args(), heads=4, k_off=256, v_off=384)
    with pytest.raises(ValueError):
        qkv_post_paged(x, *b.args(), heads=4, k_off=256, v_off=448, scales=b.scales)

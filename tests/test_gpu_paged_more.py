"""Paged attention where a wave's flag, a group's members or a plan's choice decide."""
import math

import pytest
import torch

import more_ref as M

pytestmark = pytest.mark.gpu

bf = torch.bfloat16


def rows(T, width, dev, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(T, width, generator=g).to(bf).to(dev)


def close(got, want, tol, where=slice(None)):
    got = got[:len(want)].double().cpu().view_as(want)[where]
    assert torch.isfinite(got).all()
    bad = (got - want[where]).abs() > tol[where]
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[0].tolist())


@pytest.mark.parametrize("heads", [1, 20, 40])
@pytest.mark.parametrize("bits", [8, 16])
def test_masked_nan_in_each_waves_block(dev, bits, heads):
    """Of a unit of 128 positions (eight waves of 16, or four of 32) one block has a NaN of V that no row, or the
    second alone, sees."""
    from alveare_amd import attention_paged, attention_shared_paged

    for at in range(131, 256, 16):
        b = M.Batch([2], [256], kv_heads=1, D=64, page=16, dev=dev, bits=bits, groups=[(1, 0)])
        b.put(0, 255 if at > 240 else at, v=math.nan)
        q = rows(2, heads * 64, dev)
        kw = dict(heads=heads, window=8, scale=0.2, scales=b.scales)
        want, tol = M.attention(q, b, heads, 8, 0, 0.2)
        seen = slice(0, heads if at > 240 else 2 * heads)
        for got in (attention_paged(q, *b.args(), **kw), attention_shared_paged(q, *b.args(), *b.groups(), **kw)):
            close(got, want.view(2 * heads, 64), tol.view(2 * heads, 64), seen)
            assert torch.isnan(got.view(2 * heads, 64)[seen.stop:]).all()


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("heads,kv_heads,D", [(8, 2, 128), (4, 1, 256), (16, 1, 512)])
@pytest.mark.parametrize("n", [[2, 3, 1, 2], [50, 3, 1, 70]])
@pytest.mark.parametrize("window", [0, 30])
def test_members_beside_malformed_ones(dev, bits, heads, kv_heads, D, n, window):
    """A member whose rows do not fit the batch takes its group along with it nowhere: the others' outputs are what
    they are without it. Where no rows of a group are the batch's, or not those of a member, that shares nothing."""
    from alveare_amd import attention_paged, attention_shared_paged
    from alveare_amd._lib import lib

    total = [v + 64 + i for i, v in enumerate(n)]
    at = [sum(n[:i]) for i in range(5)]
    kw = dict(heads=heads, window=window, sinks=2 if window else 0, scale=0.1)

    def run(b, q, q_start, mq):
        size = lib().alv_attention_shared_workspace(heads, kv_heads, D, 4, len(q), mq, 1)
        stale = torch.full((size,), 255, dtype=torch.uint8, device=dev)  # what the call's workspace holds
        del stale
        b.q_start.copy_(torch.tensor(q_start))
        return attention_shared_paged(q, *b.args(), *b.groups(), max_q=mq, scales=b.scales,
                                      out=torch.full_like(q, 7.0), **kw)

    b = M.Batch(n, total, kv_heads=kv_heads, D=D, page=16, dev=dev, bits=bits, groups=[(4, 64)])
    q = rows(b.T, heads * D, dev)
    want, tol = M.attention(q, b, heads, window, kw["sinks"], 0.1)
    for mq in (0, max(n)):
        close(run(b, q[:-1], at, mq), want[:at[3]], tol[:at[3]])                      # the last one's end past the rows
        close(run(b, q, [*at[:4], 2 ** 31 - 1], mq), want[:at[3]], tol[:at[3]])
        out = run(b, q, [-1, *at[1:]], mq)                                            # the first begins ahead of them
        close(out[n[0]:], want[n[0]:], tol[n[0]:])
    # with pages of their own
    b = M.Batch(n, total, kv_heads=kv_heads, D=D, page=16, dev=dev, bits=bits)
    want, tol = M.attention(q, b, heads, window, kw["sinks"], 0.1)
    b.group_start, b.shared_len = (torch.tensor(v, dtype=torch.int32, device=dev) for v in ([0, 4], [64]))
    for mq in (0, max(n)):
        close(run(b, q, [*at[:4], -5], mq), want[:at[3]], tol[:at[3]])               # the group has no rows
        close(run(b, q, [0, at[1], at[2], at[3], 1], mq)[at[2]:], want[at[2]:at[3]], tol[at[2]:at[3]])  # or one


@pytest.mark.parametrize("heads,D", [(32, 64), (64, 64), (128, 64), (128, 128), (64, 256)])
@pytest.mark.parametrize("page", [16, 64])
def test_streaming_of_many_rows_over_8_bit_pages(dev, heads, D, page):
    """Up to 64 rows of a sequence and kv head (32 at D = 256) in a batch too large for tiles."""
    from alveare_amd import attention_paged

    B = 140
    n = [i % 2 if i > 130 else 1 for i in range(B)]
    total = [1 + (i * 29) % 140 + (800 if i == 7 else 0) for i in range(B)]
    b = M.Batch(n, total, kv_heads=2, D=D, page=page, dev=dev)
    q = rows(b.T, heads * D, dev)
    for window in (0, 50):
        want, tol = M.attention(q, b, heads, window, 0, 0.1)
        close(attention_paged(q, *b.args(), heads=heads, window=window, scale=0.1, max_q=1, scales=b.scales), want, tol)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("heads,kv_heads,D", [(4, 2, 64), (8, 2, 128), (4, 1, 256), (16, 1, 512)])
@pytest.mark.parametrize("n", [[1, 1, 1, 1, 1], [1, 3, 70, 0, 140]])
def test_first_tokens_on_both_sides_of_what_is_shared(dev, bits, heads, kv_heads, D, n):
    """A window, and first tokens that end ahead of a group's shared positions, within and behind them."""
    from alveare_amd import attention_shared_paged

    own = [700, 430, 500, 90, 810]
    total = [o + s for o, s in zip(own, (64, 64, 0, 208, 208))]
    b = M.Batch(n, total, kv_heads=kv_heads, D=D, page=16, dev=dev, bits=bits, groups=[(2, 64), (1, 0), (2, 208)])
    q = rows(b.T, heads * D, dev)
    for window, sinks in ((100, 1), (100, 64), (100, 65), (30, 150), (100, 300), (600, 4), (1, 900)):
        want, tol = M.attention(q, b, heads, window, sinks, 0.1)
        for mq in (0, max(n)):
            close(attention_shared_paged(q, *b.args(), *b.groups(), heads=heads, window=window, sinks=sinks, scale=0.1,
                                         max_q=mq, scales=b.scales), want, tol)


@pytest.mark.parametrize("D,n", [(64, 1), (256, 1), (128, 64), (512, 64)])
def test_a_window_with_first_tokens_bounds_what_is_read(dev, D, n):
    """Sequences that share nothing, 40000 positions behind a window of 512: the time is attention_paged's, which
    reads some 600 (all of them would take tens of times as long)."""
    from alveare_amd import attention_paged, attention_shared_paged

    B, L, S = 16, 40000, 64
    need = (L + S - 1) // S
    k, v = (torch.randn(B * need, 1, S, D, device=dev).to(bf) for _ in range(2))
    i32 = dict(dtype=torch.int32, device=dev)
    table = torch.arange(B * need, **i32).view(B, need)
    q = rows(B * n, 4 * D, dev)
    args = q, k, v, table, torch.arange(0, B * n + 1, n, **i32), torch.full((B,), L, **i32)
    groups = torch.arange(B + 1, **i32), torch.zeros(B, **i32)
    kw = dict(heads=4, window=512, sinks=4, scale=0.1, max_q=n)

    def least(call):
        times = []
        for _ in range(8):
            a, z = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(10):
                call()
            z.record()
            z.synchronize()
            times.append(a.elapsed_time(z))
        return min(times)

    plain = least(lambda: attention_paged(*args, **kw))
    shared = least(lambda: attention_shared_paged(*args, *groups, **kw))
    assert shared < 4 * plain, (shared, plain)


@pytest.mark.parametrize("heads,kv_heads,D", [(8, 2, 64), (8, 2, 128), (4, 1, 256), (16, 1, 512)])
@pytest.mark.parametrize("n", [[1, 1, 1, 1], [3, 70, 0, 5], [130, 1, 150, 40]])
def test_powers_behind_the_end_do_not_matter(dev, heads, kv_heads, D, n):
    """Slots that no sequence holds have the largest power byte; the output is the same to the bit, and no wave
    does its rows again for it (which takes tens of times as long)."""
    from alveare_amd import attention_paged, attention_shared_paged

    total = [v + p for v, p in zip(n, (2001, 1999, 640, 830))]
    b = M.Batch(n, total, kv_heads=kv_heads, D=D, page=64, dev=dev, groups=[(2, 512), (2, 0)])
    q = rows(b.T, heads * D, dev)
    kw = dict(heads=heads, scale=0.1, max_q=max(n), scales=b.scales)
    bytes_ = b.scales.view(torch.uint8)
    held = torch.zeros(b.pages, 64, dtype=torch.bool)
    for s, t in enumerate(total):
        for p in range(b.shared[s] if b.leader[s] != s else 0, t):
            held[int(b.table[s, p // 64]), p % 64] = True
    free = (~held)[:, None, :, None].expand(bytes_.shape).to(dev)
    made = []
    for power in (127, 255):
        bytes_[free] = power
        calls = (lambda: attention_paged(q, *b.args(), **kw), lambda: attention_shared_paged(q, *b.args(), *b.groups(), **kw))
        for call in calls:
            times = []
            out = call()
            for _ in range(6):
                a, z = (torch.cuda.Event(enable_timing=True) for _ in range(2))
                a.record()
                for _ in range(5):
                    call()
                z.record()
                z.synchronize()
                times.append(a.elapsed_time(z))
            made.append((out, min(times)))
    for (a, ta), (z, tz) in zip(made[:2], made[2:]):
        assert torch.equal(a.view(torch.int16), z.view(torch.int16))
        assert tz < 3 * ta, (ta, tz)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("heads,kv_heads,D", [(8, 2, 64), (8, 2, 128), (4, 1, 256), (16, 1, 512)])
@pytest.mark.parametrize("n", [[1, 1, 1, 1], [3, 70, 0, 5], [130, 1, 150, 40]])
def test_table_entries_of_what_is_shared_do_not_matter(dev, bits, heads, kv_heads, D, n):
    """The members' own entries for shared positions name no page, or one of NaN: the same bits, and no wave does
    its rows again for it (which takes tens of times as long)."""
    from alveare_amd import attention_shared_paged

    total = [v + p for v, p in zip(n, (2001, 1999, 840, 2830))]
    b = M.Batch(n, total, kv_heads=kv_heads, D=D, page=16, dev=dev, bits=bits, groups=[(2, 528), (2, 528)])
    q = rows(b.T, heads * D, dev)
    kw = dict(heads=heads, scale=0.1, max_q=max(n), scales=b.scales)
    used = set(b.table[(b.table >= 0) & (b.table < b.pages)].tolist())
    spare = next(p for p in range(b.pages) if p not in used)
    if bits == 8:
        b.scales.view(torch.uint8)[spare] = 255
    for window, sinks in ((0, 0), (700, 600)):
        made = []
        for entry in (-1, spare):
            b.table[1, :33] = b.table[3, :33] = entry
            call = lambda: attention_shared_paged(q, *b.args(), *b.groups(), window=window, sinks=sinks, **kw)  # noqa: E731
            out = call()
            times = []
            for _ in range(6):
                a, z = (torch.cuda.Event(enable_timing=True) for _ in range(2))
                a.record()
                for _ in range(5):
                    call()
                z.record()
                z.synchronize()
                times.append(a.elapsed_time(z))
            made.append((out, min(times)))
        (a, ta), (z, tz) = made
        assert torch.equal(a.view(torch.int16), z.view(torch.int16))
        assert tz < 3 * ta, (ta, tz)

"""Argument checks of the 8-bit, shared and adjusting operators, and which groups the
page cache finds (no GPU)."""
import ctypes
import os
import random

import numpy as np
import pytest
import torch


@pytest.fixture(scope="module")
def L():
    from alveare_amd import _lib

    if not os.path.exists(_lib.LIB_PATH):
        from alveare_amd import build

        build.build()
    return _lib.lib()


P, ODD = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 2)


def attn8(L, **ch):
    a = dict(q=P, ld_q=256, k=P, v=P, ks=2 * 16 * 64, vs=2 * 16 * 64, sc=P, ss=64, pages=9, S=16, table=P, ldt=4, W=4, qs=P,
             kl=P, B=2, T=3, mq=0, heads=4, kv=2, D=64, window=0, sinks=0, scale=1.0, out=P, ldo=256, ws=None, wb=0, st=None)
    a.update(ch)
    return L.alv_attention_paged8(*a.values())


def shared(L, **ch):
    a = dict(q=P, ld_q=256, k=P, v=P, ks=2 * 16 * 64, vs=2 * 16 * 64, sc=None, ss=0, pages=9, S=16, table=P, ldt=4, W=4, qs=P,
             kl=P, B=2, T=3, mq=0, gs=P, sl=P, G=1, heads=4, kv=2, D=64, window=0, sinks=0, scale=1.0, out=P, ldo=256,
             ws=None, wb=0, st=None)
    a.update(ch)
    return L.alv_attention_shared(*a.values())


BAD = (dict(q=None), dict(k=None), dict(v=None), dict(table=None), dict(qs=None), dict(kl=None), dict(out=None), dict(S=8),
       dict(S=24), dict(S=2048), dict(B=0), dict(T=-1), dict(pages=0), dict(W=0), dict(ldt=3), dict(heads=0), dict(heads=3),
       dict(kv=0), dict(D=96), dict(D=1024), dict(window=-1), dict(sinks=-1), dict(scale=-0.5), dict(scale=float("nan")),
       dict(scale=float("inf")), dict(ld_q=255), dict(ldo=200), dict(ks=100), dict(vs=100), dict(mq=-1))
UNALIGNED = (dict(q=ODD), dict(k=ODD), dict(v=ODD), dict(out=ODD), dict(ld_q=260), dict(ldo=258), dict(ks=2052),
             dict(table=ctypes.c_void_p((1 << 20) + 1)))


def test_attention8_arguments(L):
    from alveare_amd._lib import ALV_ERR_ALIGN, ALV_ERR_ARG, ALV_ERR_RANGE, ALV_OK

    for ch in (*BAD, dict(sc=None), dict(ss=63), dict(ss=-64)):
        assert attn8(L, **ch) == ALV_ERR_ARG, ch
        assert L.alv_last_error()
    for ch in (*UNALIGNED, dict(sc=ctypes.c_void_p((1 << 20) + 8)), dict(ss=72), dict(vs=2056)):
        assert attn8(L, **ch) == ALV_ERR_ALIGN, ch
    assert attn8(L, T=(1 << 22) + 1) == ALV_ERR_RANGE
    assert attn8(L, T=1, heads=1 << 17, ld_q=1 << 23, ldo=1 << 23) == ALV_ERR_RANGE
    assert attn8(L, T=1 << 22, heads=512, ld_q=1 << 15, ldo=1 << 15) == ALV_ERR_RANGE
    assert attn8(L, W=1 << 27, ldt=1 << 27) == ALV_ERR_RANGE
    assert attn8(L, T=0, q=None, out=None) == ALV_OK


def test_shared_arguments(L):
    from alveare_amd._lib import ALV_ERR_ALIGN, ALV_ERR_ARG, ALV_ERR_RANGE, ALV_OK

    for ch in (*BAD, dict(gs=None), dict(sl=None), dict(G=-1), dict(sc=P, ss=63)):
        assert shared(L, **ch) == ALV_ERR_ARG, ch
    for ch in (*UNALIGNED, dict(sc=P, ss=72), dict(sc=P, ss=64, vs=2056), dict(gs=ODD), dict(sl=ODD)):
        assert shared(L, **ch) == ALV_ERR_ALIGN, ch
    assert shared(L, T=(1 << 22) + 1) == ALV_ERR_RANGE
    assert shared(L, T=1 << 22, heads=512, ld_q=1 << 15, ldo=1 << 15) == ALV_ERR_RANGE
    assert shared(L, T=0, q=None, out=None) == ALV_OK


def test_shared_too_many_groups(L):
    from alveare_amd._lib import ALV_ERR_RANGE

    for ch in (dict(G=(1 << 22) + 1), dict(G=2 ** 31 - 1), dict(B=(1 << 22) + 1), dict(G=2 ** 31 - 1, B=2 ** 31 - 1)):
        assert shared(L, **ch) == ALV_ERR_RANGE, ch


def test_post8_arguments(L):
    from alveare_amd._lib import ALV_ERR_ARG, ALV_ERR_RANGE, ALV_OK

    def post(**ch):
        a = dict(qkv=P, ld=512, k_off=256, v_off=384, heads=4, kv=2, D=64, qw=None, kw=None, nq=1, nk=1, nv=1, eps=1e-6,
                 rope=P, rows=100, stride=64, cos=0, sin=32, half=32, table=P, ldt=4, W=4, qs=P, kl=P, B=2, T=3, pages=9,
                 S=16, k=P, v=P, ks=2048, vs=2048, sc=P, ss=64, q=P, ldq=256, st=None)
        a.update(ch)
        return L.alv_qkv_post_paged8(*a.values())

    for ch in (dict(qkv=None), dict(k=None), dict(v=None), dict(q=None), dict(table=None), dict(sc=None), dict(ss=63),
               dict(ld=500), dict(k_off=200), dict(v_off=300), dict(D=32), dict(heads=5), dict(half=33), dict(half=0),
               dict(half=2 ** 31 - 1), dict(sin=40), dict(rows=0), dict(cos=-1), dict(S=17), dict(ks=2047), dict(ldq=255)):
        assert post(**ch) == ALV_ERR_ARG, ch
    assert post(heads=1 << 17, k_off=1 << 23, v_off=-1, ld=1 << 24, ldq=1 << 24) == ALV_ERR_RANGE
    assert post(T=0, qkv=None, q=None) == ALV_OK


def test_adjust_arguments(L):
    from alveare_amd._lib import ALV_ERR_ALIGN, ALV_ERR_ARG, ALV_ERR_RANGE, ALV_OK

    far = ctypes.c_void_p(1 << 30)

    def adjust(**ch):
        a = dict(l=P, ld=100, out=far, ldo=100, B=2, V=100, t=P, ldt=5, n=5, nt=None, np_=None, rd=None, r=1.0, fd=None,
                 f=0.0, pd=None, p=0.0, bt=P, ldbt=3, b=P, ldb=3, M=3, al=P, lda=4, st=None)
        a.update(ch)
        return L.alv_adjust_logits(*a.values())

    for ch in (dict(l=None), dict(out=None), dict(t=None), dict(bt=None), dict(b=None), dict(B=-1), dict(V=0), dict(n=-1),
               dict(M=-1), dict(ld=99), dict(ldo=99), dict(ldt=-1), dict(lda=-1), dict(r=0.0), dict(r=-1.0),
               dict(r=float("nan")), dict(out=P, ldo=101), dict(out=ctypes.c_void_p((1 << 20) + 40)),
               dict(out=ctypes.c_void_p((1 << 20) + 400)), dict(out=ctypes.c_void_p((1 << 20) - 40)),
               dict(ld=250, ldo=250, out=ctypes.c_void_p((1 << 20) + 4 * 160))):
        assert adjust(**ch) == ALV_ERR_ARG, ch
        assert L.alv_last_error()
    for ch in (dict(l=ODD), dict(t=ODD), dict(nt=ODD), dict(rd=ODD), dict(bt=ODD), dict(al=ODD)):
        assert adjust(**ch) == ALV_ERR_ALIGN, ch
    for ch in (dict(B=65536), dict(V=(1 << 24) + 1, ld=1 << 25, ldo=1 << 25), dict(n=(1 << 30) + 1),
               dict(B=4096, V=1 << 24, ld=1 << 24, ldo=1 << 24)):
        assert adjust(**ch) == ALV_ERR_RANGE, ch
    assert adjust(B=0, l=None, out=None) == ALV_OK


def test_adjust_one_row_has_no_stride(L):
    """The distance between rows counts for nothing where there is one, a zero neither; far rows and long lists of
    biases are refused."""
    from alveare_amd._lib import ALV_ERR_ARG, ALV_ERR_RANGE

    def adjust(out, ld, B=1, M=0):
        return L.alv_adjust_logits(P, ld, ctypes.c_void_p(out), ld, B, 100, None, 0, 0, None, None, None, 1.0, None, 0.0,
                                   None, 0.0, P, 0, P, 0, M, None, 0, None)

    for ld in (0, -1, 1, 100, 1000, 2 ** 62):
        assert adjust((1 << 20) + 40, ld) == ALV_ERR_ARG, ld  # within the row
        assert adjust((1 << 20) - 396, ld) == ALV_ERR_ARG, ld
    assert adjust(1 << 30, 2 ** 62, B=2) == ALV_ERR_RANGE
    assert adjust(1 << 30, 2 ** 40 + 1, B=2) == ALV_ERR_RANGE
    assert adjust(1 << 30, 100, M=2 ** 16 + 1) == ALV_ERR_RANGE


class _Host:
    """PagedCache with its pools on the host and page copies left out."""

    def __new__(cls, **kw):
        from alveare_amd import PagedCache

        class C(PagedCache):
            def _copy(self, src, dst):
                pass

        return C(layers=1, kv_heads=1, D=16, device="cpu", **kw)


def test_cache_of_8_bits():
    c = _Host(pages=8, page_size=16, slots=2, max_pages=4, dtype=torch.float8_e4m3fn)
    assert c.k[0].dtype == torch.float8_e4m3fn and c.scales[0].shape == (8, 1, 16, 2)
    assert c.scales[0].dtype == torch.float8_e8m0fnu and (c.scales[0].float() == 1).all()
    assert (c.k[0].float() == 0).all()
    assert _Host(pages=8, page_size=16, slots=2, max_pages=4).scales == [None]
    with pytest.raises(ValueError):
        _Host(pages=8, page_size=16, slots=2, max_pages=4, dtype=torch.float16)


def pages_read(cache, slots, start, length):
    S, n = cache.page_size, 0
    for a, b, s in zip(start, start[1:], length):
        n += s // S + sum(len(cache.table(slots[i])) - s // S for i in range(a, b))
    return n


def test_cache_shared_groups():
    c = _Host(pages=400, page_size=16, slots=12, max_pages=40)
    c.reserve([0], 100)
    for d in (1, 2):
        c.fork(0, d)
    c.reserve([0, 1, 2], 30)
    for d in (3, 4, 5):
        c.fork(2, d)  # what 0 and 1 share is shorter than what these share
    c.reserve([2, 3, 4, 5], 200)
    c.reserve([6, 7], [50, 3])
    c.fork(6, 8)

    def groups(slots):
        start, length = (t.tolist() for t in c.shared(slots))
        assert start[0] == 0 and start[-1] == len(slots) and all(a < b for a, b in zip(start, start[1:]))
        for a, b, s in zip(start, start[1:], length):  # what is said to be shared is
            assert s % 16 == 0
            for i in range(a, b):
                assert c.table(slots[i])[:s // 16] == c.table(slots[a])[:s // 16] and s <= c.length(slots[i])
        return start, length

    assert groups([0, 1]) == ([0, 2], [96])
    assert groups([2, 3, 4, 5]) == ([0, 4], [128])
    assert groups([0, 1, 2, 3, 4, 5]) == ([0, 2, 6], [96, 128]) or pages_read(
        c, [0, 1, 2, 3, 4, 5], *groups([0, 1, 2, 3, 4, 5])) <= pages_read(c, [0, 1, 2, 3, 4, 5], [0, 2, 6], [96, 128])
    assert groups([0, 6, 1]) == ([0, 1, 2, 3], [0, 0, 0])
    assert groups([6, 8, 7]) == ([0, 2, 3], [48, 0])  # the partly filled page is not whole
    assert groups([7]) == ([0, 1], [0])
    assert groups([10]) == ([0, 1], [0])
    for bad in ([0, 0], [12], [-1]):
        with pytest.raises((ValueError, IndexError)):
            c.shared(bad)


def test_cache_shared_groups_are_the_best():
    """Against all ways to cut a batch, for random trees of forks."""
    rng = random.Random(1)
    for _ in range(60):
        c = _Host(pages=300, page_size=16, slots=7, max_pages=20)
        c.reserve([0], rng.randint(1, 100))
        for s in range(1, 7):
            if rng.random() < 0.8:
                c.fork(rng.randrange(s), s)
            c.reserve([s], rng.randint(0, 60))
        slots = list(range(7))
        rng.shuffle(slots)
        start, length = (t.tolist() for t in c.shared(slots))
        got = pages_read(c, slots, start, length)
        best = None
        for cut in range(64):
            at = [0] + [i + 1 for i in range(6) if cut >> i & 1] + [7]
            share = []
            for a, b in zip(at, at[1:]):
                n = min(c.length(slots[i]) // 16 for i in range(a, b))
                while n and any(c.table(slots[i])[:n] != c.table(slots[a])[:n] for i in range(a, b)):
                    n -= 1
                share.append(16 * n if b - a > 1 else 0)
            r = pages_read(c, slots, at, share)
            best = r if best is None else min(best, r)
        assert got == best


def test_reference_of_codes():
    """The tests' own encoder: every code's value gives its code, halves go to the even one."""
    import more_ref as M

    v = M.code_values()
    x = torch.from_numpy(np.where(np.isnan(v), 0.0, v))[None]
    c, e = M.encode(x)
    assert int(e[0]) == 127
    assert all(int(c[0, i]) in (i, 0, 128) if i in (0, 127, 128, 255) else int(c[0, i]) == i for i in range(256))
    x = torch.tensor([[448.0, 17.0, 19.0, -17.0, 2.0 ** -10, 3 * 2.0 ** -10, 1.0625]])
    assert M.decode(*M.encode(x))[0].tolist() == [448.0, 16.0, 20.0, -16.0, 0.0, 2.0 ** -8, 1.0]
    assert int(M.encode(torch.tensor([[449.0]]))[1]) == 128
    assert int(M.encode(torch.tensor([[2.0 ** -133]]))[1]) == 1


def test_packed_calls(L):
    """alv_call gives what the entry itself gives; what it cannot pass it refuses."""
    from alveare_amd import _lib

    assert set(_lib.PACKED) <= set(_lib.SIGNATURES)
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "alveare_q4.h")).read()
    for name, (entry, n, words) in _lib.PACKED.items():
        assert f"#define ALV_CALL_{name[4:].upper()} {entry}\n" in header
        zeros = words.pack(*[0] * n)
        assert len(zeros) == 8 * n
        rc = L.alv_call(entry, zeros, n)
        message = L.alv_last_error()
        assert rc == getattr(L, name)(*[0] * n) and (rc == _lib.ALV_OK or message == L.alv_last_error())
        assert L.alv_call(entry, zeros, n - 1) == _lib.ALV_ERR_ARG
        types = _lib.SIGNATURES[name][1]
        for i, t in enumerate(types):
            if t is ctypes.c_int:
                for far in (2 ** 31, -2 ** 31 - 1, 2 ** 40):
                    assert L.alv_call(entry, words.pack(*[far if j == i else 0 for j in range(n)]), n) == _lib.ALV_ERR_RANGE
    assert L.alv_call(99, b"", 0) == _lib.ALV_ERR_ARG
    assert L.alv_call(-1, b"", 0) == _lib.ALV_ERR_ARG
    assert L.alv_call(0, None, 0) == _lib.ALV_ERR_ARG
    # every argument in its place: refused for the one that is wrong, whatever the others
    good = dict(q=1 << 20, ld_q=256, k=1 << 20, v=1 << 20, ks=2048, vs=2048, sc=1 << 20, ss=64, pages=9, S=16, table=1 << 20,
                ldt=4, W=4, qs=1 << 20, kl=1 << 20, B=2, T=0, mq=0, heads=4, kv=2, D=64, window=0, sinks=0, scale=1.0,
                out=1 << 20, ldo=256, ws=0, wb=0, st=0)
    entry, n, words = _lib.PACKED["alv_attention_paged8"]
    run = lambda **ch: L.alv_call(entry, words.pack(*{**good, **ch}.values()), n)  # noqa: E731
    assert run() == _lib.ALV_OK
    for ch in (*BAD, dict(sc=None), dict(ss=63)):
        if None not in ch.values() and "T" not in ch:
            assert run(**ch) == attn8(L, T=0, **ch) == _lib.ALV_ERR_ARG, ch
    assert run(scale=1e300) == _lib.ALV_ERR_ARG
    with pytest.raises(_lib.Q4ValueError):
        _lib.call(L, "alv_attention_paged8", *{**good, "D": 96}.values())

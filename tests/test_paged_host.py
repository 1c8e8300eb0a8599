"""The paged operators' argument checks and the page cache's bookkeeping (no GPU)."""
import ctypes
import os

import pytest
import torch


@pytest.fixture(scope="module")
def L():
    from alveare_amd import _lib

    if not os.path.exists(_lib.LIB_PATH):
        from alveare_amd import build

        build.build()
    return _lib.lib()


P = ctypes.c_void_p(1 << 20)


def attn(L, **ch):
    a = dict(q=P, ld_q=256, k=P, v=P, ks=2 * 16 * 64, vs=2 * 16 * 64, pages=9, S=16, table=P, ldt=4, W=4, qs=P, kl=P,
             B=2, T=3, mq=0, heads=4, kv=2, D=64, window=0, sinks=0, scale=1.0, out=P, ldo=256, ws=None, wb=0, st=None)
    a.update(ch)
    return L.alv_attention_paged(*a.values())


def test_attention_arguments(L):
    from alveare_amd._lib import ALV_ERR_ALIGN, ALV_ERR_ARG, ALV_ERR_RANGE, ALV_OK

    odd = ctypes.c_void_p((1 << 20) + 2)
    for ch in (dict(q=None), dict(k=None), dict(v=None), dict(table=None), dict(qs=None), dict(kl=None), dict(out=None),
               dict(S=8), dict(S=24), dict(S=2048), dict(B=0), dict(T=-1), dict(pages=0), dict(W=0), dict(ldt=3),
               dict(heads=0), dict(heads=3), dict(kv=0), dict(D=96), dict(D=1024), dict(window=-1), dict(sinks=-1),
               dict(scale=-0.5), dict(scale=float("nan")), dict(scale=float("inf")), dict(ld_q=255), dict(ldo=200),
               dict(ks=100), dict(vs=100), dict(mq=-1)):
        assert attn(L, **ch) == ALV_ERR_ARG, ch
        assert L.alv_last_error()
    for ch in (dict(q=odd), dict(k=odd), dict(v=odd), dict(out=odd), dict(ld_q=260), dict(ldo=258), dict(ks=2052),
               dict(table=ctypes.c_void_p((1 << 20) + 1))):
        assert attn(L, **ch) == ALV_ERR_ALIGN, ch
    assert attn(L, T=(1 << 22) + 1) == ALV_ERR_RANGE
    assert attn(L, T=1, heads=1 << 17, ld_q=1 << 23, ldo=1 << 23) == ALV_ERR_RANGE
    assert attn(L, T=1 << 22, heads=512, ld_q=1 << 15, ldo=1 << 15) == ALV_ERR_RANGE
    assert attn(L, W=1 << 27, ldt=1 << 27) == ALV_ERR_RANGE
    assert attn(L, T=0, q=None, out=None) == ALV_OK


def test_post_arguments(L):
    from alveare_amd._lib import ALV_ERR_ARG, ALV_ERR_RANGE, ALV_OK

    def post(**ch):
        a = dict(qkv=P, ld=512, k_off=256, v_off=384, heads=4, kv=2, D=64, qw=None, kw=None, nq=1, nk=1, nv=1, eps=1e-6,
                 rope=P, rows=100, stride=64, cos=0, sin=32, half=32, table=P, ldt=4, W=4, qs=P, kl=P, B=2, T=3, pages=9,
                 S=16, k=P, v=P, ks=2048, vs=2048, q=P, ldq=256, st=None)
        a.update(ch)
        return L.alv_qkv_post_paged(*a.values())

    for ch in (dict(qkv=None), dict(k=None), dict(v=None), dict(q=None), dict(table=None), dict(ld=500), dict(k_off=200),
               dict(v_off=300), dict(D=32), dict(heads=5), dict(half=33), dict(half=0), dict(sin=40), dict(rows=0),
               dict(cos=-1), dict(S=17), dict(ks=2047), dict(ldq=255)):
        assert post(**ch) == ALV_ERR_ARG, ch
    # heads times D, and offsets plus it, past 32 bits
    for ch in (dict(heads=1 << 26), dict(heads=1 << 27, kv=1 << 26), dict(k_off=2 ** 31 - 64, v_off=-1),
               dict(v_off=2 ** 31 - 64)):
        assert post(**ch) == ALV_ERR_ARG, ch
    assert post(heads=1 << 17, k_off=1 << 23, v_off=-1, ld=1 << 24, ldq=1 << 24) == ALV_ERR_RANGE
    assert post(T=0, qkv=None, q=None) == ALV_OK


def test_copy_arguments(L):
    from alveare_amd._lib import ALV_ERR_ALIGN, ALV_ERR_ARG, ALV_OK

    def copy(src, dst, caches=(1 << 20,), n=64, stride=64, pages=4):
        c = (ctypes.c_void_p * max(len(caches), 1))(*caches)
        s, d = ((ctypes.c_int32 * max(len(v), 1))(*v) for v in (src, dst))
        return L.alv_copy_pages(c, len(caches), n, stride, pages, s, d, len(src), None)

    for bad in (([0], [4]), ([-1], [0]), ([0, 1], [2, 2]), ([0, 2], [2, 3]), ([1], [1])):
        assert copy(*bad) == ALV_ERR_ARG, bad
    assert copy([0], [1], caches=()) == ALV_ERR_ARG
    assert copy([0], [1], caches=(0,)) == ALV_ERR_ARG
    assert copy([0], [1], n=24) == ALV_ERR_ARG
    assert copy([0], [1], stride=48) == ALV_ERR_ARG
    assert copy([0], [1], caches=((1 << 20) + 8,)) == ALV_ERR_ALIGN
    assert copy([], []) == ALV_OK


def test_sample_arguments(L):
    from alveare_amd._lib import ALV_ERR_ALIGN, ALV_ERR_ARG, ALV_ERR_RANGE, ALV_OK

    def sample(**ch):
        a = dict(x=P, ld=100, B=2, V=100, u=P, td=None, t=1.0, kd=None, k=0, pd=None, p=1.0, md=None, m=0.0, tok=P, prob=P,
                 ws=P, wb=1 << 40, st=None)
        a.update(ch)
        return L.alv_sample(*a.values())

    for ch in (dict(x=None), dict(u=None), dict(tok=None), dict(V=0), dict(ld=99), dict(B=-1)):
        assert sample(**ch) == ALV_ERR_ARG, ch
    assert sample(u=ctypes.c_void_p(1 << 20 | 2)) == ALV_ERR_ALIGN
    assert sample(V=(1 << 24) + 1, ld=1 << 25) == ALV_ERR_RANGE
    assert sample(B=70000) == ALV_ERR_RANGE
    assert sample(B=0, x=None) == ALV_OK


@pytest.fixture
def cache(monkeypatch):
    from alveare_amd import paged

    monkeypatch.setattr(paged, "copy_pages", lambda caches, src, dst: copies.append((list(src), list(dst))))
    copies = []
    c = paged.PagedCache(layers=1, kv_heads=1, D=64, pages=8, page_size=16, slots=4, max_pages=5, device="cpu")
    c.copies = copies
    return c


def test_cache_reserve_fork_and_copy_on_write(cache):
    c = cache
    c.reserve([0], 20)
    assert c.table(0) == [0, 1] and c.length(0) == 20 and c.free_pages == 6
    c.fork(0, 1)
    c.fork(0, 2)
    assert c.table(1) == c.table(2) == [0, 1] and c.free_pages == 6 and not c.copies
    c.reserve([0, 1, 2], [1, 1, 1])  # two copies; the last keeps the page
    assert c.copies == [([1, 1], [2, 3])]
    assert [c.table(s) for s in range(3)] == [[0, 2], [0, 3], [0, 1]] and c.free_pages == 4
    c.reserve([1], 0)
    assert len(c.copies) == 1
    with pytest.raises(ValueError):
        c.fork(0, 1)
    with pytest.raises(ValueError):
        c.fork(3, 3)


def test_cache_runs_out_without_a_change(cache):
    c = cache
    c.reserve([0, 1], [70, 40])  # 5 + 3 pages
    before = [c.table(s) for s in range(4)], c.free_pages
    with pytest.raises(MemoryError):
        c.reserve([2, 1], [1, 1])
    with pytest.raises(ValueError):
        c.reserve([0], 11)  # past max_pages
    with pytest.raises(ValueError):
        c.reserve([0, 0], 1)
    assert ([c.table(s) for s in range(4)], c.free_pages) == before and c.length(1) == 40
    c.free(0)
    assert c.free_pages == 5 and c.length(0) == 0
    c.fork(1, 2)
    c.reserve([2], 1)
    assert len(c.copies) == 1
    with pytest.raises(IndexError):
        c.length(4)


def test_cache_truncate_and_compact(cache):
    c = cache
    c.reserve([0, 1], [33, 33])
    c.fork(1, 2)
    c.free(0)
    c.truncate(1, 17)
    assert c.table(1) == [3, 4] and c.table(2) == [3, 4, 5]
    assert c.compact() == 3
    assert c.copies[-1] == ([3, 4, 5], [0, 1, 2])
    assert c.table(1) == [0, 1] and c.table(2) == [0, 1, 2] and c.free_pages == 5
    assert c.compact() == 0
    c.reserve([1], 1)  # position 17 is in the shared page 1
    assert c.copies[-1] == ([1], [3]) and c.table(1) == [0, 3]
    with pytest.raises(ValueError):
        c.truncate(1, 19)
    t, q, k = c.batch([2, 3, 1], [5, 0, 18])
    assert t.tolist() == [[0, 1, 2, -1, -1], [-1] * 5, [0, 3, -1, -1, -1]]
    assert q.tolist() == [0, 5, 5, 23] and k.tolist() == [33, 0, 18]
    with pytest.raises(ValueError):
        c.batch([1], [19])
    with pytest.raises(ValueError):
        c.batch([1, 1], [1, 1])


def test_operators_refuse_host_tensors():
    import alveare_amd as aa

    z = torch.zeros(1, 64, dtype=torch.bfloat16)
    pg = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, 1, dtype=torch.int32)
    for call in (lambda: aa.attention_paged(z, pg, pg, i, i[0], i[0], heads=1),
                 lambda: aa.qkv_post_paged(z, pg, pg, i, i[0], i[0], heads=1, k_off=64, v_off=128),
                 lambda: aa.copy_pages([pg], [0], [1]), lambda: aa.sample(z.float(), z[0, :1].float())):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_attention_workspace(L):
    from alveare_amd._lib import ALV_ERR_ALIGN, ALV_ERR_ARG

    need = L.alv_attention_paged_workspace(4, 2, 64, 2, 3, 0)
    assert need > 0 and L.alv_attention_paged_workspace(4, 3, 64, 2, 3, 0) == 0
    assert attn(L) == ALV_ERR_ARG and attn(L, ws=P, wb=need - 1) == ALV_ERR_ARG
    assert attn(L, ws=ctypes.c_void_p((1 << 20) + 8), wb=need) == ALV_ERR_ALIGN
    assert L.alv_sample_workspace(1, 1000) == 0 < L.alv_sample_workspace(1, 32000) < L.alv_sample_workspace(2, 32000)


def test_attention_workspace_of_any_hint(L):
    """No sequence owns more than T rows: a larger max_q is T, whatever it is multiplied by."""
    for heads, kv, D, B, T in ((65536, 1, 64, 1 << 24, 100), (65536, 1, 512, (1 << 31) - 1, 100), (16, 8, 256, 3, 7),
                               (512, 512, 64, (1 << 31) - 1, 1 << 21)):
        want = L.alv_attention_paged_workspace(heads, kv, D, B, T, T)
        assert want < 1 << 40
        for mq in (T + 1, 1 << 20, (1 << 31) - 1):
            assert L.alv_attention_paged_workspace(heads, kv, D, B, T, max(mq, T)) == want


def test_cache_is_unchanged_where_a_copy_fails(cache, monkeypatch):
    """A reserve or compaction whose copies raise leaves tables, lengths, shares and free pages as they were."""
    from alveare_amd import paged

    c = cache
    c.reserve([0, 3], [20, 33])
    c.fork(0, 1)
    c.fork(0, 2)
    state = lambda: ([c.table(s) for s in range(4)], [c.length(s) for s in range(4)], c.free_pages,  # noqa: E731
                     list(c._shared), sorted(c._free))
    before = state()

    def fail(*_):
        raise RuntimeError("no copy")

    with monkeypatch.context() as m:
        m.setattr(paged, "copy_pages", fail)
        with pytest.raises(RuntimeError, match="no copy"):
            c.reserve([3, 0, 1], [5, 13, 1])
        assert state() == before
        c.free(0)  # slots 1 and 2 hold pages 0 and 1, slot 3 pages 2, 3 and 4
        c.free(1)
        c.free(2)
        before = state()
        with pytest.raises(RuntimeError, match="no copy"):
            c.compact()
        assert state() == before
    assert c.compact() == 2 and c.copies == [([3, 4], [0, 1])] and c.table(3) == [2, 0, 1]
    c.fork(3, 1)
    c.reserve([1], 1)
    assert c.copies[-1] == ([1], [3]) and c.table(1) == [2, 0, 3] and c.free_pages == 4


def test_negative_numbers_past_32_bits(monkeypatch):
    """What a C int would turn into another number is refused before the call; any negative v_off means the raw k."""
    from alveare_amd import paged

    class Reached(Exception):
        pass

    def reach(*a):
        raise Reached(a)

    class Fake:
        alv_attention_paged = alv_qkv_post_paged = staticmethod(reach)
        alv_attention_paged_workspace = staticmethod(lambda *a: 0)

    monkeypatch.setattr(paged, "lib", Fake)
    monkeypatch.setattr(paged, "_need_gpu", lambda t: t.device)
    monkeypatch.setattr(paged, "_on", lambda dev: torch.no_grad())
    monkeypatch.setattr(paged, "_stream", lambda t: 0)
    bf = torch.bfloat16
    qkv, pg = torch.zeros(3, 256, dtype=bf), torch.zeros(4, 1, 16, 64, dtype=bf)
    batch = pg, pg, torch.zeros(2, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    out, wrap = torch.zeros(3, 128, dtype=bf), 2 ** 32
    attend = lambda **kw: paged.attention_paged(qkv[:, :128], *batch, out=out, **{"heads": 2, **kw})  # noqa: E731
    post = lambda **kw: paged.qkv_post_paged(qkv, *batch, q_out=out, rope=torch.zeros(9, 64, dtype=bf),  # noqa: E731
                                             **{"heads": 2, "k_off": 128, "v_off": 192, **kw})
    with pytest.raises(Reached):
        attend(window=5, sinks=1, max_q=3)
    with pytest.raises(Reached):
        post()
    for kw in (dict(window=-wrap), dict(window=-wrap + 7), dict(sinks=-wrap), dict(max_q=-wrap + 1), dict(heads=2 - wrap)):
        with pytest.raises(ValueError):
            attend(**kw)
    for kw in (dict(heads=2 - wrap), dict(k_off=128 - wrap), dict(k_off=128 + wrap), dict(half=32 - wrap)):
        with pytest.raises(ValueError):
            post(**kw)
    for v_off in (-1, -wrap, 192 - wrap):
        with pytest.raises(Reached) as e:
            post(v_off=v_off)
        assert e.value.args[0][3] == -1

"""Batches of sequences over a paged KV cache: prompts, drafts and decode steps.

``alveare_amd.layer`` steps one sequence by one token over a cache in one
piece. Here a call takes a packed batch: sequence b owns rows ``q_start[b] ..
q_start[b + 1] - 1`` of every activation, the last of its ``kv_len[b]``
positions (the new ones included), and position p is slot ``p % S`` of page
``page_table[b, p // S]``. The three are int32 tensors on the device, read by
the kernels, so a captured step replays with whatever they hold then. Pages are
``(pages, kv_heads, S, D)`` bfloat16, S a power of two from 16 to 1024; a table
entry outside ``[0, pages)`` holds no positions (pages a window has left behind
may be given up by writing -1 there).

With ``scales`` the pages are 8-bit, half the bytes: ``torch.float8_e4m3fn``
codes, and ``scales`` ``(pages, kv_heads, S, 2)`` ``torch.float8_e8m0fnu`` a power
of two for each slot's k and v; a value is code times power.

==========================  =================================================
``qkv_post_paged``          q/k/v norms + RoPE + insert of every new token, in
                            the bits of ``layer.qkv_post``
``attention_paged``         attention of every new token: causal, sliding
                            window, first tokens that stay visible
``attention_shared_paged``  the same where groups of sequences have their
                            first pages in common: those for many rows at once
``copy_pages``              pages copied within each of many caches
``PagedCache``              the layers' pages and the tables of a set of
                            sequences: reserve, fork, truncate, free, compact
==========================  =================================================
"""
from __future__ import annotations

import array
import functools
import heapq

import numpy as np
import torch

from ._lib import call, check, lib
from .layer import _GEMMA_EPS, _f32, _ptr
from .ops import _need_gpu, _on, _stream, _workspace


def _rows(t: torch.Tensor, name: str, width: int, dev: torch.device) -> int:
    """Checks a (T, >= width) bfloat16 tensor, contiguous along its rows; returns how far apart they are."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.bfloat16 or t.dim() != 2 or t.device != dev:
        raise TypeError(f"{name} must be a 2-D bfloat16 tensor on {dev}")
    (T, w), (ld, one) = t.shape, t.stride()
    if w < width or one != 1 and w > 1:
        raise ValueError(f"{name} rows must be contiguous and hold {width} values, got shape {tuple(t.shape)} "
                         f"strides {t.stride()}")
    return ld if T > 1 else w


def _page_stride(t: torch.Tensor, name: str, dev: torch.device, dtype: torch.dtype = torch.bfloat16) -> int:
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.dim() != 4 or t.device != dev:
        last = "2" if name == "scales" else "D"
        raise TypeError(f"{name} must be a (pages, kv_heads, page_size, {last}) {str(dtype)[6:]} tensor on {dev}")
    (n, H, S, D), (s0, s1, s2, s3) = t.shape, t.stride()
    if s3 != 1 or s2 != D or s1 != S * D and H > 1:
        raise ValueError(f"{name}: each page must be contiguous, got strides {t.stride()}")
    return s0 if n > 1 else H * S * D


def _pages(kpages: torch.Tensor, vpages: torch.Tensor, dev: torch.device, dtype: torch.dtype):
    """(shape, page strides) of the two pools: each page contiguous in itself."""
    ks, vs = _page_stride(kpages, "kpages", dev, dtype), _page_stride(vpages, "vpages", dev, dtype)
    if kpages.shape != vpages.shape:
        raise ValueError(f"kpages and vpages differ: {tuple(kpages.shape)} and {tuple(vpages.shape)}")
    return kpages.shape, ks, vs


def _batch(page_table: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor, dev: torch.device):
    """(B, max_pages, row stride of the table)."""
    for t, name, dim in ((page_table, "page_table", 2), (q_start, "q_start", 1), (kv_len, "kv_len", 1)):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.dim() != dim or t.device != dev:
            raise TypeError(f"{name} must be a {dim}-D int32 tensor on {dev}")
        if t.stride(-1) != 1 and t.shape[-1] > 1:
            raise ValueError(f"{name} must be contiguous along its rows")
    B, W = page_table.shape
    if kv_len.shape[0] != B or q_start.shape[0] != B + 1:
        raise ValueError(f"a table of {B} sequences needs kv_len of {B} and q_start of {B + 1}, got {kv_len.shape[0]} "
                         f"and {q_start.shape[0]}")
    return B, W, page_table.stride(0) if B > 1 else W


_BF16, _I32 = torch.bfloat16, torch.int32
_E4M3, _E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
_INT_MAX = 2 ** 31 - 1


def _args(t: torch.Tensor, name: str, kpages: torch.Tensor, vpages: torch.Tensor, page_table: torch.Tensor,
          q_start: torch.Tensor, kv_len: torch.Tensor, dev: torch.device, dtype: torch.dtype = _BF16):
    """((pages, kv_heads, S, D), page strides, B, max_pages, table's row stride, T, t's width and row stride): the
    checks that every call shares (dtype: the pages'). Contiguous tensors, as most are, take one test each (the
    others' take 6 us of a call whose kernel may take 5)."""
    i = dev.index
    try:
        if (t.dtype is _BF16 and kpages.dtype is dtype and vpages.dtype is dtype and page_table.dtype is _I32
                and q_start.dtype is _I32 and kv_len.dtype is _I32 and t.is_contiguous() and kpages.is_contiguous()
                and vpages.is_contiguous() and page_table.is_contiguous() and q_start.is_contiguous()
                and kv_len.is_contiguous() and kpages.get_device() == i and vpages.get_device() == i
                and page_table.get_device() == i and q_start.get_device() == i and kv_len.get_device() == i
                and t.dim() == 2 and q_start.dim() == 1 and kv_len.dim() == 1):
            shape = kpages.shape
            _, H, S, D = shape
            B, W = page_table.shape
            if vpages.shape == shape and q_start.numel() == B + 1 and kv_len.numel() == B:
                T, w = t.shape
                n = H * S * D
                return shape, n, n, B, W, W, T, w, w
    except (AttributeError, ValueError):
        pass
    return *_pages(kpages, vpages, dev, dtype), *_batch(page_table, q_start, kv_len, dev), *_shape2(t, name, dev)


def _shape2(t: torch.Tensor, name: str, dev: torch.device):
    ld = _rows(t, name, 0, dev)
    return *t.shape, ld


def _scales(scales: torch.Tensor, shape, dev: torch.device) -> int:
    """How many bytes the scales of two pages of an 8-bit pool of `shape` are apart."""
    if (isinstance(scales, torch.Tensor) and scales.dtype is _E8M0 and scales.is_contiguous() and
            scales.get_device() == dev.index and scales.shape == (*shape[:3], 2)):
        return shape[1] * shape[2] * 2
    ss = _page_stride(scales, "scales", dev, _E8M0)
    if scales.shape != (*shape[:3], 2):
        raise ValueError(f"scales of pages {tuple(shape)} are {(*shape[:3], 2)}, got {tuple(scales.shape)}")
    return ss


def _far(**numbers: int) -> None:
    raise ValueError("past 32 bits: " + ", ".join(f"{k}={v}" for k, v in numbers.items()))


def _narrow(name: str, have: int, width: int) -> None:
    raise ValueError(f"{name} rows must hold {width} values, got {have}")


def _weights(w, name: str, n: int, dev: torch.device) -> torch.Tensor | None:
    """Norm weights on a 16-byte boundary."""
    w = _f32(w, name, n, dev)
    return w.clone() if w is not None and w.data_ptr() & 15 else w


def qkv_post_paged(qkv: torch.Tensor, kpages: torch.Tensor, vpages: torch.Tensor, page_table: torch.Tensor,
                   q_start: torch.Tensor, kv_len: torch.Tensor, *, heads: int, k_off: int, v_off: int, q_w=None,
                   k_w=None, norm_q: bool = True, norm_k: bool = True, norm_v: bool = True, eps: float = _GEMMA_EPS,
                   rope: torch.Tensor | None = None, cos_off: int = 0, sin_off: int | None = None,
                   half: int | None = None, q_out: torch.Tensor | None = None,
                   scales: torch.Tensor | None = None) -> torch.Tensor:
    """``layer.qkv_post`` for every row of ``qkv`` (T, [q | k | v]): per-head
    norms, RoPE of q and k at the row's position, k and v into their pages. With
    ``scales`` the pages are 8-bit: each head's k (v) gets the smallest power of two
    that brings its largest finite magnitude to 448 or less, its values the nearest
    codes (off by at most max(2^-4 |x|, 2^-10 power)); what is not finite becomes NaN.
    ``rope`` is the (positions, width) bfloat16 table, by default [cos | sin]
    halves of its rows. Returns q (T, heads * D); rows past the last sequence are
    left as they are in ``q_out``, zeros for a sequence that does not fit its
    table (or the rope table)."""
    dev = _need_gpu(qkv)
    shape, ks, vs, B, W, ldt, T, width, ldqkv = _args(qkv, "qkv", kpages, vpages, page_table, q_start, kv_len, dev,
                                                      _BF16 if scales is None else _E4M3)
    pages, kv_heads, S, D = shape
    if v_off < 0:
        v_off = -1
    if not (0 < heads <= _INT_MAX and 0 < k_off <= _INT_MAX and v_off <= _INT_MAX and (half is None or half > 0)):
        if max(heads, k_off, v_off) > _INT_MAX or min(heads, k_off, half or 0) < -_INT_MAX:
            _far(heads=heads, k_off=k_off, v_off=v_off, half=half)
    if width < (k_off if v_off < 0 else v_off) + kv_heads * D:
        _narrow("qkv", width, (k_off if v_off < 0 else v_off) + kv_heads * D)
    ldq = heads * D
    q_w, k_w = _weights(q_w, "q_w", D, dev), _weights(k_w, "k_w", D, dev)
    rope_rows = ldr = 0
    if rope is not None:
        rope_rows, ldr = rope.shape[0], _rows(rope, "rope", 2, dev)
        half = rope.shape[1] // 2 if half is None else half
        sin_off = half if sin_off is None else sin_off
        if not (0 <= cos_off <= rope.shape[1] - half and 0 <= sin_off <= rope.shape[1] - half):
            raise ValueError(f"rope rows of {rope.shape[1]} values hold no {half} at cos_off={cos_off} and sin_off={sin_off}")
    if q_out is None:
        q_out = qkv.new_empty((T, ldq))
    else:
        ldq = _rows(q_out, "q_out", ldq, dev)
        if q_out.shape[0] < T:
            raise ValueError(f"q_out has {q_out.shape[0]} rows, qkv {T}")
    args = (qkv.data_ptr(), ldqkv, k_off, v_off, heads, kv_heads, D, _ptr(q_w), _ptr(k_w), norm_q, norm_k, norm_v, eps,
            _ptr(rope), rope_rows, ldr, cos_off, sin_off or 0, half or 0, page_table.data_ptr(), ldt, W,
            q_start.data_ptr(), kv_len.data_ptr(), B, T, pages, S, kpages.data_ptr(), vpages.data_ptr(), ks, vs)
    with _on(dev):
        if scales is None:
            call(lib(), "alv_qkv_post_paged", *args, q_out.data_ptr(), ldq, _stream(qkv))
        else:
            ss = _scales(scales, shape, dev)
            call(lib(), "alv_qkv_post_paged8", *args, scales.data_ptr(), ss, q_out.data_ptr(), ldq, _stream(qkv))
    return q_out


@functools.lru_cache(maxsize=4096)
def _size(device: int, name: str, *numbers: int) -> int:
    """Bytes of a call's workspace, a function of its numbers (asking the library is 1 us of a call). The device is
    the current one."""
    return getattr(lib(), name + "_workspace")(*numbers)


def _attention(q, kpages, vpages, page_table, q_start, kv_len, heads, window, sinks, max_q, out, scales):
    """The checks that both attentions share: (arguments of the C calls up to the batch's, from heads to sinks, out,
    its row stride, the numbers that a workspace's size goes by)."""
    dev = _need_gpu(q)
    shape, ks, vs, B, W, ldt, T, width, ldq = _args(q, "q", kpages, vpages, page_table, q_start, kv_len, dev,
                                                    _BF16 if scales is None else _E4M3)
    pages, kv_heads, S, D = shape
    ldo = heads * D
    if width < ldo:
        _narrow("q", width, ldo)
    if not (0 < heads and 0 <= window <= _INT_MAX and 0 <= sinks <= _INT_MAX and 0 <= max_q <= _INT_MAX):
        window, sinks, max_q = min(window, _INT_MAX), min(sinks, _INT_MAX), min(max_q, _INT_MAX)
        if min(heads, window, sinks, max_q) < -_INT_MAX:
            _far(heads=heads, window=window, sinks=sinks, max_q=max_q)
    if out is None:
        out = torch.empty_like(q) if width == ldo == ldq else q.new_empty((T, ldo))
    else:
        ldo = _rows(out, "out", ldo, dev)
        if out.shape[0] < T:
            raise ValueError(f"out has {out.shape[0]} rows, q {T}")
    batch = (pages, S, page_table.data_ptr(), ldt, W, q_start.data_ptr(), kv_len.data_ptr(), B, T, max_q)
    pools = (q.data_ptr(), ldq, kpages.data_ptr(), vpages.data_ptr(), ks, vs)
    if scales is not None:
        pools += scales.data_ptr(), _scales(scales, shape, dev)
    return dev, pools, batch, (heads, kv_heads, D, window, sinks), out, ldo


def attention_paged(q: torch.Tensor, kpages: torch.Tensor, vpages: torch.Tensor, page_table: torch.Tensor,
                    q_start: torch.Tensor, kv_len: torch.Tensor, *, heads: int, window: int = 0, sinks: int = 0,
                    scale: float = 1.0, max_q: int = 0, out: torch.Tensor | None = None,
                    scales: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of every row of ``q`` (T, heads * D) over the positions up to
    its own: all of them, or with ``window`` the last ``window`` and the first
    ``sinks``. A row that sees no position gets zeros; rows past the last
    sequence are left as they are in ``out``, which does not overlap ``q``.
    Scores, maxima and sums are float32; the weights are rounded to bfloat16 for
    the product with V. ``max_q``, the most rows any sequence owns, where the
    caller knows it, lets the call choose how to spread the work (1 for a decode
    step): like the other sequences' lengths it may change a row's last bits, by
    the order in which its sums are rounded, and nothing else. With ``scales`` the
    pages are 8-bit."""
    dev, pools, batch, shape, out, ldo = _attention(q, kpages, vpages, page_table, q_start, kv_len, heads, window, sinks,
                                                    max_q, out, scales)
    name = "alv_attention_paged" if scales is None else "alv_attention_paged8"
    with _on(dev):
        _, ws, n = _workspace(_size(dev.index, name, *shape[:3], *batch[-3:]), dev)
        call(lib(), name, *pools, *batch, *shape, scale, out.data_ptr(), ldo, ws or 0, n, _stream(q))
    return out


def attention_shared_paged(q: torch.Tensor, kpages: torch.Tensor, vpages: torch.Tensor, page_table: torch.Tensor,
                           q_start: torch.Tensor, kv_len: torch.Tensor, group_start: torch.Tensor,
                           shared_len: torch.Tensor, *, heads: int, window: int = 0, sinks: int = 0, scale: float = 1.0,
                           max_q: int = 0, out: torch.Tensor | None = None,
                           scales: torch.Tensor | None = None) -> torch.Tensor:
    """``attention_paged`` of a batch whose sequences come in groups with the same
    first pages (``PagedCache.shared`` finds them), which are read and multiplied
    for many of a group's rows at once. Group j is the sequences ``group_start[j] ..
    group_start[j + 1] - 1``; the first ``shared_len[j]`` positions of each (whole
    pages of them, and no more than the group's first sequence has) are taken from
    its first sequence's pages. Both are int32 tensors on the device, of groups + 1
    and groups values, read by the kernels. Every row sees what it sees in
    ``attention_paged``, its last bits may differ."""
    dev, pools, batch, shape, out, ldo = _attention(q, kpages, vpages, page_table, q_start, kv_len, heads, window, sinks,
                                                    max_q, out, scales)
    for t, name in ((group_start, "group_start"), (shared_len, "shared_len")):
        if not isinstance(t, torch.Tensor) or t.dtype != _I32 or t.dim() != 1 or t.device != dev or not t.is_contiguous():
            raise TypeError(f"{name} must be a contiguous 1-D int32 tensor on {dev}")
    G = shared_len.shape[0]
    if group_start.shape[0] != G + 1:
        raise ValueError(f"{G} shared lengths need group_start of {G + 1}, got {group_start.shape[0]}")
    if scales is None:
        pools += 0, 0
    with _on(dev):
        _, ws, n = _workspace(_size(dev.index, "alv_attention_shared", *shape[:3], *batch[-3:], G), dev)
        call(lib(), "alv_attention_shared", *pools, *batch, group_start.data_ptr(), shared_len.data_ptr(), G, *shape, scale,
             out.data_ptr(), ldo, ws or 0, n, _stream(q))
    return out


def _host_i32(v, name: str) -> array.array:
    """Page numbers as a host int32 array."""
    if isinstance(v, torch.Tensor) and v.device.type != "cpu":
        raise ValueError(f"{name} must be on the host: it is checked before anything is copied")
    if isinstance(v, (torch.Tensor, np.ndarray)):
        v = v.tolist()
    try:
        return array.array("i", v)
    except OverflowError as e:
        raise ValueError(f"{name} holds page numbers out of range") from e
    except TypeError as e:
        raise TypeError(f"{name} must be a sequence of integers: {e}") from e


def copy_pages(caches, src, dst) -> None:
    """In every cache (tensors of one shape whose first dimension counts pages,
    each page contiguous): page ``dst[i]`` = page ``src[i]``. ``src`` and ``dst``
    are host sequences; a page may be the destination of one copy and then the
    source of none. The caches do not overlap."""
    caches = list(caches)
    if not caches:
        return
    first = caches[0]
    dev = _need_gpu(first)
    shape, strides, dtype, index = first.shape, first.stride(), first.dtype, dev.index
    if len(shape) < 2 or first.numel() == 0:
        raise ValueError(f"a cache must be (pages, ...), got shape {tuple(shape)}")
    T = torch.Tensor
    try:  # (the methods mapped, and strides only where some are not contiguous: these tests are most of a small call)
        one = set(map(T.get_device, caches)) == {index}
        whole = all(map(T.is_contiguous, caches))
        ptrs = array.array("Q", map(T.data_ptr, caches))
    except TypeError:
        one = False
    if not one:
        raise ValueError(f"the caches must be tensors on one GPU, {dev}")
    if len({t.dtype for t in caches}) + len(set(map(T.size, caches))) != 2 or (
            not whole and len({t.stride() for t in caches}) != 1):
        raise ValueError(f"the caches must be alike: {dtype} {tuple(shape)} {strides}, and not all are")
    if not whole and not first[0].is_contiguous():
        raise ValueError(f"each page must be contiguous, got strides {strides}")
    src, dst = _host_i32(src, "src"), _host_i32(dst, "dst")
    if len(src) != len(dst):
        raise ValueError(f"{len(src)} sources and {len(dst)} destinations")
    esize = first.element_size()
    n = first.numel() // shape[0] * esize
    with _on(dev):
        check(lib().alv_copy_pages(ptrs.buffer_info()[0], len(caches), n, strides[0] * esize if shape[0] > 1 else n,
                                   shape[0], src.buffer_info()[0], dst.buffer_info()[0], len(src), _stream(first)),
              "alv_copy_pages")


class PagedCache:
    """The K and V pages of a model's layers and the tables of up to ``slots``
    sequences; ``dtype`` torch.float8_e4m3fn: 8-bit pages, whose ``scales`` are a
    tensor per layer (None of bfloat16 ones). One page number stands for that page of every layer, K and V:
    layers of another head layout are another cache's, and a page stays its
    sequence's until that is truncated or freed, whatever a window has left behind.

    The bookkeeping (which slot holds which pages, how often a page is shared)
    is the host's; only page copies and the tables go to the device, in the
    order of the current stream. ``batch`` gives the tensors the kernels take
    (a step of 64 slots of 4000 positions: 30 us of the host in ``reserve``, 103 in
    ``batch``, most of it the table's 64 rows; of 30000 positions 409).
    A call that needs more pages than are free raises ``MemoryError`` and changes
    nothing, nor does one whose copies raise."""

    def __init__(self, *, layers: int, kv_heads: int, D: int, pages: int, page_size: int, slots: int, max_pages: int,
                 device, dtype: torch.dtype = torch.bfloat16):
        if min(layers, kv_heads, D, pages, slots, max_pages) < 1:
            raise ValueError("layers, kv_heads, D, pages, slots and max_pages must be positive")
        if not 16 <= page_size <= 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size={page_size}: a power of two from 16 to 1024")
        self.page_size, self.pages, self.slots, self.max_pages = page_size, pages, slots, max_pages
        if dtype not in (_BF16, _E4M3):
            raise ValueError(f"dtype={dtype}: torch.bfloat16 or torch.float8_e4m3fn")
        self.pool = torch.zeros((layers, 2, pages, kv_heads, page_size, D), dtype=dtype, device=device)
        self.device, self.dtype = self.pool.device, dtype
        self.k = [self.pool[i, 0] for i in range(layers)]
        self.v = [self.pool[i, 1] for i in range(layers)]
        self.scales: list = [None] * layers
        if dtype == _E4M3:
            # (zeros would be 2^-127; of zero codes any power is one)
            powers = torch.full((layers, pages, kv_heads, page_size, 2), 127, dtype=torch.uint8, device=device)
            self.scales = list(powers.view(_E8M0).unbind(0))
        self._table: list[list[int]] = [[] for _ in range(slots)]
        self._len = [0] * slots
        self._shared = [0] * pages  # slots that hold the page
        self._free = list(range(pages))  # a heap: the lowest page first

    def _slot(self, slot: int) -> int:
        if not 0 <= slot < self.slots:
            raise IndexError(f"slot {slot} of {self.slots}")
        return slot

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, slot: int) -> int:
        return self._len[self._slot(slot)]

    def table(self, slot: int) -> list[int]:
        """The slot's pages, in the order of its positions."""
        return list(self._table[self._slot(slot)])

    def _copy(self, src: list[int], dst: list[int]) -> None:
        copy_pages(self.k + self.v, src, dst)
        if self.dtype == _E4M3:
            copy_pages(self.scales, src, dst)

    def _drop(self, page: int) -> None:
        self._shared[page] -= 1
        if self._shared[page] == 0:
            heapq.heappush(self._free, page)

    def reserve(self, slots, n) -> None:
        """Room for ``n`` more positions in each slot (one number or one per
        slot), counted in its length: a last page that is partly filled and
        shared is copied first, so that what is inserted reaches no other slot."""
        slots = [self._slot(s) for s in slots]
        n = [n] * len(slots) if isinstance(n, int) else list(n)
        if len(n) != len(slots) or len(set(slots)) != len(slots):
            raise ValueError("one count per slot, each slot once")
        if any(m < 0 for m in n):
            raise ValueError("counts must not be negative")
        S = self.page_size
        need, left, plan = 0, {}, []
        for s, m in zip(slots, n):
            total = -(-(self._len[s] + m) // S)
            if total > self.max_pages:
                raise ValueError(f"slot {s}: {self._len[s] + m} positions, its table holds {self.max_pages * S}")
            more, copied = total - len(self._table[s]), False
            if m and self._len[s] % S:
                last = self._table[s][-1]
                left[last] = left.get(last, self._shared[last]) - 1
                copied = left[last] > 0  # the last to write keeps the page
            if copied or more:
                plan.append((self._table[s], copied, more))
                need += copied + more
        if need > len(self._free):
            raise MemoryError(f"{need} pages needed, {len(self._free)} free")
        taken = [heapq.heappop(self._free) for _ in range(need)]
        src, dst, at = [], [], 0  # (a slot's copy, then the pages it grows by)
        for t, copied, more in plan:
            if copied:
                src.append(t[-1])
                dst.append(taken[at])
            at += copied + more
        if src:
            try:
                self._copy(src, dst)
            except BaseException:
                for p in taken:
                    heapq.heappush(self._free, p)
                raise
        for p in src:
            self._shared[p] -= 1
        for p in taken:
            self._shared[p] = 1
        at = 0
        for t, copied, more in plan:
            if copied:
                t.pop()
            t += taken[at:at + copied + more]
            at += copied + more
        for s, m in zip(slots, n):
            self._len[s] += m

    def fork(self, src: int, dst: int) -> None:
        """``dst`` (empty) gets the positions of ``src``: its pages, shared until
        one of the two extends into them."""
        src, dst = self._slot(src), self._slot(dst)
        if self._table[dst] or src == dst:
            raise ValueError(f"slot {dst} is in use")
        self._table[dst] = list(self._table[src])
        self._len[dst] = self._len[src]
        for p in self._table[dst]:
            self._shared[p] += 1

    def truncate(self, slot: int, length: int) -> None:
        """Only the first ``length`` positions stay (rejected drafts go)."""
        slot = self._slot(slot)
        if not 0 <= length <= self._len[slot]:
            raise ValueError(f"slot {slot} holds {self._len[slot]} positions, not {length}")
        keep = -(-length // self.page_size)
        for p in self._table[slot][keep:]:
            self._drop(p)
        del self._table[slot][keep:]
        self._len[slot] = length

    def free(self, slot: int) -> None:
        self.truncate(slot, 0)

    def compact(self) -> int:
        """Every page in use into the lowest numbers; returns how many moved."""
        used = [p for p in range(self.pages) if self._shared[p]]
        n = len(used)
        src = [p for p in used if p >= n]
        dst = [p for p in range(n) if not self._shared[p]]
        if not src:
            return 0
        self._copy(src, dst)
        to = dict(zip(src, dst))
        for t in self._table:
            t[:] = [to.get(p, p) for p in t]
        for a, b in to.items():
            self._shared[b], self._shared[a] = self._shared[a], 0
        self._free = list(range(n, self.pages))
        return len(src)

    def batch(self, slots, n):
        """(page_table, q_start, kv_len) on the device for a packed batch of the
        last ``n`` positions (one number or one per slot) of each slot."""
        slots = [self._slot(s) for s in slots]
        n = [n] * len(slots) if isinstance(n, int) else list(n)
        if len(n) != len(slots) or len(set(slots)) != len(slots):
            raise ValueError("one count per slot, each slot once")
        for s, m in zip(slots, n):
            if not 0 <= m <= self._len[s]:
                raise ValueError(f"slot {s} holds {self._len[s]} positions, not {m} new ones")
        B = len(slots)
        host = torch.full((B * self.max_pages + 2 * B + 1,), -1, dtype=torch.int32)
        a = host.numpy()
        for i, s in enumerate(slots):
            a[i * self.max_pages:i * self.max_pages + len(self._table[s])] = self._table[s]
        a[B * self.max_pages] = 0
        a[B * self.max_pages + 1:B * self.max_pages + 1 + B] = np.cumsum(n)
        a[B * self.max_pages + 1 + B:] = [self._len[s] for s in slots]
        d = host.to(self.device)
        t, q, k = d.split([B * self.max_pages, B + 1, B])
        return t.view(B, self.max_pages), q, k

    def shared(self, slots):
        """(group_start, shared_len) on the device for ``attention_shared_paged`` of a
        batch of these slots in this order: neighbours that have their first pages
        in common, grouped so that the fewest pages are read. They hold until a
        slot is forked, truncated, freed or its last shared page copied."""
        slots = [self._slot(s) for s in slots]
        if len(set(slots)) != len(slots):
            raise ValueError("each slot once")
        B, S = len(slots), self.page_size
        common = []  # whole pages that neighbours share
        for a, b in zip(slots, slots[1:]):
            ta, tb = self._table[a], self._table[b]
            most = min(self._len[a], self._len[b]) // S
            lo, hi = 0, min(most, len(ta), len(tb))
            if ta[:hi] != tb[:hi]:
                while lo + 1 < hi:  # ta[:lo] == tb[:lo], ta[:hi] != tb[:hi]
                    mid = (lo + hi) // 2
                    lo, hi = (mid, hi) if ta[:mid] == tb[:mid] else (lo, mid)
                hi = lo
            common.append(hi)
        # best[j]: (pages not read again among the first j slots, first slot of the last group, its shared pages)
        best = [(0, 0, 0)]
        for j in range(1, B + 1):
            least, top = None, (best[j - 1][0], j - 1, 0)
            for i in range(j - 2, -1, -1):
                least = common[i] if least is None else min(least, common[i])
                if least == 0:
                    break
                top = max(top, (best[i][0] + (j - 1 - i) * least, i, least), key=lambda v: v[0])
            best.append(top)
        start, length, j = [B], [], B
        while j:
            _, i, pages = best[j]
            start.append(i)
            length.append(pages * S)
            j = i
        host = torch.tensor(start[::-1] + length[::-1], dtype=torch.int32)
        return host.to(self.device).split([len(start), len(length)])

"""Batches over 8-bit and bfloat16 pages whose sequences may share their first
pages, and plain forms in 64 bits, for the tests."""
import math

import numpy as np
import torch

import paged_ref as R

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def code_values():
    """What the 256 e4m3 codes stand for."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, (1 + m / 8.0) * 2.0 ** (e - 7), m / 8.0 * 2.0 ** -6)
    v = np.where((c & 127) == 127, math.nan, v)
    return np.where(c >= 128, -v, v)


def encode(x):
    """(codes, biased exponents) uint8 of (..., D) values: the definition, by search in 64 bits."""
    x = x.double().cpu().numpy()
    fine = np.isfinite(x)
    top = np.max(np.where(fine, np.abs(x), 0.0), -1)
    e = np.full(top.shape, -126)
    for k in range(-126, 128):  # the smallest that is enough
        e = np.where((top > 448 * 2.0 ** (k - 1)), np.maximum(k, -126), e)
    y = np.where(fine, np.abs(x), 0.0) / 2.0 ** e[..., None]
    v = code_values()[:127]
    hi = np.clip(np.searchsorted(v, y), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = y - v[lo], v[hi] - y
    c = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    c = np.where(np.signbit(x), c + 128, c)
    c = np.where(fine, c, 127)
    return torch.from_numpy(c.astype(np.uint8)), torch.from_numpy((e + 127).astype(np.uint8))


def decode(codes, powers):
    v = torch.from_numpy(code_values())[codes.long()]
    return torch.ldexp(v, (powers.double() - 127)[..., None])


class Batch:
    """Sequences of `n` new rows and `total` positions. groups: (sequences, shared positions) of each group, whose
    first one owns the shared pages; the others' table entries for them are no pages. Slots that no sequence holds
    are NaN (8-bit ones with any power); k[b], v[b] are (total, kv_heads, D) float64."""

    def __init__(self, n, total, *, kv_heads, D, page, dev, bits=8, groups=(), seed=0, extra_rows=0, spare=3, width=None):
        g = torch.Generator().manual_seed(seed)
        B = len(n)
        self.n, self.total, self.page, self.kv_heads, self.D, self.dev, self.bits = n, total, page, kv_heads, D, dev, bits
        leader, shared, start, length = list(range(B)), [0] * B, [0], []
        for count, s in groups:
            b0 = start[-1]
            for b in range(b0, b0 + count):
                leader[b], shared[b] = b0, min(s, total[b0]) // page * page
            start.append(b0 + count)
            length.append(s)
        # (a sequence shorter than what its group shares reads no further than it has)
        self.shared, self.leader = shared, leader
        mine = [t if leader[b] == b else max(0, t - shared[b]) for b, t in enumerate(total)]
        need = [-(-t // page) for t in mine]
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=g).tolist()
        width = width or max(max(-(-t // page) for t in total), 1) + 1
        table = torch.full((B, width), -1, dtype=torch.int32)
        shape = (self.pages, kv_heads, page, D)
        kp, vp = torch.full(shape, math.nan), torch.full(shape, math.nan)
        powers = torch.randint(0, 256, (*shape[:3], 2), generator=g, dtype=torch.uint8)
        kc, vc = (torch.full(shape, 127, dtype=torch.uint8) for _ in range(2))
        self.k, self.v = [], []
        for b, t in enumerate(total):
            both = []
            for pool, codes, i in ((kp, kc, 0), (vp, vc, 1)):
                x = torch.randn(mine[b], kv_heads, D, generator=g) * torch.exp(0.5 * torch.randn(mine[b], kv_heads, 1, generator=g))
                x = x.bfloat16()
                if bits == 8:
                    c, e = encode(x)
                    x = decode(c, e)
                else:
                    c = e = None
                    x = x.double()
                both.append((x, c, e))
            first = 0 if leader[b] == b else shared[b] // page
            for j in range(need[b]):
                p = order.pop()
                table[b, first + j] = p
                a, z = j * page, min(mine[b], (j + 1) * page)
                for (x, c, e), pool, codes, i in ((both[0], kp, kc, 0), (both[1], vp, vc, 1)):
                    pool[p, :, :z - a] = x[a:z].float().transpose(0, 1)
                    if bits == 8:
                        codes[p, :, :z - a] = c[a:z].transpose(0, 1)
                        powers[p, :, :z - a, i] = e[a:z].transpose(0, 1)
            if leader[b] != b:
                table[b, :first] = (-1, self.pages, 2 ** 31 - 1)[b % 3]
                pre = min(t, shared[b])
                self.k.append(torch.cat([self.k[leader[b]][:pre], both[0][0]]))
                self.v.append(torch.cat([self.v[leader[b]][:pre], both[1][0]]))
            else:
                self.k.append(both[0][0])
                self.v.append(both[1][0])
        if bits == 8:
            self.kp, self.vp, self.scales = kc.to(dev).view(E4M3), vc.to(dev).view(E4M3), powers.to(dev).view(E8M0)
        else:
            self.kp, self.vp, self.scales = kp.bfloat16().to(dev), vp.bfloat16().to(dev), None
        self.table = table.to(dev)
        at = np.concatenate([[0], np.cumsum(n)])
        i32 = dict(dtype=torch.int32, device=dev)
        self.q_start, self.kv_len = torch.tensor(at, **i32), torch.tensor(total, **i32)
        self.group_start, self.shared_len = torch.tensor(start, **i32), torch.tensor(length, **i32)
        self.T = int(at[-1]) + extra_rows

    def put(self, b, p, k=None, v=None):
        """One position's k or v in the pool and in the plain copies of all that share it: a value, exact in its type."""
        at = self.leader[b] if p < self.shared[b] else b
        page, slot = int(self.table[at, p // self.page]), p % self.page
        for val, pool, plain, i in ((k, self.kp, self.k, 0), (v, self.vp, self.v, 1)):
            if val is None:
                continue
            if self.bits == 8:
                code = 127 if not math.isfinite(val) else int(encode(torch.tensor([[float(val)]]))[0])
                pool.view(torch.uint8)[page, :, slot] = code
                if math.isfinite(val):
                    self.scales.view(torch.uint8)[page, :, slot, i] = int(encode(torch.tensor([[float(val)]]))[1])
                val = val if math.isfinite(val) else math.nan
            else:
                pool[page, :, slot] = val
            for c in range(len(self.n)):
                if c == at or self.leader[c] == at and p < self.shared[c]:
                    if p < self.total[c]:
                        plain[c][p] = val

    def args(self):
        return self.kp, self.vp, self.table, self.q_start, self.kv_len

    def groups(self):
        return self.group_start, self.shared_len


def attention(q, batch, heads, window=0, sinks=0, scale=1.0, missing=()):
    """paged_ref's attention and tolerance. What a group shares is joined to a row's own part by one more factor,
    two products and a sum in float32 (and the factor's own two roundings): 8 of them cover it."""
    want, tol = R.attention(q, batch, heads, window, sinks, scale, missing)
    if any(batch.shared):
        tol = tol + 8 * R.F32 * (want.abs() + tol / R.BF16)
    return want, tol


def adjust(logits, tokens=None, n_tokens=None, n_prompt=None, repetition=1.0, frequency=0.0, presence=0.0,
           bias_tokens=None, bias=None, allowed=None):
    """One row in float64, and where it is more than the logit itself."""
    x = logits.double().cpu().numpy().copy()
    V, f32 = len(x), lambda v: float(np.float32(v))
    touched = np.zeros(V, bool)
    with np.errstate(all="ignore"):
        if tokens is not None:
            t = np.asarray(tokens)[:n_tokens]
            made = t[n_prompt or 0:]
            t, made = t[(t >= 0) & (t < V)], made[(made >= 0) & (made < V)]
            once = np.unique(t)
            r = f32(repetition)
            x[once] = np.where(x[once] > 0, x[once] / r, x[once] * r)
            touched[once] = True
            c = np.bincount(made, minlength=V)
            x -= np.where(c > 0, f32(frequency) * c + f32(presence), 0.0)
        if bias is not None:
            for i, v in zip(np.asarray(bias_tokens).tolist(), np.asarray(bias, dtype=np.float64).tolist()):
                if 0 <= i < V:
                    x[i] += v
                    touched[i] = True
        if allowed is not None:
            words = np.asarray(allowed).view(np.uint32)
            ok = (words[np.arange(V) >> 5] >> (np.arange(V) & 31).astype(np.uint32)) & 1
            x[ok == 0] = -math.inf
    return torch.from_numpy(x), torch.from_numpy(touched)

"""Plain 64-bit forms of the paged operators and of sampling, for the tests."""
import math

import numpy as np
import torch

BF16 = 2.0 ** -8   # a bf16 rounding, relative to the value (half a step)
F32 = 2.0 ** -24


class Batch:
    """Sequences of `n` new rows and `total` positions over shuffled pages. Every
    slot that no sequence holds is NaN; k[b], v[b] are (total, kv_heads, D)."""

    def __init__(self, n, total, *, kv_heads, D, page, dev, seed=0, extra_rows=0, spare=3, width=None):
        g = torch.Generator().manual_seed(seed)
        self.n, self.total, self.page, self.kv_heads, self.D, self.dev = n, total, page, kv_heads, D, dev
        need = [-(-t // page) for t in total]
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=g).tolist()
        width = width or max(max(need), 1) + 1
        table = torch.full((len(n), width), -1, dtype=torch.int32)
        shape = (self.pages, kv_heads, page, D)
        kp, vp = torch.full(shape, math.nan), torch.full(shape, math.nan)
        self.k, self.v = [], []
        for b, t in enumerate(total):
            k = torch.randn(t, kv_heads, D, generator=g).bfloat16()
            v = torch.randn(t, kv_heads, D, generator=g).bfloat16()
            self.k.append(k.double())
            self.v.append(v.double())
            for j in range(need[b]):
                p = order.pop()
                table[b, j] = p
                m = min(page, t - j * page)
                kp[p, :, :m] = k[j * page:j * page + m].float().transpose(0, 1)
                vp[p, :, :m] = v[j * page:j * page + m].float().transpose(0, 1)
        self.kp, self.vp = kp.bfloat16().to(dev), vp.bfloat16().to(dev)
        self.table = table.to(dev)
        start = np.concatenate([[0], np.cumsum(n)])
        self.q_start = torch.tensor(start, dtype=torch.int32, device=dev)
        self.kv_len = torch.tensor(total, dtype=torch.int32, device=dev)
        self.T = int(start[-1]) + extra_rows

    def put(self, b, p, k=None, v=None):
        """One position's k or v in the pool and in the plain copy."""
        page, slot = int(self.table[b, p // self.page]), p % self.page
        for val, pool, plain in ((k, self.kp, self.k), (v, self.vp, self.v)):
            if val is not None:
                pool[page, :, slot] = val
                plain[b][p] = val

    def args(self):
        return self.kp, self.vp, self.table, self.q_start, self.kv_len


def visible(L, n, window, sinks):
    p, t = np.arange(L)[None], np.arange(L - n, L)[:, None]
    m = p <= t
    if window:
        m &= (p > t - window) | (p < sinks)
    return torch.from_numpy(m)


def attention(q, batch, heads, window=0, sinks=0, scale=1.0, missing=()):
    """(out, tolerance) float64 (rows of the sequences, heads, D).

    Tolerance: the kernel multiplies weights rounded to bf16 and may add up the
    rounded ones, 2 roundings of each relative to sum w |v|; the output's own
    rounding; float32 scores, whose error (D + 2 products and sums, a scale, a
    difference and the exponential) multiplies each weight."""
    g = heads // batch.kv_heads
    outs, tols = [], []
    at = 0
    for b, (n, L) in enumerate(zip(batch.n, batch.total)):
        m = visible(L, n, window, sinks)
        for (mb, mp) in missing:
            if mb == b:
                m[:, mp * batch.page:(mp + 1) * batch.page] = False
        o = torch.zeros(n, heads, batch.D, dtype=torch.float64)
        tol = torch.zeros_like(o)
        for h in range(heads):
            k, v = batch.k[b][:, h // g], batch.v[b][:, h // g]
            x = q[at:at + n].view(n, heads, batch.D)[:, h].double().cpu()
            for i in range(n):
                idx = m[i].nonzero()[:, 0]
                if len(idx) == 0:
                    continue
                kk, vv = k[idx], v[idx]
                s = (kk @ x[i]) * scale
                ds = float((kk.abs() @ x[i].abs()).max()) * scale * (batch.D + 8) * F32 + 4 * F32
                w = torch.softmax(s, 0)
                o[i, h] = w @ vv
                a = w @ vv.abs()
                # (len + 4 float32 roundings of the sums, as many again for what chunks are joined by)
                tol[i, h] = BF16 * o[i, h].abs() + (2 * BF16 + 2 * ds + 2 * (len(idx) + 4) * F32) * a + 1e-30
        outs.append(o)
        tols.append(tol)
        at += n
    return torch.cat(outs), torch.cat(tols)


def post(qkv, batch, pos, *, heads, k_off, v_off, q_w, k_w, norm, eps, rope, half, cos_off, sin_off):
    """One row's (q, k, v) float64 (heads, D) before their last rounding and the
    size that roundings on the way are relative to."""
    D, K = batch.D, batch.kv_heads
    x = qkv.double().cpu()

    def rms(t, w):
        y = t / torch.sqrt(t.square().mean(-1, keepdim=True) + eps)
        return (y if w is None else y * w.double().cpu()).bfloat16().double()

    q = x[:heads * D].view(heads, D)
    k = x[k_off:k_off + K * D].view(K, D)
    v = k if v_off < 0 else x[v_off:v_off + K * D].view(K, D)
    q = rms(q, q_w) if norm[0] else q
    k = rms(k, k_w) if norm[1] else k
    v = rms(v, None) if norm[2] else v

    def rot(t):
        if rope is None:
            return t
        r = rope[pos].double().cpu()
        c, s = r[cos_off:cos_off + half], r[sin_off:sin_off + half]
        y = t.clone()
        y[:, :half] = t[:, :half] * c - t[:, half:2 * half] * s
        y[:, half:2 * half] = t[:, half:2 * half] * c + t[:, :half] * s
        return y

    return rot(q), rot(k), v


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, probability) of one row, as alv_sample defines it."""
    l = logits.double().cpu().numpy()
    if np.isnan(l).any():
        return int(np.argmax(np.isnan(l))), math.nan
    order = np.lexsort((np.arange(len(l)), -l))
    top = l[order[0]]
    if top == -math.inf:
        return -1, 0.0
    n = len(l)
    f32 = lambda v: float(np.float32(v))  # noqa: E731
    T = f32(temperature)
    if not T > 0:
        n = 1
        T = 1.0
    elif top_k > 0:
        n = min(n, top_k)
    with np.errstate(invalid="ignore"):
        x = np.where(l[order] == top, 0.0, (l[order] - top) / T)
    w = np.exp(x[:n])
    if f32(top_p) < 1:
        c = np.cumsum(w)
        n = max(1, int((c - w < max(f32(top_p), 0.0) * w.sum()).sum()))
    n = max(1, min(n, int((w >= min(f32(min_p), 1.0)).sum()))) if min_p > 0 else n
    c = np.cumsum(w[:n])
    uu = min(max(f32(u), 0.0), 1 - 2.0 ** -24)
    r = min(int((c <= uu * c[-1]).sum()), int((w[:n] > 0).sum()) - 1)
    return int(order[r]), w[r] / c[-1]

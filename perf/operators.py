"""The measured work of the serving operators: paged attention, paged q/k/v
post-processing, page copies, sampling.

Kinds (``case["kind"]``):

``attend``  attention of the newest tokens of a batch of sequences over a paged
            KV cache (``paged.attention_paged``).
``post``    q/k norms, RoPE and the insert of new tokens into their pages
            (``paged.qkv_post_paged``).
``copy``    pages copied in every layer's caches (``paged.copy_pages``).
``sample``  one token per row of logits from a given uniform number
            (``sample``).

Head layouts are those of the package's layers (Gemma-4 12B sliding and global,
Gemma-3 1B, Llama-3.2 1B) and generic ones.

Sequence b owns rows ``q_start[b] .. q_start[b + 1]`` of the packed batch; they
are the last of its ``kv_len[b]`` positions. Position p is slot p % S of page
``page_table[b][p // S]``; pages are (page, kv head, slot, column).
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False
DEV = "cuda"

SLIDING = {"heads": 16, "kv_heads": 8, "D": 256}  # Gemma-4 12B sliding layer
GLOBAL = {"heads": 16, "kv_heads": 1, "D": 512}   # Gemma-4 12B global layer
GEMMA1 = {"heads": 4, "kv_heads": 1, "D": 256}    # Gemma-3 1B
LLAMA1 = {"heads": 32, "kv_heads": 8, "D": 64}    # Llama-3.2 1B


# ---- cases -----------------------------------------------------------------------

def listed():
    return [
        # One sequence's next token in a sliding layer: latency of the call.
        {"name": "attend_decode_one", "kind": "attend", **SLIDING, "B": 1, "n_lo": 1, "n_hi": 1, "past_lo": 1500,
         "past_hi": 1500, "page": 16, "window": 1024, "sinks": 0},
        # A decode batch of ragged lengths, one token each: the cache's bytes.
        {"name": "attend_decode_batch", "kind": "attend", **LLAMA1, "B": 64, "n_lo": 1, "n_hi": 1, "past_lo": 100,
         "past_hi": 8000, "page": 64, "window": 0, "sinks": 0},
        # Drafted tokens verified over long contexts in a global layer.
        {"name": "attend_verify_long", "kind": "attend", **GLOBAL, "B": 4, "n_lo": 5, "n_hi": 5, "past_lo": 20011,
         "past_hi": 40009, "page": 128, "window": 0, "sinks": 0},
        # Prompt chunks of several sequences in a sliding layer whose first tokens stay visible.
        {"name": "attend_chunks_sliding", "kind": "attend", **SLIDING, "B": 3, "n_lo": 333, "n_hi": 1201, "past_lo": 0,
         "past_hi": 2500, "page": 32, "window": 1024, "sinks": 4},
        # A long prompt in a global layer, the largest attention here.
        {"name": "attend_prompt_global", "kind": "attend", **GLOBAL, "B": 1, "n_lo": 4096, "n_hi": 4096, "past_lo": 0,
         "past_hi": 0, "page": 64, "window": 0, "sinks": 0},
        # The new token of eight sequences into the cache.
        {"name": "post_decode8", "kind": "post", **SLIDING, "B": 8, "n_lo": 1, "n_hi": 1, "past_lo": 10,
         "past_hi": 3000, "page": 16, "norm_v": True, "rotated": 256},
        # A ragged prompt chunk into the cache.
        {"name": "post_chunk", "kind": "post", **SLIDING, "B": 3, "n_lo": 901, "n_hi": 2003, "past_lo": 0,
         "past_hi": 1000, "page": 64, "norm_v": True, "rotated": 256},
        # One row of logits, as after a decode step.
        {"name": "sample_one", "kind": "sample", "B": 1, "vocab": 262144, "temp": "0.8", "top_k": "64",
         "top_p": "0.95", "min_p": "0.0"},
        # A batch whose rows ask for different things (greedy among them).
        {"name": "sample_mixed", "kind": "sample", "B": 48, "vocab": 128256, "temp": "0.7,1.0,0.0,1.3",
         "top_k": "50,0,0,1000,0", "top_p": "0.9,1.0,0.95", "min_p": "0.0,0.05"},
        # Nucleus alone over a full vocabulary: no cut by count.
        {"name": "sample_nucleus", "kind": "sample", "B": 16, "vocab": 262144, "temp": "1.0", "top_k": "0",
         "top_p": "0.92", "min_p": "0.0"},
        # Partly filled last pages of forked sequences, in twelve layers' caches.
        {"name": "copy_fork", "kind": "copy", "caches": 24, "pages": 300, "kv_heads": 8, "page": 16, "D": 256,
         "pairs": 6},
        # A pool compacted: most of a small model's cache moves.
        {"name": "copy_compact", "kind": "copy", "caches": 32, "pages": 1024, "kv_heads": 8, "page": 64, "D": 64,
         "pairs": 450},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "post", "sample", "sample", "copy"])
    if kind in ("attend", "post"):
        D = rng.choice([64, 128, 256, 512])
        kv = rng.choice([1, 2, 4, 8])
        lay = rng.choice([SLIDING, GLOBAL, GEMMA1, LLAMA1, {"heads": kv * rng.choice([1, 2, 3, 4, 8]), "kv_heads": kv,
                                                            "D": D}])
        shape = rng.choice(["decode", "verify", "chunk"])
        if shape == "decode":
            c = {"B": _log(rng, 1, 64), "n_lo": 1, "n_hi": 1, "past_lo": 0, "past_hi": _log(rng, 16, 8000)}
        elif shape == "verify":
            n = rng.randint(2, 9)
            c = {"B": _log(rng, 1, 16), "n_lo": rng.choice([n, 0]), "n_hi": n, "past_lo": rng.randint(0, 20),
                 "past_hi": _log(rng, 64, 16000)}
        else:
            n = _log(rng, 17, 2048)
            c = {"B": rng.randint(1, 3), "n_lo": rng.randint(0, n), "n_hi": n, "past_lo": 0,
                 "past_hi": _log(rng, 1, 2048)}
        c = {"kind": kind, **lay, **c, "page": rng.choice([16, 32, 64, 128]), "window": 0, "sinks": 0}
        while _visible(c)[0] * c["heads"] * c["D"] > 6e10 or sum(_lens(c)[1]) * c["kv_heads"] * c["D"] > 4e8:
            c["n_hi"], c["past_hi"] = (c["n_hi"] + 1) // 2, c["past_hi"] // 2
            c["n_lo"], c["past_lo"] = min(c["n_lo"], c["n_hi"]), min(c["past_lo"], c["past_hi"])
        if kind == "attend":
            window = rng.choice([0, 0, 512, 1024, rng.randint(1, 2000)])
            return {**c, "window": window, "sinks": rng.choice([0, 1, 4]) if window else 0}
        del c["window"], c["sinks"]
        return {**c, "norm_v": rng.random() < 0.5, "rotated": rng.choice([c["D"], c["D"] // 4])}
    if kind == "sample":
        vocab = rng.choice([32000, 128256, 262144, rng.randint(1000, 262144)])
        pick = lambda *v: ",".join(str(rng.choice(v)) for _ in range(rng.randint(1, 5)))  # noqa: E731
        return {"kind": kind, "B": _log(rng, 1, 48 if vocab < 200000 else 24), "vocab": vocab,
                "temp": pick(0.0, 0.3, 0.7, 1.0, 1.5), "top_k": pick(0, 0, 1, 40, 500, 20000),
                "top_p": pick(1.0, 1.0, 0.5, 0.9, 0.99), "min_p": pick(0.0, 0.0, 0.02, 0.2)}
    page, D, kv_heads = rng.choice([16, 32, 64, 128]), rng.choice([64, 128, 256, 512]), rng.choice([1, 2, 4, 8])
    caches = 2 * rng.randint(1, 16)
    pages = max(8, min(1024, (1 << 29) // (caches * kv_heads * page * D)))
    return {"kind": kind, "caches": caches, "pages": pages, "kv_heads": kv_heads, "page": page, "D": D,
            "pairs": _log(rng, 1, pages // 2)}


# ---- inputs ----------------------------------------------------------------------

def _lens(case):
    """Rows and earlier positions of every sequence: part of the case, the same for every seed. The first
    sequence has the most of both."""
    rng = random.Random(case["past_hi"] * 1009 + case["n_hi"] * 31 + case["B"])
    n = [rng.randint(case["n_lo"], case["n_hi"]) for _ in range(case["B"])]
    past = [rng.randint(min(case["past_lo"], case["past_hi"]), case["past_hi"]) for _ in range(case["B"])]
    n[0], past[0] = case["n_hi"], case["past_hi"]
    return n, [a + b for a, b in zip(n, past)]


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _paged(case, g):
    """Page pools of earlier tokens' k and v (stale values in free slots), and the batch's tables."""
    n, total = _lens(case)
    S = case["page"]
    need = [(t + S - 1) // S for t in total]
    width = max(max(need), 1) + 2
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((case["B"], width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = order[at:at + m]
        at += m
    shape = (pages, case["kv_heads"], S, case["D"])
    start = [0]
    for v in n:
        start.append(start[-1] + v)
    return {"kpages": torch.randn(shape, generator=g, device=DEV).to(torch.bfloat16),
            "vpages": torch.randn(shape, generator=g, device=DEV).to(torch.bfloat16),
            "table": table, "q_start": _i32(start), "kv_len": _i32(total), "n": n, "total": total}


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind = case["kind"]
    st = {"case": case}
    if kind == "attend":
        st.update(_paged(case, g))
        T, D = sum(st["n"]), case["D"]
        # scores of a standard deviation of 2: some positions matter, none alone
        st["q"] = (torch.randn(T, case["heads"] * D, generator=g, device=DEV) * 2).to(torch.bfloat16)
        st["scale"] = 1.0 / math.sqrt(D)
        return st
    if kind == "post":
        st.update(_paged(case, g))
        T, D, S = sum(st["n"]), case["D"], case["heads"] * case["D"]
        K = case["kv_heads"] * D
        st["qkv"] = (torch.randn(T, S + 2 * K, generator=g, device=DEV) * 1.5).to(torch.bfloat16)
        st["q_w"] = 1 + 0.3 * torch.randn(D, generator=g, device=DEV)
        st["k_w"] = 1 + 0.3 * torch.randn(D, generator=g, device=DEV)
        # rows [cos | sin] of the first rotated / 2 angles, in the table's bf16
        half = case["rotated"] // 2
        rows = max(max(st["total"]), 1)
        freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
        ang = torch.arange(rows, dtype=torch.float64, device=DEV)[:, None] * freq
        st["rope"] = torch.cat([ang.cos(), ang.sin()], 1).to(torch.bfloat16)
        return st
    if kind == "sample":
        B, V = case["B"], case["vocab"]
        # a softcapped head's logits: a broad body and a few tokens that stand out
        x = torch.randn(B, V, generator=g, device=DEV) * 2
        top = torch.randint(0, V, (B, 40), generator=g, device=DEV)
        x.scatter_add_(1, top, torch.rand(B, 40, generator=g, device=DEV) * 14)
        st["logits"] = 30 * torch.tanh(x / 30)
        st["u"] = torch.rand(B, generator=g, device=DEV)
        # the rows take the case's values in turn
        for name in ("temp", "top_k", "top_p", "min_p"):
            v = case[name].split(",")
            v = [float(v[i % len(v)]) for i in range(B)]
            st[name] = torch.tensor(v, dtype=torch.int32 if name == "top_k" else torch.float32, device=DEV)
        return st
    shape = (case["caches"], case["pages"], case["kv_heads"], case["page"], case["D"])
    st["pool"] = torch.empty(shape, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    st["caches"] = list(st["pool"].unbind(0))
    perm = torch.randperm(case["pages"], generator=g, device=DEV).tolist()
    st["src"], st["dst"] = perm[:case["pairs"]], perm[case["pairs"]:2 * case["pairs"]]
    return st


# ---- one pass --------------------------------------------------------------------

def run(st):
    if own:
        return _run_own(st)
    return {"attend": _attend, "post": _post, "sample": _sample, "copy": _copy}[st["case"]["kind"]](st)


def _run_own(st):
    import alveare_amd as aa
    from alveare_amd import paged

    c = st["case"]
    if c["kind"] == "attend":
        return {"out": paged.attention_paged(st["q"], st["kpages"], st["vpages"], st["table"], st["q_start"],
                                             st["kv_len"], heads=c["heads"], window=c["window"], sinks=c["sinks"],
                                             scale=st["scale"], max_q=c["n_hi"])}
    if c["kind"] == "post":
        q, k = c["heads"] * c["D"], c["kv_heads"] * c["D"]
        out = paged.qkv_post_paged(st["qkv"], st["kpages"], st["vpages"], st["table"], st["q_start"], st["kv_len"],
                                   heads=c["heads"], k_off=q, v_off=q + k, q_w=st["q_w"], k_w=st["k_w"],
                                   norm_v=c["norm_v"], rope=st["rope"])
        return {"q": out, "kpages": st["kpages"], "vpages": st["vpages"]}
    if c["kind"] == "sample":
        token, prob = aa.sample(st["logits"], st["u"], temperature=st["temp"], top_k=st["top_k"], top_p=st["top_p"],
                                min_p=st["min_p"])
        return {"token": token, "prob": prob}
    paged.copy_pages(st["caches"], st["src"], st["dst"])
    return {"pool": st["pool"]}


# ---- the plain forms -------------------------------------------------------------

def _rows(st):
    """Packed row of (sequence, i) for i below the longest chunk, its position, and whether it exists."""
    first, n = st["q_start"][:-1].long(), st["q_start"].diff().long()
    i = torch.arange(max(st["n"]), device=DEV)
    there = i < n[:, None]
    return torch.where(there, first[:, None] + i, 0), (st["kv_len"].long() - n)[:, None] + i, there


def _attend(st):
    c = st["case"]
    B, S, D, H, g = c["B"], c["page"], c["D"], c["kv_heads"], c["heads"] // c["kv_heads"]
    longest = max(st["total"])
    rows, pos, there = _rows(st)
    width = (longest + S - 1) // S
    page = st["table"][:, :width].long()
    k = st["kpages"][page.clamp(min=0)].float().permute(0, 2, 1, 3, 4).reshape(B, H, width * S, D)
    v = st["vpages"][page.clamp(min=0)].float().permute(0, 2, 1, 3, 4).reshape(B, H, width * S, D)
    q = st["q"][rows].float().view(B, -1, H, g, D).permute(0, 2, 1, 3, 4).reshape(B, H, -1, D)
    at = torch.arange(width * S, device=DEV)
    seen = (at <= pos[..., None]) & (page >= 0).repeat_interleave(S, 1)[:, None]
    if c["window"]:
        seen &= (at > pos[..., None] - c["window"]) | (at < c["sinks"])
    seen = seen[:, None, :, None].expand(B, H, -1, g, -1).reshape(B, H, -1, width * S)
    s = (q @ k.transpose(2, 3).contiguous()) * st["scale"]
    s = s.masked_fill(~seen, -math.inf)
    m = s.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    e = torch.exp(s - m)
    o = (e @ v) / e.sum(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)
    o = o.view(B, H, -1, g, D).permute(0, 2, 1, 3, 4).reshape(B, -1, c["heads"] * D)
    return {"out": o[there].to(torch.bfloat16)}


def _post(st):
    c = st["case"]
    H, K, D, S = c["heads"], c["kv_heads"], c["D"], c["page"]
    _, pos, there = _rows(st)
    seq = torch.arange(c["B"], device=DEV)[:, None].expand_as(pos)[there]
    pos = pos[there]
    x = st["qkv"].float()
    q, k, v = (t.reshape(len(x), -1, D) for t in x.split([H * D, K * D, K * D], 1))

    def norm(t, w=1.0):
        # the norm's result is a bf16 activation of the layers, as run_rmsnorm returns it
        return (t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w).to(torch.bfloat16).float()

    half = st["rope"].shape[1] // 2
    cos, sin = st["rope"][pos].float()[:, None].split(half, -1)

    def rotate(t):
        a, b, rest = t.split([half, half, D - 2 * half], -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1).to(torch.bfloat16)

    page = st["table"][seq, pos // S].long()
    st["kpages"][page, :, pos % S] = rotate(norm(k, st["k_w"]))
    st["vpages"][page, :, pos % S] = (norm(v) if c["norm_v"] else v).to(torch.bfloat16)
    return {"q": rotate(norm(q, st["q_w"])).reshape(len(x), H * D), "kpages": st["kpages"], "vpages": st["vpages"]}


def _sample(st):
    # 64 bits: a token is chosen by where sums over the vocabulary cross a border
    x, order = torch.sort(st["logits"].double(), dim=1, descending=True, stable=True)
    V = x.shape[1]
    hot = st["temp"] > 0
    t = torch.where(hot, st["temp"], 1).double()[:, None]
    w = torch.exp((x - x[:, :1]) / t)
    rank = torch.arange(V, device=DEV)
    k = torch.where(st["top_k"] > 0, st["top_k"], V)
    k = torch.where(hot, k, 1)[:, None]
    w = torch.where(rank < k, w, 0)
    before = torch.cumsum(w, 1) - w
    keep = (before < st["top_p"].double()[:, None] * w.sum(1, keepdim=True)) | (st["top_p"] >= 1)[:, None]
    keep &= w >= st["min_p"].double()[:, None]
    keep[:, 0] = True
    w = torch.where(keep, w, 0)
    total = torch.cumsum(w, 1)
    z = total[:, -1:]
    r = (total <= st["u"].double()[:, None] * z).sum(1, keepdim=True)
    r = torch.minimum(r, (w > 0).sum(1, keepdim=True) - 1)
    return {"token": order.gather(1, r)[:, 0].to(torch.int32), "prob": (w.gather(1, r) / z)[:, 0].float()}


def _copy(st):
    st["pool"][:, st["dst"]] = st["pool"][:, st["src"]]
    return {"pool": st["pool"]}


# ---- what a pass cannot do without ------------------------------------------------

def _visible(case):
    """Over all sequences: (row, position) pairs that are visible, and positions that some row sees."""
    pairs = union = 0
    for n, total in zip(*_lens(case)):
        if n == 0:
            continue
        t = np.arange(total - n, total)
        w, s = case["window"], case["sinks"]
        lo = np.maximum(t + 1 - w, 0) if w else np.zeros_like(t)
        pairs += int((t + 1 - lo + np.minimum(lo, s)).sum())
        union += total - int(lo[0]) + min(int(lo[0]), s)
    return pairs, union


def work(case):
    kind = case["kind"]
    if kind == "attend":
        pairs, union = _visible(case)
        T, D = sum(_lens(case)[0]), case["D"]
        return {"bytes": 2 * 2 * T * case["heads"] * D + 2 * 2 * union * case["kv_heads"] * D,
                "flops": 4 * pairs * case["heads"] * D}
    if kind == "post":
        T, D = sum(_lens(case)[0]), case["D"]
        values = T * (case["heads"] + 2 * case["kv_heads"]) * D
        return {"bytes": 2 * 2 * values + 2 * T * case["rotated"], "flops": 10 * values}
    if kind == "sample":
        return {"bytes": 4 * case["B"] * case["vocab"], "flops": 4 * case["B"] * case["vocab"]}
    return {"bytes": 2 * 2 * case["caches"] * case["pairs"] * case["kv_heads"] * case["page"] * case["D"], "flops": 0}


# ---- in 64 bits ------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "copy":
        pool = st["pool"].clone()
        for s, d in zip(st["src"], st["dst"]):
            pool[:, d] = st["pool"][:, s]
        return {"pool": pool.double()}
    if kind == "sample":
        return _exact_sample(st)
    D, S, H = case["D"], case["page"], case["kv_heads"]
    if kind == "attend":
        g = case["heads"] // H
        out = torch.empty(sum(st["n"]), case["heads"], D, dtype=torch.float64, device=DEV)
        at = 0
        for b, (n, total) in enumerate(zip(st["n"], st["total"])):
            p = torch.arange(total, device=DEV)
            pages, slots = st["table"][b].long()[p // S], p % S
            for i0 in range(0, n, 512):
                i1 = min(n, i0 + 512)
                t = torch.arange(total - n + i0, total - n + i1, device=DEV)[:, None]
                off = p > t
                if case["window"]:
                    off |= (p <= t - case["window"]) & (p >= case["sinks"])
                for h in range(H):
                    k, v = st["kpages"][pages, h, slots].double(), st["vpages"][pages, h, slots].double()
                    for hq in range(h * g, h * g + g):
                        q = st["q"].view(-1, case["heads"], D)[at + i0:at + i1, hq].double()
                        s = torch.mm(q, k.t()) * st["scale"]
                        out[at + i0:at + i1, hq] = torch.softmax(s.masked_fill(off, -math.inf), 1) @ v
            at += n
        return {"out": out.view(len(out), -1)}
    kp, vp = st["kpages"].double(), st["vpages"].double()
    x = st["qkv"].double().view(-1, case["heads"] + 2 * H, D)
    rms = lambda t: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6)  # noqa: E731
    qk = rms(x[:, :-H])
    qk = torch.cat([qk[:, :-H] * st["q_w"].double(), qk[:, -H:] * st["k_w"].double()], 1)
    qk = qk.to(torch.bfloat16).double()  # the definition's own bf16 between norm and rotation
    v = rms(x[:, -H:]) if case["norm_v"] else x[:, -H:]
    half = case["rotated"] // 2
    at = 0
    for b, (n, total) in enumerate(zip(st["n"], st["total"])):
        p = torch.arange(total - n, total, device=DEV)
        z = torch.complex(st["rope"][p, :half].double(), st["rope"][p, half:].double())[:, None]
        y = torch.complex(qk[at:at + n, :, :half].contiguous(), qk[at:at + n, :, half:2 * half].contiguous()) * z
        qk[at:at + n, :, :half], qk[at:at + n, :, half:2 * half] = y.real, y.imag
        pages, slots = st["table"][b].long()[p // S], p % S
        kp[pages, :, slots], vp[pages, :, slots] = qk[at:at + n, -H:], v[at:at + n]
        at += n
    return {"q": qk[:, :-H].reshape(len(x), -1), "kpages": kp, "vpages": vp}


def _exact_sample(st):
    tokens, probs = [], []
    for b in range(st["case"]["B"]):
        l = st["logits"][b].cpu().numpy().astype(np.float64)
        order = np.lexsort((np.arange(len(l)), -l))
        T, k = float(st["temp"][b]), int(st["top_k"][b])
        n = 1 if T <= 0 else (min(k, len(l)) if k > 0 else len(l))
        w = np.exp((l[order[:n]] - l[order[0]]) / (T if T > 0 else 1.0))
        p = float(st["top_p"][b])
        if p < 1:
            n = min(n, 1 + int(np.searchsorted(np.cumsum(w), p * w.sum(), side="left")))
        n = max(1, min(n, int((w >= float(st["min_p"][b])).sum())))
        c = np.cumsum(w[:n])
        r = min(int(np.searchsorted(c, float(st["u"][b]) * c[-1], side="right")), n - 1)
        tokens.append(int(order[r]))
        probs.append(w[r] / c[-1])
    return {"token": np.array(tokens, np.int32), "prob": np.array(probs, np.float64)}

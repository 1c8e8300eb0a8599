"""The measured work of the operators that a served batch needs beside those of
``perf/operators.py``: a KV cache in 8 bits, attention of sequences that share
their first pages, and what is done to logits before a token is drawn.

Kinds (``case["kind"]``):

``post8``   q/k norms, RoPE and the insert of new tokens into 8-bit pages
            (``paged.qkv_post_paged`` with ``scales``).
``attend8`` attention of the newest tokens over 8-bit pages
            (``paged.attention_paged`` with ``scales``).
``shared``  attention of a batch whose sequences come in groups with the same
            first positions, 8-bit pages or bfloat16
            (``paged.attention_shared_paged``).
``adjust``  penalties for tokens that occurred, biases and the tokens that a
            grammar allows, on rows of logits (``adjust_logits``).

An 8-bit page holds e4m3 codes; position s of kv head h in page p has the two
powers of two ``scales[p, h, s]`` = (k's, v's), and a value is code times power.
The power is the smallest that brings the head's largest magnitude to 448 or
less, 2^-126 at least.

Head layouts are those of the package's layers (Gemma-4 12B sliding and global,
Gemma-3 1B, Llama-3.2 1B) and generic ones. Sequence b owns rows ``q_start[b] ..
q_start[b + 1]`` of the packed batch, the last of its ``kv_len[b]`` positions;
position p is slot p % S of page ``page_table[b][p // S]``. Group j of a shared
batch is the sequences ``group_start[j] .. group_start[j + 1]``, whose first
``shared_len[j]`` positions are the same pages.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False
DEV = "cuda"
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu

SLIDING = {"heads": 16, "kv_heads": 8, "D": 256}  # Gemma-4 12B sliding layer
GLOBAL = {"heads": 16, "kv_heads": 1, "D": 512}   # Gemma-4 12B global layer
GEMMA1 = {"heads": 4, "kv_heads": 1, "D": 256}    # Gemma-3 1B
LLAMA1 = {"heads": 32, "kv_heads": 8, "D": 64}    # Llama-3.2 1B


# ---- cases -----------------------------------------------------------------------

def listed():
    return [
        # The new token of eight sequences into an 8-bit cache: latency of the call.
        {"name": "post8_decode8", "kind": "post8", **SLIDING, "B": 8, "n_lo": 1, "n_hi": 1, "past_lo": 10,
         "past_hi": 3000, "page": 16, "norm_v": True, "rotated": 256},
        # A ragged prompt chunk into an 8-bit cache.
        {"name": "post8_chunk", "kind": "post8", **SLIDING, "B": 3, "n_lo": 901, "n_hi": 2003, "past_lo": 0,
         "past_hi": 1000, "page": 64, "norm_v": True, "rotated": 256},
        # One sequence's next token in a sliding layer: latency of the call.
        {"name": "attend8_decode_one", "kind": "attend8", **SLIDING, "B": 1, "n_lo": 1, "n_hi": 1, "past_lo": 1500,
         "past_hi": 1500, "page": 16, "window": 1024, "sinks": 0},
        # A decode batch of ragged lengths, one token each: the cache's bytes.
        {"name": "attend8_decode_batch", "kind": "attend8", **LLAMA1, "B": 64, "n_lo": 1, "n_hi": 1, "past_lo": 100,
         "past_hi": 8000, "page": 64, "window": 0, "sinks": 0},
        # Drafted tokens verified over long contexts in a global layer.
        {"name": "attend8_verify_long", "kind": "attend8", **GLOBAL, "B": 4, "n_lo": 5, "n_hi": 5, "past_lo": 20011,
         "past_hi": 40009, "page": 128, "window": 0, "sinks": 0},
        # A prompt's later chunk in a global layer: matrix products, the largest attention here.
        {"name": "attend8_prompt", "kind": "attend8", **GLOBAL, "B": 1, "n_lo": 4096, "n_hi": 4096, "past_lo": 2048,
         "past_hi": 2048, "page": 64, "window": 0, "sinks": 0},
        # Eight answers sampled from one prompt.
        {"name": "shared_samples", "kind": "shared", **GEMMA1, "bits": 16, "B": 8, "groups": 1, "share_lo": 4096,
         "share_hi": 4096, "n_lo": 1, "n_hi": 1, "past_lo": 3, "past_hi": 400, "page": 16, "window": 0, "sinks": 0},
        # A decode batch of three system prompts, each with its users.
        {"name": "shared_system", "kind": "shared", **LLAMA1, "bits": 16, "B": 64, "groups": 3, "share_lo": 2000,
         "share_hi": 8000, "n_lo": 1, "n_hi": 1, "past_lo": 20, "past_hi": 1500, "page": 64, "window": 0, "sinks": 0},
        # Drafts of sixteen sequences over one long document, in 8 bits.
        {"name": "shared_document8", "kind": "shared", **GLOBAL, "bits": 8, "B": 16, "groups": 1, "share_lo": 20032,
         "share_hi": 20032, "n_lo": 0, "n_hi": 5, "past_lo": 0, "past_hi": 700, "page": 32, "window": 0, "sinks": 0},
        # One row of logits after a decode step: penalties and a grammar that allows a part of the vocabulary.
        {"name": "adjust_one", "kind": "adjust", "B": 1, "vocab": 262144, "history": 1500, "prompt": 1000, "bias": 10,
         "repetition": "1.1", "frequency": "0.2", "presence": "0.1", "allowed": 0.3, "in_place": False},
        # A batch with long histories; its rows ask for different things.
        {"name": "adjust_batch", "kind": "adjust", "B": 48, "vocab": 128256, "history": 8000, "prompt": 6000,
         "bias": 300, "repetition": "1.0,1.2,1.05", "frequency": "0.0,0.5", "presence": "0.0,0.0,0.4,-0.2",
         "allowed": 0.0, "in_place": False},
        # Grammars alone, few tokens allowed, in the head's own buffer.
        {"name": "adjust_grammar", "kind": "adjust", "B": 64, "vocab": 262144, "history": 0, "prompt": 0, "bias": 0,
         "repetition": "1.0", "frequency": "0.0", "presence": "0.0", "allowed": 0.01, "in_place": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend8", "attend8", "shared", "shared", "post8", "adjust"])
    if kind == "adjust":
        vocab = rng.choice([32000, 128256, 262144, rng.randint(1000, 262144)])
        pick = lambda *v: ",".join(str(rng.choice(v)) for _ in range(rng.randint(1, 5)))  # noqa: E731
        history = rng.choice([0, _log(rng, 1, 16000)])
        mask = rng.choice([0.0, rng.choice([0.001, 0.05, 0.5, 0.97])])
        return {"kind": kind, "B": _log(rng, 1, 64), "vocab": vocab, "history": history,
                "prompt": rng.randint(0, history), "bias": rng.randint(1, 1000) if rng.random() < 0.5 or not history else 0,
                "repetition": pick(1.0, 1.0, 1.02, 1.3, 0.9), "frequency": pick(0.0, 0.0, 0.3, -0.1),
                "presence": pick(0.0, 0.0, 0.6, -0.4), "allowed": mask, "in_place": False}
    D = rng.choice([64, 128, 256, 512])
    kv = rng.choice([1, 2, 4, 8])
    lay = rng.choice([SLIDING, GLOBAL, GEMMA1, LLAMA1, {"heads": kv * rng.choice([1, 2, 3, 4, 8]), "kv_heads": kv,
                                                        "D": D}])
    page = rng.choice([16, 32, 64, 128])
    window = rng.choice([0, 0, 0, 512, 1024, rng.randint(1, 2000)])
    win = {"window": window, "sinks": rng.choice([0, 1, 4]) if window else 0}
    if kind == "shared":
        n = rng.choice([1, 1, 1, rng.randint(2, 9), _log(rng, 10, 200)])
        B = _log(rng, 2, 64 if n < 10 else 8)
        c = {"kind": kind, **lay, "bits": rng.choice([8, 16]), "B": B, "groups": rng.randint(1, max(1, B // 3)),
             "share_lo": rng.choice([0, 16]), "share_hi": _log(rng, 64, 20000), "n_lo": rng.choice([n, 0]), "n_hi": n,
             "past_lo": 0, "past_hi": _log(rng, 1, 2000), "page": page, **win}
        while _cost(c) > 5e10 or sum(_lens(c)[1]) * c["kv_heads"] * c["D"] > 4e8:
            c["share_hi"], c["past_hi"] = (c["share_hi"] + 1) // 2, (c["past_hi"] + 1) // 2
            c["share_lo"] = min(c["share_lo"], c["share_hi"])
        return c
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
    c = {"kind": kind, **lay, **c, "page": page, **win}
    while _cost(c) > 5e10 or sum(_lens(c)[1]) * c["kv_heads"] * c["D"] > 4e8:
        c["n_hi"], c["past_hi"] = (c["n_hi"] + 1) // 2, c["past_hi"] // 2
        c["n_lo"], c["past_lo"] = min(c["n_lo"], c["n_hi"]), min(c["past_lo"], c["past_hi"])
    if kind == "attend8":
        return c
    del c["window"], c["sinks"]
    return {**c, "norm_v": rng.random() < 0.5, "rotated": rng.choice([c["D"], c["D"] // 4])}


# ---- inputs ----------------------------------------------------------------------

def _groups(case):
    """First sequence of every group (and B), and the groups' shared positions, whole pages."""
    if case["kind"] != "shared":
        return list(range(case["B"] + 1)), [0] * case["B"]
    rng = random.Random(case["share_hi"] * 7 + case["B"])
    cuts = [0] + sorted(rng.sample(range(1, case["B"]), case["groups"] - 1)) + [case["B"]]
    S = case["page"]
    return cuts, [rng.randint(case["share_lo"], case["share_hi"]) // S * S for _ in range(case["groups"] - 1)] + [
        case["share_hi"] // S * S]


def _lens(case):
    """Rows, positions and (of these) shared positions of every sequence: part of the case, the same for every
    seed. The first sequence has the most rows and the longest own past."""
    rng = random.Random(case["past_hi"] * 1009 + case["n_hi"] * 31 + case["B"])
    n = [rng.randint(case["n_lo"], case["n_hi"]) for _ in range(case["B"])]
    past = [rng.randint(min(case["past_lo"], case["past_hi"]), case["past_hi"]) for _ in range(case["B"])]
    n[0], past[0] = case["n_hi"], case["past_hi"]
    cuts, share = _groups(case)
    shared = [s for a, b, s in zip(cuts, cuts[1:], share) for _ in range(b - a)]
    return n, [a + b + s for a, b, s in zip(n, past, shared)], shared


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _power(amax):
    """The biased exponent of a head's power of two."""
    m, e = torch.frexp(amax.float())  # 448 = 0.875 * 2^9
    return (e - 9 + (m > 0.875) + 127).clamp(1, 254).to(torch.uint8)


def _encode(x):
    """(codes, biased exponents) of rows of values."""
    e = _power(x.abs().amax(-1))
    return (x.float() * torch.exp2(127.0 - e.float())[..., None]).to(E4M3), e


def _pool(shape, bits, g):
    """Two page pools of earlier tokens' k and v (stale values in free slots), and the powers of 8-bit ones."""
    if bits == 16:
        return [torch.randn(shape, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2)] + [None]
    pools, powers = [], torch.empty((*shape[:3], 2), dtype=torch.uint8, device=DEV)
    for i in range(2):
        codes = torch.empty(shape, dtype=torch.uint8, device=DEV)
        for p0 in range(0, shape[0], 256):  # heads of different sizes
            x = torch.randn((min(256, shape[0] - p0), *shape[1:]), generator=g, device=DEV)
            x *= torch.exp(0.3 * torch.randn(x.shape[:3], generator=g, device=DEV))[..., None]
            c, powers[p0:p0 + 256, ..., i] = _encode(x)
            codes[p0:p0 + 256] = c.view(torch.uint8)
        pools.append(codes.view(E4M3))
    return pools + [powers.view(E8M0)]


def _paged(case, g):
    n, total, shared = _lens(case)
    cuts, _ = _groups(case)
    S = case["page"]
    need = [(t + S - 1) // S for t in total]
    width = max(max(need), 1) + 2
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((case["B"], width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for a, b in zip(cuts, cuts[1:]):
        for i in range(a, b):
            k = shared[i] // S
            if i == a:
                table[i, :need[i]] = order[at:at + need[i]]
                at += need[i]
            else:
                table[i, :k] = table[a, :k]
                table[i, k:need[i]] = order[at:at + need[i] - k]
                at += need[i] - k
    start = [0]
    for v in n:
        start.append(start[-1] + v)
    pools = _pool((max(at, 1) + 3, case["kv_heads"], S, case["D"]), case.get("bits", 8), g)
    # the pool holds no more pages than are used (and three): the table's numbers within it
    rank = torch.full((pages,), -1, dtype=torch.int32, device=DEV)
    used = table[table >= 0].long().unique()
    rank[used] = torch.randperm(len(pools[0]), generator=g, device=DEV)[:len(used)].to(torch.int32)
    table = torch.where(table >= 0, rank[table.clamp(min=0).long()], table)
    return {"kpages": pools[0], "vpages": pools[1], "scales": pools[2], "table": table, "q_start": _i32(start),
            "kv_len": _i32(total), "n": n, "total": total}


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind = case["kind"]
    st = {"case": case}
    if kind in ("attend8", "shared"):
        st.update(_paged(case, g))
        T, D = sum(st["n"]), case["D"]
        # scores of a standard deviation of 2: some positions matter, none alone
        st["q"] = (torch.randn(T, case["heads"] * D, generator=g, device=DEV) * 2).to(torch.bfloat16)
        st["scale"] = 1.0 / math.sqrt(D)
        cuts, share = _groups(case)
        st["group_start"], st["shared_len"] = _i32(cuts), _i32(share)
        return st
    if kind == "post8":
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
    B, V, L = case["B"], case["vocab"], case["history"]
    # a softcapped head's logits
    st["logits"] = 30 * torch.tanh(torch.randn(B, V, generator=g, device=DEV) / 10)
    if L:
        # tokens as texts have them: a few often, most once (ranks by a power law), rows of different lengths
        r = torch.rand(B, L, generator=g, device=DEV)
        rank = torch.exp(r * math.log(V)).long().clamp(max=V - 1)
        st["tokens"] = torch.randperm(V, generator=g, device=DEV)[rank].to(torch.int32)
        n = (L - (torch.rand(B, generator=g, device=DEV) * 0.4 * L).int()).to(torch.int32)
        n[0] = L
        st["n_tokens"], st["n_prompt"] = n, torch.minimum(n, torch.full_like(n, case["prompt"]))
    for name in ("repetition", "frequency", "presence"):
        v = case[name].split(",")
        st[name] = torch.tensor([float(v[i % len(v)]) for i in range(B)], device=DEV)
    if case["bias"]:
        st["bias_tokens"] = torch.randint(0, V, (B, case["bias"]), generator=g, device=DEV, dtype=torch.int32)
        st["bias"] = torch.randn(B, case["bias"], generator=g, device=DEV) * 5
    if case["allowed"]:
        W = (V + 31) // 32
        m = torch.rand(B, W, 32, generator=g, device=DEV) < case["allowed"]
        m = (m.long() << torch.arange(32, device=DEV)).sum(-1)
        st["allowed"] = torch.where(m >= 1 << 31, m - (1 << 32), m).to(torch.int32)
    return st


# ---- one pass --------------------------------------------------------------------

def run(st):
    if own:
        return _run_own(st)
    return {"attend8": _attend, "shared": _attend, "post8": _post, "adjust": _adjust}[st["case"]["kind"]](st)


def _run_own(st):
    import alveare_amd as aa
    from alveare_amd import paged

    c = st["case"]
    if c["kind"] == "adjust":
        return {"logits": aa.adjust_logits(
            st["logits"], tokens=st.get("tokens"), n_tokens=st.get("n_tokens"), n_prompt=st.get("n_prompt"),
            repetition=st["repetition"], frequency=st["frequency"], presence=st["presence"],
            bias_tokens=st.get("bias_tokens"), bias=st.get("bias"), allowed=st.get("allowed"),
            out=st["logits"] if c["in_place"] else None)}
    batch = st["kpages"], st["vpages"], st["table"], st["q_start"], st["kv_len"]
    if c["kind"] == "attend8":
        return {"out": paged.attention_paged(st["q"], *batch, heads=c["heads"], window=c["window"], sinks=c["sinks"],
                                             scale=st["scale"], max_q=c["n_hi"], scales=st["scales"])}
    if c["kind"] == "shared":
        return {"out": paged.attention_shared_paged(st["q"], *batch, st["group_start"], st["shared_len"],
                                                    heads=c["heads"], window=c["window"], sinks=c["sinks"],
                                                    scale=st["scale"], max_q=c["n_hi"], scales=st["scales"])}
    q, k = c["heads"] * c["D"], c["kv_heads"] * c["D"]
    out = paged.qkv_post_paged(st["qkv"], *batch, heads=c["heads"], k_off=q, v_off=q + k, q_w=st["q_w"], k_w=st["k_w"],
                               norm_v=c["norm_v"], rope=st["rope"], scales=st["scales"])
    return {"q": out, "kpages": st["kpages"], "vpages": st["vpages"], "scales": st["scales"]}


# ---- the plain forms -------------------------------------------------------------

def _rows(st):
    """Packed row of (sequence, i) for i below the longest chunk, its position, and whether it exists."""
    first, n = st["q_start"][:-1].long(), st["q_start"].diff().long()
    i = torch.arange(max(st["n"]), device=DEV)
    there = i < n[:, None]
    return torch.where(there, first[:, None] + i, 0), (st["kv_len"].long() - n)[:, None] + i, there


def _values(st, name, page):
    """The values of pages (by number), float32: codes times powers."""
    x = st[name]
    if st["scales"] is None:
        return x[page].float()
    e = st["scales"].view(torch.uint8)[..., 0 if name == "kpages" else 1][page].float()
    return x.view(torch.uint8)[page].view(E4M3).float() * torch.exp2(e - 127)[..., None]


def _attend(st):
    c = st["case"]
    B, S, D, H, g = c["B"], c["page"], c["D"], c["kv_heads"], c["heads"] // c["kv_heads"]
    width = (max(st["total"]) + S - 1) // S
    rows, pos, there = _rows(st)
    page = st["table"][:, :width].long()
    k, v = (_values(st, name, page.clamp(min=0)).permute(0, 2, 1, 3, 4).reshape(B, H, width * S, D)
            for name in ("kpages", "vpages"))
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
    for i, (name, t) in enumerate((("kpages", rotate(norm(k, st["k_w"]))),
                                   ("vpages", (norm(v) if c["norm_v"] else v).to(torch.bfloat16)))):
        codes, e = _encode(t)
        st[name].view(torch.uint8)[page, :, pos % S] = codes.view(torch.uint8)
        st["scales"].view(torch.uint8)[page, :, pos % S, i] = e
    return {"q": rotate(norm(q, st["q_w"])).reshape(len(x), H * D), "kpages": st["kpages"], "vpages": st["vpages"],
            "scales": st["scales"]}


def _adjust(st):
    x = st["logits"]
    B, V = x.shape
    if "tokens" in st:
        at = torch.arange(st["tokens"].shape[1], device=DEV)
        here, made = at < st["n_tokens"][:, None], at >= st["n_prompt"][:, None]
        t = st["tokens"].long()
        seen = torch.zeros(B, V, dtype=torch.int32, device=DEV).scatter_add_(1, t, here.int()) > 0
        count = torch.zeros(B, V, dtype=torch.int32, device=DEV).scatter_add_(1, t, (here & made).int())
        r, f, p = (st[k][:, None] for k in ("repetition", "frequency", "presence"))
        x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
        x = x - f * count - p * (count > 0)
    if "bias" in st:
        x = x + torch.zeros_like(x).scatter_add_(1, st["bias_tokens"].long(), st["bias"])
    if "allowed" in st:
        bits = st["allowed"][:, :, None] >> torch.arange(32, dtype=torch.int32, device=DEV) & 1
        x = torch.where(bits.view(B, -1)[:, :V] != 0, x, -math.inf)
    if st["case"]["in_place"]:
        st["logits"].copy_(x)
        x = st["logits"]
    return {"logits": x}


# ---- what a pass cannot do without ------------------------------------------------

def _visible(case):
    """Over all sequences: (row, position) pairs that are visible; positions that some row sees, those that a group
    shares counted once."""
    pairs = 0
    cuts, share = _groups(case)
    n, total, shared = _lens(case)
    w, s = case.get("window", 0), case.get("sinks", 0)
    own_part, first = 0, [None] * len(share)
    group = [j for j, (a, b) in enumerate(zip(cuts, cuts[1:])) for _ in range(b - a)]
    for b in range(case["B"]):
        if n[b] == 0:
            continue
        t = np.arange(total[b] - n[b], total[b])
        lo = np.maximum(t + 1 - w, 0) if w else np.zeros_like(t)
        pairs += int((t + 1 - lo + np.minimum(lo, s)).sum())
        own_part += total[b] - max(int(lo[0]), shared[b])
        j = group[b]
        first[j] = int(lo[0]) if first[j] is None else min(first[j], int(lo[0]))
    both = sum(max(0, h - lo) + min(lo, s, h) for h, lo in zip(share, first) if lo is not None)
    if case["kind"] != "shared":
        both = sum(min(lo, s) for lo in first if lo is not None)
    return pairs, own_part + both


def _cost(case):
    return _visible(case)[0] * case["heads"] * case["D"]


def work(case):
    kind = case["kind"]
    if kind == "adjust":
        B, V, L = case["B"], case["vocab"], case["history"]
        off = 1 - case["allowed"] if case["allowed"] else 0
        side = 4 * L * B + 8 * case["bias"] * B + (V // 8 * B if case["allowed"] else 0)
        # in place, what a grammar leaves alone is neither read nor written
        rows = 4 * V * off if case["in_place"] else 4 * V * (2 - off)
        return {"bytes": int(side + rows * B), "flops": B * V}
    T, D, K = sum(_lens(case)[0]), case["D"], case["kv_heads"]
    if kind == "post8":
        q, kv = T * case["heads"] * D, 2 * T * K * D
        return {"bytes": 2 * 2 * q + 3 * kv + 2 * T * K + 2 * T * case["rotated"], "flops": 10 * (q + kv)}
    pairs, union = _visible(case)
    per = 2 * (D + 1) if case.get("bits", 8) == 8 else 4 * D
    return {"bytes": 2 * 2 * T * case["heads"] * D + per * union * K, "flops": 4 * pairs * case["heads"] * D}


# ---- in 64 bits ------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "adjust":
        return _exact_adjust(st)
    D, S, H = case["D"], case["page"], case["kv_heads"]
    if kind == "post8":
        return _exact_post(st)
    g = case["heads"] // H
    out = torch.empty(sum(st["n"]), case["heads"], D, dtype=torch.float64, device=DEV)
    at = 0
    for b, (n, total) in enumerate(zip(st["n"], st["total"])):
        p = torch.arange(total, device=DEV)
        pages, slots = st["table"][b].long()[p // S], p % S
        for h in range(H if n else 0):
            k, v = (st[name].view(torch.uint8 if st["scales"] is not None else torch.int16)[pages, h, slots]
                    for name in ("kpages", "vpages"))
            if st["scales"] is None:
                k, v = k.view(torch.bfloat16).double(), v.view(torch.bfloat16).double()
            else:
                e = st["scales"].view(torch.uint8)[pages, h, slots].double() - 127
                k = torch.ldexp(k.view(E4M3).double(), e[:, :1])
                v = torch.ldexp(v.view(E4M3).double(), e[:, 1:])
            for i0 in range(0, n, 512):
                i1 = min(n, i0 + 512)
                t = torch.arange(total - n + i0, total - n + i1, device=DEV)[:, None]
                off = p > t
                if case["window"]:
                    off |= (p <= t - case["window"]) & (p >= case["sinks"])
                for hq in range(h * g, h * g + g):
                    q = st["q"].view(-1, case["heads"], D)[at + i0:at + i1, hq].double()
                    s = torch.mm(q, k.t()) * st["scale"]
                    out[at + i0:at + i1, hq] = torch.softmax(s.masked_fill(off, -math.inf), 1) @ v
        at += n
    return {"out": out.view(len(out), -1)}


def _exact_post(st):
    """The codes before their rounding to e4m3."""
    case = st["case"]
    D, S, H = case["D"], case["page"], case["kv_heads"]
    kp, vp, sc = (st[k].float().double() for k in ("kpages", "vpages", "scales"))
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
        for i, (pool, t) in enumerate(((kp, qk[at:at + n, -H:]), (vp, v[at:at + n]))):
            top = t.to(torch.bfloat16).double().abs().amax(-1)  # (and between rotation and powers)
            e = torch.ceil(torch.log2(top / 448)).clamp(-126, 127)
            pool[pages, :, slots], sc[pages, :, slots, i] = torch.ldexp(t, -e[..., None]), torch.exp2(e)
        at += n
    return {"q": qk[:, :-H].reshape(len(x), -1), "kpages": kp, "vpages": vp, "scales": sc}


def _exact_adjust(st):
    x = st["logits"].cpu().numpy().astype(np.float64)
    for b in range(st["case"]["B"]):
        if "tokens" in st:
            t = st["tokens"][b, :int(st["n_tokens"][b])].cpu().numpy()
            r, f, p = (float(st[k][b]) for k in ("repetition", "frequency", "presence"))
            once = np.unique(t)
            x[b, once] = np.where(x[b, once] > 0, x[b, once] / r, x[b, once] * r)
            made, count = np.unique(t[int(st["n_prompt"][b]):], return_counts=True)
            x[b, made] -= f * count + p
        if "bias" in st:
            np.add.at(x[b], st["bias_tokens"][b].cpu().numpy(), st["bias"][b].double().cpu().numpy())
        if "allowed" in st:
            bits = np.unpackbits(st["allowed"][b].cpu().numpy().view(np.uint8), bitorder="little")
            x[b, bits[:x.shape[1]] == 0] = -np.inf
    return {"logits": x}

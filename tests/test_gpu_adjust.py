"""Penalties, biases and allowed tokens on rows of logits, against a plain form in
64 bits. The float64 steps (a product or quotient, a difference of a product and a
sum, the sum of M biases and its addition: M + 5 roundings of 2^-53, each relative to
no more than the sum of the terms' sizes) and one rounding to float32, 2^-24."""
import math

import numpy as np
import pytest
import torch

import more_ref as M

pytestmark = pytest.mark.gpu


def make(B, V, L, Mb, dev, seed=0, repeat=20):
    g = torch.Generator().manual_seed(seed)
    c = {"logits": torch.randn(B, V, generator=g) * 5}
    c["logits"][:, V // 2] = 0.0
    c["tokens"] = torch.randint(0, max(1, V // repeat), (B, L), generator=g).to(torch.int32) * min(repeat, V)
    c["tokens"][:, 1::5] = torch.randint(0, V, c["tokens"][:, 1::5].shape, generator=g).to(torch.int32)
    if L > 3:
        c["tokens"][:, 3] = torch.tensor([-1, V, 2 ** 31 - 1, -2 ** 31])[torch.arange(B) % 4].to(torch.int32)
    c["n_tokens"] = torch.randint(0, L + 1, (B,), generator=g).to(torch.int32)
    c["n_tokens"][0] = L
    c["n_prompt"] = (c["n_tokens"] * torch.rand(B, generator=g)).to(torch.int32)
    c["repetition"] = torch.tensor([1.2, 1.0, 0.7])[torch.arange(B) % 3]
    c["frequency"] = torch.tensor([0.3, 0.0, -0.25, 0.0])[torch.arange(B) % 4]
    c["presence"] = torch.tensor([0.0, 0.0, 0.5, 0.0, -1.0])[torch.arange(B) % 5]
    if Mb:
        c["bias_tokens"] = torch.randint(0, V, (B, Mb), generator=g).to(torch.int32)
        c["bias_tokens"][:, Mb // 2:] = c["bias_tokens"][:, :Mb - Mb // 2]  # each twice
        c["bias_tokens"][:, 0] = c["tokens"][:, 0] if L else 0
        c["bias"] = torch.randn(B, Mb, generator=g) * 3
    c["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (B, (V + 31) // 32), generator=g).to(torch.int32)
    return {k: v.to(dev) for k, v in c.items()}


def check(c, in_place=False, **ch):
    from alveare_amd import adjust_logits

    c = {**c, **ch}
    logits = c.pop("logits")
    keep = logits.clone()
    got = adjust_logits(logits, **c, out=logits if in_place else None)
    assert (got.data_ptr() == logits.data_ptr()) == in_place
    if not in_place:
        assert torch.equal(logits.nan_to_num(), keep.nan_to_num())
    keep, out = keep.view(-1, keep.shape[-1]), got.view(-1, keep.shape[-1]).cpu()
    for b in range(len(keep)):
        row = {}
        for k, v in c.items():
            if v is None or not isinstance(v, torch.Tensor):
                row[k] = v
            elif k in ("bias_tokens", "bias", "allowed", "tokens"):
                row[k] = (v if v.dim() == 1 else v[b % v.shape[0]]).cpu().numpy()
            else:
                row[k] = v[b].item()
        want, touched = M.adjust(keep[b], **row)
        size = keep[b].double().abs().cpu() * 2 + want.abs() + 50
        tol = torch.where(touched, 2.0 ** -24 * want.abs() + 2.0 ** -53 * 2000 * size, 0.0)
        g = out[b].double()
        same = (g == want) | (torch.isnan(g) & torch.isnan(want)) | ((g - want).abs() <= tol)
        assert same.all(), (b, (~same).nonzero()[:4].tolist(), g[~same][:4], want[~same][:4])
    return got


@pytest.mark.parametrize("V", [1, 31, 32, 1000, 4095, 4096, 4097, 32000, 128256, 262144])
@pytest.mark.parametrize("L,Mb", [(0, 0), (1, 1), (700, 0), (5000, 40), (0, 300)])
def test_adjust(dev, V, L, Mb):
    c = make(5, V, L, Mb, dev, seed=V + L)
    check(c)
    check(c, allowed=None)
    check(c, in_place=True)


@pytest.mark.parametrize("in_place", [False, True])
def test_adjust_what_is_given(dev, in_place):
    """Each part alone and none, one row, numbers in place of arrays, lists and words for all rows at once."""
    c = make(6, 9001, 300, 16, dev)
    part = lambda *k: {n: c[n].clone() for n in ("logits", *k)}  # noqa: E731
    check(part(), in_place)
    check(part("allowed"), in_place)
    check(part("bias_tokens", "bias"), in_place)
    check(part("tokens"), in_place, repetition=1.5)
    check(part("tokens", "n_tokens"), in_place, frequency=0.5)
    check(part("tokens", "n_prompt"), in_place, presence=-0.5, repetition=2.0)
    check(part("tokens", "n_tokens", "n_prompt"), in_place)  # nothing is asked for
    one = {k: v[:1].clone() for k, v in c.items()}
    check(one, in_place)
    check({**part("tokens", "n_tokens", "n_prompt", "repetition", "frequency"), "bias_tokens": c["bias_tokens"][2],
           "bias": c["bias"][2], "allowed": c["allowed"][3:4]}, in_place)
    flat = check({"logits": c["logits"][0].clone(), "tokens": c["tokens"][:1], "repetition": 1.1}, in_place)
    assert flat.dim() == 1


def test_adjust_not_finite(dev):
    """Infinities and NaN in the logits; every token forbidden; and what sample makes of such a row."""
    from alveare_amd import sample

    c = make(4, 5000, 200, 8, dev)
    c["logits"][:, :600:7] = math.inf
    c["logits"][:, 1:600:7] = -math.inf
    c["logits"][:, 2:600:7] = math.nan
    c["bias"][0, 1], c["bias"][1, 2] = -math.inf, math.inf
    check(c)
    check(c, in_place=True)
    c = make(3, 5000, 200, 8, dev)
    c["allowed"][0], c["allowed"][1] = 0, 0
    c["allowed"][1, 70] = 1 << 9
    out = check(c)
    assert (out[0] == -math.inf).all()
    token, prob = sample(out, torch.full((3,), 0.5, device=dev))
    assert token[:2].tolist() == [-1, 70 * 32 + 9] and prob[:2].tolist() == [0.0, 1.0]


def test_adjust_counts(dev):
    """Thousands of one token, all tokens once, a token in prompt and answer."""
    V, L = 3000, 9000
    logits = torch.linspace(-4, 4, V).repeat(3, 1).to(dev)
    t = torch.zeros(3, L, dtype=torch.int32)
    t[0] = 17
    t[1, :V] = torch.arange(V)
    t[1, V:] = 5
    t[2] = torch.arange(L) % V
    n_prompt = torch.tensor([0, 3000, 4500], dtype=torch.int32)
    check({"logits": logits, "tokens": t.to(dev), "n_prompt": n_prompt.to(dev)}, frequency=0.01, presence=0.5, repetition=1.25)
    over = torch.tensor([L + 5, -3, 10], dtype=torch.int32, device=dev)  # counted as all, as none
    got = check({"logits": logits, "tokens": t.to(dev), "n_tokens": over.clamp(0, L)}, frequency=1.0)
    from alveare_amd import adjust_logits

    assert torch.equal(got, adjust_logits(logits, tokens=t.to(dev), n_tokens=over, frequency=1.0))


@pytest.mark.parametrize("V,L,Mb", [(50000, 140000, 0), (3000, 131071, 8191), (3000, 131072, 8191), (3000, 40, 8192),
                                    (262144, 140000, 65536)])
def test_adjust_long_histories_and_lists(dev, V, L, Mb):
    """On both sides of what 32 bits a token hold."""
    c = make(2, V, L, Mb, dev, seed=L)
    if V == 3000:
        c["tokens"][0] = 7  # as often as there are tokens
        c["n_prompt"][0] = 0
    check(c, frequency=0.001)
    check(c, in_place=True, frequency=0.001)


def test_adjust_strides_and_alignment(dev):
    """Rows that start anywhere, columns of wider arrays, logits and out side by side in one array."""
    c = make(4, 2051, 90, 6, dev)
    wide = torch.full((4, 4200), 9.0, device=dev)
    for a, o in ((0, 2060), (1, 2063), (3, 2100)):
        wide[:, a:a + 2051] = c["logits"]
        from alveare_amd import adjust_logits

        rest = {k: v for k, v in c.items() if k != "logits"}
        tok = torch.full((4, 101), 5, dtype=torch.int32, device=dev)
        tok[:, 3:93] = c["tokens"]
        words = torch.zeros(4, 80, dtype=torch.int32, device=dev)
        words[:, 1:1 + c["allowed"].shape[1]] = c["allowed"]
        want = adjust_logits(c["logits"], **rest)
        rest.update(tokens=tok[:, 3:93], allowed=words[:, 1:1 + c["allowed"].shape[1]])
        got = adjust_logits(wide[:, a:a + 2051], **rest, out=wide[:, o:o + 2051])
        assert torch.equal(got, want) and torch.equal(wide[:, a:a + 2051], c["logits"])
        keep = wide.clone()
        adjust_logits(wide[:, a:a + 2051], **rest, out=wide[:, a:a + 2051])
        keep[:, a:a + 2051] = want
        assert torch.equal(wide, keep)


def test_adjust_same_bits_and_graph(dev):
    """Duplicates in lists give the same bits each time; a captured call sees what its tensors hold then."""
    from alveare_amd import adjust_logits

    c = make(7, 30000, 4000, 200, dev)
    first = adjust_logits(**c)
    for _ in range(3):
        assert torch.equal(adjust_logits(**c), first)
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    g = torch.cuda.CUDAGraph()
    out = torch.empty_like(c["logits"])
    with torch.cuda.graph(g, stream=s):
        adjust_logits(**c, out=out)
    for turn in range(4):
        n = make(7, 30000, 4000, 200, dev, seed=100 + turn)
        for k, v in n.items():
            c[k].copy_(v)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, adjust_logits(**c)), turn


def test_adjust_refusals(dev):
    from alveare_amd import Q4ValueError, adjust_logits

    l = torch.zeros(2, 100, device=dev)
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)  # noqa: E731
    for kw in (dict(tokens=i(3, 5)), dict(tokens=i(5)), dict(bias_tokens=i(2, 4)), dict(bias=l),
               dict(bias_tokens=i(2, 4), bias=l[:, :3]), dict(allowed=i(2, 3)), dict(allowed=i(3, 4))):
        with pytest.raises(ValueError):
            adjust_logits(l, **kw)
    for kw in (dict(tokens=i(2, 5).long()), dict(allowed=l), dict(tokens=i(2, 5), n_tokens=i(1)), dict(out=l[:1]),
               dict(tokens=i(2, 5), n_prompt=i(2).cpu()), dict(tokens=i(2, 5), repetition=l[0].double())):
        with pytest.raises(TypeError):
            adjust_logits(l, **kw)
    with pytest.raises(TypeError):
        adjust_logits(l.double())
    with pytest.raises(Q4ValueError):
        adjust_logits(l, tokens=i(2, 5), repetition=0.0)
    wide = torch.zeros(2, 250, device=dev)
    with pytest.raises(Q4ValueError):
        adjust_logits(wide[:, :100], out=wide[:, 50:150])
    with pytest.raises(Q4ValueError):
        adjust_logits(wide[:, :100], out=wide[:, 200:].reshape(-1)[:100].expand(2, 100))
    assert adjust_logits(l[:0]).shape == (0, 100)

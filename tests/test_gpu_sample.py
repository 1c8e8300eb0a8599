"""Sampling against its definition in 64 bits: tokens are equal, probabilities
within float32's rounding (2^-24 of the float64 quotient, and the fixed-point
weights' 2^-36)."""
import math

import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu


def check(dev, logits, u, **kw):
    import alveare_amd as aa

    B = logits.shape[0]
    dt = {"top_k": torch.int32}
    full = {k: v if isinstance(v, list) else [v] * B for k, v in kw.items()}
    args = {k: torch.tensor(v, dtype=dt.get(k, torch.float32), device=dev) if isinstance(kw[k], list) else kw[k]
            for k, v in full.items()}
    token, prob = aa.sample(logits.to(dev), torch.tensor(u, dtype=torch.float32, device=dev), **args)
    for b in range(B):
        want, p = R.sample(logits[b], u[b], **{k: v[b] for k, v in full.items()})
        assert int(token[b]) == want, (b, int(token[b]), want, {k: v[b] for k, v in full.items()}, u[b])
        if math.isnan(p):
            assert math.isnan(float(prob[b]))
        else:
            assert abs(float(prob[b]) - p) <= p * (2.0 ** -24 + 2.0 ** -35) + 2.0 ** -149
    return token


def normal(B, V, seed=0, std=3.0):
    return torch.randn(B, V, generator=torch.Generator().manual_seed(seed)) * std


@pytest.mark.parametrize("V", [1, 2, 63, 64, 1000, 1025, 32000, 128256, 262144, 300001])
def test_sizes(dev, V):
    x = normal(6, V, V)
    u = [0.0, 0.25, 0.5, 0.77, 0.999, 1 - 2.0 ** -24]
    check(dev, x, u)
    check(dev, x, u, temperature=0.7, top_k=50, top_p=0.9, min_p=0.02)
    check(dev, x, u, top_p=0.95)


@pytest.mark.parametrize("top_k", [0, 1, 2, 17, 1000, 5000, 40000, 10 ** 6])
@pytest.mark.parametrize("top_p", [1.0, 0.0, 0.3, 0.9, 0.9999])
@pytest.mark.parametrize("min_p", [0.0, 0.1, 1.0])
def test_cuts(dev, top_k, top_p, min_p):
    x = normal(4, 50000, 7, 2.0)
    check(dev, x, [0.01, 0.4, 0.8, 0.9999], temperature=1.2, top_k=top_k, top_p=top_p, min_p=min_p)


def test_parameters_per_row(dev):
    x = normal(7, 20011, 3)
    check(dev, x, [0.5, 0.1, 0.9, 0.3, 0.6, 0.99, 0.2], temperature=[0.0, 1.0, 0.5, -1.0, 2.0, math.nan, math.inf],
          top_k=[5, 0, 3, -1, 100, 7, 4], top_p=[0.5, 2.0, 1.0, 0.1, -3.0, 0.9, 0.95],
          min_p=[0.0, -1.0, 0.3, 2.0, 0.001, 0.0, 0.0])


@pytest.mark.parametrize("V", [5, 4096, 100000])
def test_ties(dev, V):
    """Equal logits keep their order by index across every cut, zeros of both signs alike."""
    x = torch.zeros(6, V)
    x[1, V // 2:] = -0.0
    x[2, ::2] = 1.0
    x[3, V // 3:] = -2.0
    x[4] = torch.arange(V).remainder(3).float()
    x[5] = 5.0
    x[5, 0] = -math.inf
    for u in (0.0, 0.3, 0.5, 0.75, 0.999):
        check(dev, x, [u] * 6)
        check(dev, x, [u] * 6, top_p=0.5)
        check(dev, x, [u] * 6, top_k=max(1, V // 4))
        check(dev, x, [u] * 6, min_p=0.5, top_k=3, top_p=0.7)


@pytest.mark.parametrize("V", [100, 5000, 262144])
def test_extreme_values(dev, V):
    inf = math.inf
    big = 3.0e38
    x = normal(8, V, 5)
    x[0, 1:] = -inf                 # one token left
    x[1, :] = -inf                  # none
    x[2, 7] = inf                   # one infinity
    x[3, [3, V - 1]] = inf          # two share the weight
    x[4, V // 2] = math.nan
    x[5, ::2] = -big                # masked by the type's lowest values
    x[5, 1] = big
    x[6, V // 3:] = torch.finfo(torch.float32).min
    x[7, :] = torch.where(torch.arange(V) % 2 == 0, 1e30, -1e30)
    for kw in ({}, dict(top_k=20), dict(top_p=0.8), dict(min_p=0.2), dict(temperature=1e-30), dict(temperature=1e30),
               dict(temperature=0.0)):
        check(dev, x, [0.6, 0.3, 0.1, 0.7, 0.5, 0.2, 0.9, 0.4], **kw)


def test_one_bin_distributions(dev):
    """Logits that differ in their last bits only, and outliers far above the rest."""
    V = 60000
    x = torch.empty(3, V)
    x[0] = 1.0 + torch.arange(V).float() * 2.0 ** -23
    x[1] = normal(1, V, 1, 1e-6)[0]
    x[1, 5] = 40.0
    x[2] = normal(1, V, 2, 50.0)[0]
    for kw in ({}, dict(top_k=30000), dict(top_p=0.4), dict(top_k=50000, top_p=0.6), dict(temperature=100.0, top_p=0.9)):
        for u in (0.001, 0.5, 0.97):
            check(dev, x, [u] * 3, **kw)


def test_strided_rows_and_given_outputs(dev):
    import alveare_amd as aa

    x = normal(5, 3000, 9).to(dev)
    u = torch.rand(5, generator=torch.Generator().manual_seed(1)).to(dev)
    want = aa.sample(x[:, :2500].contiguous(), u, top_k=100)
    token, prob = torch.full((8,), 9, dtype=torch.int32, device=dev), torch.full((8,), 9.0, device=dev)
    got = aa.sample(x[:, :2500], u, top_k=100, token=token, prob=prob)
    assert got[0] is token and torch.equal(token[:5], want[0]) and (token[5:] == 9).all()
    assert torch.equal(prob[:5], want[1]) and (prob[5:] == 9).all()
    one = aa.sample(x[2, :2500], u[2:3], top_k=100)
    assert int(one[0]) == int(want[0][2])
    assert aa.sample(x[:0], u)[0].shape == (0,)
    for off in (1, 2, 3):  # rows that start off a 16-byte boundary
        y = aa.sample(x[:, off:2500], u, top_p=0.9)
        z = aa.sample(x[:, off:2500].contiguous(), u, top_p=0.9)
        assert torch.equal(y[0], z[0]) and torch.equal(y[1], z[1])


def test_large_batch(dev):
    import alveare_amd as aa

    x = normal(300, 777, 2)
    u = torch.rand(300, generator=torch.Generator().manual_seed(5))
    check(dev, x, u.tolist(), top_p=0.9, temperature=0.8)
    a = aa.sample(x.to(dev), u.to(dev))
    for _ in range(2):
        b = aa.sample(x.to(dev), u.to(dev))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_frequencies(dev):
    """Even numbers over [0, 1) give every token its share: of N, token r is drawn
    within one of N times its probability (an interval of u)."""
    import alveare_amd as aa

    x = torch.tensor([[0.0, 1.0, -1.0, 2.0, 0.5, -3.0]])
    N = 4096
    u = (torch.arange(N, dtype=torch.float32) + 0.5) / N
    token, _ = aa.sample(x.expand(N, 6).contiguous().to(dev), u.to(dev))
    share = torch.softmax(x[0].double(), 0) * N
    assert ((torch.bincount(token.cpu(), minlength=6) - share).abs() <= 1).all()


def test_graphs_and_streams(dev):
    import alveare_amd as aa

    made = []
    for seed, V in ((1, 262144), (2, 5000)):
        x = normal(3, V, seed).to(dev)
        u = torch.rand(3, device=dev)
        s = torch.cuda.Stream(dev)
        s.wait_stream(torch.cuda.current_stream(dev))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = aa.sample(x, u, top_k=300, top_p=0.9)
        made.append((x, u, s, g, out))
    for turn in range(5):
        for i, (x, u, s, g, out) in enumerate(made):
            x.copy_(normal(3, x.shape[1], 20 + turn + i))
            u.uniform_()
        torch.cuda.synchronize()
        for x, u, s, g, out in made:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for x, u, s, g, out in made:
            want = aa.sample(x, u, top_k=300, top_p=0.9)
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_greedy_is_the_heads_argmax(dev):
    import alveare_amd as aa
    import numpy as np

    x = normal(4, 9000, 6)
    x[1, 400] = x[1].max()
    x[2, [70, 8000]] = math.nan
    token, _ = aa.sample(x.to(dev), torch.rand(4, device=dev), temperature=0.0)
    assert token.tolist() == [int(np.argmax(r)) for r in x.numpy()]


def test_refusals(dev):
    import alveare_amd as aa

    x, u = normal(2, 100).to(dev), torch.rand(2, device=dev)
    for a, b, kw in ((x.double(), u, {}), (x.cpu(), u, {}), (x, u.double(), {}), (x, u[:1], {}), (x.t(), u, {}),
                     (x, u, dict(top_k=torch.zeros(2, device=dev))), (x, u, dict(temperature=u[:1])),
                     (x, u, dict(top_p=torch.zeros(2))), (x, u, dict(token=torch.zeros(2, device=dev))),
                     (x, u, dict(prob=torch.zeros(1, device=dev))), (x[:, :0], u, {})):
        with pytest.raises((TypeError, ValueError)):
            aa.sample(a, b, **kw)


def test_top_k_of_any_size(dev):
    import alveare_amd as aa

    x, u = normal(4, 5000).to(dev), torch.tensor([0.1, 0.5, 0.9, 0.999], device=dev)
    want = aa.sample(x, u)
    for k in (5000, 2 ** 31, 2 ** 32 + 1, -2 ** 40):
        for a, b in zip(aa.sample(x, u, top_k=k), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("V", [1024, 1025, 4095, 4097, 8192, 8193, 16383, 16384, 16385])
def test_sizes_around_the_variants_ends(dev, V):
    """Cuts of every kind, ties past what a bin compares, and -infinity among them."""
    x = normal(6, V, seed=V)
    x[1] = (x[1] * 2).round() / 2       # a few dozen values
    x[2, ::3] = -math.inf
    x[3] = 0.25                         # one value
    x[4] = x[4] * 1e-3
    x[4, V // 2] = 40.0                 # one far above the rest
    u = [0.3, 0.7, 0.999, 0.5, 0.9999999, 0.0]
    check(dev, x, u, temperature=0.7, top_k=[0, 50, 0, 700, 0, 3], top_p=[0.95, 1.0, 0.6, 0.9, 0.999999, 0.5],
          min_p=[0.0, 0.0, 0.05, 0.0, 0.0, 0.2])
    check(dev, x, u)


def bf16_rounded(B, V, seed, std=2.0):
    """Logits as a bf16 product leaves them: hundreds of each value."""
    return normal(B, V, seed, std).bfloat16().float()


@pytest.mark.parametrize("V", [4000, 16384, 32000, 128256, 262144])
def test_logits_that_were_bf16(dev, V):
    for seed, std in ((1, 1.0), (2, 2.5)):
        x = bf16_rounded(5, V, seed, std)
        for kw in ({}, dict(top_p=0.92), dict(top_k=V // 3), dict(temperature=2.0, top_k=V // 6, top_p=0.95),
                   dict(min_p=0.01, top_p=0.99, temperature=0.8)):
            check(dev, x, [0.0, 0.2, 0.55, 0.9, 0.9999], **kw)


def test_neighbouring_logits_of_which_each_is_held_by_many(dev):
    """Runs of equal logits a last bit apart, around zero and the type's smallest among them."""
    V = 49998
    x = torch.full((4, V), -9.0)
    x[0, ::2] = (1.0 + torch.arange(V // 2).remainder(5).float() * 2.0 ** -23)
    x[1, 1::3] = torch.arange(V // 3).remainder(7).float() * 2.0 ** -149
    x[1, 2::3] = -torch.arange(V // 3).remainder(3).float() * 2.0 ** -149
    x[2] = (torch.arange(V) * 7919 % V).remainder(300).float() * 2.0 ** -12
    x[3, :4000] = 2.0
    x[3, 4000:] = 2.0 - torch.arange(V - 4000).remainder(200).float() * 2.0 ** -10
    for kw in ({}, dict(top_p=0.7), dict(top_k=4001), dict(top_k=20000, top_p=0.6, min_p=0.3)):
        for u in (0.0, 0.35, 0.8, 0.9999):
            check(dev, x, [u] * 4, **kw)


def us_with_top_p(dev, x):
    import alveare_amd as aa

    x, u = x.to(dev), torch.full((x.shape[0],), 0.7, device=dev)
    best = math.inf
    for turn in range(6):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        for _ in range(10):
            aa.sample(x, u, top_p=0.92)
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b)) if turn else best
    return best * 100


@pytest.mark.parametrize("V,B", [(16384, 256), (262144, 1), (128256, 48)])
def test_ties_cost_no_second_way(dev, V, B):
    """A row of tied logits takes the launches of any other (and, at the crossings, two or three rounds of a
    histogram in shared memory): less than three times its time, not the twenty of a row read again by one workgroup."""
    free, tied = us_with_top_p(dev, normal(B, V, 1, 2.0)), us_with_top_p(dev, bf16_rounded(B, V, 1))
    assert tied < 3 * free, (free, tied)


@pytest.mark.parametrize("V,B,step,times", [(128256, 48, 0.25, 6), (262144, 1, 0.25, 12), (262144, 1, 1e9, 25)])
def test_what_thousands_of_ties_cost(dev, V, B, step, times):
    """One workgroup reads such a row a few times over for each crossing (measured 2.8, 6 and 11 times a row without
    ties; nine passes of atomics for each were 9, 24 and 82)."""
    x = normal(B, V, 1, 2.0)
    free, tied = us_with_top_p(dev, x), us_with_top_p(dev, (x / step).round() * step)
    assert tied < times * free, (free, tied)


@pytest.mark.parametrize("V,step", [(40000, 1.0), (262144, 0.25), (262144, 4.0), (300001, 1e9), (1500000, 0.0), (3000001, 2.0 ** -7)])
def test_thousands_of_tokens_at_a_border(dev, V, step):
    """More tokens in the bins of the crossings than are collected: logits of a few values, and very many."""
    x = normal(3, V, seed=V, std=2.0)
    x = (x / step).round() * step if step else x
    x[1, V // 3: V // 2] = -math.inf
    x[2, ::5] = x[2].max() + 0.5
    for kw in ({}, dict(top_p=0.9), dict(top_k=V // 2, top_p=0.8, temperature=1.5), dict(top_k=V // 50, min_p=0.2)):
        for u in (0.0, 0.43, 0.99999):
            check(dev, x, [u] * 3, **kw)


@pytest.mark.parametrize("V", [3000, 20000, 262144])
def test_many_infinities_and_zeros(dev, V):
    """Infinities, or zeros of both signs, more than a border's tokens are compared or collected."""
    import alveare_amd as aa

    x = normal(4, V, seed=V)
    x[0, ::2] = math.inf
    x[1, V // 3:] = math.inf
    x[1, :V // 4] = -math.inf
    x[2, ::2] = 0.0
    x[2, 1::2] = -0.0
    x[3, ::2] = -0.0
    x[3, 1::4] = 0.0
    for kw in ({}, dict(top_p=0.6), dict(top_k=V // 3)):
        for u in (0.0, 0.5, 0.97):
            check(dev, x, [u] * 4, **kw)
    # An infinite temperature: as 3e38, of which every finite (l - l_0) / T here leaves exp 1 in 64 bits too, and
    # -infinity 0 (the plain form's own -infinity / infinity is no number).
    for u in (0.0, 0.5, 0.97):
        token, prob = aa.sample(x.to(dev), torch.full((4,), u, device=dev), temperature=math.inf, top_k=V - 7, top_p=0.9)
        for b in range(4):
            want, p = R.sample(x[b], u, temperature=3e38, top_k=V - 7, top_p=0.9)
            assert int(token[b]) == want and abs(float(prob[b]) - p) <= p * (2.0 ** -24 + 2.0 ** -35)


def test_ties_replayed(dev):
    """A captured call over rows that change between free, tied and constant ones."""
    import alveare_amd as aa

    V = 262144
    x, u = normal(3, V, 1).to(dev), torch.tensor([0.2, 0.6, 0.95], device=dev)
    aa.sample(x, u, top_p=0.9)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = aa.sample(x, u, top_p=0.9)
    for seed in range(4):
        y = normal(3, V, 10 + seed)
        y[seed % 3] = y[seed % 3].bfloat16().float()
        y[(seed + 1) % 3] = (y[(seed + 1) % 3] * 4).round() / 4 if seed else 0.25
        x.copy_(y)
        g.replay()
        torch.cuda.synchronize()
        want = aa.sample(x, u, top_p=0.9)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        for b in range(3):
            assert int(out[0][b]) == R.sample(y[b], float(u[b]), top_p=0.9)[0]

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

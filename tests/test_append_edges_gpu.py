"""paged_append at the ends of a sequence's table, on a real MI355X."""
import pytest
import torch

from tests.test_paged_cache_gpu import BF16, I32, Case, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('page,layout', [(16, 'head'), (1, 'row'), (64, 'qkv')])
def test_append_drops_only_the_rows_outside(page, layout):
    """rows that start before position 0 or reach behind the table: those inside are written"""
    from pixparse_amd import ops
    dev, kv, T = torch.device('cuda:0'), 3, 9
    c = Case(dev, 6, kv, kv, page, [70] * 6, layout, seed=page, pages=-(-70 // page))
    starts = [-2, -9, -8, c.cap - 4, -2 ** 31, 2 ** 31 - 1]
    g = torch.Generator().manual_seed(page)
    k, v = (torch.randn(6, T, kv * 64, generator=g).to(BF16) for _ in range(2))
    k0, v0, w0 = c.k.clone(), c.v.clone(), c.weights.clone()
    for b, s in enumerate(starts):
        for t in range(T):
            p = s + t
            if 0 <= p < c.cap:
                at = (int(c.table[b, p // page]), p % page)
                k0[at], v0[at] = c.d(k[b, t].view(kv, 64)), c.d(v[b, t].view(kv, 64))
                w0[b, :, p] = 0
    w = c.d(c.weights)
    ops.paged_append(c.d(k), c.d(v), c.k, c.v, c.d(c.table), torch.tensor(starts, dtype=I32, device=dev), torch.full((6,), T, dtype=I32, device=dev), weights=w)
    assert same(c.k, k0) and same(c.v, v0) and torch.equal(w.cpu(), w0)

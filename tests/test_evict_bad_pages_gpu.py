"""cache_evict on sequences whose page table leads outside the pool, on a real MI355X: they stay as they are, as a whole."""
import math

import pytest
import torch

from tests.test_paged_cache_gpu import BF16, I32, Case, evict_reference, same

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def dev():
    assert torch.cuda.is_available(), 'these tests need the MI355X'
    from pixparse_amd import hip
    hip.load()
    return torch.device('cuda:0')


@pytest.mark.parametrize('in_place', [True, False])
@pytest.mark.parametrize('kv,page,n,budget,recent', [
    (2, 16, 100, 50, 10),
    (2, 1, 1500, 700, 0),           # more entries of the table than threads of a workgroup
    (1, 64, 9000, 300, 300),        # the window alone: nothing is selected
    (1, 16, 9000, 2000, 7),         # more positions than a workgroup holds at once
    (43, 32, 1500, 1100, 100),      # heads for every CU: the rows move in the selecting launch
])
def test_evict_leaves_sequences_with_bad_pages(dev, kv, page, n, budget, recent, in_place):
    """page ids -1, n_pages and 2^31 - 1, inside the budget, behind it and in the last page of the length: rows, weights and length stay, kept is -1.
    A bad page behind the length, or under a sequence that is not cut, changes nothing."""
    from pixparse_amd import ops
    c = Case(dev, 6, kv, kv, page, [n] * 5 + [budget - 1], 'head', seed=n, pages=-(-n // page) + 2)
    good = c.table.clone()
    last = (n - 1) // page
    c.table[0, 0], c.table[1, last - 1], c.table[2, last], c.table[5, 0] = -1, c.k.shape[0], 2 ** 31 - 1, -1
    c.table[3, last + 1:] = 2 ** 31 - 1
    bad = c.table
    n_dev, new = c.lengths, torch.full((6,), -9, dtype=I32, device=dev)
    w, kept = c.d(c.weights), torch.full((6, kv, budget), 5, dtype=I32, device=dev)
    c.table, c.n = good, [-5, -5, -5] + c.n[3:]             # (the reference leaves lengths outside the table alone)
    kept_ref, k_ref, v_ref, w_ref = evict_reference(c, c.weights, budget, recent)
    out = n_dev if in_place else new
    ops.cache_evict(c.k, c.v, c.d(bad), n_dev, w, budget, recent, out, kept=kept)
    assert out.tolist() == [n, n, n, budget, budget, budget - 1]
    assert torch.equal(kept.cpu(), kept_ref)
    assert torch.equal(w.cpu().view(I32), w_ref.view(I32))
    assert same(c.k.cpu(), k_ref) and same(c.v.cpu(), v_ref)


def test_a_bad_page_stays_visible_over_an_eviction(dev):
    """attention answers NaN before the cut and after it"""
    from pixparse_amd import ops
    c = Case(dev, 2, 2, 2, 16, [100, 100], 'head', seed=1)
    c.table[0, 5] = -1
    table, n, w = c.d(c.table), c.lengths, torch.zeros(2, 2, c.cap, device=dev)
    o = torch.zeros(2, 128, dtype=BF16, device=dev)
    for i in range(2):
        ops.paged_attn_decode(c.d(c.q), c.k, c.v, table, n, o, 2, 0.125, weights=w if i == 0 else None)
        assert bool(o[0].isnan().all()) and bool(torch.isfinite(o[1]).all())
        ops.cache_evict(c.k, c.v, table, n, w, 48, 8, n)
    assert n.tolist() == [100, 48] and math.isnan(float(w[0, 0, 0]))

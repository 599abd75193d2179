"""Infinite value rows under ordinary probabilities, on a real MI355X: what the formula gives, infinity, and no NaN from the way a probability is held."""
import math

import pytest
import torch

from tests.test_paged_cache_gpu import BF16, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('sign', [1, -1])
@pytest.mark.parametrize('H,kv,lengths', [(8, 8, [64, 200]), (16, 2, [1500, 90])])
def test_infinite_value_rows(H, kv, lengths, sign):
    """channel c is infinite in the row of one key of its own: p > 0, so o[c] is infinite, whatever bits p has.  (Scores of under 40 in base 2: no p
    is small enough to vanish.)"""
    from pixparse_amd import ops
    dev = torch.device('cuda:0')
    c = Case(dev, 2, H, kv, 32, lengths, 'head', seed=H)
    for b, n in enumerate(lengths):
        at = torch.randperm(n, generator=torch.Generator().manual_seed(b))[:64].tolist()
        for ch, p in enumerate(at):
            c.v[int(c.table[b, p // 32]), p % 32, :, ch] = sign * math.inf
    o = torch.zeros(2, H * 64, dtype=BF16, device=dev)
    for q in (c.q, c.q * 0.5, c.q * 0.25):
        ops.paged_attn_decode(c.d(q), c.k, c.v, c.d(c.table), c.lengths, o, H, 0.125)
        assert bool((o == sign * math.inf).all()), f'{int(o.isnan().sum())} of {o.numel()} are NaN'

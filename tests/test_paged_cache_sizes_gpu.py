"""Sizes of the paged cache at which its kernels take other ways, on a real MI355X: more query heads on a key-value head than one workgroup takes (16),
sequences longer than one the selecting workgroup of an eviction holds (8192), rows that take three or more tiles to move.  References and
tolerances are those of test_paged_cache_gpu."""
import pytest
import torch

import tests.test_paged_cache_gpu as paged

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def dev():
    assert torch.cuda.is_available(), 'these tests need the MI355X'
    from pixparse_amd import hip
    hip.load()
    return torch.device('cuda:0')


@pytest.mark.parametrize('append', [False, True])
@pytest.mark.parametrize('weights', [False, True])
@pytest.mark.parametrize('B,H,kv,page,lengths,layout', [
    (2, 17, 1, 16, [77, 0], 'head'),                # two workgroups, the second of one head; few enough keys for one launch without weights
    (3, 32, 1, 64, [200, 256, 1], 'row'),           # two whole ones
    (2, 34, 2, 32, [600, 1000], 'qkv'),             # eight waves a workgroup
    (1, 40, 1, 64, [3000], 'head'),                 # three, split over the length
    (2, 51, 3, 16, [1025, 2100], 'row'),
])
def test_more_query_heads_than_a_workgroup_takes(dev, B, H, kv, page, lengths, layout, append, weights):
    paged.test_paged_attention(dev, B, H, kv, page, lengths, layout, append, weights)


@pytest.mark.parametrize('in_place', [True, False])
@pytest.mark.parametrize('B,kv,page,lengths,layout,budget,recent,kind', [
    (2, 1, 64, [8193, 8192], 'head', 4000, 100, 'random'),
    (2, 2, 64, [8193, 16400], 'head', 1000, 20, 'odd'),             # moved from registers
    (1, 2, 16, [17000], 'row', 8500, 500, 'ties'),                  # quarter rows, three tiles; equal weights on both sides of a tile's border
    (1, 1, 32, [17000], 'qkv', 12500, 0, 'zeros'),                  # four tiles, all weights equal
    (1, 1, 128, [24935], 'head', 2048, 0, 'close'),
    (1, 36, 64, [4500], 'head', 4200, 30, 'random'),                # half rows, three tiles
    (2, 35, 16, [2600, 2500], 'row', 2300, 9, 'ties'),              # whole rows, three tiles
    (2, 130, 16, [3200, 60], 'head', 3100, 7, 'random'),            # heads for every CU: whole rows in the selecting launch, four tiles
])
def test_evict_long_sequences(dev, B, kv, page, lengths, layout, budget, recent, kind, in_place):
    paged.test_evict(dev, B, kv, page, lengths, layout, budget, recent, kind, in_place)


@pytest.mark.parametrize('append', [False, True])
@pytest.mark.parametrize('weights', [False, True])
@pytest.mark.parametrize('H,kv,pages', [(4, 4, 20), (12, 2, 70), (2, 1, 2000)])
def test_lengths_far_below_the_capacity(dev, H, kv, pages, append, weights, monkeypatch):
    """a table that covers what sequences may still reach (320 to 32000 positions), most splits without a key; entries behind the length hold no page"""
    made = paged.Case.__init__

    def init(self, dev, B, H, kv, page, lengths, layout, seed=0):
        made(self, dev, B, H, kv, page, lengths, layout, seed, pages=pages)
        for b, n in enumerate(lengths):
            self.table[b, -(-n // page):] = -1
    monkeypatch.setattr(paged.Case, '__init__', init)
    paged.test_paged_attention(dev, 5, H, kv, 16, [0, 1, 64, 130, 310], 'head', append, weights)

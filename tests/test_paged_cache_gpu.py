"""The paged key-value cache on a real MI355X: ops.paged_attn_decode, paged_append and cache_evict against plain forms in 64 bits.

Tolerance of the attention output, derived: the scores are fp32 sums of 64 exact products, off by at most 64 * 2^-24 of the sum of their magnitudes;
the base-2 exponent adds its own rounding (2^-24 of the score) and v_exp 2^-22, so every probability is off by at most a factor 1 +- delta with
delta = (64 + 1) 2^-24 A + 2^-21, A = the largest sum of magnitudes; sums of n positive terms add n 2^-24 at most.  The output moves by at most
2 (delta + n 2^-24) max|v| and is rounded to bf16 once: half a step, 2^-8 of the value.  In P.V (not in the weights) a probability is the sum of two
bf16 numbers, the second at most 2^-8 of it: off by 2^-17 more, the same for all of its products, so another 2^-17 max|v|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
HALF_STEP = torch.finfo(BF16).eps / 2


@pytest.fixture(scope='module')
def dev():
    assert torch.cuda.is_available(), 'these tests need the MI355X'
    from pixparse_amd import hip
    hip.load()
    return torch.device('cuda:0')


class Case:
    """pool, page table and lengths on the device; unused rows of the pool hold NaN, which nothing may read into a result"""

    def __init__(self, dev, B, H, kv, page, lengths, layout='head', seed=0, extra=3, pages=None):
        g = torch.Generator().manual_seed(seed)
        self.B, self.H, self.kv, self.page = B, H, kv, page
        self.n = list(lengths)
        per = pages or max(1, -(-max(self.n + [1]) // page))
        self.cap = per * page
        total = B * per + extra
        self.table = torch.randperm(total, generator=g)[:B * per].view(B, per).to(I32)
        k, v = (torch.randn(B, self.cap, kv, 64, generator=g).to(BF16) for _ in range(2))
        pools = []
        for rows in (k, v):
            pool = torch.full((total, page, kv, 64), math.nan, dtype=BF16)
            for b in range(B):
                for p in range(self.n[b]):
                    pool[int(self.table[b, p // page]), p % page] = rows[b, p]
            pools.append(pool)
        self.k_rows, self.v_rows = k, v
        if layout == 'head':
            self.k, self.v = (p.permute(0, 2, 1, 3).contiguous().to(dev).permute(0, 2, 1, 3) for p in pools)
        elif layout == 'qkv':          # heads of k and v as column blocks of a wider row, behind a third block
            wide = torch.full((total, page, 3 * kv * 64), math.nan, dtype=BF16, device=dev)
            self.k, self.v = (wide[:, :, i * kv * 64:(i + 1) * kv * 64].unflatten(2, (kv, 64)) for i in (1, 2))
            self.k.copy_(pools[0])
            self.v.copy_(pools[1])
        else:
            self.k, self.v = (p.to(dev) for p in pools)
        self.q = (torch.randn(B, H * 64, generator=g) * 2).to(BF16)
        self.k_new, self.v_new = (torch.randn(B, kv * 64, generator=g).to(BF16) for _ in range(2))
        self.weights = torch.rand(B, kv, self.cap, generator=g)
        self.dev = dev

    def d(self, t):
        return t.to(self.dev)

    @property
    def lengths(self):
        return torch.tensor(self.n, dtype=I32, device=self.dev)

    def reference(self, append=False):
        """o [B, H, 64] and weights in 64 bits, the bound of every o"""
        o = torch.zeros(self.B, self.H, 64, dtype=F64)
        w = self.weights.double()
        bound = torch.zeros_like(o)
        wb = torch.zeros_like(w)
        for b, n in enumerate(self.n):
            if n == 0:
                continue
            k, v = self.k_rows[b, :n].double(), self.v_rows[b, :n].double()
            if append:
                k, v = k.clone(), v.clone()
                k[n - 1], v[n - 1] = self.k_new[b].double().view(self.kv, 64), self.v_new[b].double().view(self.kv, 64)
                w[b, :, n - 1] = 0
            for h in range(self.H):
                hk = h // (self.H // self.kv)
                q = self.q[b, h * 64:(h + 1) * 64].double()
                p = torch.softmax(k[:, hk] @ q / 8, 0)
                o[b, h] = p @ v[:, hk]
                delta = 65 * 2 ** -24 * float((k[:, hk].abs() @ q.abs()).max()) / 8 * math.log2(math.e) + 2 ** -21 + n * 2 ** -24
                bound[b, h] = (2 * delta + 2 ** -17) * float(v[:, hk].abs().max()) + HALF_STEP * o[b, h].abs()
                w[b, hk, :n] += p
                wb[b, hk, :n] += 2 * delta * p + 2 ** -23 * w[b, hk, :n]
        return o.view(self.B, -1), bound.view(self.B, -1), w, wb


def within(a, ref, bound, what):
    err = (a.double().cpu() - ref).abs()
    assert bool((err <= bound).all()), f'{what}: {float((err - bound).max()):.3g} over its bound'


def same(a, b):
    """bit for bit, NaN included"""
    return torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))


SHAPES = [
    # B, H, kv, page, lengths, layout
    (1, 2, 2, 16, [1], 'head'),
    (3, 3, 3, 1, [0, 1, 5], 'row'),
    (2, 12, 12, 8, [63, 64], 'qkv'),
    (4, 4, 4, 64, [65, 0, 128, 200], 'head'),
    (2, 16, 4, 32, [300, 257], 'row'),
    (2, 6, 2, 16, [511, 30], 'head'),           # three query heads a key-value head, of the 16 that a workgroup takes
    (1, 20, 2, 16, [77], 'qkv'),                # ten
    (2, 8, 1, 128, [1025, 1024], 'head'),       # eight, split over the length
    (3, 2, 1, 64, [2049, 0, 1], 'row'),         # two, split, one sequence with fewer keys than splits
    (1, 1, 1, 256, [6189], 'head'),
    (1, 5, 5, 4096, [4097], 'row'),
]


@pytest.mark.parametrize('append', [False, True])
@pytest.mark.parametrize('weights', [False, True])
@pytest.mark.parametrize('B,H,kv,page,lengths,layout', SHAPES)
def test_paged_attention(dev, B, H, kv, page, lengths, layout, append, weights):
    from pixparse_amd import ops
    c = Case(dev, B, H, kv, page, lengths, layout, seed=sum(lengths) + H)
    ref, bound, wref, wbound = c.reference(append)
    k0, v0 = c.k.clone(), c.v.clone()
    o = torch.full((B, H * 64), 7.0, dtype=BF16, device=dev)
    w = c.d(c.weights) if weights else None
    kw = dict(k_new=c.d(c.k_new), v_new=c.d(c.v_new)) if append else {}
    ops.paged_attn_decode(c.d(c.q), c.k, c.v, c.d(c.table), c.lengths, o, H, 0.125, weights=w, **kw)
    within(o, ref, bound, 'o')
    for b, n in enumerate(lengths):
        if n == 0:
            assert not o[b].any()
        elif append:
            page_id, slot = int(c.table[b, (n - 1) // page]), (n - 1) % page
            k0[page_id, slot], v0[page_id, slot] = c.d(c.k_new[b].view(kv, 64)), c.d(c.v_new[b].view(kv, 64))
    assert same(c.k, k0) and same(c.v, v0), 'rows other than the appended ones have changed'
    if weights:
        within(w, wref, wbound + 1e-30, 'weights')
        for b, n in enumerate(lengths):
            assert torch.equal(w[b, :, n:].cpu(), c.weights[b, :, n:]), 'weights behind the length have changed'


@pytest.mark.parametrize('lengths', [[40, 45, 37], [4100, 4109, 4097]])
def test_shared_prefix_and_strided_operands(dev, lengths):
    """sequences that share the pages they only read and append to pages of their own; every operand a view into a wider tensor"""
    from pixparse_amd import ops
    c = Case(dev, 3, 4, 2, 16, lengths, 'head', seed=4)
    shared = min(lengths) // 16 - 1
    for b in (1, 2):
        c.table[b, :shared] = c.table[0, :shared]
        c.k_rows[b, :shared * 16], c.v_rows[b, :shared * 16] = c.k_rows[0, :shared * 16], c.v_rows[0, :shared * 16]
    ref, bound, wref, wbound = c.reference(append=True)
    per = c.table.shape[1]
    wide = lambda t, extra: torch.cat([c.d(t), torch.full((*t.shape[:-1], extra), -1, dtype=t.dtype, device=dev)], -1)
    qkv = torch.cat([c.d(c.q), c.d(c.k_new), c.d(c.v_new)], 1)
    table, w, o = wide(c.table, 3), wide(c.weights, 5), torch.full((3, 300), 7.0, dtype=BF16, device=dev)
    ops.paged_attn_decode(qkv[:, :256], c.k, c.v, table[:, :per], c.lengths, o[:, 20:276], 4, 0.125, k_new=qkv[:, 256:384], v_new=qkv[:, 384:],
                          weights=w[:, :, :c.cap])
    within(o[:, 20:276], ref, bound, 'o')
    within(w[:, :, :c.cap], wref, wbound + 1e-30, 'weights')
    assert bool((o[:, :20] == 7).all()) and bool((o[:, 276:] == 7).all()) and bool((w[:, :, c.cap:] == -1).all())


def test_paged_attention_matches_the_contiguous_kernel(dev):
    """the same cache as one page a sequence through attn_decode: both round once, the contiguous one its probabilities too (2^-8 each)"""
    from pixparse_amd import ops
    B, H, n = 3, 4, 1000
    g = torch.Generator(device=dev).manual_seed(1)
    q = torch.randn(B, H * 64, generator=g, device=dev).to(BF16)
    kv = torch.randn(B, 1024, 2 * H * 64, generator=g, device=dev).to(BF16)
    a, b = torch.empty_like(q), torch.empty_like(q)
    ops.attn_decode(q, kv[:, :n, :H * 64], kv[:, :n, H * 64:], a, H, 0.125)
    pages = kv.view(B * 16, 64, 2, H, 64)
    table = torch.arange(B * 16, dtype=I32, device=dev).view(B, 16)
    ops.paged_attn_decode(q, pages[:, :, 0], pages[:, :, 1], table, torch.full((B,), n, dtype=I32, device=dev), b, H, 0.125)
    vmax = float(kv[:, :, H * 64:].abs().max())
    assert float((a.float() - b.float()).abs().max()) <= 2 * HALF_STEP * float(a.abs().max()) + HALF_STEP * vmax


def test_bad_pages_and_lengths_reach_no_memory(dev):
    """(the address arithmetic itself is tested on the host) a sequence whose table or length leads outside comes out NaN, the others as ever"""
    from pixparse_amd import ops
    c = Case(dev, 6, 4, 2, 16, [40, 40, 40, 40, 40, 2000], 'head', seed=9)
    table, n = c.table.clone(), c.lengths
    table[0, 1], table[1, 2], table[2, 0] = -1, c.k.shape[0], 2 ** 31 - 1
    n[3], n[4] = c.cap + 1, -1
    ref, bound, _, _ = c.reference()
    o = torch.zeros(6, 256, dtype=BF16, device=dev)
    w = c.d(c.weights)
    ops.paged_attn_decode(c.d(c.q), c.k, c.v, c.d(table), n, o, 4, 0.125, weights=w)
    assert bool(o[:5].isnan().all())
    within(o[5:], ref[5:], bound[5:], 'o of the sound sequence')
    assert torch.equal(w[3:5].cpu(), c.weights[3:5])
    k0, v0 = c.k.clone(), c.v.clone()
    ops.paged_append(c.d(c.k_new)[:, None], c.d(c.v_new)[:, None], c.k, c.v, c.d(table), torch.tensor([20, 33, 3, c.cap, -1, 5], dtype=I32, device=dev),
                     torch.ones(6, dtype=I32, device=dev))
    for pool, row in ((k0, c.k_new), (v0, c.v_new)):
        pool[int(c.table[5, 0]), 5] = c.d(row[5].view(2, 64))
    assert same(c.k, k0) and same(c.v, v0)


def test_pool_beyond_32_bits(dev):
    """pages whose rows start more than 2^32 elements behind the base"""
    from pixparse_amd import ops
    page, kv, stride = 16, 2, 1 << 28
    base = torch.empty((1 << 32) + (1 << 20), dtype=BF16, device=dev)
    k = base.as_strided((17, page, kv, 64), (stride, kv * 128, 128, 1))
    v = base.as_strided((17, page, kv, 64), (stride, kv * 128, 128, 1), 64)
    c = Case(dev, 1, 4, kv, page, [page * 17 - 3], 'row', seed=3, extra=0)
    k.copy_(c.k)
    v.copy_(c.v)
    ref, bound, _, _ = c.reference(True)
    o = torch.empty(1, 256, dtype=BF16, device=dev)
    ops.paged_attn_decode(c.d(c.q), k, v, c.d(c.table), c.lengths, o, 4, 0.125, k_new=c.d(c.k_new), v_new=c.d(c.v_new))
    within(o, ref, bound, 'o')
    last = (c.n[0] - 1)
    assert torch.equal(k[int(c.table[0, last // page]), last % page].cpu().view(-1), c.k_new[0])


@pytest.mark.parametrize('seed', range(3))
def test_peaked_and_infinite_scores(dev, seed):
    """one key that takes everything, keys of the type's lowest value, +inf in a value row"""
    from pixparse_amd import ops
    c = Case(dev, 2, 2, 2, 32, [100, 1500], 'head', seed=seed)
    lowest = torch.finfo(BF16).min
    for b in range(2):
        c.k_rows[b, 7] = 30.0 * c.q[b, :128].view(2, 64).sign()
        c.k_rows[b, 20] = lowest * c.q[b, :128].view(2, 64).sign()
        c.v_rows[b, 7, 0, 5] = math.inf
        for pool, rows in ((c.k, c.k_rows), (c.v, c.v_rows)):
            for p in (7, 20):
                pool[int(c.table[b, p // 32]), p % 32] = c.d(rows[b, p])
    o = torch.empty(2, 128, dtype=BF16, device=dev)
    ops.paged_attn_decode(c.d(c.q), c.k, c.v, c.d(c.table), c.lengths, o, 2, 0.125)
    # (the peaked key's score is above 600 and every other's under 60: its probability is 1 in 64 bits and in 32)
    want = c.v_rows[:, 7].reshape(2, 128)
    assert torch.equal(o.cpu(), want)


@pytest.mark.parametrize('n', [5, 3000])
def test_scores_that_are_all_minus_infinity(dev, n):
    """no softmax exists: NaN as the formula has it, not the zeros of an empty sequence"""
    from pixparse_amd import ops
    c = Case(dev, 2, 1, 1, 64, [n, 0], 'head', seed=n)
    c.k[:, :, :, 0] = -math.inf
    q = c.q.clone()
    q[:, 0] = 1.0
    o = torch.zeros(2, 64, dtype=BF16, device=dev)
    ops.paged_attn_decode(c.d(q), c.k, c.v, c.d(c.table), c.lengths, o, 1, 0.125)
    assert bool(o[0].isnan().all()) and not o[1].any()


@pytest.mark.parametrize('kv,page,layout,T', [(2, 16, 'head', 1), (12, 1, 'row', 33), (3, 64, 'qkv', 130)])
def test_append(dev, kv, page, layout, T):
    from pixparse_amd import ops
    n = [200, 150, 131, 0]
    c = Case(dev, 4, kv, kv, page, n, layout, seed=T, pages=-(-340 // page))
    g = torch.Generator().manual_seed(T)
    rows = torch.randn(4, T, 3 * kv * 64, generator=g).to(BF16)
    counts = torch.tensor([T, T // 2, 0, T], dtype=I32)
    k0, v0, w0 = c.k.clone(), c.v.clone(), c.weights.clone()
    for b in range(4):
        for t in range(int(counts[b])):
            p = n[b] + t
            at = (int(c.table[b, p // page]), p % page)
            k0[at], v0[at] = (c.d(rows[b, t, i * kv * 64:(i + 1) * kv * 64].view(kv, 64)) for i in (1, 2))
            w0[b, :, p] = 0
    d, w = c.d(rows), c.d(c.weights)
    ops.paged_append(d[:, :, kv * 64:2 * kv * 64], d[:, :, 2 * kv * 64:], c.k, c.v, c.d(c.table), c.lengths, c.d(counts), weights=w)
    assert same(c.k, k0) and same(c.v, v0) and torch.equal(w.cpu(), w0)


def evict_reference(c, w, budget, recent):
    """by the definition, on the host: kept lists, then rows and weights moved"""
    k, v = c.k.cpu().clone(), c.v.cpu().clone()
    w = w.clone()
    kept = torch.full((c.B, c.kv, budget), -1, dtype=I32)
    for b, n in enumerate(c.n):
        if not 0 <= n <= c.cap:
            continue
        for h in range(c.kv):
            if n <= budget:
                kept[b, h, :n] = torch.arange(n)
                continue
            rank = lambda p: (0 if w[b, h, p] != w[b, h, p] else 1, 0.0 if w[b, h, p] != w[b, h, p] else -float(w[b, h, p]), p)
            old = sorted(range(n - recent), key=rank)[:budget - recent]
            at = sorted(old) + list(range(n - recent, n))
            kept[b, h] = torch.tensor(at)
            page = lambda p: (c.table[b].long()[torch.as_tensor(p) // c.page], torch.as_tensor(p) % c.page, h)
            for pool in (k, v):
                pool[page(list(range(budget)))] = pool[page(at)]
            w[b, h, :budget] = w[b, h, at]
    return kept, k, v, w


@pytest.mark.parametrize('in_place', [True, False])
@pytest.mark.parametrize('B,kv,page,lengths,layout,budget,recent,kind', [
    (2, 130, 16, [120, 61], 'row', 60, 7, 'random'),        # more heads than CUs
    (3, 2, 16, [100, 40, 0], 'head', 64, 16, 'random'),
    (2, 3, 1, [17, 9], 'row', 1, 0, 'random'),
    (2, 1, 8, [300, 299], 'qkv', 299, 299, 'random'),       # the window alone
    (1, 2, 64, [1500], 'head', 700, 0, 'ties'),             # more equal weights than places
    (2, 2, 32, [2100, 1024], 'row', 1023, 23, 'zeros'),     # nothing was ever looked at
    (1, 1, 128, [5000], 'head', 4999, 1, 'random'),
    (2, 2, 16, [260, 333], 'head', 77, 5, 'odd'),           # NaN, infinities, -0, subnormal and negative weights
    (1, 1, 16, [2500], 'head', 1300, 300, 'close'),         # weights that differ in their last bit
    (2, 35, 16, [1500, 1400], 'head', 1300, 9, 'random'),   # a workgroup moves whole rows, in more than one tile
    (2, 24, 64, [2600, 40], 'row', 2300, 100, 'random'),    # half rows
    (1, 32, 32, [4700], 'qkv', 4500, 100, 'random'),        # quarter rows
])
def test_evict(dev, B, kv, page, lengths, layout, budget, recent, kind, in_place):
    from pixparse_amd import ops
    c = Case(dev, B, kv, kv, page, lengths, layout, seed=budget)
    g = torch.Generator().manual_seed(budget + 1)
    w = torch.randn(c.weights.shape, generator=g).exp()
    if kind == 'ties':
        w = (w * 2).floor() / 2
    elif kind == 'zeros':
        w.zero_()
    elif kind == 'close':
        w = (torch.full(w.shape, 1.5).view(I32) + torch.randint(0, 900, w.shape, generator=g, dtype=I32)).view(F32)
    elif kind == 'odd':
        odd = torch.tensor([math.nan, math.inf, -math.inf, -0.0, 0.0, 1e-40, -1e-40, -3.0, 3.4e38])
        w = torch.where(torch.rand(w.shape, generator=g) < 0.7, odd[torch.randint(0, 9, w.shape, generator=g)], w)
    kept_ref, k_ref, v_ref, w_ref = evict_reference(c, w, budget, recent)
    n, wd, kept = c.lengths, c.d(w), torch.full((B, kv, budget), 5, dtype=I32, device=dev)
    new = n if in_place else torch.full_like(n, -9)
    ops.cache_evict(c.k, c.v, c.d(c.table), n, wd, budget, recent, new, kept=kept)
    assert torch.equal(kept.cpu(), kept_ref)
    assert new.tolist() == [min(x, budget) for x in lengths]
    assert same(c.k.cpu(), k_ref) and same(c.v.cpu(), v_ref)
    assert torch.equal(wd.cpu().view(I32), w_ref.view(I32))


def test_evict_to_more_than_there_is(dev):
    """a budget that no sequence can reach cuts nothing, and takes no memory for a list of that length"""
    from pixparse_amd import ops
    c = Case(dev, 2, 2, 2, 16, [100, 40], 'head', seed=1)
    k, v, n, new = c.k.clone(), c.v.clone(), c.lengths, torch.full_like(c.lengths, -9)
    w = c.d(torch.randn(c.weights.shape).exp())
    before = w.clone()
    for recent in (0, 10 ** 10):
        ops.cache_evict(c.k, c.v, c.d(c.table), n, w, 10 ** 12, recent, new)
        assert new.tolist() == [100, 40] and same(c.k, k) and same(c.v, v) and torch.equal(w, before)


def test_evict_leaves_bad_sequences(dev):
    from pixparse_amd import ops
    c = Case(dev, 3, 2, 2, 16, [100, 100, 100], 'head', seed=4)
    w = c.d(c.weights)
    n = torch.tensor([c.cap + 1, -5, 100], dtype=I32, device=dev)
    c.n = n.tolist()
    kept_ref, k_ref, v_ref, w_ref = evict_reference(c, c.weights, 50, 10)
    new, kept = torch.empty_like(n), torch.empty(3, 2, 50, dtype=I32, device=dev)
    ops.cache_evict(c.k, c.v, c.d(c.table), n, w, 50, 10, new, kept=kept)
    assert new.tolist() == [c.cap + 1, -5, 50] and torch.equal(kept.cpu(), kept_ref)
    assert same(c.k.cpu(), k_ref) and same(c.v.cpu(), v_ref) and torch.equal(w.cpu(), w_ref)


def _loop(c, steps, budget):
    """append + attend + gather weights, evict when the cache is full: what one layer of a generation program does"""
    from pixparse_amd import ops
    dev, B = c.dev, c.B
    g = torch.Generator(device=dev).manual_seed(11)
    rows = torch.randn(steps, 3, B, c.kv * 64, generator=g, device=dev).to(BF16)
    q = torch.randn(steps, B, c.H * 64, generator=g, device=dev).to(BF16)
    table, n, w = c.d(c.table), c.lengths, c.d(c.weights)
    outs = torch.zeros(steps, B, c.H * 64, dtype=BF16, device=dev)

    def step(q, k, v, o):
        n.add_(1)
        ops.paged_attn_decode(q, c.k, c.v, table, n, o, c.H, 0.125, k_new=k, v_new=v, weights=w)
        ops.cache_evict(c.k, c.v, table, n, w, budget, 8, n)
    return step, rows, q, outs, (n, w)


def test_loop_of_steps_captured_and_replayed(dev):
    """the loop eagerly, and as one captured step replayed with the program's own work between the replays: the same bits"""
    def fresh():
        c = Case(dev, 3, 4, 2, 16, [60, 0, 33], 'head', seed=8, pages=5)
        return c, _loop(c, 12, 64)
    c, (step, rows, q, outs, state) = fresh()
    for i in range(12):
        step(q[i], rows[i, 0], rows[i, 1], outs[i])
    torch.cuda.synchronize()
    c2, (step2, rows2, q2, outs2, state2) = fresh()
    qs, ks, vs, os = q2[0].clone(), rows2[0, 0].clone(), rows2[0, 1].clone(), outs2[0].clone()
    saved = [t.clone() for t in (c2.k, c2.v, *state2)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step2(qs, ks, vs, os)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step2(qs, ks, vs, os)
    for t, s in zip((c2.k, c2.v, *state2), saved):
        t.copy_(s)
    for i in range(12):
        qs.copy_(q2[i])
        ks.copy_(rows2[i, 0])
        vs.copy_(rows2[i, 1])
        graph.replay()
        outs2[i].copy_(os)
        assert float((outs2[i].float() * 2).sum()) == float((outs2[i].float() * 2).sum())
    torch.cuda.synchronize()
    assert torch.equal(outs, outs2) and all(torch.equal(a, b) for a, b in zip(state, state2)) and same(c.k, c2.k) and same(c.v, c2.v)
    assert state[0].tolist() == [64, 12, 45]


def test_two_streams_at_once(dev):
    """split calls of two streams, none waiting for the other: workspaces are their own"""
    from pixparse_amd import ops
    cases = [Case(dev, 4, 4, 4, 64, [3000 + i, 2500, 100, 2999], 'head', seed=i) for i in range(2)]
    args = [(c.d(c.q), c.k, c.v, c.d(c.table), c.lengths) for c in cases]
    once = []
    for c, a in zip(cases, args):
        o, w = torch.empty(4, 256, dtype=BF16, device=dev), torch.zeros(4, 4, c.cap, device=dev)
        ops.paged_attn_decode(*a, o, 4, 0.125, weights=w)
        once.append((o, w))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    many = [[(torch.empty(4, 256, dtype=BF16, device=dev), torch.zeros(4, 4, c.cap, device=dev)) for _ in range(20)] for c in cases]
    torch.cuda.synchronize()
    for i in range(20):
        for s, a, m in zip(streams, args, many):
            with torch.cuda.stream(s):
                ops.paged_attn_decode(*a, m[i][0], 4, 0.125, weights=m[i][1])
    torch.cuda.synchronize()
    for (o, w), m in zip(once, many):
        assert all(torch.equal(o, x) and torch.equal(w, y) for x, y in m)

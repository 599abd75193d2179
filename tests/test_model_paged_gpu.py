"""Generation over the paged cache and training on token scores through the model on a real MI355X."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
V, LAYERS = 515, 2


@pytest.fixture(scope='module')
def dev():
    assert torch.cuda.is_available()
    return torch.device('cuda:0')


def build(dev, L=64, B=3, seed=12):
    """a small model whose logits are spread out, its parameters for the oracle, encoder outputs of B images"""
    from oracle import ref_cpu as R
    from pixparse_amd.models import Cruller, ImageEncoderCfg, ModelCfg, TextDecoderCfg
    from pixparse_amd.models.archs import register_arch
    vit = dict(patch=8, dim=128, depth=2, heads=2, mlp_ratio=4, ln_eps=1e-6, pre_norm=False, mean=(0.5,) * 3, std=(0.5,) * 3)
    bart = dict(d_model=128, heads=2, ffn=256, ln_eps=1e-5, vocab=509, dropout=0.0)
    register_arch('vit', 'vit_test', vit)
    register_arch('bart', 'bart_test', bart)
    R.VIT_ARCHS['vit_test'], R.BART_ARCHS['bart_test'] = vit, bart
    cfg = ModelCfg(image_encoder=ImageEncoderCfg(name='vit_test', image_fmt='RGB', image_size=(37, 50), pretrained=False),
                   text_decoder=TextDecoderCfg(name='bart_test', pretrained=False, num_decoder_layers=LAYERS, max_length=L))
    torch.manual_seed(seed)
    model = Cruller(cfg, vocab_size=V)
    with torch.no_grad():
        for n, p in model.named_parameters():
            if n.endswith('.bias'):
                p.normal_(0, 0.05)
            elif p.dim() >= 2:
                p.mul_(4.0)
    params = {k: v.detach().clone() for k, v in model.state_dict().items() if not k.endswith('lm_head.weight')}
    spec = R.ModelSpec('vit_test', 'bart_test', LAYERS, L, (37, 50), 3, vocab=V)
    image, tokens, target = R.synthetic_sample(spec, B, seed=seed)
    model.to(dev)
    model._ensure_engines()
    model.refresh_shadows(full=True)
    return model, params, spec, image, tokens, target


PROMPTS = [[514, 7, 301, 44, 9, 120, 77, 300, 5, 63, 410, 513], [514], [514, 31, 8, 400, 2]]


def same(a, b):
    return all(x['ids'] == y['ids'] and torch.equal(x['logprob'], y['logprob']) and torch.equal(x['entropy'], y['entropy'])
               and torch.equal(x['top_ids'], y['top_ids']) for x, y in zip(a, b))


def test_ragged_prompts_vs_oracle(dev):
    """prompts of 12, 1 and 5 tokens in one batch: against the oracle's whole decoder on every prefix.  The bf16 policy's tolerance of the
    existing generation tests (3e-2 of the largest logit) holds for the chosen token; its log probability differs by at most twice
    that, the chosen logit's share and the log-sum-exp's."""
    from oracle import ref_cpu as R
    model, params, spec, image, _, _ = build(dev)
    enc = model.image_encoder(image.to(dev)).clone()
    steps = 10
    got = model.generate_paged(enc, PROMPTS, 2, steps, top=3, page_size=16, use_graph=False)
    assert same(got, model.generate_paged(enc, PROMPTS, 2, steps, top=3, page_size=16, use_graph=True))
    assert same(got, model.generate_paged(enc, PROMPTS, 2, steps, top=3, page_size=1, use_graph=True))
    oenc = R.encode_image(params, spec, image, 'bf16')
    for b, (prompt, g) in enumerate(zip(PROMPTS, got)):
        n = len(g['ids'])
        assert 1 <= n <= steps and g['logprob'].shape == g['entropy'].shape == (n,) and g['top_ids'].shape == (n, 3)
        assert 2 not in g['ids'][:-1] and (n == steps or g['ids'][-1] == 2)
        seq = torch.tensor([prompt + g['ids']])
        logits = R.bart_decoder_forward(params, spec.dec_arch, LAYERS, seq[:, :-1], oenc[b:b + 1], 'bf16', prefix='text_decoder.trunk.')[0].float()
        for t in range(n):
            o = logits[len(prompt) - 1 + t]
            tol = 3e-2 * max(1.0, float(o.abs().max()))
            assert float(o.max() - o[g['ids'][t]]) <= tol, (b, t)
            assert abs(float(torch.log_softmax(o, 0)[g['ids'][t]]) - float(g['logprob'][t])) <= 2 * tol, (b, t)
            assert int(g['top_ids'][t, 0]) == g['ids'][t] and bool((g['top_logprob'][t, :-1] >= g['top_logprob'][t, 1:]).all())


def test_batches_wider_than_sixteen(dev):
    """20 sequences (the contiguous cache takes 16): every sequence as it comes out of a smaller batch.  The projections run on another kernel there
    (fp32 sums in another order), so up to the bf16 tolerance of the scores of the same tokens: compared while the tokens agree"""
    model, _, _, image, _, _ = build(dev)
    enc = model.image_encoder(image.to(dev)).clone()
    many = enc.repeat(7, 1, 1)[:20]
    prompts = [PROMPTS[i % 3] for i in range(20)]
    got = model.generate_paged(many, prompts, -1, 8)
    few = model.generate_paged(enc, PROMPTS, -1, 8)
    for i, g in enumerate(got):
        ref = few[i % 3]
        assert len(g['ids']) == 8 and bool(torch.isfinite(g['logprob']).all())
        agree = next((t for t in range(8) if g['ids'][t] != ref['ids'][t]), 8)
        assert agree >= 1
        scale = 3e-2 * max(1.0, float(few[i % 3]['top_logprob'].abs().max()))
        assert float((g['logprob'][:agree] - ref['logprob'][:agree]).abs().max()) <= 2 * scale


def test_budgets(dev):
    """a budget that nothing exceeds changes nothing; one that cuts keeps the run whole: eager and replayed alike, finite scores, and the first tokens
    (before any cut) those of the uncut run"""
    model, _, _, image, _, _ = build(dev)
    enc = model.image_encoder(image.to(dev)).clone()
    S = enc.shape[1]
    plain = model.generate_paged(enc, PROMPTS, -1, 30)
    assert same(plain, model.generate_paged(enc, PROMPTS, -1, 30, self_budget=64, cross_budget=S))
    cut = dict(self_budget=16, self_recent=6, evict_every=8, cross_budget=S // 2, cross_after=5)
    a = model.generate_paged(enc, PROMPTS, -1, 30, use_graph=False, **cut)
    b = model.generate_paged(enc, PROMPTS, -1, 30, use_graph=True, **cut)
    assert same(a, b)
    for x, y in zip(a, plain):
        assert len(x['ids']) == 30 and bool(torch.isfinite(x['logprob']).all()) and x['ids'][:5] == y['ids'][:5]
    cache, cross = model._engines[1].gen['cache'], model._engines[1].gen['cross']
    assert all(16 <= n <= 24 for n in cache.lengths.tolist()) and cross.lengths.tolist() == [S // 2] * 3
    long = [p * 3 for p in PROMPTS]                     # a prompt of 36 tokens is cut to the budget after eight steps
    c = model.generate_paged(enc, long, -1, 12, **cut)
    assert all(len(x['ids']) == 12 and bool(torch.isfinite(x['logprob']).all()) for x in c)


def test_refusals(dev):
    model, _, _, image, _, _ = build(dev)
    enc = model.image_encoder(image.to(dev)).clone()
    for kw, match in ((dict(prompts=PROMPTS[:2]), 'prompts'), (dict(prompts=[[1], [], [1]]), 'prompts'), (dict(max_steps=0), 'max_steps'), (dict(max_steps=60), 'positions'),
                      (dict(top=0), 'top'), (dict(top=33), 'top'), (dict(page_size=24), 'page_size'), (dict(self_budget=4, self_recent=5), 'self_recent'), (dict(cross_budget=0), 'cross_budget')):
        with pytest.raises(ValueError, match=match):
            model.generate_paged(enc, **{**dict(prompts=PROMPTS, eos_id=2, max_steps=5), **kw})


def test_embedding_at_positions_of_their_own(dev):
    from pixparse_amd import ops
    g = torch.Generator(device=dev).manual_seed(0)
    tok, pos = torch.randn(50, 128, generator=g, device=dev), torch.randn(12, 128, generator=g, device=dev)
    ids = torch.tensor([[3], [49], [50], [-1], [0], [7]], device=dev)
    at = torch.tensor([0, 9, 1, 1, 10, -3], dtype=torch.int32, device=dev)
    out = torch.zeros(6, 128, device=dev)
    ops.embed_decode_rows(ids, tok, pos, out, at, 2)
    assert torch.equal(out[0], tok[3] + pos[2]) and torch.equal(out[1], tok[49] + pos[11]) and bool(out[2:].isnan().all())


def test_training_on_scores_is_training_on_the_loss(dev):
    """d_logprob = -1 / n_valid is the gradient of the mean cross-entropy: the same logit gradients up to one bf16 rounding of either (2^-8 of a
    value at most, so of a norm), which every later product carries linearly: 2 * 2^-8 of each gradient, with half as much again for the roundings
    of the backward pass that fall differently"""
    from oracle import ref_cpu as R
    model, _, spec, image, tokens, target = build(dev, L=32, B=2)
    ti, tt = R.shift_tokens(tokens, target)
    image, ti, tt = image.to(dev), ti.to(dev), tt.to(dev)
    model.arena.alloc_training_state()
    model.arena.g.zero_()
    loss = float(model.forward_loss(image, ti, tt))
    model.backward()
    want = model.arena.g.clone()
    model.arena.g.zero_()
    logprob, entropy = model.forward_logprobs(image, ti, tt)
    n = int((tt != -100).sum())
    logits = model._engines[2].t['dec.logits'][:, :V].double()
    ref = torch.log_softmax(logits, 1)
    valid = tt.reshape(-1) != -100
    lp = torch.where(valid, torch.gather(ref, 1, tt.reshape(-1).clamp_min(0)[:, None])[:, 0], 0.0)
    assert float((logprob.reshape(-1).double() - lp).abs().max()) <= 2e-5 and float((entropy.reshape(-1).double() + (ref.exp() * ref).sum(1)).abs().max()) <= 1e-4
    assert abs(float(-logprob.sum() / n) - loss) <= 1e-5 * max(1.0, loss)
    model.backward_logprobs(torch.full_like(logprob, -1.0 / n))
    for name in model.arena.entries:
        a, b = model.arena.grad(name).float(), None
        e = model.arena.entries[name]
        b = want[e.offset:e.offset + e.numel].view_as(a)
        norm = float(b.norm())
        assert norm == 0 and float(a.norm()) == 0 or float((a - b).norm()) <= 3 * 2 ** -8 * norm, name
    model.arena.g.zero_()
    model.forward_logprobs(image, ti, tt)
    model.backward_logprobs(None, torch.full_like(logprob, 0.1 / n))
    assert bool(torch.isfinite(model.arena.g).all()) and float(model.arena.g.norm()) > 0


def test_a_gradient_follows_the_scores_it_belongs_to(dev):
    """once, right after forward_logprobs(), in its shape; anything else is refused before a gradient is touched"""
    from oracle import ref_cpu as R
    model, _, spec, image, tokens, target = build(dev, L=32, B=2)
    ti, tt = R.shift_tokens(tokens, target)
    image, ti, tt = image.to(dev), ti.to(dev), tt.to(dev)
    model.arena.alloc_training_state()
    model.arena.g.zero_()
    d = torch.full(tt.shape, -0.1, device=dev)
    with pytest.raises(RuntimeError, match='forward_logprobs'):
        model.backward_logprobs(d)
    model.forward_logprobs(image, ti, tt)
    with pytest.raises(ValueError, match='d_logprob'):
        model.backward_logprobs(d.t())
    with pytest.raises(ValueError, match='d_entropy'):
        model.backward_logprobs(d, d.reshape(-1))
    model.forward_loss(image, ti, tt)
    with pytest.raises(RuntimeError, match='forward_logprobs'):
        model.backward_logprobs(d)
    assert not bool(model.arena.g.any())
    model.forward_logprobs(image, ti, tt)
    model.backward_logprobs(d)
    got = model.arena.g.clone()
    with pytest.raises(RuntimeError, match='forward_logprobs'):
        model.backward_logprobs(d)
    assert torch.equal(model.arena.g, got) and bool(got.any())

"""Scores of given tokens and their backward pass, and the cuts of a bounded cache, through the model on a real MI355X."""
import pytest
import torch

from tests.test_model_paged_gpu import PROMPTS, build

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def dev():
    assert torch.cuda.is_available()
    return torch.device('cuda:0')


def training(dev, seed=12):
    from oracle import ref_cpu as R
    model, _, _, image, tokens, target = build(dev, L=32, B=2, seed=seed)
    ti, tt = R.shift_tokens(tokens, target)
    model.arena.alloc_training_state()
    model.arena.g.zero_()
    return model, image.to(dev), ti.to(dev).clone(), tt.to(dev).clone()


def test_a_prompt_is_cut_by_the_attention_it_got(dev, monkeypatch):
    """A prompt longer than the budget is held whole until attention weights exist: up to the first regular cut the tokens are those of the uncut run,
    their scores up to the bf16 policy's tolerance.  At that cut every one of the 8 steps has given every head weights of sum 1: base-2 scores under 64
    less their maximum round by 2^-18 at most, once for the sum and once for the weight, v_exp by 2^-22, 43 additions by 2^-18 in all: within 2^-16
    of 1.  It keeps the positions that the definition keeps, which are not the lowest everywhere."""
    from pixparse_amd.layers import paged_cache
    model, _, _, image, _, _ = build(dev)
    enc = model.image_encoder(image.to(dev)).clone()
    long = [p * 3 for p in PROMPTS]                        # 36, 3 and 15 tokens
    budget, recent, every, steps = 16, 6, 8, 20
    plain = model.generate_paged(enc, long, -1, steps)
    cuts = []
    evict = paged_cache.PagedCache.evict

    def spy(self, b, r):
        before = [w.clone() for w in self.weights], self.lengths.clone()
        k = [t.clone() for t in self.k]
        evict(self, b, r)
        cuts.append((before, [t.clone() for t in self.k], k, self.table.clone()))
    monkeypatch.setattr(paged_cache.PagedCache, 'evict', spy)
    got = model.generate_paged(enc, long, -1, steps, self_budget=budget, self_recent=recent, evict_every=every)
    for a, b in zip(got, plain):
        assert a['ids'][:every] == b['ids'][:every]
        assert float((a['logprob'][:every] - b['logprob'][:every]).abs().max()) <= 2 * 3e-2 * max(1.0, float(b['top_logprob'].abs().max()))
        assert len(a['ids']) == steps and bool(torch.isfinite(a['logprob']).all())
    (weights, lengths), after, k, table = next(c for c in cuts if int(c[0][1].max()) > budget)
    assert lengths.tolist() == [len(p) - 1 + every for p in long]
    n = int(lengths[0])
    lowest = list(range(budget - recent)) + list(range(n - recent, n))
    others = 0
    for layer, w in enumerate(weights):
        for h in range(w.shape[1]):
            x = w[0, h, :n].double().cpu()
            assert abs(float(x.sum()) - every) <= every * 2 ** -16
            at = sorted(sorted(range(n - recent), key=lambda p: (-float(x[p]), p))[:budget - recent]) + list(range(n - recent, n))
            others += at != lowest
            size = k[layer].shape[1]
            row = lambda pool, p: pool[layer][int(table[0, p // size]), p % size, h]
            for i, p in enumerate(at):
                assert torch.equal(row(after, i), row(k, p))
    assert others > 0


def test_no_gradient_through_another_forward(dev):
    """an encoder pass in between leaves its own activations behind, and a plain backward() has no logit gradients to start from: both are refused
    before a gradient is touched, and what is still sound goes on"""
    model, image, ti, tt = training(dev)
    d = torch.full(tt.shape, -0.1, device=dev)
    model.forward_logprobs(image, ti, tt)
    model.backward_logprobs(d)
    want = model.arena.g.clone()
    model.arena.g.zero_()
    for between in (lambda: model.image_encoder(image.flip(0)), lambda: model.encode_image(image[:1]), lambda: model.encode(image)):
        model.forward_logprobs(image, ti, tt)
        between()
        for backward in (lambda: model.backward_logprobs(d), model.backward):
            with pytest.raises(RuntimeError, match='forward_logprobs'):
                backward()
    model.forward_logprobs(image, ti, tt)
    with pytest.raises(RuntimeError, match='backward_logprobs'):
        model.backward()
    assert not bool(model.arena.g.any())
    model.backward_logprobs(d)
    assert torch.equal(model.arena.g, want)
    model.forward_loss(image, ti, tt)
    model.backward()


def test_scores_belong_to_the_caller(dev):
    """the next call leaves them alone; changing them, or the targets, in place changes no gradient"""
    model, image, ti, tt = training(dev)
    logprob, entropy = model.forward_logprobs(image, ti, tt)
    kept = logprob.clone(), entropy.clone()
    d = torch.linspace(-1, 1, tt.numel(), device=dev).view(tt.shape)
    model.backward_logprobs(d, 0.1 * d)
    want = model.arena.g.clone()
    other = model.forward_logprobs(image.flip(0), ti, tt)
    assert torch.equal(logprob, kept[0]) and torch.equal(entropy, kept[1])
    assert not torch.equal(other[0], logprob) and not torch.equal(other[1], entropy)
    model.arena.g.zero_()
    logprob, entropy = model.forward_logprobs(image, ti, tt)
    logprob.zero_()
    entropy.fill_(7.0)
    tt.fill_(3)
    model.backward_logprobs(d, 0.1 * d)
    assert torch.equal(model.arena.g, want) and bool(want.any())


def test_targets_of_another_shape_are_refused(dev):
    model, image, ti, tt = training(dev)
    for bad in (tt.t(), tt.reshape(-1), tt[:, :-1]):
        with pytest.raises(ValueError, match='text_target'):
            model.forward_logprobs(image, ti, bad)


def test_training_on_scores_uses_the_configured_dropout(dev):
    """the masks of forward_loss() at the same micro-step, in both directions, also where tokens are generated in between; none with dropout=False.
    (The bounds are those of the comparison without dropout: one bf16 rounding of either logit gradient, 2^-8 of a gradient, and half as much
    again for the roundings of the backward pass.)"""
    model, image, ti, tt = training(dev)
    n = int((tt != -100).sum())
    clean = model.forward_logprobs(image, ti, tt)
    enc = model.image_encoder(image).clone()
    model.dec_arch = dict(model.dec_arch, dropout=0.25)
    model.set_train_dropout(True, seed=5)
    loss = float(model.forward_loss(image, ti, tt))
    model.backward()
    want = model.arena.g.clone()
    for generate in (False, True):
        model.set_train_dropout(True, seed=5)
        model.arena.g.zero_()
        logprob, entropy = model.forward_logprobs(image, ti, tt)
        assert abs(float(-logprob.sum() / n) - loss) <= 1e-5 * max(1.0, loss)
        if generate:
            model.generate_paged(enc, [[3, 4], [5]], -1, 3)
        model.backward_logprobs(torch.full_like(logprob, -1.0 / n))
        for name, e in model.arena.entries.items():
            a, b = model.arena.grad(name).float(), want[e.offset:e.offset + e.numel].view_as(model.arena.grad(name))
            assert float((a - b).norm()) <= 3 * 2 ** -8 * float(b.norm()), name
    # micro-steps count on as forward_loss() does: the next masks are others
    assert not torch.equal(model.forward_logprobs(image, ti, tt)[0], logprob)
    same = model.forward_logprobs(image, ti, tt, dropout=False)
    assert torch.equal(same[0], clean[0]) and torch.equal(same[1], clean[1])
    model.set_train_dropout(False)
    same = model.forward_logprobs(image, ti, tt)
    assert torch.equal(same[0], clean[0]) and torch.equal(same[1], clean[1])

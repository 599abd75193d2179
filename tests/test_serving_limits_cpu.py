"""Refusals of the serving operators that come before anything is launched, without a GPU."""
import pytest
import torch

from pixparse_amd import hip


def test_too_many_positions_for_weights_are_refused_before_the_launch():
    """2^27 positions: more blocks of 1024 than one launch takes, for the weights only.  (Nothing is launched, so no address is used.)"""
    at, page, pages = 4096, 4096, 2 ** 15
    need = hip.query('crl_paged_attn_decode_ws_bytes', 1, 1, 1, page, pages, 1)
    rc = hip.load().crl_paged_attn_decode(at, 64, at, at, page * 64, 64, page * 64, 1, page, at, pages, pages, at, 0, 0, 0, 0, at, 64, at, page * pages,
                                          page * pages, 1, 1, 1, 0.125, at, need, 0)
    assert rc == -1 and 'too many' in hip.last_error()


@pytest.mark.parametrize('check_every', [0, -1])
def test_generation_needs_steps_between_its_looks_at_the_end(check_every):
    """no steps between two looks would go round for ever"""
    from pixparse_amd.models import Cruller, ImageEncoderCfg, ModelCfg, TextDecoderCfg
    from pixparse_amd.models.archs import register_arch
    register_arch('vit', 'vit_limits', dict(patch=8, dim=128, depth=1, heads=2, mlp_ratio=4, ln_eps=1e-6, pre_norm=False, mean=(0.5,) * 3, std=(0.5,) * 3))
    register_arch('bart', 'bart_limits', dict(d_model=128, heads=2, ffn=256, ln_eps=1e-5, vocab=61, dropout=0.0))
    model = Cruller(ModelCfg(image_encoder=ImageEncoderCfg(name='vit_limits', image_fmt='RGB', image_size=(16, 16), pretrained=False),
                             text_decoder=TextDecoderCfg(name='bart_limits', pretrained=False, num_decoder_layers=1, max_length=16)), vocab_size=64)
    with pytest.raises(ValueError, match='check_every'):
        model.generate_paged(torch.zeros(1, 5, 128), [[3]], 2, 4, check_every=check_every)

"""Refusals of the serving operators that come before anything is launched, without a GPU."""
from pixparse_amd import hip


def test_too_many_positions_for_weights_are_refused_before_the_launch():
    """2^27 positions: more blocks of 1024 than one launch takes, for the weights only.  (Nothing is launched, so no address is used.)"""
    at, page, pages = 4096, 4096, 2 ** 15
    need = hip.query('crl_paged_attn_decode_ws_bytes', 1, 1, 1, page, pages, 1)
    rc = hip.load().crl_paged_attn_decode(at, 64, at, at, page * 64, 64, page * 64, 1, page, at, pages, pages, at, 0, 0, 0, 0, at, 64, at, page * pages,
                                          page * pages, 1, 1, 1, 0.125, at, need, 0)
    assert rc == -1 and 'too many' in hip.last_error()

"""Token scores and their gradient where all logits of a row share a large offset, on a real MI355X."""
import pytest
import torch

from tests.test_logprobs_gpu import F32, check, close, forward, make, reference, rel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('offset', [300.0, -3000.0, 2.0 ** 17])
def test_gradient_of_logits_with_a_large_offset(offset):
    """The scores take deviations from the maximum first, so their bounds are those of the usual logits.  The gradient starts from lse in fp32, whose
    rounding is 2^-24 |lse| at most: by that much log p is off and, relatively, p, beside the bounds of the usual case (3 rel of p, 4 rel (2 + spread) of
    log p + H).  2^17 with 2^-24: 2^-7 of p, so e^x - 1 <= 1.01 x."""
    from pixparse_amd import ops
    dev, M, V = torch.device('cuda:0'), 4, 3001
    x, target = make(M, V, F32, dev, seed=4)
    x += offset
    check(x, target, V, 3)
    _, H, lse, _, _ = forward(x, target, V)
    g = torch.Generator(device=dev).manual_seed(1)
    dl, dh = torch.randn(M, generator=g, device=dev), torch.randn(M, generator=g, device=dev)
    _, rH, rlse, logp, p, spread = reference(x, target, V)
    hit = torch.arange(V, device=dev)[None] == target[:, None]
    lpH = logp + rH[:, None]
    want = dl.double()[:, None] * (hit.double() - p) - dh.double()[:, None] * p * lpH
    e, far = rel(V), (2 ** -24 * rlse.abs())[:, None]
    g64, h64 = dl.double().abs()[:, None], dh.double().abs()[:, None]
    bound = (3 * e + 1.01 * far) * p * (g64 + h64 * lpH.abs()) + 1.01 * h64 * p * (4 * e * (2 + spread[:, None]) + far) + 2 ** -22 * (hit * g64) \
        + want.abs() * (2 ** -24 + 2 ** -22) + 2 ** -140
    d = torch.full_like(x, 3.0)
    ops.token_logprobs_bwd(x, target, V, lse, H, dl, dh, d)
    close(d[:, :V], want, bound, 'dlogits')

"""Where the scan's, the convolution's and the norm's operators can go wrong beyond ordinary calls: quotients on the border of two 8-bit numbers, rows and launches at their limits, offsets that
do not ascend, values that are not finite beside lanes and channels that are not there."""
import pytest
import torch

import vision_rwkv_amd as vr

DEV = "cuda"
pytestmark = pytest.mark.gpu


# ---- the norm ------------------------------------------------------------------------------------------------------------

def _borders(kind, C, unit):
    """Rows of results that are whole, half and quarter steps of the 8-bit type times `unit`, rounded to fp32: next to the border of two numbers, or on it."""
    if kind == torch.int8:
        t = (torch.arange(C) % 509 - 254).float() / 2
        t[0] = 127
    else:
        t = (16 + (torch.arange(C) % 64).float() / 4) * 2.0 ** ((torch.arange(C) // 64 % 12) - 8)
        t[0] = 448
    return t * unit


@pytest.mark.parametrize("kind", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("C", [64, 768, 1024, 2048, 4096, 8192, 70, 1021])
def test_eight_bits_are_the_quotient_by_the_scale(C, kind):
    """Rows of one and minus one have a root of exactly one and results that are the weights, so that scale and quotient can be said to the bit: both rounded once to fp32, the quotient then to 8 bits."""
    top = 127 if kind == torch.int8 else 448
    x = torch.where(torch.arange(3 * C).view(3, C) % 3 == 1, -1.0, 1.0)
    for unit in (1.1, 0.013, 777.7, 1.0 + 2.0 ** -23, 1.9999998, 3e33, 2e-33):
        w = _borders(kind, C, unit)
        q, scale = vr.rms_norm(x.to(DEV), w.to(DEV), eps=0.0, quantize=kind)
        want_scale = w.abs().max() / torch.tensor(float(top))
        ratio = (x * w / want_scale).clamp(-top, top)
        want = ratio.round().to(kind) if kind == torch.int8 else ratio.to(kind)
        assert (scale.cpu() == want_scale).all()
        assert torch.equal(q.cpu().view(torch.uint8), want.view(torch.uint8)), unit


@pytest.mark.parametrize("C", [768, 70])
def test_eight_bits_beside_an_infinity(C):
    """A row with an infinite result has an infinite scale: the others are zeros, the infinite one is NaN (0 in int8)."""
    x, w = torch.ones(2, C, device=DEV), torch.ones(C, device=DEV)
    w[3] = float("inf")
    for kind in (torch.float8_e4m3fn, torch.int8):
        q, scale = vr.rms_norm(x, w, eps=0.0, quantize=kind)
        others = torch.arange(C) != 3
        assert torch.isinf(scale).all() and not q.float().cpu()[:, others].any()
        assert torch.isnan(q[:, 3].float()).all() if kind != torch.int8 else not q[:, 3].any()

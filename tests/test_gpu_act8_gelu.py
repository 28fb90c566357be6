"""GPU: relative precision of the 8-bit layers' GELU where it is small.

z Phi(z) for z < 0: the tail is exp2(-(log2 e / 2) z z) t Q(t).  The constant, its product with z and the next product are rounded once each, 3 x 2^-24 of an exponent of
z^2 / 2 nats: 1.5 z^2 2^-24 of the tail.  The rest is within 2^-21: the fitted Q (5e-8), exp2 and the reciprocal (2^-23 each at most), t's own argument (two roundings, in a Q t that moves
by less than its argument: 2 x 2^-24), and the last of seven steps of the polynomial, the three products (4 x 2^-24)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_gelu_of_negative_numbers():
    from airv2x_perception_amd.opencood_iface import act8_ops as A
    z = -torch.linspace(1, 12, 64 * 1024, dtype=torch.double).float().view(64, 1024)
    want = z.double() * torch.special.erfc(-z.double() / math.sqrt(2)) / 2
    with torch.no_grad():
        got = A.gelu(z.cuda()).double().cpu()
    far = ((got - want).abs() / want.abs() / (2.0 ** -21 + 1.5 * z.double() ** 2 * 2.0 ** -24)).max()
    assert float(far) <= 1, float(far)
    # how far the claim is from the measured error, in ranges
    e = ((got - want) / want).abs()
    assert float(e[z > -2].max()) <= 2.0 ** -21 + 6 * 2.0 ** -24 and float(e.max()) <= 2.0 ** -21 + 216 * 2.0 ** -24


def test_gelu_of_large_numbers():
    from airv2x_perception_amd.opencood_iface import act8_ops as A
    z = torch.tensor([0.0, 1e-30, -1e-30, 14.0, -14.0, 1e4, -1e4, 3e38, -3e38, math.inf], dtype=torch.float32)
    z = torch.cat([z, torch.zeros(6)])[None]
    with torch.no_grad():
        got = A.gelu(z.cuda()).cpu()[0]
    assert torch.equal(got[[0, 3, 5, 7, 9]], z[0, [0, 3, 5, 7, 9]]) and (got[[4, 6, 8]].abs() <= 1e-38).all()
    assert torch.allclose(got[1:3], z[0, 1:3] / 2, rtol=1e-6, atol=0)

"""The scale of a block is its largest magnitude / 448 rounded to nearest: for every significand of exponents over the whole range."""
import pytest
import torch

from smallframework_b200 import interface as S

pytestmark = pytest.mark.gpu


# biased exponents: subnormal numbers, the smallest normal ones, those around 448 * 2^-126 (from where on a scale is above its least), ordinary ones, the largest
@pytest.mark.parametrize("exponent", [0, 1, 2, 8, 9, 10, 64, 126, 127, 128, 135, 200, 253, 254])
def test_every_significand(exponent):
    n = 1 << 21
    x, q = torch.zeros(n, 16, device="cuda"), S.Float8Buffer(n, 16)
    for part in range(4):
        bits = torch.arange(part * n, (part + 1) * n, device="cuda", dtype=torch.int32) + (exponent << 23)
        largest = bits.view(torch.float32)
        x[:, 3] = torch.where(bits % 3 == 0, -largest, largest)
        S.QuantizeBlocks(n, 16, S.FloatBuffer(data=x), q)
        # a quotient by 7 * 2^6 is a 7th of a step away from the middle between two fp32 numbers or on it, so rounding it twice rounds it right
        want = torch.where(largest > 0, (largest.double() / 448).float().clamp_min(2.0 ** -126), 1.0)
        assert torch.equal(q.scales, want)
        if exponent >= 10:
            assert (q.t.view(n, 16)[:, 3].float().abs() == 448).all()

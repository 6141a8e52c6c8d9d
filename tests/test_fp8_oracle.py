"""The FP8 oracle against torch's E4M3 conversion and against the definition of the scale (CPU)."""

import torch

from oracle import fp8_ref as ref


def test_rounding_is_e4m3s_for_every_bf16_value():
    bits = torch.arange(0, 1 << 16, dtype=torch.int32).to(torch.int16)
    x = bits.view(torch.bfloat16).double()
    x = x[x.isfinite() & (x.abs() <= 448)]
    assert torch.equal(ref.e4m3(x), x.float().to(torch.float8_e4m3fn).double())


def test_scale_is_the_smallest_power_of_two_that_fits():
    a = torch.cat([torch.exp2(torch.arange(-140, 128).double()) * m for m in (1.0, 1.5, 1.75, 1.7500001, 1.9999999)])
    a = a[(a > 0) & (a < 3.4e38)]
    s = ref.scale_of(a)
    assert (a <= 448 * s).all()
    assert ((a > 448 * s / 2) | (s == 2.0 ** -126)).all()
    assert torch.equal(torch.frexp(s)[0], torch.full_like(s, 0.5))
    assert ref.scale_of(torch.zeros(3).double()).eq(1).all()

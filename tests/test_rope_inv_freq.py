"""decoder.rope_inv_freq on the CPU, against the two published scalings for long
contexts written out one frequency at a time."""
import math

import pytest
import torch

from python.kinetic_rt.decoder import rope_inv_freq


def by_turns(f, stretch, context):
    """Wavelengths longer than the trained context are stretched, those shorter than a quarter of it kept."""
    wave = 2 * math.pi / f
    if wave < context / 4:
        return f
    if wave > context:
        return f / stretch
    smooth = (context / wave - 1) / (4 - 1)
    return (1 - smooth) * f / stretch + smooth * f


def by_index(i, f, dim, theta, stretch, context):
    """Linear in the index between the last dimension of 32 turns or more and the first of one or fewer."""
    def where(turns):
        # theta ** (-2 i / dim) * context = 2 pi turns
        return dim / 2 * math.log(context / (2 * math.pi * turns), theta)
    low, high = max(math.floor(where(32)), 0), min(math.ceil(where(1)), dim - 1)
    if low == high:
        high += 1e-3
    ramp = min(max((i - low) / (high - low), 0.0), 1.0)
    return f / stretch * ramp + f * (1 - ramp)


CASES = [(128, 500000.0, 8.0, 8192), (128, 10000.0, 16.0, 4096), (64, 10000.0, 2.0, 2048), (96, 1e6, 4.0, 32768),
         (2, 10000.0, 8.0, 8192), (128, 500000.0, 1.0, 8192)]


@pytest.mark.parametrize("dim,theta,stretch,context", CASES)
def test_llama3(dim, theta, stretch, context):
    f, factor = rope_inv_freq(torch, dim, theta, stretch, context, device="cpu", scaling="llama3")
    want = [by_turns(theta ** (-2 * i / dim), stretch, context) for i in range(dim // 2)]
    assert f.dtype == torch.float64 and f.tolist() == pytest.approx(want, rel=1e-13)
    assert factor == 1.0  # cos and sin are not scaled
    assert torch.equal(f, rope_inv_freq(torch, dim, theta, stretch, context, device="cpu")[0])


@pytest.mark.parametrize("dim,theta,stretch,context", CASES)
def test_yarn(dim, theta, stretch, context):
    f, factor = rope_inv_freq(torch, dim, theta, stretch, context, device="cpu", scaling="yarn")
    want = [by_index(i, theta ** (-2 * i / dim), dim, theta, stretch, context) for i in range(dim // 2)]
    assert f.dtype == torch.float64 and f.tolist() == pytest.approx(want, rel=1e-13)
    assert factor == pytest.approx(0.1 * math.log(stretch) + 1, rel=1e-15)


def test_yarn_bounds():
    """128 dims, base 10000, 4096 trained tokens: indexes up to 20 are kept, from 46 on divided."""
    f, _ = rope_inv_freq(torch, 128, 10000.0, 16.0, 4096, device="cpu", scaling="yarn")
    plain, factor = rope_inv_freq(torch, 128, 10000.0, device="cpu")
    assert factor == 1.0
    ratio = (f / plain).tolist()
    assert ratio[:21] == pytest.approx([1.0] * 21) and ratio[46:] == pytest.approx([1 / 16] * 18)
    assert all(a > b for a, b in zip(ratio[20:46], ratio[21:47]))


def test_refusals():
    for kw in (dict(scaling="other"), dict(stretch=0.5), dict(stretch=float("nan"))):
        with pytest.raises(ValueError, match="rope_inv_freq"):
            rope_inv_freq(torch, 128, 10000.0, device="cpu", **kw)

"""Norms and clipping factors at the ends of fp32's range (ops/clip.py, csrc/kernels/clip.hip).

The norm and the factor are 64-bit numbers.  Returned as fp32 the norm may round to infinity while the clipped values are
ordinary numbers; a factor may be subnormal in fp32 (limit 1e-3, norm 1e38) or beyond it (a large `scale`) while its products
are not.  A product is off by the factor's rounding and its own (2 x 2^-24), plus half of the type's for bf16 (2^-8) and fp16
(2^-11), plus half of the smallest step of the type below its normal range."""
import math

import pytest
import torch

from distributed_tensorflow_amd.ops import GlobalNormClip
from distributed_tensorflow_amd.ops import reference as R

gpu = pytest.mark.gpu
F, B, H = torch.float32, torch.bfloat16, torch.float16
HALF = {F: 0.0, B: 2.0 ** -8, H: 2.0 ** -11}
LEAST = {F: 2.0 ** -150, B: 2.0 ** -134 + 2.0 ** -150, H: 2.0 ** -25}        # (bf16 is rounded from fp32)


def check(got, want):
    tol = want.abs() * (2.0 ** -23 + HALF[got.dtype]) + LEAST[got.dtype]
    d = (got.double() - want).abs()
    assert bool((d <= tol).all()), f"off by {float((d / want.abs()).max()):.3g} of the value"


def values(n, top, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return ((torch.rand(n, device="cuda", generator=g) * 2 - 1) * top).to(dtype)


def lists(top):
    """A vector with a tail, an unaligned slice, a strided matrix of whole vectors and one of odd rows"""
    buf = values(4096, top, F, 1)
    return [values(70001, top, F, 2), values(4099, top, B, 3), buf[5:1000], values(64 * 40, top, F, 4).view(64, 40)[:, :16],
            values(33 * 21, top, B, 5).view(33, 21)[:, 2:19]]


@gpu
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("top,limit,scale", [
    (1e38, 1e-3, 1.0),          # factor about 1e-44: two digits in fp32
    (1e38, 3e-10, 1.0),         # about 1e-50: zero in fp32, products 1e-12
    (1e36, 1e-37, 1.0),         # products below the normal range
    (1e-30, 1e40, 1e60),        # beyond fp32
    (1e-30, 1e3, 1e60),         # scaled up, then clipped down: a factor of about 1e31
    (1e30, 1e-3, 1e-40)])       # subnormal by the scale alone
def test_factors_beyond_fp32(gpu_lib, top, limit, scale, in_place):
    tensors = lists(top)
    before = [t.double() for t in tensors]
    norm = scale * math.sqrt(sum(float(t.square().sum()) for t in before))
    factor = scale * min(1.0, limit / norm)
    got, n = GlobalNormClip(tensors, out=None if in_place else [torch.full_like(t, 7.0) for t in tensors]).clip(limit, scale=scale)
    assert float(n) == math.inf if norm > 3.5e38 else abs(float(n) - norm) <= norm * 2.0 ** -23
    for o, b in zip(got, before):
        check(o, b * factor)


@gpu
@pytest.mark.parametrize("factor_at", [2.0 ** -126, 2.0 ** -127])
def test_products_around_the_smallest_normal_factor(gpu_lib, factor_at):
    t = torch.full((1000,), 3.0e37, device="cuda")
    norm = math.sqrt(float(t.double().square().sum()))
    (got,), _ = GlobalNormClip([t], out=[torch.empty_like(t)]).clip(1.7 * factor_at * norm)
    check(got, t.double() * (1.7 * factor_at))


@gpu
def test_fp16_with_a_factor_beyond_fp32(gpu_lib):
    t = values(5000, 6e4, H)
    norm = math.sqrt(float(t.double().square().sum()))
    (got,), n = GlobalNormClip([t], out=[torch.empty_like(t)]).clip(1e-300)
    assert bool((got == 0).all()) and abs(float(n) - norm) <= norm * 2.0 ** -23
    (got,), _ = GlobalNormClip([t], out=[torch.empty_like(t)]).clip(1e300, scale=0.0)
    assert bool((got == 0).all())


# ---------------------------------------------------------------------- a norm that fp32 does not hold
def two(device):
    return [torch.full((2,), 3e38, device=device), torch.full((3,), -2e38, device=device)]


def test_reference_goes_by_the_norm_in_64_bits():
    out, norm = R.clip_by_global_norm(two("cpu"), 1.0)
    want = math.sqrt(2 * 9.0 + 3 * 4.0) * 1e38
    assert float(norm) == pytest.approx(want, rel=1e-6)
    assert torch.allclose(out[0].double(), torch.full((2,), 3e38 / want, dtype=torch.float64), rtol=1e-6)


@gpu
@pytest.mark.parametrize("in_place", [False, True])
def test_a_norm_beyond_fp32_is_returned_as_infinity_and_clips(gpu_lib, in_place):
    tensors = two("cuda")
    norm = math.sqrt(2 * float(tensors[0][0]) ** 2 + 3 * float(tensors[1][0]) ** 2)
    before = [t.double() for t in tensors]
    got, n = GlobalNormClip(tensors, out=None if in_place else [torch.empty_like(t) for t in tensors]).clip(2.0)
    assert float(n) == math.inf and float(GlobalNormClip([t.clone() for t in two("cuda")]).norm()) == math.inf
    for o, b in zip(got, before):
        check(o, b * (2.0 / norm))
    # within the limit nothing changes
    tensors = two("cuda")
    got, n = GlobalNormClip(tensors).clip(1e39)
    assert float(n) == math.inf and all(torch.equal(o, b) for o, b in zip(got, two("cuda")))

"""CPU: the polynomials of the score modifiers, restated in numpy float32: the
decode's tanh cap (mod_cap in paged_decode_impl.cuh), the prefill's
(chunked_prefill_impl.cuh) and its quartic exp2 (exp2_fma4)."""
import numpy as np
import pytest

f32 = np.float32


def fma(a, b, c):
    return (np.float64(a) * np.float64(b) + np.float64(c)).astype(f32)


def decode_cap(z, cap2):
    """mod_cap with an exact exponential: z and the cap in the exp2 domain."""
    z, cap2 = np.asarray(z, f32), f32(cap2)
    with np.errstate(over="ignore", under="ignore"):
        u = (z * (f32(1) / cap2)).astype(f32)
        t = u * u
        p = fma(fma(fma(f32(0.017241478), t, f32(-0.05304549)), t, f32(0.13325879)), t, f32(-0.33333144))
        near = fma(z * t, p, z)
        e = np.exp2((u * f32(2.8853900817779268)).astype(np.float64)).astype(f32)
        far = fma(f32(-2) * cap2, f32(1) / (f32(1) + e), cap2)
    return np.where(np.abs(u) <= f32(0.5), near, far)


@pytest.mark.parametrize("cap2", [1e-30, 1e-9, 1e-3, 1.0, 72.0, 1.4e4, 1.4e6, 1.4e30, 1.6e38])
def test_decode_cap_error_follows_the_score(cap2):
    """Relative to the score: 2^-21 (each rounding in the polynomial form is one of a number near it; the
    exponential form's roundings are of numbers up to 2 c, and its score is above 0.46 c)."""
    z = np.concatenate([np.geomspace(1e-6, 1e5, 200_001), np.geomspace(1e-3, 30.0, 200_001) * min(cap2, 1e37)]).astype(f32)
    z = np.concatenate([z, -z])
    ref = cap2 * np.tanh(z.astype(np.float64) / np.float64(f32(cap2)))
    got = decode_cap(z, cap2).astype(np.float64)
    assert np.isfinite(got).all()
    normal = np.abs(ref) > 1e-36
    assert (np.abs(got - ref)[normal] <= 2.0 ** -21 * np.abs(ref)[normal]).all()
    assert decode_cap(f32(0), cap2) == 0


def test_prefill_tanh_polynomial():
    u = np.linspace(1e-4, 0.5, 500_001)
    t = u * u
    got = u * (((-0.044402227 * t + 0.13190296) * t - 0.3332632) * t + 0.99999946)
    assert np.abs(got / np.tanh(u) - 1).max() < 5.6e-7


def test_prefill_quartic_exp2():
    x = np.linspace(-125.9, 9.0, 2_000_001, dtype=f32)
    t = x + f32(12582912.0)
    f = (x - (t - f32(12582912.0))).astype(f32)
    p = fma(fma(fma(fma(f32(0.0095701), f, f32(0.05591786)), f, f32(0.24024745)), f, f32(0.69312181)), f, f32(0.99999926))
    got = (p.view(np.int32) + ((t.view(np.int32) - np.int32(0x4B400000)) << 23)).view(f32).astype(np.float64)
    assert np.abs(got / np.exp2(x.astype(np.float64)) - 1).max() < 2.7e-6

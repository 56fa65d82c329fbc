"""The accuracy mode's masked attention (fp32) is fp32 arithmetic: bounds that operands rounded
to fewer bits, or a coarser exponential, do not meet (shown here on the CPU), and the kernels
against them on the B200."""

import math

import pytest
import torch

import fp8_reference as ref
import ltx_nn

U = 2.0 ** -24  # half a step of fp32, relative
NORM = 1e-5


def inputs(seed, b, tq, tk, h, d, std, dev="cpu"):
    g = torch.Generator(device=dev).manual_seed(seed)
    q, k, v = (torch.randn(b, t, h * d, generator=g, device=dev) for t in (tq, tk, tk))
    keep = torch.rand(b, tk, generator=g, device=dev) < 0.7
    keep[:, 0] = True
    return q * std, k, v, keep


def errors(got, q, k, v, h, keep, scale):
    """(largest error in units of its bound, error of the norm) of got against float64.

    Elements: a score is a sum of d products (off by (d + 4) U of sum|q k| scale: the additions,
    and the roundings of the scale and of q or the result by it), reduced by the maximum (U of
    both) and exponentiated (4 U), so a weight is off by E = U ((d + 4) sum|q k| scale + 2 max|s| + 4),
    numerator and denominator; their sums add Tk + 8 roundings: (2 E + (Tk + 8) U) sum w|v| / sum w.
    Norm: these roundings are independent. For unit k and |q| up to 3 the root mean square of a
    weight's error is below 30 U (scores below 40: their own rounding is 0.3 U 40, the dot
    product's 0.3 U sqrt(d) 3), a sum's over 9000 keys below 0.3 U sqrt(9000) = 30 U of the
    result, so 1e-5 = 168 U is passed with room to spare."""
    cpu = [t.double().cpu() for t in (q, k, v)]
    lo = ~keep.cpu()
    d = q.shape[-1] // h
    want = ref.attention(*cpu, h, lo, None, None, scale)
    size = ref.attention(cpu[0], cpu[1], cpu[2].abs(), h, lo, None, None, scale)
    bound = torch.empty_like(size)
    for i in range(q.shape[0]):
        for c in range(0, q.shape[-1], d):
            qa, ka = cpu[0][i, :, c:c + d], cpu[1][i, keep[i].cpu(), c:c + d]
            s = (qa.abs() @ ka.abs().t()).amax(1) * scale
            m = (qa @ ka.t()).abs().amax(1) * scale
            bound[i, :, c:c + d] = (2 * U * ((d + 4) * s + 2 * m + 4) + (k.shape[1] + 8) * U)[:, None]
    err = got.double().cpu() - want
    return float((err.abs() / (bound * size)).max()), float(err.norm() / want.norm())


def rounded(x, bits):
    """x rounded to `bits` significant bits."""
    m, e = torch.frexp(x.double())
    return torch.ldexp(torch.round(torch.ldexp(m, torch.full_like(e, bits))), e - bits)


CASES = [(1, 3, 300, 2, 64), (2, 40, 129, 2, 128), (1, 5, 4000, 1, 64), (2, 60, 200, 2, 32)]


@pytest.mark.parametrize("std", [1.0, 3.0])
@pytest.mark.parametrize("b,tq,tk,h,d", CASES)
def test_the_bounds_tell_fp32_from_less(b, tq, tk, h, d, std):
    q, k, v, keep = inputs(b + tk, b, tq, tk, h, d, std)
    scale = d ** -0.5

    def norm_error(o):
        return errors(o, q, k, v, h, keep, scale)[1]

    # fp32 all the way passes both
    o = torch.empty_like(q)
    for i in range(b):
        for c in range(0, h * d, d):
            s = (q[i, :, c:c + d] @ k[i, keep[i], c:c + d].t()) * scale
            p = torch.exp(s - s.amax(1, keepdim=True))
            o[i, :, c:c + d] = (p @ v[i, keep[i], c:c + d]) / p.sum(1, keepdim=True)
    worst, norm = errors(o, q, k, v, h, keep, scale)
    assert worst <= 1 and norm <= NORM
    # operands of 11 bits (TF32) and 8 (bf16) do not
    for bits in (11, 8):
        t = [rounded(x, bits) for x in (q, k, v)]
        assert norm_error(ref.attention(*t, h, ~keep, None, None, scale)) > 2 * NORM
        t = [rounded(q, bits), rounded(k, bits), v.double()]
        assert norm_error(ref.attention(*t, h, ~keep, None, None, scale)) > 2 * NORM
    # nor does an exponential of 2^-13 relative error
    o = torch.empty(b, tq, h * d, dtype=torch.float64)
    for i in range(b):
        for c in range(0, h * d, d):
            s = (q[i, :, c:c + d].double() @ k[i, keep[i], c:c + d].double().t()) * scale
            x = (s - s.amax(1, keepdim=True)) / math.log(2)
            f = x - torch.round(x)
            p = torch.ldexp(((0.0551708005 * f + 0.242609262) * f + 0.693260968) * f + 0.999928176, torch.round(x))
            o[i, :, c:c + d] = (p @ v[i, keep[i], c:c + d].double()) / p.sum(1, keepdim=True)
    assert norm_error(o) > 1.5 * NORM


@pytest.mark.gpu
@pytest.mark.parametrize("std", [1.0, 3.0])
@pytest.mark.parametrize("b,tq,tk,h,d", [*CASES, (1, 1, 9000, 2, 128), (2, 300, 129, 3, 64), (10, 129, 70, 8, 64),
                                         (20, 129, 40, 15, 128), (19, 5, 33, 8, 32), (30, 200, 100, 6, 32),
                                         (1, 480, 200, 8, 64)])
def test_fp32_masked_attention_is_fp32(b, tq, tk, h, d, std):
    q, k, v, keep = inputs(b + tk, b, tq, tk, h, d, std, "cuda")
    got = ltx_nn.cross_attention(q, k, v, h, mask=keep)
    worst, norm = errors(got, q, k, v, h, keep, d ** -0.5)
    assert worst <= 1 and norm <= NORM, (worst, norm)

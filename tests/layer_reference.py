"""Plain 64-bit forms of the operators in ``liteform_ae_b200.layer`` and bounds on what 32-bit sums and one rounding
may be off, for the tests.  ``U`` is half a step of a type (torch.finfo(t).eps / 2); terms below the smallest normal
number add ``TINY``."""
import math

import torch

U = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn)}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh"]


def act(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "silu":
        return z * torch.special.expit(z)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def slope(z, name):
    z = z.detach().clone().requires_grad_(True)
    y = act(z, name)
    g, = torch.autograd.grad(y.sum(), z)
    return torch.where(z > 0, 1.0, 0.0).double() if name == "relu" else g


def dense(indptr, indices, vals, shape):
    """A as a dense 64-bit matrix (CPU)."""
    a = torch.zeros(shape, dtype=torch.float64)
    rows = torch.repeat_interleave(torch.arange(shape[0]), torch.diff(indptr))
    a[rows, indices.long()] = vals.double() if vals is not None else 1.0
    return a


# Errors of the activations in 32 bits, absolute, for |z| as given: the special function unit's 2^x and 1 / x are off by
# at most 2^-22 relative (4 units of 2^-24) and the series for the normal distribution by 7.5e-8 (1.3 units), 1 + e and
# the products by half a unit; where the exponential's argument is rounded (|t| 2^-24 relative in e^t, and |t| e^-t / (1 +
# e^-t) <= 0.28) or the distribution is near 1 the error is absolute in what z is multiplied with.  16 units cover each
# form with room; the slopes add products of the same terms with factors up to |z| (silu, gelu) and 1.6 |z| (1 + 0.134 z^2)
# where the sigmoid's complement is not 0 (the product of both stays below 3), for which 64 units are allowed.
def act_error(z):
    return 16 * U[torch.float32] * z.abs()


SLOPE_ERROR = 64 * 2.0 ** -24


def rounded(value, off, dtype):
    """What a value known to +- `off` may be off after its rounding to `dtype`."""
    return off + U[dtype] * (value.abs() + off) + TINY[dtype]


def product(A, B, bias, name, residual, out_dtype):
    """(z, y, bound of z, bound of y), A dense in 64 bits; B the rows as they stand (scaled)."""
    n = (A != 0).sum(1, keepdim=True).double()
    z = A @ B
    size = A.abs() @ B.abs()
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs()
    # n products and n additions in any order, the scale's product and the bias: at most n + 3 roundings a term
    zoff = (n + 3) * U[torch.float32] * 1.01 * size + n * TINY[torch.float32]
    y = act(z, name)
    yoff = 1.13 * zoff + (act_error(z) if name not in ("none", "relu") else 0)     # slopes stay within 1.13
    if residual is not None:
        y = y + residual.double()
        yoff = yoff + U[torch.float32] * (y.abs() + yoff)
    return z, y, rounded(z, zoff, out_dtype), rounded(y, yoff, out_dtype)


def close(got, want, bound, what=""):
    got = got.detach().cpu().double()
    off = (got - want).abs()
    bad = ~(off <= bound)
    if bool(bad.any()):
        i = tuple(int(v) for v in torch.nonzero(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; first at {i}: {float(got[i])!r} for "
                             f"{float(want[i])!r}, bound {float(bound.expand_as(want)[i])!r}")

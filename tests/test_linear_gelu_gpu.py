"""gelu and its slope where they are small: relative to their own value, over all of f32's range."""
import importlib
import math

import pytest

from test_linear_gpu import dt

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def wl():
    return importlib.import_module("7_b200.wave_linear")


def values(torch, io):
    """Both signs, from 2^-20 to where the normal distribution's tail leaves f32 (|z| = 13), as they are in the type."""
    far = torch.arange(1, 417, device="cuda", dtype=torch.float64) / 32
    near = 2.0 ** -torch.arange(1, 21, device="cuda", dtype=torch.float64)
    z = torch.cat([far, near]).to(dt(torch, io))
    z = torch.cat([z, -z, torch.zeros(8, device="cuda", dtype=z.dtype)])
    return z[: z.numel() // 8 * 8]


def tail_error(z):
    """Bound of the relative error of the kernels' tail Q(|z|) = e^(-z^2/2) t P(t), t = 1 / (1 + 0.3 |z|):
    the exponent -z^2/2 log2 e is off by its constant's and two products' roundings, 3 * 2^-24 of itself, so its power
    by 3 * 2^-24 z^2/2, and by 2^-22 for the unit that raises it; t by three roundings and the unit's 2^-23, which t P(t)
    takes at most 2.7-fold (t (t P)' / t P <= 2.66, at t = 1); P's eight steps round by 2^-24 each of at most 1.84 P
    (the sum of magnitudes at t = 1); the polynomial is off by 1.5e-7; three more products."""
    return 3 * 2.0 ** -24 * z * z / 2 + 2.0 ** -22 + 2.7 * (3 * 2.0 ** -24 + 2.0 ** -23) + 1.84 * 8 * 2.0 ** -24 + 1.5e-7 + 3 * 2.0 ** -24


@pytest.mark.parametrize("tokens", [1, 436])  # features on the tile's rows and on its columns
@pytest.mark.parametrize("io", ["bf16", "f16"])
def test_gelu_of_far_values(cuda, wc, wl, io, tokens):
    torch = cuda
    z = values(torch, io)
    eye = torch.eye(8, device="cuda", dtype=z.dtype)
    x = z.reshape(-1, 8)
    for rows in ([x.repeat(4, 1)] if tokens > 1 else x[::7].split(1)):
        a = rows.double().abs()
        q = torch.special.erfc(a / math.sqrt(2)) / 2
        exact = torch.where(rows < 0, -a * q, a - a * q)
        for out in (torch.float32, z.dtype):
            y = wl.linear(rows, eye, activation="gelu", out_dtype=out)
            # (a tail that leaves f32's range of normal numbers is 0: 16 * 2^-126; the sum for z > 0 rounds once more)
            limit = a * q * tail_error(a) + 2.0 ** -24 * exact.abs() + 16 * 2.0 ** -126
            if out != torch.float32:
                limit = limit + torch.finfo(out).eps / 2 * exact.abs() + torch.finfo(out).smallest_normal * torch.finfo(out).eps
            assert bool(((y.double() - exact).abs() <= limit).all()), float(((y.double() - exact).abs() / limit).max())
    wc.check_device_status()


@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("io", ["bf16", "f16"])
def test_gelu_slope_of_far_values(cuda, wc, wl, io, rows):
    """dbias in f32 of one row of dy = 1 is the slope itself, unrounded (of 300 rows, 299 of them 0: the same)."""
    torch = cuda
    z = values(torch, io)
    n = z.numel()
    dy = torch.zeros(rows, n, device="cuda", dtype=z.dtype)
    dy[rows // 2] = 1
    x, w = torch.zeros(rows, 8, device="cuda", dtype=z.dtype), torch.zeros(n, 8, device="cuda", dtype=z.dtype)
    db = wl.linear_backward(dy, x, w, activation="gelu", pre_activation=z.expand(rows, n).contiguous(), need_dx=False,
                            need_dweight=False)[2].double()
    a = z.double().abs()
    q, phi = torch.special.erfc(a / math.sqrt(2)) / 2, torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)
    exact = torch.where(z < 0, q - a * phi, 1 - q + a * phi)
    # both parts by the tail's error (phi has the power's part of it, and a constant), their sum and 1 - q round once more each
    limit = (q + a * phi) * (tail_error(a) + 2 * 2.0 ** -24) + 2 * 2.0 ** -24 * exact.abs() + 32 * 2.0 ** -126
    assert bool(((db - exact).abs() <= limit).all()), float(((db - exact).abs() / limit).max())
    wc.check_device_status()

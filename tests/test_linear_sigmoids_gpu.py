"""silu, gelu_tanh and their slopes relative to their own value, over all of f32's range."""
import importlib
import math

import pytest

from test_linear_gpu import dt
from test_linear_gelu_gpu import values

pytestmark = pytest.mark.gpu
H = 2.0 ** -24  # half a step of f32


@pytest.fixture(scope="module")
def wl():
    return importlib.import_module("7_b200.wave_linear")


def parts(torch, act, z):
    """In 64 bits: s = 1 / (1 + e^-v), 1 - s, z v' and a bound of s' relative error.  y = z s, slope = s (1 + (1 - s) z v').

    v = z for silu, 2 sqrt(2/pi) (z + 0.044715 z^3) for gelu_tanh; the kernels raise 2 to -v log2 e, which is off by the
    roundings on the way: 2 of them (the constant, the product), or 8 (z^2, two constants of up to three products each,
    their sum, the product with z), 2^-24 of v each.  2^-22 for the unit that raises it, half a step for 1 + e, 2^-23
    for the reciprocal."""
    z = z.double()
    c, a = 2 * math.sqrt(2 / math.pi), 0.044715
    v = z if act == "silu" else c * (z + a * z ** 3)
    zv = z if act == "silu" else c * (z + 3 * a * z ** 3)
    s, rest = 1 / (1 + torch.exp(-v)), 1 / (1 + torch.exp(v))
    return z, s, rest, zv, (2 if act == "silu" else 8) * H * v.abs() + 2.0 ** -22 + H + 2.0 ** -23


def wide(torch, io, act):
    z = values(torch, io)
    return z if act == "gelu_tanh" else torch.cat([z, z * 8])  # e^z leaves f32 at 88


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("io", ["bf16", "f16"])
def test_values(cuda, wc, wl, io, act):
    torch = cuda
    x = wide(torch, io, act).reshape(-1, 8)
    eye = torch.eye(8, device="cuda", dtype=x.dtype)
    z, s, _, _, es = parts(torch, act, x)
    exact = z * s
    for out in (torch.float32, x.dtype):
        y = wl.linear(x, eye, activation=act, out_dtype=out)
        # (an e^-v beyond f32 makes s 0: below 2^-126 times |z| <= 104)
        limit = exact.abs() * (es + H) + 104 * 2.0 ** -126
        if out != torch.float32:
            limit = limit + torch.finfo(out).eps / 2 * exact.abs() + torch.finfo(out).smallest_normal * torch.finfo(out).eps
        assert bool(((y.double() - exact).abs() <= limit).all()), float(((y.double() - exact).abs() / limit).max())
    wc.check_device_status()


@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("io", ["bf16", "f16"])
def test_slopes(cuda, wc, wl, io, act, rows):
    """dbias in f32 of one row of dy = 1 is the slope itself, unrounded."""
    torch = cuda
    x = wide(torch, io, act)
    n = x.numel()
    dy = torch.zeros(rows, n, device="cuda", dtype=x.dtype)
    dy[rows // 2] = 1
    zeros = torch.zeros(max(rows, n), 8, device="cuda", dtype=x.dtype)
    db = wl.linear_backward(dy, zeros[:rows], zeros[:n], activation=act, pre_activation=x.expand(rows, n).contiguous(),
                            need_dx=False, need_dweight=False)[2].double()
    _, s, rest, zv, es = parts(torch, act, x)
    exact = s * (1 + rest * zv)
    size = s * (1 + rest * zv.abs())
    # s once in front; 1 - s is off by s' error and a rounding of its own; z v' by at most five roundings; the sum and the
    # product round once each.  (s and s z v' below 2^-126 may be 0; |z v'| <= 104 where s is not.)
    limit = es * exact.abs() + s * zv.abs() * (s * es + H * rest) + 7 * H * size + (1 + 2 * 300) * 2.0 ** -126
    assert bool(((db - exact).abs() <= limit).all()), float(((db - exact).abs() / limit).max())
    wc.check_device_status()

"""The linear layers on the GPU against plain 64-bit arithmetic.

Most inputs are multiples of 1/4 in [-2, 2]: products are multiples of 1/16, and
with up to 2^17 of them every partial sum is below 2^24 sixteenths, exact in f32
in any order and with any rounding.  What the kernels return must then be the
exact value rounded once -- compared bit for bit, in every layout, tile and
split.  The smooth activations are compared with tolerances derived beside them.
"""
import importlib
import math

import pytest

from _util import env_knobs

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def wl():
    return importlib.import_module("7_b200.wave_linear")


def dt(torch, name):
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


def quarters(torch, gen, *shape, io):
    return (torch.randint(-8, 9, shape, generator=gen, device="cuda") / 4).to(dt(torch, io))


def make_gen(torch, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def activate(torch, z, act):
    if act == "none":
        return z
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    u = z if act == "silu" else 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    return z * torch.sigmoid(u)


def slope(torch, z, act):
    z = z.detach().clone().requires_grad_(True)
    if act == "relu":
        return (z.detach() > 0).double()
    activate(torch, z, act).sum().backward()
    return z.grad


def same(torch, got, want, what):
    """`want` in 64 bits, rounded once to got's type: equal bit for bit (0 and -0 alike)."""
    want = want.to(torch.float32).to(got.dtype)
    assert got.shape == want.shape
    differ = int((got != want).sum())
    assert differ == 0, f"{what}: {differ} of {want.numel()} values differ, largest by {float((got.double() - want.double()).abs().max())}"


def strided(torch, t, gap):
    """The same values with `gap` more elements (of NaN) between rows."""
    if not gap:
        return t
    wide = torch.full((*t.shape[:-1], t.shape[-1] + gap), float("nan"), dtype=t.dtype, device=t.device)
    wide[..., : t.shape[-1]] = t
    return wide[..., : t.shape[-1]]


def offsets_of(torch, sizes, front=0):
    o = torch.zeros(len(sizes) + 1, dtype=torch.int64)
    o[1:] = torch.tensor(sizes).cumsum(0)
    return (o + front).to(torch.int32).cuda()


def forward_want(torch, x, w, b, r, act):
    z = x.double() @ w.double().t()
    if b is not None:
        z = z + b.double()
    y = activate(torch, z, act)
    return z, y if r is None else y + r.double()


SIZES = [(1, 1, 1), (1, 8, 8), (1, 200, 1000), (2, 129, 63), (15, 128, 64), (16, 130, 72), (17, 257, 65), (33, 64, 640),
         (64, 1000, 200), (65, 384, 136), (127, 255, 129), (128, 128, 1), (129, 511, 40), (200, 72, 2050), (300, 640, 264),
         (515, 1032, 776)]


@pytest.mark.parametrize("io,out", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_forward_exact(cuda, wc, wl, m, n, k, io, out):
    torch, gen = cuda, make_gen(cuda, m + n + k)
    x, w = quarters(torch, gen, m, k, io=io), quarters(torch, gen, n, k, io=io)
    b, r = quarters(torch, gen, n, io=io), quarters(torch, gen, m, n, io=io)
    for bias, res, act in ((None, None, "none"), (b, None, "relu"), (b.float(), r, "none"), (None, r, "relu")):
        z, y = forward_want(torch, x, w, bias, res, act)
        got, got_z = wl.linear(x, w, bias, res, activation=act, out_dtype=dt(torch, out), save_pre_activation=True)
        same(torch, got, y, "y")
        same(torch, got_z, z, "z")
    wc.check_device_status()


@pytest.mark.parametrize("gap", [1, 3, 7, 8, 40])
@pytest.mark.parametrize("m,n,k", [(5, 40, 64), (140, 96, 200), (300, 33, 65)])
def test_forward_strided_rows(cuda, wc, wl, m, n, k, gap):
    """Every operand with gaps between its rows (filled with NaN), outputs written between guard values."""
    torch, gen = cuda, make_gen(cuda, gap)
    x, w = (strided(torch, quarters(torch, gen, a, k, io="f16"), gap) for a in (m, n))
    r = strided(torch, quarters(torch, gen, m, n, io="f16"), gap)
    for t in (torch.float16, torch.float32):
        wide = torch.full((m, n + gap), 7.0, dtype=t, device="cuda")
        _, y = forward_want(torch, x, w, None, r, "relu")
        got = wl.linear(x, w, None, r, activation="relu", out=wide[:, :n])
        assert got.data_ptr() == wide.data_ptr()
        same(torch, got, y, "y")
        assert bool((wide[:, n:] == 7).all())
    # views that start off a 16-byte boundary
    x1, w1 = x[:, 1:], w[:, 1:]
    same(torch, wl.linear(x1, w1), x1.double() @ w1.double().t(), "off a boundary")
    wc.check_device_status()


@pytest.mark.parametrize("swap", [0, 1])
@pytest.mark.parametrize("tile", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("splits", [1, 2, 3, 5, 8])
def test_every_tile_and_split(cuda, wc, wl, tile, splits, swap):
    """Forward and backward in each variant of the one-CTA kernel, sizes that divide by nothing."""
    gen = make_gen(cuda, tile * 10 + splits)
    with env_knobs(wc, WAVE_CUDA_LINEAR_TILE=tile, WAVE_CUDA_LINEAR_SPLITS=splits, WAVE_CUDA_LINEAR_SWAP=swap):
        check_all(cuda, wc, wl, gen, ((45, 300, 712), (261, 136, 330)))


def test_pairs(cuda, wc, wl):
    """The same on CTA pairs: one tile and less, ragged edges, several tiles, experts with a handful of rows."""
    with env_knobs(wc, WAVE_CUDA_LINEAR_SWAP=0, WAVE_CUDA_LINEAR_PAIR=1):
        check_all(cuda, wc, wl, make_gen(cuda, 3), ((45, 300, 712), (261, 136, 330), (1000, 520, 1032), (513, 1001, 777)))
        # more tiles than pairs, several cut stages of one expert after the other in the ring
        check_all(cuda, wc, wl, make_gen(cuda, 4), ((300, 2504, 2568),), [3, 17, 0, 5, 33, 1, 2, 64, 80, 15, 16, 40])


@pytest.mark.parametrize("pair", [0, 1])
def test_bands_of_tiles(cuda, wc, wl, pair):
    """More row blocks than a band of the walk over the tiles has, with a last band that is cut short."""
    with env_knobs(wc, WAVE_CUDA_LINEAR_SWAP=0, WAVE_CUDA_LINEAR_PAIR=pair):
        check_all(cuda, wc, wl, make_gen(cuda, 5), ((4700, 328, 72), (2700, 1160, 136)), [2500, 0, 60, 17])
    with env_knobs(wc, WAVE_CUDA_LINEAR_SWAP=1, WAVE_CUDA_LINEAR_TILE=16):
        check_all(cuda, wc, wl, make_gen(cuda, 6), ((700, 2440, 72),), [500, 0, 60, 17])


def check_all(torch, wc, wl, gen, shapes, rows=None):
    for m, n, k in shapes:
        x, w, dy = (quarters(torch, gen, *s, io="bf16") for s in ((m, k), (n, k), (m, n)))
        b, r = quarters(torch, gen, n, io="bf16"), quarters(torch, gen, m, n, io="bf16")
        z, y = forward_want(torch, x, w, b, r, "relu")
        for out in (torch.bfloat16, torch.float32):
            got, got_z = wl.linear(x, w, b, r, activation="relu", out_dtype=out, save_pre_activation=True)
            same(torch, got, y, "y")
            same(torch, got_z, z, "z")
            dx, dw, db = wl.linear_backward(dy, x, w, dweight_dtype=out)
            same(torch, dx, dy.double() @ w.double(), "dx")
            same(torch, dw, dy.double().t() @ x.double(), "dw")
            same(torch, db, dy.double().sum(0), "db")
        sizes = rows or [0, 17, 0, 1, m - 20, 0]
        off = offsets_of(torch, sizes, 1)
        wg = quarters(torch, gen, len(sizes), n, k, io="bf16")
        want_y, want_dx, want_dw, want_db = grouped_want(torch, x, wg, off, None, "none", dy)
        for out in (torch.bfloat16, torch.float32):
            same(torch, wl.grouped_linear(x, wg, off, out_dtype=out), want_y, "grouped y")
            dx, dw, db = wl.grouped_linear_backward(dy, x, wg, off, dweight_dtype=out)
            same(torch, dx, want_dx, "grouped dx")
            same(torch, dw, want_dw, "grouped dw")
            same(torch, db, want_db, "grouped db")
    wc.check_device_status()


def grouped_want(torch, x, w, off, b, act, dy=None, z_in=None):
    """By loops over the experts: y (and z), or with dy the gradients; zero where no expert has rows."""
    ends = torch.cummax(off.long().clamp(0, x.shape[0]), 0).values.tolist()
    y = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device="cuda")
    z = y.clone()
    dx = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    dw = torch.zeros(w.shape, dtype=torch.float64, device="cuda")
    db = torch.zeros(w.shape[:2], dtype=torch.float64, device="cuda")
    for g, (lo, hi) in enumerate(zip(ends[:-1], ends[1:])):
        if hi <= lo:
            continue
        z[lo:hi] = x[lo:hi].double() @ w[g].double().t()
        if b is not None:
            z[lo:hi] += b[g].double()
        y[lo:hi] = activate(torch, z[lo:hi], act)
        if dy is not None:
            dz = dy[lo:hi].double()
            if z_in is not None:
                dz = dz * slope(torch, z_in[lo:hi].double(), act)
            dx[lo:hi] = dz @ w[g].double()
            dw[g] = dz.t() @ x[lo:hi].double()
            db[g] = dz.sum(0)
    return (z, y) if dy is None and b is not None else (y, dx, dw, db) if dy is not None else y


@pytest.mark.parametrize("io", ["bf16", "f16"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_backward_exact(cuda, wc, wl, m, n, k, io):
    """relu passes dy or nothing, so dz and every sum are exact."""
    torch, gen = cuda, make_gen(cuda, m * n + k)
    x, w, dy, z = (quarters(torch, gen, *s, io=io) for s in ((m, k), (n, k), (m, n), (m, n)))
    dz = dy.double() * slope(torch, z.double(), "relu")
    want = dz @ w.double(), dz.t() @ x.double(), dz.sum(0)
    for dw_t, db_t, dy_t in ((dt(torch, io), torch.float32, dt(torch, io)), (torch.float32, dt(torch, io), torch.float32)):
        got = wl.linear_backward(dy.to(dy_t), x, w, activation="relu", pre_activation=z, dweight_dtype=dw_t, dbias_dtype=db_t)
        for g, e, t, name in zip(got, want, (dt(torch, io), dw_t, db_t), ("dx", "dw", "db")):
            assert g.dtype == t
            same(torch, g, e, name)
    plain = wl.linear_backward(dy, x, w)
    for g, e, name in zip(plain, (dy.double() @ w.double(), dy.double().t() @ x.double(), dy.double().sum(0)), ("dx", "dw", "db")):
        same(torch, g, e, name + " without an activation")
    for i in range(3):
        needs = [j == i for j in range(3)]
        got = wl.linear_backward(dy, x, w, activation="relu", pre_activation=z, need_dx=needs[0], need_dweight=needs[1],
                                 need_dbias=needs[2])
        assert [g is not None for g in got] == needs
        same(torch, got[i], want[i], "one gradient alone")
    wc.check_device_status()


@pytest.mark.parametrize("gap", [1, 6, 8])
def test_backward_strided_rows(cuda, wc, wl, gap):
    torch, gen = cuda, make_gen(cuda, 5)
    m, n, k = 70, 130, 90
    x, w, dy, z = (strided(torch, quarters(torch, gen, *s, io="bf16"), gap) for s in ((m, k), (n, k), (m, n), (m, n)))
    dz = dy.double() * slope(torch, z.double(), "relu")
    got = wl.linear_backward(dy, x, w, activation="relu", pre_activation=z)
    for g, e in zip(got, (dz @ w.double(), dz.t() @ x.double(), dz.sum(0))):
        same(torch, g, e, "strided")
    got = wl.linear_backward(dy[:, 1:], x, w[1:], need_dbias=True)
    for g, e in zip(got, (dy[:, 1:].double() @ w[1:].double(), dy[:, 1:].double().t() @ x.double(), dy[:, 1:].double().sum(0))):
        same(torch, g, e, "off a boundary")
    wc.check_device_status()


GROUPS = [
    (64, 96, 72, [64], 0),                              # one expert has everything
    (64, 96, 72, [0, 0, 64, 0], 0),
    (1, 40, 200, [0, 1, 0], 0),                         # one token
    (30, 130, 65, [1] * 30, 0),                         # one row each
    (9, 64, 64, [0, 0, 0], 4),                          # nobody has a row
    (300, 129, 328, [0, 127, 1, 128, 0, 30, 3], 5),     # rows in front and behind
    (700, 72, 136, [16, 15, 17, 0, 63, 65, 64, 200, 129, 99], 2),
    (513, 264, 64, [513 // 64 + (i < 513 % 64) for i in range(64)], 0),
]


@pytest.mark.parametrize("io,out", [("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("m,n,k,sizes,front", GROUPS)
def test_grouped_exact(cuda, wc, wl, m, n, k, sizes, front, io, out):
    torch, gen = cuda, make_gen(cuda, m + n)
    G, t = len(sizes), dt(torch, out)
    off = offsets_of(torch, sizes, front)
    x, w, dy, z_in = (quarters(torch, gen, *s, io=io) for s in ((m, k), (G, n, k), (m, n), (m, n)))
    b = quarters(torch, gen, G, n, io=io)
    last = front + sum(sizes)
    for v in (x, dy, z_in):  # rows that nobody has are never used
        v[:front] = float("nan")
        v[last:] = float("inf")
    for g, s in enumerate(sizes):
        if s == 0:
            w[g] = float("nan")
    z, y = grouped_want(torch, x, w, off, b, "relu")
    got, got_z = wl.grouped_linear(x, w, off, b, activation="relu", out_dtype=t, save_pre_activation=True)
    same(torch, got, y, "y")
    same(torch, got_z, z, "z")
    kept = torch.full((m, n), 3.0, dtype=t, device="cuda")
    wl.grouped_linear(x, w, off, b.float(), activation="relu", out=kept)
    same(torch, kept[front:last], y[front:last], "out")
    assert bool((kept[:front] == 3).all()) and bool((kept[last:] == 3).all())
    _, dx, dw, db = grouped_want(torch, x, w, off, None, "relu", dy, z_in)
    got = wl.grouped_linear_backward(dy, x, w, off, activation="relu", pre_activation=z_in, dweight_dtype=t)
    for g, e, name in zip(got, (dx, dw, db), ("dx", "dw", "db")):
        same(torch, g, e, name)
    _, dx, dw, db = grouped_want(torch, x, w, off, None, "none", dy)
    got = wl.grouped_linear_backward(dy, x, w, off, dbias_dtype=dt(torch, io))
    for g, e, name in zip(got, (dx, dw, db), ("dx", "dw", "db")):
        same(torch, g, e, name + " without an activation")
    wc.check_device_status()


@pytest.mark.parametrize("columns,io", [(64, "bf16"), (128, "f16"), (160, "f16"), (256, "bf16")])
@pytest.mark.parametrize("m,n,k,sizes,front", GROUPS + [
    (1400, 264, 520, [1, 0, 32, 33, 64, 255, 256, 257, 5], 3), (2900, 1001, 330, [513, 600, 0, 700, 1, 1023], 0),
    (300, 40, 8, [300], 0), (5200, 2312, 136, [2600, 17, 0, 2300], 21)])
def test_grouped_pairs_with_tokens_on_columns(cuda, wc, wl, m, n, k, sizes, front, columns, io):
    """Tiles as wide as the experts have tokens; the last one has more tiles than pairs and more blocks than a band."""
    with env_knobs(wc, WAVE_CUDA_LINEAR_PAIR=1, WAVE_CUDA_LINEAR_SWAP=1, WAVE_CUDA_LINEAR_COLUMNS=columns):
        d = wc.LinearDesc(m, n, k, len(sizes), wc.BF16, wc.BF16, wc.BF16, wc.BF16, wc.F32)
        for product in (0, 1):
            plan = wc.linear_plan_for_sms(d, product, 148)
            assert plan["tile_rows"] == 256 and plan["tokens_on_columns"] and plan["tile_columns"] == columns
        test_grouped_exact(cuda, wc, wl, m, n, k, sizes, front, io, io)


@pytest.mark.parametrize("gap", [1, 8])
def test_grouped_strided(cuda, wc, wl, gap):
    """Gaps between rows and between the experts' matrices."""
    torch, gen = cuda, make_gen(cuda, 6)
    m, n, k, sizes = 90, 48, 80, [20, 0, 41, 29]
    off = offsets_of(torch, sizes)
    x, dy = strided(torch, quarters(torch, gen, m, k, io="bf16"), gap), strided(torch, quarters(torch, gen, m, n, io="bf16"), gap)
    wide = torch.full((4, n + 3, k + gap), float("nan"), dtype=torch.bfloat16, device="cuda")
    w = wide[:, :n, :k]
    w.copy_(quarters(torch, gen, 4, n, k, io="bf16"))
    y, dx, dw, db = grouped_want(torch, x, w, off, None, "none", dy)
    same(torch, wl.grouped_linear(x, w, off), y, "y")
    for g, e in zip(wl.grouped_linear_backward(dy, x, w, off), (dx, dw, db)):
        same(torch, g, e, "gradients")
    wc.check_device_status()


@pytest.mark.parametrize("bad", [[0, 40, 20, 64], [-5, 10, 30, 64], [0, 10, 500, 700], [64, 0, 0, 64], [70, 80, 90, 99], [-9, -8, -7, -1]])
def test_bad_offsets_are_cut(cuda, wc, wl, bad):
    """Offsets outside the tokens or out of order: cut and read with a running maximum, as the header says."""
    torch, gen = cuda, make_gen(cuda, 8)
    m, n, k = 64, 72, 136
    off = torch.tensor(bad, dtype=torch.int32, device="cuda")
    x, w, dy = (quarters(torch, gen, *s, io="bf16") for s in ((m, k), (3, n, k), (m, n)))
    y, dx, dw, db = grouped_want(torch, x, w, off, None, "none", dy)
    same(torch, wl.grouped_linear(x, w, off), y, "y")
    for g, e in zip(wl.grouped_linear_backward(dy, x, w, off), (dx, dw, db)):
        same(torch, g, e, "gradients")
    wc.check_device_status()


def test_many_experts(cuda, wc, wl):
    """1024 experts, most without rows."""
    torch, gen = cuda, make_gen(cuda, 9)
    sizes = torch.zeros(1024, dtype=torch.int64)
    sizes[torch.randperm(1024, generator=torch.Generator().manual_seed(1))[:200]] = torch.arange(200) % 7
    m, n, k = int(sizes.sum()), 40, 64
    off = offsets_of(torch, sizes.tolist())
    x, w, dy = (quarters(torch, gen, *s, io="f16") for s in ((m, k), (1024, n, k), (m, n)))
    y, dx, dw, db = grouped_want(torch, x, w, off, None, "none", dy)
    same(torch, wl.grouped_linear(x, w, off), y, "y")
    for g, e in zip(wl.grouped_linear_backward(dy, x, w, off), (dx, dw, db)):
        same(torch, g, e, "gradients")
    with pytest.raises(ValueError, match="experts must be between"):
        wl.grouped_linear(x, torch.zeros(1025, n, k, dtype=torch.float16, device="cuda"),
                          torch.zeros(1026, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("io", ["bf16", "f16"])
def test_smooth_activations(cuda, wc, wl, act, io):
    """z runs over [-30, 30] exactly (x is a row of values, W the identity), so all that is off is the activation's own
    arithmetic: f32 functions of a few steps (2^-24 each) and an exponential of the special-function unit, whose argument
    x log2 e <= 44 is off by 44 * 2^-24 and whose result by 2^-22 -- together below 4e-6 of the value where the sigmoid is
    not small, and below 4e-6 |z| / 2 ... absolutely where 1 + erf cancels.  8e-6 (|y| + |z| 2^-3) covers both;
    16-bit results add half a step of their type."""
    torch = cuda
    step = 2.0 ** -5
    z = (torch.arange(-960, 960, device="cuda") * step).reshape(16, 120).to(dt(torch, io))
    eye = torch.eye(120, device="cuda", dtype=dt(torch, io))
    exact = activate(torch, z.double(), act)
    for out in (torch.float32, dt(torch, io)):
        got, got_z = wl.linear(z, eye, activation=act, out_dtype=out, save_pre_activation=True)
        assert torch.equal(got_z, z)
        limit = 8e-6 * (exact.abs() + z.double().abs() / 8)
        if out != torch.float32:
            limit = limit + torch.finfo(out).eps / 2 * exact.abs() + torch.finfo(out).smallest_normal * torch.finfo(out).eps
        assert bool(((got.double() - exact).abs() <= limit).all()), float(((got.double() - exact).abs() - limit).max())
    # the slope: dy = 1 makes the input gradient dz itself (W is the identity), rounded to the type twice (as an operand
    # and as dx, the second time exactly); slopes are below 1.13, their parts below 2, errors as above
    s = slope(torch, z.double(), act)
    one = torch.ones_like(z)
    dx, _, db = wl.linear_backward(one, z, eye, activation=act, pre_activation=z, need_dweight=False)
    limit = 8e-6 * (1 + z.double().abs() / 8)
    t = dt(torch, io)
    assert bool(((dx.double() - s).abs() <= limit + torch.finfo(t).eps / 2 * s.abs() + torch.finfo(t).smallest_normal * torch.finfo(t).eps).all())
    # column sums of 16 unrounded slopes, 4 additions deep
    assert bool(((db.double() - s.sum(0)).abs() <= limit.sum(0) + 16 * 2.0 ** -24 * s.abs().sum(0)).all())


def test_f32_results_of_long_sums(cuda, wc, wl):
    """f32 results are summed from pieces of 512 products.  The tensor core truncates where it aligns and adds 16
    products to its accumulator: at most 17 steps of 2^-23 of the piece's sum of magnitudes, 32 times; the pieces are
    rounded to nearest: K / 512 half steps of 2^-23 of the whole.  In all (17 * 32 + K / 1024) 2^-23 of sum |x w|."""
    torch, gen = cuda, make_gen(cuda, 10)
    for m, n, k in ((4, 64, 16384), (200, 136, 16384)):
        x = torch.randn(m, k, generator=gen, device="cuda").to(torch.bfloat16)
        w = torch.randn(n, k, generator=gen, device="cuda").to(torch.bfloat16)
        y = wl.linear(x, w, out_dtype=torch.float32).double()
        limit = (17 * 32 + k / 1024) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t())
        assert bool(((y - x.double() @ w.double().t()).abs() <= limit).all())
        # and what it is in practice: 2e-6 of the norm where one accumulator has 1.9e-5
        e = x.double() @ w.double().t()
        assert float((y - e).norm() / e.norm()) < 2e-6


def test_special_values(cuda, wc, wl):
    """A NaN or an infinity stays in its token's row; relu keeps a NaN; f16 overflows to infinity."""
    torch, gen = cuda, make_gen(cuda, 11)
    for m in (20, 200):
        x, w = quarters(torch, gen, m, 72, io="f16"), quarters(torch, gen, 136, 72, io="f16")
        _, y = forward_want(torch, x, w, None, None, "relu")
        bad = x.clone()
        bad[3, 5], bad[7, 6] = float("nan"), float("inf")
        got = wl.linear(bad, w, activation="relu")
        keep = [i for i in range(m) if i not in (3, 7)]
        same(torch, got[keep], y[keep], "other rows")
        assert bool(got[3].isnan().all())
        big = wl.linear(torch.full((m, 64), 200.0, dtype=torch.float16, device="cuda"),
                        torch.full((24, 64), 200.0, dtype=torch.float16, device="cuda"))
        assert bool(big.isinf().all())


@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
def test_far_pre_activations(cuda, wc, wl, act):
    """Pre-activations of any size in bf16: values and slopes are the limits, a NaN stays one."""
    torch = cuda
    far = torch.tensor([3e38, 1e20, 1e6, 300.0, -300.0, -1e6, -1e20, -3e38], device="cuda").to(torch.bfloat16)[None]
    eye = torch.eye(8, device="cuda", dtype=torch.bfloat16)
    # (one value to a token: 0 * 3e38 in the other products is 0)
    z = torch.diag(far[0])
    y = wl.linear(z, eye, activation=act)
    assert torch.equal(torch.diag(y), torch.where(far[0] > 0, far[0], torch.zeros_like(far[0])))
    dy = torch.ones_like(z)
    dx = wl.linear_backward(dy, z, eye, activation=act, pre_activation=far.expand(8, 8).contiguous(), need_dweight=False,
                            need_dbias=False)[0]
    want = (far > 0).to(torch.bfloat16).expand(8, 8)
    assert bool(((dx - want).abs() <= 1e-20).all())
    nan = torch.full_like(z, float("nan"))
    assert bool(wl.linear_backward(dy, z, eye, activation=act, pre_activation=nan, need_dweight=False)[2].isnan().all())
    inf = torch.full_like(z, float("inf"))
    assert bool((wl.linear_backward(dy, z, eye, activation=act, pre_activation=inf, need_dweight=False)[2] == 8).all())
    assert bool((wl.linear_backward(dy, z, eye, activation=act, pre_activation=-inf, need_dweight=False)[2].abs() <= 1e-20).all())


def test_no_tokens(cuda, wc, wl):
    torch = cuda
    w, wg = (torch.ones(*s, 16, 24, dtype=torch.bfloat16, device="cuda") for s in ((), (3,)))
    x, dy = (torch.ones(0, c, dtype=torch.bfloat16, device="cuda") for c in (24, 16))
    off = torch.zeros(4, dtype=torch.int32, device="cuda")
    assert wl.linear(x, w).shape == (0, 16) and wl.grouped_linear(x, wg, off).shape == (0, 16)
    for got, lead in ((wl.linear_backward(dy, x, w), ()), (wl.grouped_linear_backward(dy, x, wg, off), (3,))):
        assert got[0].shape == (0, 24)
        assert got[1].shape == (*lead, 16, 24) and not bool(got[1].any())
        assert got[2].shape == (*lead, 16) and not bool(got[2].any())


def test_residual_in_place(cuda, wc, wl):
    torch, gen = cuda, make_gen(cuda, 12)
    for m in (3, 150, 700):
        x, w, r = (quarters(torch, gen, *s, io="bf16") for s in ((m, 520), (264, 520), (m, 264)))
        _, y = forward_want(torch, x, w, None, r, "none")
        stream_in = r.clone()
        wl.linear(x, w, None, stream_in, out=stream_in)
        same(torch, stream_in, y, "in place")


def test_refusals(cuda, wc, wl):
    torch = cuda
    z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
    x, w, off = z(8, 32), z(16, 32), z(3, t=torch.int32)
    cases = [
        (lambda: wl.linear(x[0], w), "x must be"),
        (lambda: wl.linear(x, w[None]), "x must be"),
        (lambda: wl.linear(x, z(16, 31)), "x has 32 features"),
        (lambda: wl.linear(x.float(), w.float()), "x must have dtype"),
        (lambda: wl.linear(x, w.half()), "share dtype"),
        (lambda: wl.linear(z(32, 8).t(), w), "contiguous rows"),
        (lambda: wl.linear(x, z(32, 16).t()), "contiguous rows"),
        (lambda: wl.linear(z(1, 32).expand(8, 32), w), "must not overlap"),
        (lambda: wl.linear(x, w, z(15)), "bias must be"),
        (lambda: wl.linear(x, w, z(16, t=torch.float16)), "bias must have dtype"),
        (lambda: wl.linear(x, w, None, z(8, 15)), "residual must have shape"),
        (lambda: wl.linear(x, w, None, z(8, 16, t=torch.float32)), "residual must have dtype"),
        (lambda: wl.linear(x, w, None, z(16).expand(8, 16)), "must not overlap"),
        (lambda: wl.linear(x, w, activation="tanh"), "activation must be one of"),
        (lambda: wl.linear(x, w, out_dtype=torch.float16), "out_dtype must be"),
        (lambda: wl.linear(x, w, out=z(8, 17)), "out must have shape"),
        (lambda: wl.linear(x, w, out=z(8, 16), out_dtype=torch.float32), "out has dtype"),
        (lambda: wl.linear(x, w.cpu()), "share dtype and device"),
        (lambda: wl.linear_backward(z(8, 15), x, w), "dy must have shape"),
        (lambda: wl.linear_backward(z(8, 16), x, w, activation="relu"), "needs the pre-activation"),
        (lambda: wl.linear_backward(z(8, 16), x, w, activation="relu", pre_activation=z(8, 16, t=torch.float32)), "pre_activation must have dtype"),
        (lambda: wl.linear_backward(z(8, 16), x, w, dweight_dtype=torch.float16), "dweight_dtype must be"),
        (lambda: wl.grouped_linear(x, z(2, 16, 32), off.long()), "offsets must be"),
        (lambda: wl.grouped_linear(x, z(3, 16, 32), off), "offsets must be"),
        (lambda: wl.grouped_linear(x, w, off), "x must be"),
        (lambda: wl.grouped_linear(x, z(2, 16, 32), off, z(16)), "bias must be"),
        (lambda: wl.grouped_linear(x, z(1, 16, 32).expand(2, 16, 32), off), "must not overlap"),
        (lambda: wl.grouped_linear_backward(z(8, 16), x, z(2, 16, 32), None), "offsets must be given"),
    ]
    for call, message in cases:
        with pytest.raises(ValueError, match=message):
            call()


def test_streams(cuda, wc, wl):
    """Calls on two streams at once, tensors made on another stream than the call's."""
    torch, gen = cuda, make_gen(cuda, 13)
    m, n, k = 40, 520, 1032
    data = [tuple(quarters(torch, gen, *s, io="bf16") for s in ((m, k), (n, k), (m, n))) for _ in range(4)]
    want = [(x.double() @ w.double().t(), dy.double() @ w.double(), dy.double().t() @ x.double()) for x, w, dy in data]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for rep in range(8):
        for i, (x, w, dy) in enumerate(data):
            with torch.cuda.stream(streams[i % 2]):
                got.append((i, wl.linear(x, w), *wl.linear_backward(dy, x, w)[:2]))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for i, *g in got:
        for a, b in zip(g, want[i]):
            same(torch, a, b, "on a stream")
    wc.check_device_status()


def test_graph_capture_and_replay(cuda, wc, wl):
    """A captured forward and backward pass, dense and grouped, replayed on new inputs; two graphs, replayed in turn and
    at once; the experts' offsets change between replays."""
    torch, gen = cuda, make_gen(cuda, 14)
    m, n, k, G = 70, 137, 201, 5  # odd features: the calls lay their operands out in workspaces of their own
    x, w, dy, wg = (quarters(torch, gen, *s, io="f16") for s in ((m, k), (n, k), (m, n), (G, n, k)))
    off = offsets_of(torch, [10, 0, 30, 5, 20], 2)

    def calls():
        y, z = wl.linear(x, w, activation="relu", save_pre_activation=True)
        yg, zg = wl.grouped_linear(x, wg, off, activation="relu", save_pre_activation=True)
        return [y, *wl.linear_backward(dy, x, w, activation="relu", pre_activation=z), yg,
                *wl.grouped_linear_backward(dy, x, wg, off, activation="relu", pre_activation=zg)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = calls()
        graphs.append((g, out))

    def wanted():
        z, y = forward_want(torch, x, w, None, None, "relu")
        dz = dy.double() * (z > 0)
        zb = torch.zeros(G, n, dtype=torch.float64, device="cuda")
        zg, yg = grouped_want(torch, x, wg, off, zb, "relu")
        _, dx, dw, db = grouped_want(torch, x, wg, off, None, "relu", dy, zg)
        return [y, dz @ w.double(), dz.t() @ x.double(), dz.sum(0), yg, dx, dw, db]

    for sizes, front in (([10, 0, 30, 5, 20], 2), ([0, 0, 70, 0, 0], 0), ([1, 2, 3, 4, 5], 40)):
        for t in (x, w, dy, wg):
            t.copy_(quarters(torch, gen, *t.shape, io="f16"))
        off.copy_(offsets_of(torch, sizes, front))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0][0].replay()
        graphs[1][0].replay()
        torch.cuda.synchronize()
        want = wanted()
        for _, out in graphs:
            for a, b in zip(out, want):
                same(torch, a, b, "replayed")
    wc.check_device_status()


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("m,n,k,experts", [(515, 1032, 776, 0), (300, 136, 4096, 0), (2304, 2048, 1024, 0), (700, 520, 1288, 6), (4096, 72, 2568, 3)])
def test_launches_side_by_side(cuda, wc, wl, m, n, k, experts, captured):
    """The backward pass' products overlap: what follows on the stream (another layer, the inputs written anew) sees all of
    them finished, and the next call does not disturb them."""
    torch, gen = cuda, make_gen(cuda, m)
    lead = (experts,) if experts else ()
    x, w, dy, z = (torch.randn(s, generator=gen, device="cuda").to(torch.bfloat16) for s in ((m, k), (*lead, n, k), (m, n), (m, n)))
    v = torch.randn(64, k, generator=gen, device="cuda").to(torch.bfloat16)
    off = offsets_of(torch, [m // experts] * (experts - 1) + [m - m // experts * (experts - 1)]) if experts else None

    def backward(dy, x, z, **need):
        if experts:
            return wl.grouped_linear_backward(dy, x, w, off, activation="silu", pre_activation=z, **need)
        return wl.linear_backward(dy, x, w, activation="silu", pre_activation=z, **need)

    alone = []
    for i, name in enumerate(("need_dx", "need_dweight", "need_dbias")):
        alone.append(backward(dy, x, z, **{o: o == name for o in ("need_dx", "need_dweight", "need_dbias")})[i])
        torch.cuda.synchronize()
    alone.append(wl.linear(alone[0], v))
    torch.cuda.synchronize()
    dy1, x1, z1 = (torch.empty_like(t) for t in (dy, x, z))

    def step():
        for to, t in ((dy1, dy), (x1, x), (z1, z)):
            to.copy_(t)
        dx, dw, db = backward(dy1, x1, z1)
        y = wl.linear(dx, v)  # another layer reads dx at once
        for t in (dy1, x1, z1):
            t.fill_(float("nan"))
        again = backward(dy, x, z)
        return [dx, dw, db, y, *again]

    if captured:
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
    for _ in range(5):
        if captured:
            graph.replay()
        else:
            got = step()
        torch.cuda.synchronize()
        for g, e in zip(got, alone + alone[:3]):
            assert torch.equal(g, e)
    wc.check_device_status()


def test_same_call_same_bits(cuda, wc, wl):
    torch, gen = cuda, make_gen(cuda, 15)
    for m, n, k in ((3, 2048, 2048), (200, 520, 1000)):
        x, w, dy = (torch.randn(*s, generator=gen, device="cuda").to(torch.bfloat16) for s in ((m, k), (n, k), (m, n)))
        first = None
        for _ in range(5):
            got = [wl.linear(x, w, out_dtype=torch.float32), *wl.linear_backward(dy, x, w, dweight_dtype=torch.float32)]
            if first is not None:
                assert all(torch.equal(a, b) for a, b in zip(first, got))
            first = got


def test_offsets_beyond_32_bits(cuda, wc, wl):
    """More than 2^31 elements in y, x and dw; weights of the last expert behind 2^31 elements."""
    torch, gen = cuda, make_gen(cuda, 16)
    m, n, k = 66000, 32784, 16
    x, w = quarters(torch, gen, m, k, io="bf16"), quarters(torch, gen, n, k, io="bf16")
    y = wl.linear(x, w)
    for at in (slice(0, 300), slice(m - 300, m)):
        same(torch, y[at], x[at].double() @ w.double().t(), "far rows")
    # the wide matrix as dy: its column sums over the last columns, and dx of the last rows
    dx, dw, db = wl.linear_backward(y, x, w, need_dweight=True)
    # y is bf16-rounded multiples of 1/16 and the columns' sums of magnitudes stay below 2^24 of them: exact
    same(torch, db[-64:], y[:, -64:].double().sum(0), "far columns")
    e = y[-100:].double() @ w.double()
    scale = y[-100:].double().abs() @ w.double().abs()
    # 2049 accumulations of 16 products each, 17 truncations of 2^-23 in each, and half a bf16 step
    assert bool(((dx[-100:].double() - e).abs() <= 2049 * 17 * 2.0 ** -23 * scale + 2.0 ** -8 * e.abs()).all())
    del y, dx, dw, db
    torch.cuda.empty_cache()
    G, n, k = 36, 8192, 8192
    wg = torch.zeros(G, n, k, dtype=torch.bfloat16, device="cuda")
    wg[-1] = quarters(torch, gen, n, k, io="bf16")
    x = quarters(torch, gen, 5, k, io="bf16")
    off = offsets_of(torch, [2] + [0] * (G - 2) + [3])
    y = wl.grouped_linear(x, wg, off)
    same(torch, y[2:], x[2:].double() @ wg[-1].double().t(), "last expert")
    assert not bool(y[:2].any())
    dy = quarters(torch, gen, 5, n, io="bf16")
    dx, dw, _ = wl.grouped_linear_backward(dy, x, wg, off)
    same(torch, dw[-1], dy[2:].double().t() @ x[2:].double(), "last expert's gradient")
    assert not bool(dw[1:-1].any())
    wc.check_device_status()


def test_gradients_against_differences(cuda, wc, wl):
    """<dx, u> + <dW, v> + <db, e> against the change of sum(y * g) along (u, v, e), central differences of the forward
    kernel's f32 results.  Inputs and steps are multiples of 1/64, exact in f16, so the two points are what they say."""
    torch, gen = cuda, make_gen(cuda, 17)
    m, n, k, h = 24, 40, 64, 1 / 64
    for act in ("gelu", "gelu_tanh", "silu"):
        x, w, b, u, v, e, g = (quarters(torch, gen, *s, io="f16") / 4 for s in ((m, k), (n, k), (n,), (m, k), (n, k), (n,), (m, n)))

        def value(t):
            y = wl.linear((x.float() + t * u.float()).half(), (w.float() + t * v.float()).half(),
                          b.float() + t * e.float(), activation=act, out_dtype=torch.float32)
            return float((y.double() * g.double()).sum())

        h_big = 4 * h  # x + t u: multiples of 1/16 * 1/16, below 1: exact
        d1, d2 = ((value(s) - value(-s)) / (2 * s) for s in (h_big, 2 * h_big))
        diff = (4 * d1 - d2) / 3  # the error's h^2 term removed: what is left is of the order of h^4
        _, z = wl.linear(x, w, b.float(), activation=act, save_pre_activation=True)
        dx, dw, db = wl.linear_backward(g, x, w, activation=act, pre_activation=z, dweight_dtype=torch.float32)
        grad = float((dx.double() * u.double()).sum() + (dw.double() * v.double()).sum() + (db.double() * e.double()).sum())
        # z and dz rounded to f16 (2^-11 each, and dx once more): 3 half steps of every term's magnitude
        z64 = x.double() @ w.double().t() + b.double()
        dz = g.double() * slope(torch, z64, act)
        size = float((dz.abs() @ w.double().abs() * u.double().abs()).sum() + (dz.abs().t() @ x.double().abs() * v.double().abs()).sum()
                     + (dz.abs().sum(0) * e.double().abs()).sum())
        exact = float((dz @ w.double() * u.double()).sum() + (dz.t() @ x.double() * v.double()).sum() + (dz.sum(0) * e.double()).sum())
        assert abs(grad - exact) <= 3 * 2.0 ** -11 * size
        # the differences' own error: the fourth-order term, measured in 64 bits at the same points
        f = lambda t: float((activate(torch, (x.double() + t * u.double()) @ (w.double() + t * v.double()).t() + b.double() + t * e.double(), act) * g.double()).sum())  # noqa: E731
        e1, e2 = ((f(s) - f(-s)) / (2 * s) for s in (h_big, 2 * h_big))
        rest = abs((4 * e1 - e2) / 3 - exact)
        noise = 2 * 8e-6 * float((g.double().abs() * (1 + z64.abs())).sum()) / h_big
        assert abs(diff - exact) <= rest + noise


def test_a_layer_as_it_is_used(cuda, wc, wl):
    """Projections, attention, the projection back onto the residual stream, a dense feed-forward layer and one of
    experts behind a router, forward and backward: each step against the formula on the values that went into it."""
    torch, gen = cuda, make_gen(cuda, 18)
    wa = importlib.import_module("7_b200.wave_attention")
    B, S, H, D, F, G = 2, 64, 4, 32, 264, 6
    E, T = H * D, B * S
    rand = lambda *s, scale=1.0: (scale * torch.randn(*s, generator=gen, device="cuda")).to(torch.bfloat16)  # noqa: E731
    near = lambda got, want, steps, what: _near(torch, got, want, steps, what)  # noqa: E731
    x = rand(T, E)
    wq, wk, wv, wo = (rand(E, E, scale=E ** -0.5) for _ in range(4))
    heads = lambda t: t.reshape(B, S, H, D).transpose(1, 2).contiguous()  # noqa: E731
    q, k, v = (heads(wl.linear(x, w)) for w in (wq, wk, wv))
    o = wa.attention(q, k, v, causal=True).transpose(1, 2).reshape(T, E)
    h = wl.linear(o, wo, None, x)
    near(h, o.double() @ wo.double().t() + x.double(), 1, "projection")
    # dense feed-forward
    w1, b1, w2, b2 = rand(F, E, scale=E ** -0.5), rand(F), rand(E, F, scale=F ** -0.5), rand(E)
    up, z1 = wl.linear(h, w1, b1, activation="gelu", save_pre_activation=True)
    h2 = wl.linear(up, w2, b2, h)
    near(up, activate(torch, h.double() @ w1.double().t() + b1.double(), "gelu"), 1, "up")
    near(h2, up.double() @ w2.double().t() + b2.double() + h.double(), 1, "down")
    # experts: one for each token, the largest of the router's scores
    router = rand(G, E, scale=E ** -0.5)
    scores = wl.linear(h2, router, out_dtype=torch.float32)
    expert = scores.argmax(1)
    order = expert.argsort(stable=True)
    off = torch.zeros(G + 1, dtype=torch.int32, device="cuda")
    off[1:] = torch.bincount(expert, minlength=G).cumsum(0)
    we1, we2 = rand(G, F, E, scale=E ** -0.5), rand(G, E, F, scale=F ** -0.5)
    rows = h2[order]
    mid, zm = wl.grouped_linear(rows, we1, off, activation="silu", save_pre_activation=True)
    back = wl.grouped_linear(mid, we2, off)
    y = h2.clone()
    y[order] += back
    for t in range(0, T, 17):
        g, row = int(expert[order[t]]), rows[t].double()
        near(mid[t], activate(torch, we1[g].double() @ row, "silu"), 1, "expert up")
        near(back[t], we2[g].double() @ mid[t].double(), 1, "expert down")
    # the way back through both feed-forward layers
    dy = rand(T, E)
    dmid, dwe2, _ = wl.grouped_linear_backward(dy[order], mid, we2, off, need_dbias=False)
    drows, dwe1, dbe1 = wl.grouped_linear_backward(dmid, rows, we1, off, activation="silu", pre_activation=zm)
    dh2 = dy.clone()
    dh2[order] += drows
    dup, dw2, db2 = wl.linear_backward(dh2, up, w2)
    dh, dw1, db1 = wl.linear_backward(dup, h, w1, activation="gelu", pre_activation=z1)
    _, ex, ew, eb = grouped_want(torch, rows, we1, off, None, "silu", dmid, zm)
    near(drows, ex, 2, "experts' dx")
    near(dwe1, ew, 2, "experts' dw")
    near(dbe1, eb, 1, "experts' db")
    dz = dup.double() * slope(torch, z1.double(), "gelu")
    near(dh, dz @ w1.double(), 2, "dx")
    near(dw1, dz.t() @ h.double(), 2, "dw")
    near(dw2, dh2.double().t() @ up.double(), 1, "dw2")
    near(db2, dh2.double().sum(0), 1, "db2")
    assert dwe2.shape == we2.shape and db1.shape == b1.shape
    wc.check_device_status()


def _near(torch, got, want, roundings, what):
    """Each rounding to bf16 is off by 2^-9 of its value's size (relative to the norm, at most half a step 2^-8 / 2 ... 2^-8);
    independent ones add up at most linearly."""
    err = float((got.double() - want).norm() / want.norm())
    assert err <= roundings * 2.0 ** -8, f"{what}: {err}"

"""Rows and matrices far apart: element offsets beyond 32 bits in every operand and result, strides beyond 2^31 bytes."""
import ctypes as C
import importlib

import pytest

from test_linear_gpu import forward_want, grouped_want, make_gen, offsets_of, quarters, same

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def wl():
    return importlib.import_module("7_b200.wave_linear")


def test_no_tokens_and_far_rows(cuda, wc):
    """Without tokens dW is zero, whatever the distance of its rows; what lies between them stays."""
    torch = cuda
    n, k, G = 3, 64, 2
    for ld, elem, t in (((1 << 29) + 8, wc.F32, torch.float32), (72, wc.F32, torch.float32), (64, wc.BF16, torch.bfloat16)):
        for experts in (0, G):
            if experts and ld > 1000:
                continue
            matrices = max(experts, 1)
            flat = torch.full((ld * n * matrices,), 7.0, dtype=t, device="cuda")
            d = wc.LinearDesc(0, n, k, experts, wc.BF16, wc.BF16, wc.BF16, elem, wc.F32)
            d.lddw = ld
            off = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
            wc.check(wc.lib().wave_cuda_linear_bwd(C.byref(d), None, None, None, None, off.data_ptr(), None, flat.data_ptr(), None,
                                                   None, torch.cuda.current_stream().cuda_stream or None))
            rows = flat.view(matrices * n, ld)
            assert not bool(rows[:, :k].any())
            assert bool((rows[:, k:k + 1000] == 7).all()) and bool((rows[:, -8:] == 7).all() or ld == 64)
            del flat, rows
    torch.cuda.empty_cache()


def far(torch, rows, cols, dtype):
    """[rows, cols] of which the last row starts beyond 2^31 elements; 16-byte rows."""
    ld = max(cols, ((1 << 31) // (rows - 1) + 8) // 8 * 8 + 8)
    flat = torch.empty(ld * (rows - 1) + cols, dtype=dtype, device="cuda")
    view = flat.as_strided((rows, cols), (ld, 1))
    assert (rows - 1) * ld > 1 << 31
    return view


@pytest.mark.parametrize("m,knobs", [(9, {}), (3000, {}), (3000, dict(PAIR=1, SWAP=0)), (600, dict(PAIR=0, SWAP=0, TILE=64, SPLITS=2))])
def test_every_row_far(cuda, wc, m, knobs):
    """x, W, y, z, the residual, dy, dx and dW all with their last rows beyond 2^31 elements."""
    from _util import env_knobs
    torch, gen = cuda, make_gen(cuda, m)
    n, k = 136, 72
    bf = torch.bfloat16
    stream = torch.cuda.current_stream().cuda_stream or None

    def put(rows, cols):
        t = far(torch, rows, cols, bf)
        return t.copy_(quarters(torch, gen, rows, cols, io="bf16"))

    x, w, r, dy, z = put(m, k), put(n, k), put(m, n), put(m, n), put(m, n)
    y, z_out, dx, dw = far(torch, m, n, bf), far(torch, m, n, bf), far(torch, m, k, bf), far(torch, n, k, bf)
    d = wc.LinearDesc(m, n, k, 0, wc.BF16, wc.BF16, wc.BF16, wc.BF16, wc.F32, 1)
    d.ldx, d.ldw, d.ldy, d.ldr, d.ldz, d.lddx, d.lddw = (t.stride(0) for t in (x, w, y, r, z, dx, dw))
    with env_knobs(wc, **{f"WAVE_CUDA_LINEAR_{a}": v for a, v in knobs.items()}):
        wc.check(wc.lib().wave_cuda_linear_fwd(C.byref(d), x.data_ptr(), w.data_ptr(), None, r.data_ptr(), None, y.data_ptr(),
                                               z_out.data_ptr(), None, stream))
        want_z, want_y = forward_want(torch, x, w, None, r, "relu")
        same(torch, y, want_y, "y")
        same(torch, z_out, want_z, "z")
        ws = torch.empty(max(1, wc.linear_workspace_bytes(d, True)), dtype=torch.uint8, device="cuda")
        db = torch.empty(n, device="cuda")
        wc.check(wc.lib().wave_cuda_linear_bwd(C.byref(d), dy.data_ptr(), x.data_ptr(), w.data_ptr(), z.data_ptr(), None,
                                               dx.data_ptr(), dw.data_ptr(), db.data_ptr(), ws.data_ptr(), stream))
        dz = dy.double() * (z.double() > 0)
        same(torch, dx, dz @ w.double(), "dx")
        same(torch, dw, dz.t() @ x.double(), "dw")
        same(torch, db, dz.sum(0), "db")
    wc.check_device_status()
    del x, w, r, dy, z, y, z_out, dx, dw
    torch.cuda.empty_cache()


def test_far_rows_of_other_layouts(cuda, wc, wl):
    """Rows that have to be laid out first, and experts' rows and matrices, beyond 2^31 elements."""
    torch, gen = cuda, make_gen(cuda, 7)
    m, n, k, G = 700, 72, 65, 5
    x, dy = far(torch, m, k, torch.bfloat16), far(torch, m, n, torch.bfloat16)
    for t in (x, dy):
        t.copy_(quarters(torch, gen, *t.shape, io="bf16"))
    step = (1 << 31) // (G - 1) + 16
    w = torch.empty(step * (G - 1) + n * k, dtype=torch.bfloat16, device="cuda").as_strided((G, n, k), (step, k, 1))
    w.copy_(quarters(torch, gen, G, n, k, io="bf16"))
    off = offsets_of(torch, [0, 300, 1, 0, 390], 3)
    want_y, want_dx, want_dw, want_db = grouped_want(torch, x, w, off, None, "none", dy)
    out = far(torch, m, n, torch.float32)
    out.zero_()
    same(torch, wl.grouped_linear(x, w, off, out=out), want_y, "y")
    for g, e, name in zip(wl.grouped_linear_backward(dy, x, w, off), (want_dx, want_dw, want_db), ("dx", "dw", "db")):
        same(torch, g, e, name)
    wc.check_device_status()
    del x, dy, w, out
    torch.cuda.empty_cache()


def test_weight_gradients_of_far_columns_and_experts(cuda, wc, wl):
    """dW where dy has more than 2^31 elements, and of the first and the last of experts whose matrices have.

    The first is summed from pieces of 512 products in f32: 17 truncations of 2^-23 of the piece's magnitudes in each of its
    32 steps, and m / 512 roundings of 2^-24 of the whole."""
    torch, gen = cuda, make_gen(cuda, 8)
    m, n, k = 66000, 32784, 16
    x = quarters(torch, gen, m, k, io="bf16")
    dy = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    for at in range(0, m, 6000):
        dy[at: at + 6000] = quarters(torch, gen, 6000, n, io="bf16")
    dw = wl.linear_backward(dy, x, torch.zeros(n, k, dtype=torch.bfloat16, device="cuda"), dweight_dtype=torch.float32,
                            need_dx=False, need_dbias=False)[1]
    for cols in (slice(0, 128), slice(n - 128, n)):
        d = dy[:, cols].double()
        limit = (17 * 32 + m / 1024) * 2.0 ** -23 * (d.abs().t() @ x.double().abs())
        assert bool(((dw[cols].double() - d.t() @ x.double()).abs() <= limit).all())
    del dy, dw
    torch.cuda.empty_cache()
    G, n, k = 36, 8192, 8192
    wg = torch.zeros(G, n, k, dtype=torch.bfloat16, device="cuda")
    wg[0] = quarters(torch, gen, n, k, io="bf16")
    wg[-1] = quarters(torch, gen, n, k, io="bf16")
    x, dy = quarters(torch, gen, 5, k, io="bf16"), quarters(torch, gen, 5, n, io="bf16")
    off = offsets_of(torch, [2] + [0] * (G - 2) + [3])
    dx, dw, db = wl.grouped_linear_backward(dy, x, wg, off)
    for g, rows in ((0, slice(0, 2)), (G - 1, slice(2, 5))):
        same(torch, dx[rows], dy[rows].double() @ wg[g].double(), "dx")
        same(torch, dw[g], dy[rows].double().t() @ x[rows].double(), "dw")
        same(torch, db[g], dy[rows].double().sum(0), "db")
    assert not bool(dw[1:-1].any()) and not bool(db[1:-1].any())
    wc.check_device_status()
    del wg, dw
    torch.cuda.empty_cache()

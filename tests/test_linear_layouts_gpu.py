"""What the linear layers lay out in their workspace, where rows are no multiple of 16 bytes apart."""
import ctypes as C
import importlib

import pytest

from test_linear_gpu import grouped_want, make_gen, offsets_of, quarters, same

pytestmark = pytest.mark.gpu
PATTERN = -21931  # of the workspace before the call; no quarter in [-2, 2] has these bits


@pytest.fixture(scope="module")
def wl():
    return importlib.import_module("7_b200.wave_linear")


def laid_out(torch, wc, d, backward, call):
    """Runs `call(workspace, stream)` over a workspace of a known pattern; returns it as 16-bit words."""
    need = wc.linear_workspace_bytes(d, backward)
    ws = torch.full((need // 2,), PATTERN, dtype=torch.int16, device="cuda")
    wc.check(call(ws.data_ptr(), torch.cuda.current_stream().cuda_stream or None))
    wc.check_device_status()
    return ws


ROUTES = [
    ([0, 0, 2, 0, 3, 0, 0, 0], 0),   # a few of the experts
    ([5, 0, 0, 0, 0, 0, 0, 4], 2),   # the first and the last, rows in front that belong to nobody
    ([0] * 8, 0),                    # none
    ([1] * 8, 0),                    # all
]


@pytest.mark.parametrize("sizes,front", ROUTES)
@pytest.mark.parametrize("k,gap", [(65, 0), (1021, 0), (64, 4)])
def test_experts_without_rows_are_not_laid_out(cuda, wc, k, gap, sizes, front):
    """Their place in the workspace keeps what it held, forward and backward; the others' rows are there, padded with zeros."""
    torch, gen = cuda, make_gen(cuda, k)
    n, m, G = 40, 12, len(sizes)
    off = offsets_of(torch, sizes, front)
    x = quarters(torch, gen, m, k, io="bf16")
    w = torch.full((G, n, k + gap), float("nan"), dtype=torch.bfloat16, device="cuda")
    w[..., :k] = quarters(torch, gen, G, n, k, io="bf16")
    dy = quarters(torch, gen, m, n, io="bf16")
    for g, s in enumerate(sizes):
        if s == 0:
            w[g] = float("nan")
    d = wc.LinearDesc(m, n, k, G, wc.BF16, wc.BF16, wc.BF16, wc.BF16, wc.F32, 0, 1)
    d.ldw = k + gap
    ld = (k + 7) // 8 * 8
    y, dx = torch.empty(m, n, dtype=torch.bfloat16, device="cuda"), torch.empty(m, k, dtype=torch.bfloat16, device="cuda")
    want_y, want_dx, _, _ = grouped_want(torch, x, w[..., :k], off, None, "none", dy)
    # forward: x, then the weights; backward without dW and dbias: the weights first (dy is loaded as it is)
    x_words = 0 if k % 8 == 0 else (m * ld * 2 + 255) // 256 * 128
    fwd = laid_out(torch, wc, d, False, lambda ws, st: wc.lib().wave_cuda_linear_fwd(
        C.byref(d), x.data_ptr(), w.data_ptr(), None, None, off.data_ptr(), y.data_ptr(), None, ws, st))
    bwd = laid_out(torch, wc, d, True, lambda ws, st: wc.lib().wave_cuda_linear_bwd(
        C.byref(d), dy.data_ptr(), None, w.data_ptr(), None, off.data_ptr(), dx.data_ptr(), None, None, ws, st))
    same(torch, y, want_y, "y")
    same(torch, dx, want_dx, "dx")
    for ws, at, what in ((fwd, x_words, "forward"), (bwd, 0, "backward")):
        place = ws[at: at + G * n * ld].view(G, n, ld)
        for g, s in enumerate(sizes):
            if s == 0:
                assert bool((place[g] == PATTERN).all()), f"{what}: expert {g} has no rows and was laid out"
            else:
                assert torch.equal(place[g, :, :k], w[g, :, :k].view(torch.int16)), f"{what}: expert {g}"
                assert not bool(place[g, :, k:].any())


def test_many_experts_of_odd_sizes(cuda, wc, wl):
    """1024 experts, most without rows (their weights NaN), operands that have to be laid out; offsets that decrease."""
    torch, gen = cuda, make_gen(cuda, 3)
    sizes = torch.zeros(1024, dtype=torch.int64)
    sizes[torch.randperm(1024, generator=torch.Generator().manual_seed(2))[:90]] = torch.arange(90) % 5
    m, n, k = int(sizes.sum()), 33, 61
    off = offsets_of(torch, sizes.tolist())
    x, w, dy = (quarters(torch, gen, *s, io="f16") for s in ((m, k), (1024, n, k), (m, n)))
    w[(sizes == 0).cuda()] = float("nan")
    y, dx, dw, db = grouped_want(torch, x, w, off, None, "none", dy)
    same(torch, wl.grouped_linear(x, w, off), y, "y")
    for g, e in zip(wl.grouped_linear_backward(dy, x, w, off), (dx, dw, db)):
        same(torch, g, e, "gradients")
    bad = torch.tensor([3, 40, 20, 200, 64, 64, 10, 7], dtype=torch.int32, device="cuda")
    w7 = quarters(torch, gen, 7, n, k, io="f16")
    y, dx, dw, db = grouped_want(torch, x, w7, bad, None, "none", dy)
    same(torch, wl.grouped_linear(x, w7, bad), y, "bad offsets")
    for g, e in zip(wl.grouped_linear_backward(dy, x, w7, bad), (dx, dw, db)):
        same(torch, g, e, "bad offsets")
    wc.check_device_status()


def test_laid_out_over_many_blocks(cuda, wc, wl):
    """More pieces than the launch has threads: dense operands, and experts of several turns each."""
    torch, gen = cuda, make_gen(cuda, 4)
    m, n, k = 3001, 1501, 1021
    x, w = quarters(torch, gen, m, k, io="bf16"), quarters(torch, gen, n, k, io="bf16")
    same(torch, wl.linear(x, w), x.double() @ w.double().t(), "y")
    wg = quarters(torch, gen, 5, n, k, io="bf16")
    off = offsets_of(torch, [1000, 0, 1, 1990, 0], 3)
    same(torch, wl.grouped_linear(x, wg, off), grouped_want(torch, x, wg, off, None, "none"), "grouped y")
    wc.check_device_status()

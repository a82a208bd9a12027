"""Gradients by expert where the mean of the experts' rows says little: one expert with nearly all of them."""
import importlib

import pytest

from test_linear_gpu import dt, grouped_want, make_gen, offsets_of, quarters, same

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def wl():
    return importlib.import_module("7_b200.wave_linear")


ROUTES = [
    [0, 0, 8000, 3, 0, 189, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0],    # one has nearly all
    [8192] + [0] * 15,
    [0] * 15 + [8192],
    [1023, 1024, 1025, 0, 2047, 2048, 2049, 1],              # around whole blocks
    [1025, 1, 1, 1, 1, 1],
    [700, 0, 324],                                           # as many as one block takes
    [3000, 2500, 0, 0, 0, 0, 0, 0, 0, 0],
]


@pytest.mark.parametrize("front", [0, 7])
@pytest.mark.parametrize("sizes", ROUTES)
@pytest.mark.parametrize("n,k,io,dy_type", [(136, 40, "bf16", "bf16"), (33, 72, "f16", "f32"), (1100, 24, "f16", "f16")])
def test_gradients_exact(cuda, wc, wl, n, k, io, dy_type, sizes, front):
    """relu passes dy or nothing: every sum is exact."""
    torch, gen = cuda, make_gen(cuda, n + len(sizes))
    G, m = len(sizes), sum(sizes) + 2 * front
    off = offsets_of(torch, sizes, front)
    x, w, dy, z = (quarters(torch, gen, *s, io=io) for s in ((m, k), (G, n, k), (m, n), (m, n)))
    for t in (x, dy, z):
        t[:front] = float("nan")
        t[m - front:] = float("nan")
    _, dx, dw, db = grouped_want(torch, x, w, off, None, "relu", dy, z)
    for need in (True, False):
        got = wl.grouped_linear_backward(dy.to(dt(torch, dy_type)), x, w, off, activation="relu", pre_activation=z,
                                         dweight_dtype=torch.float32, need_dbias=need)
        for g, e, name in zip(got, (dx, dw, db) if need else (dx, dw), ("dx", "dw", "db")):
            same(torch, g, e, name)
    got = wl.grouped_linear_backward(dy, x, w, off, need_dx=False, need_dweight=False, dbias_dtype=dt(torch, io))[2]
    same(torch, got, grouped_want(torch, x, w, off, None, "none", dy)[3], "db alone")
    wc.check_device_status()


def test_one_experts_column_sums(cuda, wc, wl):
    """The sum over an expert's rows is taken in pieces: with values of one sign, 2^-24 of the result for each addition that
    a value goes through.  A piece is of 1024 rows, 32 or more of them side by side: at most 32 additions, 3 within a
    warp, 8 over the warps; 40 more pieces by 8 strands, 6 additions, and 8 over the strands: 57.  (One running sum for
    each 32nd of the 40960 rows is off by 10 times as much.)"""
    torch, gen = cuda, make_gen(cuda, 1)
    G, n, k = 64, 256, 8
    sizes = [0] * 20 + [40950] + [1] * 10 + [0] * 33
    m = sum(sizes)
    off = offsets_of(torch, sizes)
    row = torch.rand(n, generator=gen, device="cuda") + 1  # the same in every row
    dy = row.expand(m, n).contiguous()
    x, w = torch.ones(m, k, device="cuda", dtype=torch.bfloat16), torch.ones(G, n, k, device="cuda", dtype=torch.bfloat16)
    db = wl.grouped_linear_backward(dy, x, w, off, need_dx=False, need_dweight=False)[2]
    for g, s in enumerate(sizes):
        want = s * row.double()
        assert bool(((db[g].double() - want).abs() <= 57 * 2.0 ** -24 * want).all()), float(((db[g].double() - want).abs() / want).max())
    wc.check_device_status()


@pytest.mark.parametrize("captured", [False, True])
def test_side_by_side(cuda, wc, wl, captured):
    """The sums' second step, dx and dW overlap: what follows on the stream sees them finished, and inputs written anew at
    once disturb nothing; routing changes from call to call."""
    torch, gen = cuda, make_gen(cuda, 2)
    G, n, k = 16, 520, 264
    routes = [[0, 5000, 1] + [0] * 13, [312] * 15 + [321], [0] * 14 + [1000, 4001]]
    m = 5001
    w = torch.randn(G, n, k, generator=gen, device="cuda").to(torch.bfloat16)
    x, dy, z = (torch.randn(m, c, generator=gen, device="cuda").to(torch.bfloat16) for c in (k, n, n))
    tables = [offsets_of(torch, r) for r in routes]
    need = ("need_dx", "need_dweight", "need_dbias")
    alone = []
    for off in tables:
        for i in range(3):
            alone.append(wl.grouped_linear_backward(dy, x, w, off, activation="silu", pre_activation=z,
                                                    **{o: o == need[i] for o in need})[i])
            torch.cuda.synchronize()
    x1, dy1, z1, off1 = (torch.empty_like(t) for t in (x, dy, z, tables[0]))

    def step():
        got = []
        for off in tables:
            for to, t in ((x1, x), (dy1, dy), (z1, z), (off1, off)):
                to.copy_(t)
            got += wl.grouped_linear_backward(dy1, x1, w, off1, activation="silu", pre_activation=z1)
            for t in (x1, dy1, z1):
                t.fill_(float("nan"))
            off1.zero_()
        return got

    step()
    torch.cuda.synchronize()
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
    for _ in range(5):
        if captured:
            graph.replay()
        else:
            got = step()
        torch.cuda.synchronize()
        for a, b in zip(got, alone):
            assert torch.equal(a, b)
    wc.check_device_status()

"""The epilogue's slots of shared memory: the order of their uses on the host, and forward passes in which blocks that
leave by bulk stores and blocks that do not follow one another in a slot."""
import importlib
import os
import subprocess

import pytest

from _util import env_knobs
from conftest import ROOT
from test_linear_gpu import dt, forward_want, grouped_want, make_gen, offsets_of, quarters, same

DRIVER = os.path.join(ROOT, "tests", "drivers", "slot_turns_host_test.cpp")


@pytest.fixture(scope="module")
def wl():
    return importlib.import_module("7_b200.wave_linear")


def test_no_place_is_taken_while_a_store_reads_it(tmp_path):
    exe = str(tmp_path / "slot_turns")
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "7_b200", "csrc"), DRIVER, "-o", exe], check=True)
    run = subprocess.run([exe], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout


@pytest.mark.gpu
@pytest.mark.parametrize("io", ["bf16", "f16"])
@pytest.mark.parametrize("y_gap,z_gap", [(1, 0), (0, 1), (4, 0), (0, 4), (0, 0), (1, 1)])
@pytest.mark.parametrize("m,n,k,pair", [(4500, 520, 64, 0), (4500, 520, 64, 1), (1900, 264, 72, 0)])
def test_one_of_y_and_z_by_bulk_stores(cuda, wc, m, n, k, pair, y_gap, z_gap, io):
    """Rows of y or z that no bulk store can write, beside rows of the other that one can: short contractions, so that
    uses of a slot follow closely, and more tiles than CTAs."""
    torch, gen = cuda, make_gen(cuda, m + n + y_gap)
    t = dt(torch, io)
    x, w, b, r = (quarters(torch, gen, *s, io=io) for s in ((m, k), (n, k), (n,), (m, n)))
    z, y = forward_want(torch, x, w, b, r, "relu")
    code = wc.BF16 if io == "bf16" else wc.F16
    d = wc.LinearDesc(m, n, k, 0, code, code, code, code, wc.F32, 1)
    d.ldy, d.ldz = n + y_gap, n + z_gap
    import ctypes as C
    with env_knobs(wc, WAVE_CUDA_LINEAR_SWAP=0, WAVE_CUDA_LINEAR_PAIR=pair):
        for _ in range(3):
            got_y, got_z = (torch.full((m, n + gap), 7.0, dtype=t, device="cuda") for gap in (y_gap, z_gap))
            wc.check(wc.lib().wave_cuda_linear_fwd(C.byref(d), x.data_ptr(), w.data_ptr(), b.data_ptr(), r.data_ptr(), None,
                                                   got_y.data_ptr(), got_z.data_ptr(), None,
                                                   torch.cuda.current_stream().cuda_stream or None))
            same(torch, got_y[:, :n], y, "y")
            same(torch, got_z[:, :n], z, "z")
            assert bool((got_y[:, n:] == 7).all()) and bool((got_z[:, n:] == 7).all())
    wc.check_device_status()


@pytest.mark.gpu
def test_out_with_odd_rows_beside_z(cuda, wc, wl):
    """The same from Python: a caller's buffer with gaps, and z of the call's own."""
    torch, gen = cuda, make_gen(cuda, 2)
    m, n, k = 3000, 328, 136
    x, w = quarters(torch, gen, m, k, io="bf16"), quarters(torch, gen, n, k, io="bf16")
    z, y = forward_want(torch, x, w, None, None, "relu")
    wide = torch.full((m, n + 3), 7.0, dtype=torch.bfloat16, device="cuda")
    _, got_z = wl.linear(x, w, activation="relu", out=wide[:, :n], save_pre_activation=True)
    same(torch, wide[:, :n], y, "y")
    same(torch, got_z, z, "z")
    assert bool((wide[:, n:] == 7).all())
    wc.check_device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("pair", [0, 1])
@pytest.mark.parametrize("columns", [0, 48, 80, 208])
@pytest.mark.parametrize("save", [False, True])
def test_last_chunks_of_other_widths(cuda, wc, wl, columns, pair, save):
    """Tiles whose last chunk is narrower than 32 columns, features in whole pieces of 16 bytes."""
    torch, gen = cuda, make_gen(cuda, 3 + columns)
    knobs = dict(WAVE_CUDA_LINEAR_SWAP=0, WAVE_CUDA_LINEAR_PAIR=pair, WAVE_CUDA_LINEAR_SPLITS=1)
    if columns:
        knobs["WAVE_CUDA_LINEAR_COLUMNS"] = columns
    with env_knobs(wc, **knobs):
        for m, n, k in ((1528, 424, 216), (5370, 152, 408), (557, 2872, 200)):
            x, w, r = (quarters(torch, gen, *s, io="f16") for s in ((m, k), (n, k), (m, n)))
            z, y = forward_want(torch, x, w, None, r, "none")
            got = wl.linear(x, w, None, r, save_pre_activation=save)
            if save:
                same(torch, got[1], z, "z")
                got = got[0]
            same(torch, got, y, "y")
    wc.check_device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("pair", [0, 1])
@pytest.mark.parametrize("k", [8, 64, 200])
@pytest.mark.parametrize("save", [False, True])
def test_cut_blocks_behind_whole_ones(cuda, wc, wl, k, pair, save):
    """Experts' last blocks, written row by row, between whole blocks of others in the same warp's next tiles."""
    torch, gen = cuda, make_gen(cuda, 4 + k)
    n, sizes = 776, [300, 129, 0, 64, 1, 511, 33, 256, 95, 700, 161, 5, 1027, 128, 31]
    m = sum(sizes) + 9
    off = offsets_of(torch, sizes, 4)
    x, w, b = (quarters(torch, gen, *s, io="bf16") for s in ((m, k), (len(sizes), n, k), (len(sizes), n)))
    z, y = grouped_want(torch, x, w, off, b, "relu")
    with env_knobs(wc, WAVE_CUDA_LINEAR_SWAP=0, WAVE_CUDA_LINEAR_PAIR=pair):
        for _ in range(3):
            got = wl.grouped_linear(x, w, off, b, activation="relu", save_pre_activation=save)
            if save:
                same(torch, got[1], z, "z")
                got = got[0]
            same(torch, got, y, "y")
    wc.check_device_status()

"""The linear layers without a GPU: what the C ABI and the Python functions refuse, and the workspace they ask for."""
import ctypes as C
import importlib

import pytest


@pytest.fixture(scope="module")
def wl():
    return importlib.import_module("7_b200.wave_linear")


def desc(wc, tokens=8, n=32, k=64, **fields):
    d = wc.LinearDesc()
    wc.lib().wave_cuda_linear_desc_init(C.byref(d), tokens, n, k)
    for name, value in fields.items():
        setattr(d, name, value)
    return d


def test_desc_init(wc):
    d = desc(wc, 3, 5, 7)
    assert (d.tokens, d.out_features, d.in_features, d.experts) == (3, 5, 7, 0)
    assert (d.io_type, d.y_type, d.bias_type, d.dweight_type, d.dbias_type) == (wc.BF16,) * 4 + (wc.F32,)
    assert d.activation == 0 and d.ldx == 0 and d.expert_stride_w == 0
    wc.linear_validate(d)


@pytest.mark.parametrize("fields,code,message", [
    (dict(tokens=-1), "E_INVALID", "tokens must be >= 0; got -1"),
    (dict(out_features=0), "E_INVALID", "out_features and in_features must be >= 1; got 0 and 64"),
    (dict(in_features=-3), "E_INVALID", "out_features and in_features must be >= 1; got 32 and -3"),
    (dict(experts=1025), "E_INVALID", "experts must be between 0 (one weight matrix) and 1024; got 1025"),
    (dict(experts=-1), "E_INVALID", "experts must be between 0"),
    (dict(io_type=2), "E_UNSUPPORTED", "io_type must be bf16 or f16; got 2"),
    (dict(y_type=0), "E_UNSUPPORTED", "y_type must be io_type or f32; got 0"),
    (dict(bias_type=0), "E_UNSUPPORTED", "bias_type must be io_type or f32"),
    (dict(dweight_type=7), "E_UNSUPPORTED", "dweight_type must be io_type or f32"),
    (dict(dbias_type=0), "E_UNSUPPORTED", "dbias_type must be io_type or f32"),
    (dict(activation=5), "E_INVALID", "activation must be one of none, relu, gelu, gelu_tanh, silu; got 5"),
    (dict(activation=-1), "E_INVALID", "activation must be one of"),
    (dict(ldx=63), "E_INVALID", "ldx must be 0 or between 64 and 2^36 elements; got 63"),
    (dict(ldw=1), "E_INVALID", "ldw must be 0 or between 64"),
    (dict(ldy=31), "E_INVALID", "ldy must be 0 or between 32"),
    (dict(ldr=-32), "E_INVALID", "ldr must be 0 or between 32"),
    (dict(ldz=(1 << 36) + 1), "E_INVALID", "ldz must be 0 or between 32"),
    (dict(lddx=2), "E_INVALID", "lddx must be 0 or between 64"),
    (dict(lddw=2), "E_INVALID", "lddw must be 0 or between 64"),
    (dict(experts=2, expert_stride_w=32 * 64 - 1), "E_INVALID", "expert_stride_w must be 0 or hold a whole matrix"),
    (dict(experts=2, lddw=72, expert_stride_dw=32 * 64), "E_INVALID", "expert_stride_dw must be 0 or hold a whole matrix"),
    (dict(tokens=2**30, out_features=2**20), "E_INVALID", "too many output tiles"),
    (dict(tokens=2**30 + 1), "E_INVALID", "tokens and features must be at most 2^30"),
    (dict(in_features=2**31 - 1), "E_INVALID", "tokens and features must be at most 2^30"),
])
def test_descriptor_refusals(wc, fields, code, message):
    with pytest.raises(wc.WaveCudaError) as err:
        wc.linear_validate(desc(wc, **fields))
    assert err.value.code == getattr(wc, code)
    assert message in err.value.message


def test_forward_workspace_is_for_operands_that_are_laid_out(wc):
    assert wc.linear_workspace_bytes(desc(wc), False) == 0
    # 8 rows of 65 features padded to 72, and 32 of them for the weights; each rounded up to 256 bytes
    assert wc.linear_workspace_bytes(desc(wc, k=65), False) == 1280 + 4608
    assert wc.linear_workspace_bytes(desc(wc, ldx=68), False) == 1024
    assert wc.linear_workspace_bytes(desc(wc, tokens=1, k=65), False) == 4608  # a single row has no stride
    assert wc.linear_workspace_bytes(desc(wc, experts=3, expert_stride_w=32 * 64 + 4), False) == 3 * 4096


def fwd(wc, d, *ptrs, workspace=None):
    return wc.lib().wave_cuda_linear_fwd(C.byref(d), *ptrs, workspace, None)


X, W, Y, OFF = 0x10000, 0x20000, 0x30000, 0x40000  # never read: every call below is refused first


@pytest.mark.parametrize("fields,args,message", [
    (dict(), (0, W, 0, 0, 0, Y, 0), "X, W and Y must be non-null"),
    (dict(), (X, 0, 0, 0, 0, Y, 0), "X, W and Y must be non-null"),
    (dict(), (X, W, 0, 0, 0, 0, 0), "X, W and Y must be non-null"),
    (dict(), (X + 2, W, 0, 0, 0, Y, 0), "X and W must be 16-byte aligned"),
    (dict(experts=2), (X, W, 0, 0, 0, Y, 0), "grouped layers need the experts' offsets"),
    (dict(experts=2), (X, W, 0, Y, OFF, Y, 0), "a residual goes with one weight matrix"),
])
def test_forward_refuses_before_any_launch(wc, fields, args, message):
    rc = fwd(wc, desc(wc, **fields), *(a or None for a in args))
    assert rc in (wc.E_INVALID, wc.E_UNSUPPORTED)
    assert message in wc.lib().wave_cuda_last_error().decode()


@pytest.mark.parametrize("fields,args,message", [
    (dict(), (0, X, W, 0, 0, Y, Y, 0), "must be non-null device pointers"),
    (dict(), (Y, 0, W, 0, 0, Y, Y, 0), "must be non-null device pointers"),
    (dict(), (Y, X, 0, 0, 0, Y, Y, 0), "must be non-null device pointers"),
    (dict(activation=4), (Y, X, W, 0, 0, Y, Y, 0), "needs the pre-activation Z"),
    (dict(), (Y + 2, X, W, 0, 0, Y, Y, 0), "dY, X and W must be 16-byte aligned"),
    (dict(experts=2), (Y, X, W, 0, 0, Y, Y, 0), "grouped layers need the experts' offsets"),
])
def test_backward_refuses_before_any_launch(wc, fields, args, message):
    rc = wc.lib().wave_cuda_linear_bwd(C.byref(desc(wc, **fields)), *(a or None for a in args), None, None)
    assert rc == wc.E_INVALID
    assert message in wc.lib().wave_cuda_last_error().decode()


def test_no_device_is_an_error(wc):
    import torch
    if torch.cuda.is_available():
        pytest.skip("this machine has a device")
    assert fwd(wc, desc(wc), X, W, None, None, None, Y, None) == wc.E_CUDA


def test_no_tokens_needs_no_device(wc):
    assert fwd(wc, desc(wc, tokens=0), *([None] * 7)) == wc.OK


def test_python_refuses_cpu_tensors(wl):
    import torch
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(16, 8, dtype=torch.bfloat16)
    offsets = torch.zeros(3, dtype=torch.int32)
    for call in (lambda: wl.linear(x, w), lambda: wl.linear_backward(x, x, w),
                 lambda: wl.grouped_linear(x, w[None], offsets), lambda: wl.grouped_linear_backward(x, x, w[None], offsets)):
        with pytest.raises(ValueError, match="no CPU path"):
            call()
    with pytest.raises(ValueError, match="offsets must be given"):
        wl.grouped_linear(x, w[None], None)


@pytest.mark.parametrize("knobs", [{}, dict(TILE=16), dict(TILE=256, SWAP=1), dict(SPLITS=5), dict(PAIR=1), dict(PAIR=0, SWAP=0),
                                   dict(PAIR=1, SWAP=1, TILE=64), dict(PAIR=1, SPLITS=8)])
def test_every_plan_can_run(wc, knobs):
    """Whatever the sizes: a tile the kernels have, whole clusters, a ring of at least three stages, a block for every tile."""
    import math
    import random

    from _util import env_knobs

    rng = random.Random(7)
    size = lambda hi: int(math.exp(rng.uniform(0, math.log(hi))))  # noqa: E731
    with env_knobs(wc, **{f"WAVE_CUDA_LINEAR_{k}": v for k, v in knobs.items()}):
        for _ in range(400):
            m, n, k = size(200000), size(40000), size(40000)
            d = desc(wc, m if rng.random() > 0.02 else 0, n, k, experts=rng.choice([0, size(1024)]))
            if rng.random() < 0.3:
                d.y_type = d.dweight_type = wc.F32
            for product in range(3):
                sms = rng.choice([2, 16, 100, 132, 148])
                p = wc.linear_plan_for_sms(d, product, sms)
                pair = p["tile_rows"] == 256
                f32 = product != 1 and d.y_type == wc.F32
                unit = (128 if pair else 64) if product and not p["tokens_on_columns"] else (32 if pair else 16)
                assert p["tile_columns"] % unit == 0 and unit <= p["tile_columns"] <= (128 if f32 else 256), (m, n, k, p)
                assert 1 <= p["splits"] <= 8 and p["grid"] >= 1 and p["grid"] % p["splits"] == 0
                assert 3 <= p["stages"] <= 12
                assert not pair or (p["splits"] == 1 and p["grid"] % 2 == 0 and not f32)
                assert not p["tokens_on_columns"] or (product == 0 and p["tile_columns"] <= 128) or (
                    pair and product < 2 and d.experts > 0)
                if p["splits"] > 1:  # one cluster to a tile
                    rows, cols = p["tile_rows"], p["tile_columns"]
                    up = lambda a, b: -(-a // b)  # noqa: E731
                    P, Q = [((n, d.tokens) if p["tokens_on_columns"] else (d.tokens, n)), (d.tokens, k), (n, k)][product]
                    if not d.experts:
                        tiles = up(P, rows) * up(Q, cols)
                    elif product == 2:
                        tiles = up(P, rows) * up(Q, cols) * d.experts
                    else:
                        tokens, other = (cols, up(P, rows)) if p["tokens_on_columns"] else (rows, up(Q, cols))
                        # experts that each have one token more than whole tiles
                        tiles = other * max((d.tokens - e) // tokens + e for e in range(min(d.experts, d.tokens) + 1))
                    assert p["grid"] >= tiles * p["splits"], (m, n, k, p)


def test_plan_refusals(wc):
    for product, sms in ((-1, 148), (3, 148), (0, 1)):
        with pytest.raises(wc.WaveCudaError, match="product must be"):
            wc.linear_plan_for_sms(desc(wc), product, sms)

"""The longest sums of the linear layers' 16-bit results: refused on the host, before any launch."""
import ctypes as C

import pytest

from test_linear_host import OFF, W, X, Y, desc, fwd

FAR = (1 << 26) + 1


@pytest.mark.parametrize("fields,args,message", [
    (dict(k=FAR), (X, W, None, None, None, Y, None), "y in 16 bits takes sums of at most 2^26 products; got 67108865"),
    (dict(k=FAR, experts=2), (X, W, None, None, OFF, Y, None), "y in 16 bits takes sums"),
])
def test_forward(wc, fields, args, message):
    assert fwd(wc, desc(wc, n=1, **fields), *args) == wc.E_UNSUPPORTED
    assert message in wc.lib().wave_cuda_last_error().decode()


@pytest.mark.parametrize("fields,results,message", [
    (dict(n=FAR, k=1), (Y, None, None), "dX in 16 bits takes sums of at most 2^26 products; got 67108865"),
    (dict(tokens=FAR, n=8, k=8), (None, Y, None), "dW in 16 bits takes sums of at most 2^26 products; got 67108865"),
    (dict(tokens=FAR, n=8, k=8, experts=2), (None, Y, None), "dW in 16 bits takes sums"),
])
def test_backward(wc, fields, results, message):
    offsets = OFF if fields.get("experts") else None
    rc = wc.lib().wave_cuda_linear_bwd(C.byref(desc(wc, **fields)), Y, X, W, None, offsets, *results, Y, None)
    assert rc == wc.E_UNSUPPORTED
    assert message in wc.lib().wave_cuda_last_error().decode()


def test_what_is_not_asked_for_is_not_refused(wc):
    """f32 weight gradients, gradients that are left out and calls without tokens pass these checks (what they then lack here
    is a device)."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("this machine has a device")
    for d, results in ((desc(wc, tokens=FAR, n=8, k=8, dweight_type=wc.F32), (None, Y, None)),
                       (desc(wc, tokens=FAR, n=8, k=8), (None, None, Y)), (desc(wc, n=FAR, k=1), (None, Y, None)),
                       (desc(wc, tokens=0, n=FAR, k=1), (Y, None, None))):
        assert wc.lib().wave_cuda_linear_bwd(C.byref(d), Y, X, W, None, None, *results, Y, None) == wc.E_CUDA


@pytest.mark.gpu
def test_python_says_so_as_a_value_error(cuda, wc):
    import importlib
    wl = importlib.import_module("7_b200.wave_linear")
    torch = cuda
    x = torch.zeros(FAR, 1, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(1, 1, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="dW in 16 bits takes sums of at most"):
        wl.linear_backward(x, x, w)
    with pytest.raises(ValueError, match="y in 16 bits takes sums of at most"):
        wl.linear(x.view(1, FAR), x.view(1, FAR))
    dx, dw, db = wl.linear_backward(x, x, w, need_dweight=False)
    assert dw is None and not bool(dx.any()) and not bool(db.any())
    wc.check_device_status()

"""More refusals of the feed-forward operators, on the host: what a caller of the C entries or of the registered operators can pass by
the Python checks.  Nothing is launched."""
import ctypes
import math

import pytest

INVALID = 1
one, null = ctypes.c_void_p(64), None


@pytest.fixture(scope="module")
def lib():
    from verace_amd import _lib
    return _lib.load()


def test_betas_out_of_range(lib):
    """beta1 and beta2 of the SiTU forms are 2^-64 to 2^64; the other activations do not read them.  No rows: nothing is launched."""
    def forward(act, b1, b2):
        return lib.vmi_gated_linear(one, 16, null, one, 16, null, one, 16, null, 1, act, b1, b2, one, 8, 1, null, 0, 8, 16, null)

    def backward(act, b1, b2):
        return lib.vmi_gated_linear_bwd(one, 16, one, 16, one, 16, 1, act, b1, b2, null, one, 8, null, null, 0, 8, 16, one, 1 << 30, null)

    for call in (forward, backward):
        for bad in (0.0, -4.0, 2.0 ** -65, 2.0 ** 65, math.inf, -math.inf, math.nan):
            assert call(3, bad, 25.0) == INVALID and call(3, 4.0, bad) == INVALID, bad
            assert call(1, bad, bad) == 0
        for b1, b2 in ((2.0 ** -64, 2.0 ** 64), (2.0 ** 64, 2.0 ** -64), (4.0, 25.0)):
            assert call(3, b1, b2) == 0


def test_eps_out_of_range(lib):
    """eps of the 8-bit norm is a finite fp32 number, 0 or more, at the C entry (which the registered operator calls) and in Python; rows
    as they are do not read it."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    import torch
    import verace_amd as va

    def quant(norm, eps):
        return lib.vmi_norm_add_quant(one, 16, null, 0, null, 1, 1, norm, eps, null, one, one, 0, 16, null)

    for bad in (-1e-6, math.inf, -math.inf, math.nan):
        assert quant(1, bad) == INVALID and quant(0, bad) == 0
    assert quant(1, 0.0) == 0 and quant(1, 1e38) == 0
    with FakeTensorMode(allow_non_fake_inputs=True):
        a = torch.empty(3, 16, dtype=torch.bfloat16, device="cuda")
        for bad in (-1e-6, math.inf, math.nan, 1e39):
            with pytest.raises(RuntimeError, match="eps"):
                va.norm_add_quant(a, eps=bad)
        va.norm_add_quant(a, eps=3e38)

"""The packed product's kernels ask for their dynamic LDS on the device that they are launched on; a refusal is the call's error."""
import pytest
import torch

from biomedkg_amd import _lib as L
from biomedkg_amd import ops


@pytest.mark.skipif(torch.cuda.is_available(), reason="the buffers are the host's: nothing may be launched")
@pytest.mark.parametrize("times", [1, 2])
def test_a_refused_grant_is_the_calls_error(times):
    """without a device there is nothing to grant: every call that needs more LDS than a kernel gets unasked says so, the second
    one as well"""
    lib = L.lib()
    host = torch.zeros(1 << 12, dtype=torch.uint8)
    p = (host.data_ptr() + 255) // 256 * 256
    m, n, cols = 4000, 4000, 4000                            # 256 x 256 tiles
    for _ in range(times):
        assert lib.bkg_mx4_matmul(p, p, m, p, p, n, cols, None, p, 1, n, p, 1 << 40, None) != 0
        assert b"dynamic LDS" in lib.bkg_last_error()
    # one row of 64 panels, packed within the launch, and of 26 panels: 57 KB beside 12 KB of the kernel's own
    for n, cols in ((256, 8192), (100000, 8192), (256, 3300)):
        assert lib.bkg_mx4_linear(p, 1, cols, 1, p, p, n, cols, None, p, 1, n, p, 1 << 40, None) != 0
        assert b"dynamic LDS" in lib.bkg_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [2700, 3300, 3840, 3900, 8192])
@pytest.mark.parametrize("n", [40, 70000])
def test_rows_packed_within_the_launch_on_both_sides_of_what_is_asked_for(cols, n):
    gen = torch.Generator().manual_seed(cols + n)
    x = torch.randn(8192 // ((cols + 127) // 128 * 128), cols, generator=gen).cuda()
    table = ops.mx4_quantize(torch.randn(n, cols, generator=gen).cuda())
    got = ops.mx4_linear(x, table).double()
    xv, wv = ops.mx4_dequantize(ops.mx4_quantize(x)).double(), ops.mx4_dequantize(table).double()
    mag = xv.abs() @ wv.abs().t()
    assert float(((got - xv @ wv.t()).abs() - (cols + 5) * 2.0 ** -24 * mag).max()) <= 0

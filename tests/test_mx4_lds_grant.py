"""The packed product's kernels ask for their dynamic LDS on the device that they are launched on; a refusal is the call's error."""
import pytest
import torch

from biomedkg_amd import _lib as L


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
    for n in (256, 100000):                                  # one row of 64 panels, packed within the launch
        assert lib.bkg_mx4_linear(p, 1, 8192, 1, p, p, n, 8192, None, p, 1, n, p, 1 << 40, None) != 0
        assert b"dynamic LDS" in lib.bkg_last_error()

"""4-bit products at the edges of what they promise: long work ahead of them on the stream, and numbers and scales at the ends of their
ranges (see test_mx4_gpu.py for how a product is compared and its tolerance)."""
import pytest
import torch

from tests.test_mx4_gpu import check_product, layers, random_mx4, values64

pytestmark = pytest.mark.gpu


def test_the_time_of_the_kernel_ahead_is_not_the_products_own():
    """A kernel of 2.5 seconds that lets the next one start beside it: a product behind it is right, although every wait in it ends
    after two.  (The kernel ahead is the hook whose own wait runs out: bit 3 is its.)"""
    from crucible_strix_halo_b200 import capi
    L = layers()
    x, w = torch.randn(24, 256, device="cuda"), random_mx4(96, 256, 1)
    xq = random_mx4(200, 256, 2)
    one, many, y = (torch.empty(r, 96, device="cuda") for r in (1, 24, 200))
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    L.mx4_rows(x[:1], w, [one])
    torch.cuda.synchronize()
    assert capi.lib.cr_device_status() == 0
    one.zero_()
    capi.check(capi.lib.cr_debug_wait_timeout(status.data_ptr(), 2500000, torch.cuda.current_stream().cuda_stream))
    L.mx4_rows(x[:1], w, [one])                              # digits of its own
    L.mx4_rows(x, w, [many])                                 # digits from a kernel before it
    L.mx4_gemm(xq, w, [y])
    torch.cuda.synchronize()
    word = capi.lib.cr_device_status()
    capi.check(capi.lib.cr_device_status_clear())
    assert word == 8 and int(status) == 1
    check_product(x[:1].double().cpu(), values64(w), [one], 256)
    check_product(x.double().cpu(), values64(w), [many], 256)
    check_product(values64(xq), values64(w), [y], 256)

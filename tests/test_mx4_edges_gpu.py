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


def _ones(K, byte):
    """K x K, the identity times 2^(byte - 127)."""
    w = layers().Mx4.empty(K, K)
    w.codes.zero_()
    i = torch.arange(K, device="cuda")
    w.codes[i, i // 2] = torch.where(i % 2 == 0, 2, 32).to(torch.uint8)       # code 2 is 1.0
    w.scales.fill_(byte)
    return w


def _rows_of_sizes(exponents, K, dtype, seed):
    """A row for each exponent: its largest element is in [2^e, 2^(e + 1)), the others are of that size and of every smaller one."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    e = torch.tensor(exponents, device="cuda", dtype=torch.float64)[:, None]
    u = lambda: torch.rand(len(exponents), K, device="cuda", generator=gen, dtype=torch.float64)
    down = torch.floor(40 * u() ** 2)
    x = (1 + u()) * torch.exp2(e - down) * torch.where(u() < 0.5, -1.0, 1.0)
    x[:, ::32] = torch.exp2(e)                                                # one of every block has the exponent, and is exact
    x[:, 5] = (2 - 2.0 ** -7) * torch.exp2(e)[:, 0]                           # the largest of a 16-bit type with it
    x = torch.where(x.abs() < torch.exp2(e + 1) * (1 - 2.0 ** -9), x, torch.exp2(e))
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("exponents,byte", [(range(-126, -84), 187), (range(-84, -60), 127), (range(100, 128), 127), (range(118, 128), 100)])
def test_every_element_is_as_near_as_the_header_says(exponents, byte, dtype):
    """Products with the identity give the elements back, each with the error of its digits alone: what the digits hold of an element is a
    multiple of the last one's weight or of the element's own last bit, so that their sums are exact but for the final one."""
    L = layers()
    K, exponents = 128, list(exponents)
    x, w = _rows_of_sizes(exponents, K, dtype, 1), _ones(K, byte)
    y = torch.empty(len(exponents), K, device="cuda")
    L.mx4_rows(x, w, [y])
    digits = 12 if dtype == torch.float32 else 10
    e = torch.tensor(exponents, dtype=torch.float64)[:, None]
    limit = torch.exp2(e + 1 - 3 * digits) * torch.where(e == 127, 2, 1)
    limit = limit.clamp(min=2.0 ** -128)
    x64, got = x.double().cpu(), y.double().cpu() * 2.0 ** (127 - byte)
    assert torch.isfinite(got).all()
    # one rounding of the sum, and one where it lies under fp32's normal numbers
    over = (got - x64).abs() - limit - 2.0 ** -24 * x64.abs() - 2.0 ** (-150 + 127 - byte)
    assert over.max() <= 0, "row %d of exponent %d" % (int(over.amax(1).argmax()), exponents[int(over.amax(1).argmax())])
    for r in range(0, len(exponents), 5):                                     # a row alone makes its digits itself
        one = torch.empty(1, K, device="cuda")
        L.mx4_rows(x[r:r + 1], w, [one])
        assert torch.equal(one[0], y[r])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_types_largest_numbers(dtype):
    """Products of the largest numbers with ones do not overflow, and have their bits."""
    L = layers()
    top = torch.finfo(dtype).max
    x = torch.zeros(3, 64, device="cuda", dtype=dtype)
    x[0, 3], x[1, 40], x[2, 63] = top, -top, top * 0.875
    w, y = _ones(64, 127), torch.empty(3, 64, device="cuda")
    L.mx4_rows(x, w, [y])
    assert torch.equal(y, x.float())

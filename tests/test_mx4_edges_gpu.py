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


def _scaled(m, byte):
    """Gives block b of row r of a 4-bit matrix the scale byte[r, b]."""
    r, b = torch.arange(m.rows, device="cuda")[:, None], torch.arange(m.inner // 32, device="cuda")[None]
    m.scales[r // 128 * ((m.inner + 127) // 128) * 512 + b // 4 * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4] = byte.to(torch.uint8)


def _launched(name, call):
    """The kernels that `call` launches hold one of that name."""
    from crucible_strix_halo_b200 import capi
    stream = torch.cuda.current_stream().cuda_stream
    capi.check(capi.lib.cr_profile_enable(1))
    try:
        capi.check(capi.lib.cr_profile_begin(stream))
        call()
        return name in capi.profile_collect()
    finally:
        capi.check(capi.lib.cr_profile_enable(0))


@pytest.mark.parametrize("R,K,N,kernel", [
    (4000, 1088, 4128, "mx4_gemm_pair_kernel"),                  # 16 x 17 tiles of 256 x 256: what is left of the last wave whole,
    (2040, 1088, 9824, "mx4_gemm_pair_kernel"),                  # in four
    (2000, 1088, 5632, "mx4_gemm_pair_kernel"),                  # and in two
    (300, 1088, 2048, "mx4_gemm_split_kernel"),
])
def test_scales_that_differ_from_row_to_row_and_block_to_block(R, K, N, kernel):
    """Scales from 0 to 254: those of a block are far from its neighbours' in X and as far the other way in W, and every row of X and of W
    has an offset of its own, so that the products of an output are of one size, and another output's are of another."""
    L = layers()
    x, w = random_mx4(R, K, 1), random_mx4(N, K, 2)
    b = torch.arange(K // 32, device="cuda")[None]
    size = b * 97 % 34 * 7                                       # 0..231, all different
    t, u = (torch.arange(n, device="cuda")[:, None] * 5 % 23 for n in (R, N))
    _scaled(x, size + t)                                         # 0..253
    _scaled(w, 254 - size - u)
    y = torch.empty(R, N, device="cuda")
    assert _launched(kernel, lambda: L.mx4_gemm(x, w, [y]))
    check_product(values64(x), values64(w), [y], K)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("low", [0, 54])
@pytest.mark.parametrize("R,N", [(1, 96), (9, 9632), (16, 9632), (24, 9632), (50, 9632)])
def test_rows_with_weights_of_every_scale(R, N, low, dtype):
    """Scales of W from 0 to 199 and from 54 to 253, elements of X as much larger or smaller."""
    L = layers()
    K = 1088
    gen = torch.Generator(device="cuda").manual_seed(R)
    w = random_mx4(N, K, 2)
    b = torch.arange(K // 32, device="cuda")[None]
    size = b * 97 % 34 * 53 // 10                                # 0..174
    u = torch.arange(N, device="cuda")[:, None] * 5 % 26
    _scaled(w, low + size + u)                                   # low..low + 199
    e = (110 if low == 0 else 56) - size.double().repeat_interleave(32, 1)
    x = ((1 + torch.rand(R, K, device="cuda", generator=gen, dtype=torch.float64)) * torch.exp2(e)).to(dtype)
    x = torch.where(torch.rand(R, K, device="cuda", generator=gen) < 0.5, -x, x)
    y = torch.empty(R, N, device="cuda")
    L.mx4_rows(x, w, [y])
    x64, w64 = x.double().cpu(), values64(w)
    limit = K * 2.0 ** -24 * (x64.abs() @ w64.abs().t()) + 2.0 ** -128 * w64.abs().sum(1)
    assert ((y.double().cpu() - x64 @ w64.t()).abs() <= limit).all()

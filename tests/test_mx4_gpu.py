"""Microscaled 4-bit floats (cr_mx4_quant, cr_mx4_dequant) and the products with them (cr_mx4_gemm, cr_mx4_rows) against the
definition in 64 bits.

Tolerances.  Quantisation is exact.  A product's sums are fp32: in any order, K terms are off by at most K 2^-24 of the sum of their
magnitudes, which is counted for every element; a bf16 output adds half a step, 2^-8 of its value."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def layers():
    from crucible_strix_halo_b200 import layers
    return layers


def values64(m):
    """The numbers an Mx4 stands for, element by element from the layout's definition."""
    codes, scales = m.codes.cpu().long(), m.scales.cpu().long()
    nib = torch.stack([codes & 15, codes >> 4], -1).reshape(m.rows, m.inner)
    r, b = torch.arange(m.rows)[:, None], torch.arange(m.inner // 32)[None]
    byte = scales[(r // 128 * ((m.inner + 127) // 128) + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4]
    unit = torch.where(byte == 255, torch.full(byte.shape, math.nan, dtype=torch.float64), torch.exp2(byte.double() - 127))
    return (torch.where(nib >= 8, -1.0, 1.0).double() * GRID[nib & 7]) * unit.repeat_interleave(32, 1)


def quantised64(x):
    """The specification's conversion: nearest grid point, ties to the even code; NaN for blocks that are not finite."""
    b = x.double().cpu().reshape(x.shape[0], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    s = torch.where(top > 0, torch.floor(torch.log2(torch.where(top > 0, top, 1.0))) - 2, -127.0)
    # log2 of a number just below a power of two may round up
    s = torch.where(torch.exp2(s + 2) > top, s - 1, s).clamp(-127, 127)
    s = torch.where(top > 0, s, -127.0)
    y = b / torch.exp2(s)
    dist = (y.abs()[..., None] - GRID).abs()
    near = dist.argmin(-1)                                                # of two as near the lower code ...
    up = (near + 1).clamp(max=7)
    tie = (dist.gather(-1, up[..., None]) == dist.gather(-1, near[..., None]))[..., 0]
    near = torch.where(tie & (near % 2 == 1), up, near)                   # ... unless the upper one is even
    v = torch.copysign(GRID[near], y) * torch.exp2(s)
    return torch.where(torch.isfinite(top), v, torch.full_like(v, math.nan)).reshape(x.shape)


def random_mx4(rows, inner, seed, low=118, high=124):
    """Random codes; scales of a few sizes; what belongs to no row or block holds NaN scales."""
    L, gen = layers(), torch.Generator(device="cuda").manual_seed(seed)
    m = L.Mx4.empty(rows, inner)
    m.codes.copy_(torch.randint(0, 256, m.codes.shape, device="cuda", generator=gen, dtype=torch.uint8))
    m.scales.fill_(255)
    r, b = torch.arange(rows, device="cuda")[:, None], torch.arange(inner // 32, device="cuda")[None]
    at = (r // 128 * ((inner + 127) // 128) + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4
    m.scales[at.flatten()] = torch.randint(low, high, (at.numel(),), device="cuda", generator=gen, dtype=torch.uint8)
    return m


def check_product(x64, w64, outs, K):
    want, size = x64 @ w64.t(), x64.abs() @ w64.abs().t()
    col = 0
    for o in outs:
        got, y, s = o.double().cpu(), want[:, col:col + o.shape[1]], size[:, col:col + o.shape[1]]
        limit = K * 2.0 ** -24 * s
        if o.dtype == torch.bfloat16:
            limit = limit * (1 + 2.0 ** -8) + 2.0 ** -8 * y.abs()
        assert torch.equal(got.isnan(), y.isnan())
        over = ((got - y).abs() - limit).nan_to_num(nan=-1.0)
        assert over.max().item() <= 0, "off by %g more than %g" % (over.max().item(), limit.flatten()[over.argmax()].item())
        col += o.shape[1]
    status()


def status():
    from crucible_strix_halo_b200 import capi
    torch.cuda.synchronize()
    assert capi.lib.cr_device_status() == 0


# ---- quantisation ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner", [(1, 64), (13, 192), (129, 320), (300, 2048)])
def test_quantisation_is_the_definition(rows, inner, dtype):
    L = layers()
    gen = torch.Generator(device="cuda").manual_seed(rows)
    x = (torch.randn(rows, inner, device="cuda", generator=gen) * torch.exp(2 * torch.randn(inner, device="cuda", generator=gen))).to(dtype)
    x[0, :32] = 0
    q = L.mx4_quant(x)
    want = quantised64(x)
    assert torch.equal(values64(q), want)
    for t in TYPES:
        assert torch.equal(L.mx4_dequant(q, t).cpu(), want.float().to(t))


def test_quantisation_of_every_border():
    """Points of the grid, the ties between them and their neighbours, at several scales; the largest and smallest numbers."""
    L = layers()
    g = [0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7]
    t = torch.tensor(g, dtype=torch.float32)
    rows = []
    for e in (-126, -30, 0, 1, 60, 124):
        v = t * 2.0 ** e
        for w in (v, torch.nextafter(v, torch.zeros(16)), torch.nextafter(v, torch.full((16,), math.inf)).clamp(max=float(v.max()))):
            rows.append(torch.cat([w, -w]))
    tiny = torch.arange(1, 33, dtype=torch.float32) * 2.0 ** -149
    big = torch.full((32,), torch.finfo(torch.float32).max)
    one = torch.zeros(32)
    one[31] = -2.0 ** -149
    rows += [tiny, big, one, torch.zeros(32)]
    x = torch.stack(rows).reshape(-1, 64).cuda()
    q = L.mx4_quant(x)
    want = quantised64(x)
    assert torch.equal(values64(q), want)
    assert torch.equal(L.mx4_dequant(q).cpu(), want.float())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_blocks_that_are_not_finite(bad, dtype):
    L = layers()
    x = torch.ones(3, 128, device="cuda", dtype=dtype)
    x[1, 40] = bad
    got = L.mx4_dequant(L.mx4_quant(x))
    assert got[1, 32:64].isnan().all()
    got[1, 32:64] = 1
    assert torch.equal(got, torch.ones_like(got))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset,pitch", [(0, 200), (1, 193), (8, 256)])
def test_rows_at_any_pitch_and_address(offset, pitch, dtype):
    L = layers()
    buf = torch.randn(40 * pitch + offset, device="cuda").to(dtype)
    x = buf[offset:offset + 40 * pitch].view(40, pitch)[:, :192]
    q = L.mx4_quant(x)
    assert torch.equal(values64(q), quantised64(x))
    back = torch.full((40 * pitch + offset,), 7.0, device="cuda", dtype=dtype)
    y = back[offset:offset + 40 * pitch].view(40, pitch)
    L.mx4_dequant(q, out=y[:, :192])
    assert torch.equal(y[:, :192].cpu(), quantised64(x).float().to(dtype))
    assert (y[:, 192:] == 7).all() and (back[:offset] == 7).all()


def test_scale_bytes_of_no_row_are_left():
    L = layers()
    q = L.Mx4.empty(5, 192)
    q.scales.fill_(99)
    q.codes.fill_(99)
    L.mx4_quant(torch.ones(5, 192, device="cuda"), q)
    r, b = torch.arange(5)[:, None], torch.arange(6)[None]
    at = (b // 4 * 512 + r % 32 * 16 + b % 4).flatten()
    s = q.scales.cpu()
    assert (s[at] == 125).all()
    s[at] = 99
    assert (s == 99).all()


# ---- products ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("R,K,widths,f32", [
    (1, 64, [32], [True]),                                       # the smallest
    (1, 2048, [2048], [False]),
    (7, 128, [32], [False]),
    (64, 192, [96], [True]),                                     # half a group of scales at the end of K
    (127, 256, [128], [True]),
    (128, 320, [256, 32], [False, True]),
    (129, 448, [128, 64, 32], [True, False, True]),
    (200, 6144, [160], [True]),                                  # long K, few tiles: K is split
    (300, 2048, [1024, 512, 32], [True, False, True]),
    (257, 512, [544], [True]),
    (2100, 1088, [2080, 288], [False, True]),                    # several waves of tiles, ragged both ways
    (5000, 128, [4128], [True]),                                 # more tiles than CTAs, short K
    (2040, 320, [9792, 32], [True, False]),                      # the last wave's few tiles are cut into four
    (2000, 192, [5536, 96], [False, True]),                      # and into two
])
def test_product_of_two_4_bit_matrices(R, K, widths, f32):
    L = layers()
    x, w = random_mx4(R, K, R + K), random_mx4(sum(widths), K, R + K + 1)
    outs = [torch.full((R, c), math.nan, device="cuda", dtype=torch.float32 if f else torch.bfloat16) for c, f in zip(widths, f32)]
    L.mx4_gemm(x, w, outs)
    check_product(values64(x), values64(w), outs, K)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,K,widths,f32", [
    (1, 64, [32], [True]),
    (1, 4096, [2048], [True]),
    (2, 192, [64, 32], [False, True]),
    (8, 320, [160], [True]),
    (9, 2048, [1024, 32], [True, False]),
    (13, 2560, [4128], [True]),
    (16, 448, [288], [True]),
    (17, 6144, [96], [True]),
    (33, 1088, [544], [False]),
    (72, 2048, [8224], [True]),
    (100, 256, [128], [True]),
    (11, 320, [9632], [True]),                                   # more tiles than a wave of clusters, by the number of digit rows:
    (13, 576, [9568, 32], [False, True]),
    (17, 192, [9632], [True]),
    (20, 1088, [9600, 64], [True, False]),
    (21, 512, [9632], [True]),
    (24, 320, [9632], [True]),
    (25, 448, [9760], [True]),
    (50, 192, [19232], [True]),                                  # several tiles a pair, several passes
])
def test_product_of_rows_as_they_are(R, K, widths, f32, dtype):
    L = layers()
    gen = torch.Generator(device="cuda").manual_seed(R)
    x = (torch.randn(R, K, device="cuda", generator=gen) * torch.exp(torch.randn(K, device="cuda", generator=gen))).to(dtype)
    w = random_mx4(sum(widths), K, R + K)
    outs = [torch.full((R, c), math.nan, device="cuda", dtype=torch.float32 if f else torch.bfloat16) for c, f in zip(widths, f32)]
    L.mx4_rows(x, w, outs)
    check_product(x.double().cpu(), values64(w), outs, K)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K,N", [(64, 96), (2048, 2048), (2560, 13952)])
def test_a_row_has_the_same_bits_in_every_call(K, N, dtype):
    L = layers()
    w = random_mx4(N, K, N)
    x = torch.randn(45, K, device="cuda").to(dtype)
    whole = torch.empty(45, N, device="cuda")
    L.mx4_rows(x, w, [whole])
    for r0, n in ((0, 1), (3, 2), (5, 4), (7, 8), (11, 13), (20, 20), (20, 24), (1, 16), (44, 1)):
        part = torch.empty(n, N, device="cuda")
        L.mx4_rows(x[r0:r0 + n], w, [part])
        assert torch.equal(part, whole[r0:r0 + n])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_very_large_and_very_small_numbers(dtype):
    """Each row of X has a size of its own, and so has each block of W: the sums stay those of the numbers, subnormal results apart."""
    L = layers()
    e = torch.tensor([-100, -40, -14, 0, 15, 40, 60], device="cuda")
    x = (torch.randn(7, 256, device="cuda") * torch.exp2(e.float())[:, None]).to(dtype)
    w = random_mx4(64, 256, 3, low=100, high=160)
    y = torch.empty(7, 64, device="cuda")
    L.mx4_rows(x, w, [y])
    check_product(x.double().cpu(), values64(w), [y], 256)


def test_rows_of_numbers_near_the_ends_of_the_range():
    """Rows of numbers down to 2^-126 and up to 2^127 with weights of the other size: what lies under 2^-127 in X is left out, 2^-128 an
    element."""
    L = layers()
    K = 256
    gen = torch.Generator(device="cuda").manual_seed(3)
    for e, low in ((-126, 220), (-110, 200), (126, 40)):
        x = (1 + torch.rand(4, K, device="cuda", generator=gen)) * 2.0 ** e * (1 - 2 * torch.randint(0, 2, (4, K), device="cuda", generator=gen))
        w = random_mx4(64, K, 5, low=low, high=low + 3)
        y = torch.empty(4, 64, device="cuda")
        L.mx4_rows(x, w, [y])
        x64, w64 = x.double().cpu(), values64(w)
        limit = K * 2.0 ** -24 * (x64.abs() @ w64.abs().t()) + 2.0 ** -127 * w64.abs().sum(1)
        assert ((y.double().cpu() - x64 @ w64.t()).abs() <= limit).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_with_an_outlier_keep_their_small_elements(dtype):
    """One element 2^13 times the others: the products of the others with it left out of the weights are as exact as ever."""
    L = layers()
    x = torch.randn(3, 256, device="cuda")
    x[:, 100] = 2.0 ** 13
    x = x.to(dtype)
    w = random_mx4(64, 256, 4)
    w.codes[:, 50] = 0                                       # elements 100 and 101
    y = torch.empty(3, 64, device="cuda")
    L.mx4_rows(x, w, [y])
    x64 = x.double().cpu()
    x64[:, 100:102] = 0
    want, size = x64 @ values64(w).t(), x64.abs() @ values64(w).abs().t()
    assert ((y.double().cpu() - want).abs() <= 256 * 2.0 ** -24 * size).all()


@pytest.mark.parametrize("R", [5, 300])
def test_scales_of_every_size(R):
    """Blocks of X and W whose scales go over the whole range of the byte, 0 and 254 among them, and whose products are of one size."""
    L = layers()
    K, N = 32 * 256, 96
    x, w = random_mx4(R, K, 1), random_mx4(N, K, 2)
    up = (torch.arange(256, device="cuda") * 97 % 255).to(torch.uint8)                  # every value of 0..254 (and one twice)
    for m, byte in ((x, up), (w, 254 - up)):
        r, b = torch.arange(m.rows, device="cuda")[:, None], torch.arange(256, device="cuda")[None]
        m.scales[(r // 128 * 64 + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4] = byte[None].expand(m.rows, 256)
    y = torch.empty(R, N, device="cuda")
    L.mx4_gemm(x, w, [y])
    check_product(values64(x), values64(w), [y], K)


@pytest.mark.parametrize("call", ["gemm", "rows"])
@pytest.mark.parametrize("R", [5, 300])
def test_blocks_that_are_nan_reach_their_own_outputs_alone(call, R):
    L = layers()
    K, N = 320, 160
    x, w = random_mx4(R, K, 1), random_mx4(N, K, 2)
    w.scales[(37 % 32) * 16 + 37 // 32 * 4 + 1] = 255          # block 1 of row 37
    w64, x64 = values64(w), values64(x)
    y = torch.empty(R, N, device="cuda")
    if call == "gemm":
        x.scales[512 + 3 * 16] = 255                           # block 4 of row 3
        x64 = values64(x)
        L.mx4_gemm(x, w, [y])
    else:
        rows = x64.float().cuda()
        rows[4, 7] = math.nan
        x64[4, 7] = math.nan
        L.mx4_rows(rows, w, [y])
    check_product(x64, w64, [y], K)


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_a_row_that_is_not_finite_is_nan_and_leaves_the_others(value):
    L = layers()
    x, w = torch.randn(9, 128, device="cuda"), random_mx4(64, 128, 2)
    x[4, 20] = value
    y = torch.empty(9, 64, device="cuda")
    L.mx4_rows(x, w, [y])
    assert y[4].isnan().all()
    keep = [0, 1, 2, 3, 5, 6, 7, 8]
    check_product(x[keep].double().cpu(), values64(w), [y[keep]], 128)


@pytest.mark.parametrize("value", [math.inf, math.nan])
@pytest.mark.parametrize("R", [13, 24, 60])
def test_many_rows_of_which_one_is_not_finite(R, value):
    L = layers()
    x, w = torch.randn(R, 192, device="cuda").bfloat16(), random_mx4(288, 192, 2)
    x[R - 2, 190] = value
    y = torch.empty(R, 288, device="cuda")
    L.mx4_rows(x, w, [y])
    assert y[R - 2].isnan().all()
    keep = [r for r in range(R) if r != R - 2]
    check_product(x[keep].double().cpu(), values64(w), [y[keep]], 192)


def test_many_rows_captured_and_beside_another_stream():
    """24 rows at a time, the weights made by the call before: replayed with new rows and weights, another stream's calls in between."""
    L = layers()
    R, K, N = 24, 320, 9632
    x, plain = torch.zeros(R, K, device="cuda", dtype=torch.bfloat16), torch.zeros(N, K, device="cuda")
    w, y = L.Mx4.empty(N, K), torch.empty(R, N, device="cuda")
    other, side = random_mx4(N, K, 8), torch.cuda.Stream()
    xo = torch.randn(R, K, device="cuda")
    want = torch.empty(R, N, device="cuda")
    L.mx4_rows(xo, other, [want])
    L.mx4_rows(x, L.mx4_quant(plain, out=w), [y])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(2):
            L.mx4_rows(x, L.mx4_quant(plain, out=w), [y])
    for seed in (1, 2):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        x.copy_(torch.randn(R, K, device="cuda", generator=gen))
        plain.copy_(torch.randn(N, K, device="cuda", generator=gen))
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            yo = torch.empty(R, N, device="cuda")
            L.mx4_rows(xo, other, [yo])
        torch.cuda.synchronize()
        check_product(x.double().cpu(), values64(w), [y], K)
        assert torch.equal(yo, want)


@pytest.mark.parametrize("call", ["gemm", "rows"])
@pytest.mark.parametrize("R", [3, 130, 700])
def test_outputs_at_a_pitch_leave_what_is_beside_them(call, R):
    L = layers()
    K, widths = 192, [64, 96]
    x, w = random_mx4(R, K, 5), random_mx4(160, K, 6)
    bufs = [torch.full((R + 2, 160), 7.0, device="cuda", dtype=t) for t in (torch.float32, torch.bfloat16)]
    outs = [b[1:R + 1, 16:16 + c] for b, c in zip(bufs, widths)]
    if call == "gemm":
        L.mx4_gemm(x, w, outs)
    else:
        L.mx4_rows(values64(x).float().cuda(), w, outs)
    check_product(values64(x), values64(w), outs, K)
    for b, c in zip(bufs, widths):
        b[1:R + 1, 16:16 + c] = 7
        assert (b == 7).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset,pitch", [(0, 200), (1, 193), (8, 256)])
def test_rows_product_at_any_pitch_and_address(offset, pitch, dtype):
    L = layers()
    buf = torch.randn(11 * pitch + offset, device="cuda").to(dtype)
    x = buf[offset:offset + 11 * pitch].view(11, pitch)[:, :192]
    w, y = random_mx4(96, 192, 8), torch.empty(11, 96, device="cuda")
    L.mx4_rows(x, w, [y])
    check_product(x.double().cpu(), values64(w), [y], 192)


def test_weights_past_32_bits_of_bytes():
    """A matrix whose codes pass 2^31 bytes: its last rows are multiplied, and quantised, as the first ones are."""
    L = layers()
    N, K = 1 << 20, 4288
    m = L.Mx4(torch.zeros(N, K // 2, device="cuda", dtype=torch.uint8), torch.full((N // 128 * 34 * 512,), 127, device="cuda", dtype=torch.uint8), N, K)
    tail = random_mx4(128, K, 3)
    m.codes[-128:] = tail.codes
    m.scales[-tail.scales.numel():] = tail.scales
    x = torch.randn(3, K, device="cuda")
    want = x.double().cpu()
    y = torch.empty(3, N, device="cuda")
    L.mx4_rows(x, m, [y])
    assert not y[:, :-128].any()
    check_product(want, values64(tail), [y[:, -128:]], K)
    xq = random_mx4(3, K, 4)
    L.mx4_gemm(xq, m, [y])
    assert not y[:, :-128].any()
    check_product(values64(xq), values64(tail), [y[:, -128:]], K)


# ---- streams, graphs, refusals -------------------------------------------------------------------------------------------

def test_captured_calls_replay_on_new_inputs():
    L = layers()
    K, N = 512, 288
    w = random_mx4(N, K, 1)
    x, small = torch.zeros(150, K, device="cuda"), torch.zeros(5, K, device="cuda")
    xq, y, z = L.Mx4.empty(150, K), torch.empty(150, N, device="cuda"), torch.empty(5, N, device="cuda")

    def calls():
        L.mx4_quant(x, xq)
        L.mx4_gemm(xq, w, [y])
        L.mx4_rows(small, w, [z])
    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    for seed in (1, 2):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        x.normal_(generator=gen)
        small.normal_(generator=gen)
        graph.replay()
        check_product(quantised64(x), values64(w), [y], K)
        check_product(small.double().cpu(), values64(w), [z], K)


def test_calls_on_two_streams_do_not_disturb_each_other():
    L = layers()
    K, N = 2048, 2048
    w = random_mx4(N, K, 1)
    xs = [random_mx4(R, K, R) for R in (40, 900)]
    rows = [torch.randn(9, K, device="cuda") for _ in range(2)]
    want = [(L.mx4_gemm(x, w, [torch.empty(x.rows, N, device="cuda")])[0], L.mx4_rows(r, w, [torch.empty(9, N, device="cuda")])[0]) for x, r in zip(xs, rows)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(20):
        for s, x, r in zip(streams, xs, rows):
            with torch.cuda.stream(s):
                got.append((L.mx4_gemm(x, w, [torch.empty(x.rows, N, device="cuda")])[0], L.mx4_rows(r, w, [torch.empty(9, N, device="cuda")])[0]))
    status()
    for i, (a, b) in enumerate(got):
        assert torch.equal(a, want[i % 2][0]) and torch.equal(b, want[i % 2][1])


def test_plain_launches_give_the_same_bits():
    """Without programmatic dependent launches the same kernels run one after the other."""
    from crucible_strix_halo_b200 import capi
    L = layers()
    K, N = 2560, 4128
    x, w = torch.randn(60, K, device="cuda").bfloat16(), random_mx4(N, K, 1)
    xq = random_mx4(300, K, 2)

    def calls():
        y = [torch.empty(r, N, device="cuda") for r in (1, 9, 60, 300)]
        L.mx4_rows(x[:1], w, y[:1])
        L.mx4_rows(x[:9], w, y[1:2])
        L.mx4_rows(x, w, y[2:3])
        L.mx4_gemm(xq, w, y[3:])
        return y + [L.mx4_dequant(L.mx4_quant(x))]
    want = calls()
    capi.set_options(pdl=0)
    try:
        got = calls()
    finally:
        capi.set_options(pdl=1)
    status()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_projection_chain_as_a_prompt_and_as_steps():
    """Prompt rows through quantise, 4-bit input projection and the GDN core; the input projection of the same rows as verify rows
    gives the core's rows of the same numbers."""
    from crucible_strix_halo_b200 import capi
    L = layers()
    g = capi.Geometry(256, 16, 2, 4, 2)
    gen = torch.Generator(device="cuda").manual_seed(9)
    rn = lambda *s, std=1.0: torch.randn(*s, device="cuda", generator=gen) * std
    R, C, Z = 517, g.gdn_channels, 512
    x = rn(R, 256).bfloat16()
    w = L.mx4_quant(rn(C + Z + 32, 256, std=1 / 16))
    gw = L.GdnWeights(g, rn(C, 4, std=0.5), rn(4) - 1, rn(4, std=0.5), 1 + rn(128, std=0.1))
    qkv, z, ab = (torch.empty(R, c, device="cuda", dtype=torch.bfloat16) for c in (C, Z, 32))
    xq = L.mx4_quant(x)
    L.mx4_gemm(xq, w, [qkv, z, ab])
    check_product(values64(xq), values64(w), [qkv, z, ab], 256)
    rows = [torch.empty(13, c, device="cuda", dtype=torch.bfloat16) for c in (C, Z, 32)]
    L.mx4_rows(L.mx4_dequant(xq)[:13], w, rows)
    for a, b in zip(rows, (qkv, z, ab)):                      # two orders of the same exact products, each rounded once
        assert (a.float() - b[:13].float()).abs().max() <= 2.0 ** -7 * b[:13].float().abs().max()
    out = L.GdnPrefillPlan(gw, R, in_dtype=capi.IN_BF16).run(L.GdnSession(g), qkv, z, ab[:, :8].contiguous(), 0, capi.GDN_CHUNK_TC)
    status()
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("call,error", [
    ("L.mx4_quant(torch.ones(2, 96, device='cuda'))", ValueError),                                     # inner not a multiple of 64
    ("L.mx4_quant(torch.ones(0, 64, device='cuda'))", ValueError),
    ("L.mx4_quant(torch.ones(2, 64, device='cuda').double())", TypeError),
    ("L.mx4_quant(torch.ones(64, 2, device='cuda').t())", ValueError),
    ("L.mx4_quant(torch.ones(2, 64))", ValueError),
    ("L.mx4_quant(torch.ones(64, device='cuda'))", ValueError),
    ("L.mx4_quant(torch.ones(3, 64, device='cuda'), m(2, 64))", ValueError),
    ("L.mx4_dequant(m(2, 64), out=torch.ones(2, 32, device='cuda'))", ValueError),
    ("L.mx4_gemm(m(2, 64), m(32, 128), [o(2, 32)])", RuntimeError),
    ("L.mx4_gemm(m(2, 64), m(32, 64), [o(3, 32)])", ValueError),
    ("L.mx4_gemm(m(2, 64), m(32, 64), [o(2, 64)])", RuntimeError),
    ("L.mx4_gemm(m(2, 64), m(32, 64), [o(2, 32).half()])", TypeError),
    ("L.mx4_gemm(m(2, 64), m(32, 64), [])", RuntimeError),
    ("L.mx4_rows(torch.ones(2, 128, device='cuda'), m(32, 64), [o(2, 32)])", ValueError),
    ("L.mx4_rows(torch.ones(0, 64, device='cuda'), m(32, 64), [o(0, 32)])", RuntimeError),
    ("L.mx4_rows(torch.ones(2, 64, device='cuda').int(), m(32, 64), [o(2, 32)])", TypeError),
    ("L.mx4_rows(torch.ones(2, 64, device='cuda'), L.Mx4(m(32, 64).codes, m(32, 64).scales[:100], 32, 64), [o(2, 32)])", ValueError),
    ("L.mx4_rows(torch.ones(2, 64, device='cuda'), L.Mx4(m(32, 64).codes, m(32, 64).scales, 64, 64), [o(2, 64)])", ValueError),
    ("L.mx4_rows(torch.ones(2, 64, device='cuda'), m(33, 64), [o(2, 33)])", RuntimeError),
])
def test_refusals(call, error):
    L = layers()
    scope = dict(L=L, torch=torch, m=L.Mx4.empty, o=lambda *s: torch.empty(*s, device="cuda"))
    with pytest.raises(error):
        eval(call, scope)
    status()

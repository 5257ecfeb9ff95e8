"""4-bit matrices, products and choices of a token whose offsets pass 32 bits, and calls of very many rows: what lies at the end is as
right as what lies at the start (see test_mx4_gpu.py for the tolerance of a product)."""
import pytest
import torch

from tests.test_mx4_gpu import check_product, layers, quantised64, random_mx4, status, values64

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def free():
    yield
    torch.cuda.empty_cache()


def _part(m, r0):
    """The rows of a 4-bit matrix from r0, a multiple of 128, on."""
    groups = (m.inner + 127) // 128
    return layers().Mx4(m.codes[r0:], m.scales[r0 // 128 * groups * 512:], m.rows - r0, m.inner)


def test_quantisation_past_32_bits_of_elements():
    L = layers()
    rows, inner = (1 << 20) + 5, 4160
    x = torch.zeros(rows, inner, device="cuda", dtype=torch.bfloat16)
    x[-133:] = torch.randn(133, inner, device="cuda")
    x[:3] = x[-3:]
    q = L.mx4_quant(x)
    want = quantised64(x[-133:])
    tail = _part(q, 1 << 20)
    assert torch.equal(values64(tail), want[-5:])
    y = torch.empty(rows, inner, device="cuda", dtype=torch.bfloat16)
    L.mx4_dequant(q, out=y)
    assert torch.equal(y[-133:].cpu(), want.bfloat16()) and torch.equal(y[:3].cpu(), want[-3:].bfloat16())
    assert not y[3:-133].any()
    status()


def test_outputs_past_32_bits_of_elements():
    L = layers()
    R, K, N = 70001, 64, 32800
    x, w = random_mx4(R, K, 1), random_mx4(N, K, 2)
    y = torch.empty(R, N, device="cuda", dtype=torch.bfloat16)
    L.mx4_gemm(x, w, [y])
    w64 = values64(w)
    check_product(values64(_part(x, 69888)), w64, [y[69888:]], K)
    rows = L.mx4_dequant(x)
    y.fill_(0)
    L.mx4_rows(rows, w, [y])
    check_product(rows[-50:].double().cpu(), w64, [y[-50:]], K)
    check_product(rows[:50].double().cpu(), w64, [y[:50]], K)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_the_most_rows_of_a_call(dtype):
    L = layers()
    R, K, N = (1 << 20) - 1, 64, 32
    x, w, y = torch.randn(R, K, device="cuda").to(dtype), random_mx4(N, K, 1), torch.empty(R, N, device="cuda")
    L.mx4_rows(x, w, [y])
    check_product(x.double().cpu(), values64(w), [y], K)


def test_choices_past_32_bits_of_bytes():
    """Three rows of a gigabyte each: the choice is found at the start, in the middle and at the end of a row."""
    L = layers()
    V = (1 << 29) + 7
    logits = torch.zeros(3, V, device="cuda", dtype=torch.float16)
    at = [0, 1 << 28, V - 1]
    logits[torch.arange(3, device="cuda"), torch.tensor(at, device="cuda")] = 2.0
    counts = torch.zeros(V, device="cuda", dtype=torch.int32)
    counts[-1] = 1
    out = torch.empty(3, V, device="cuda")
    choice = L.logits_choose([dict(logits=logits, counts=counts, repetition=1.25, out=out)])[0]
    assert choice.tolist() == at
    assert out[2, -1].item() == torch.tensor(2.0).div(1.25).item() and out[1, 1 << 28].item() == 2.0 and not out[0, 1:].any()
    mask = torch.full(((V + 31) // 32,), -1, device="cuda", dtype=torch.int32)
    mask[-1] = 1                                             # of the last word's seven tokens the first one
    logits[2, V - 7] = 1.0
    assert L.logits_choose([dict(logits=logits, mask=mask)])[0].tolist() == [0, 1 << 28, V - 7]


def test_choices_of_very_many_rows():
    L = layers()
    R, V = 300001, 37
    logits = torch.randn(R, V, device="cuda")
    assert torch.equal(L.logits_choose([dict(logits=logits)])[0].long(), logits.argmax(1))

"""speculative.Head with a vocabulary that is no multiple of 32: the rows of its matrix behind the vocabulary are never chosen."""
import pytest
import torch

from tests.test_mx4_gpu import layers, values64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grammar", [False, True])
@pytest.mark.parametrize("vocabulary,rows", [(1003, 1024), (1, 32), (4097, 4128)])
def test_tokens_come_from_the_vocabulary(vocabulary, rows, grammar):
    """All logits of the vocabulary are below 0, those of the rows behind it are 0."""
    from crucible_strix_halo_b200 import speculative
    L = layers()
    gen = torch.Generator(device="cuda").manual_seed(vocabulary)
    weights = torch.zeros(rows, 128, device="cuda")
    weights[:vocabulary] = -1 - torch.rand(vocabulary, 128, device="cuda", generator=gen)
    w = L.mx4_quant(weights)
    words = (vocabulary + 31) // 32
    mask = torch.randint(-2 ** 31, 2 ** 31, (5, words), device="cuda", generator=gen).to(torch.int32)
    mask[:, 0] |= 1                                          # at least token 0
    bias = torch.randn(vocabulary, device="cuda", generator=gen)
    head = speculative.Head(w, repetition=1.25, frequency=0.5, presence=0.25, bias=bias, allowed=(lambda tokens, drafts: mask) if grammar else None,
                            vocabulary=vocabulary)
    tokens, drafts = [vocabulary - 1, 0, vocabulary // 2], [vocabulary - 1, 0, 0, vocabulary // 3]
    head.accept(tokens)
    out = 0.5 + torch.rand(5, 128, device="cuda", generator=gen)
    got = head.choose(out, tokens, drafts)
    counts = torch.bincount(torch.tensor(tokens), minlength=vocabulary).double()
    assert torch.equal(head.counts.cpu().double(), counts)
    logits = (out.double().cpu() @ values64(w).t())[:, :vocabulary]
    assert (logits < 0).all()
    for r in range(5):
        if r:
            counts[drafts[r - 1]] += 1
        x = logits[r]
        y = torch.where(counts > 0, x * 1.25 - 0.5 * counts - 0.25, x) + bias.double().cpu()
        if grammar:
            v = torch.arange(vocabulary)
            y = torch.where((mask[r].cpu().long()[v // 32] >> (v % 32)) & 1 == 1, y, -torch.inf)
        # Logits are below 400: an fp32 sum of 128 terms is off by less than 128 2^-24 400 = 0.0031, times 1.25 and a few roundings of
        # 2^-24 500 less than 0.0041; of the best and the chosen one together less than 0.01.
        assert y[got[r]] >= y.max() - 0.01

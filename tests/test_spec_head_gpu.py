"""A stream whose tokens the framework's own head chooses (speculative.Head): 4-bit head product, penalties, bias, grammar, choice,
in plain decoding and in verify spans, against the same steps in 64 bits and against one another."""
import numpy as np
import pytest
import torch

from tests.test_mx4_gpu import values64
from tests.test_spec_loop_gpu import Glue, V

pytestmark = pytest.mark.gpu


def _grammar(tokens, drafts):
    """At position p a token t is allowed unless (t + p) % 3 == 0."""
    rows = []
    for r in range(len(drafts) + 1):
        p = len(tokens) + r
        word = sum(1 << t for t in range(V) if (t + p) % 3)
        rows.append([word - (1 << 32) if word >= 1 << 31 else word])
    return torch.tensor(rows, device="cuda", dtype=torch.int32)


def _make(seed, ctx, span, allowed=_grammar):
    from crucible_strix_halo_b200 import capi, layers, speculative
    g = capi.Geometry(256, 16, 2, 4, 2)
    rng = np.random.default_rng(seed)
    gw = [layers.GdnWeights(g, 0.5 * rng.normal(size=(g.gdn_channels, 4)), rng.normal(size=4) - 1, 0.5 * rng.normal(size=4),
                            1 + 0.1 * rng.normal(size=128), ab=0.05 * rng.normal(size=(8, 256)))]
    qw, mw = (layers.QsaWeights(g, *[1 + 0.1 * rng.normal(size=n) for n in (256, 256, 128, 128)]) for _ in range(2))
    glue = Glue(g, seed)
    w = layers.mx4_quant(glue.head.t().contiguous())
    bias = torch.zeros(V, device="cuda")
    bias[7] = 2.0

    def stream():
        head = speculative.Head(w, repetition=1.2, frequency=0.5, presence=1.0, bias=bias, allowed=allowed)
        return speculative.SpecStream(g, gw, qw, mw, glue, ctx, span=span, head=head)
    return glue, w, bias, stream


def test_rounds_with_a_head_equal_plain_decoding():
    span, total, prompt = 5, 60, [3, 17, 4, 9, 30, 1]
    glue, w, bias, stream = _make(2, 128, span)
    plain = stream()
    plain.feed(prompt)
    while len(plain.tokens) < total:
        plain.decode_one()
    truth = list(plain.tokens)
    assert all((t + p) % 3 for p, t in enumerate(truth) if p >= len(prompt)), "a token that the grammar does not allow"
    assert len(set(truth[len(prompt):])) > 8                                   # the penalties keep it from repeating itself
    glue.truth = truth
    glue.wrong = set(int(p) for p in np.random.default_rng(5).choice(np.arange(len(prompt), total), size=12, replace=False))
    spec = stream()
    spec.feed(prompt)
    while len(spec.tokens) < total - span:
        spec.round()
    assert spec.tokens == truth[:len(spec.tokens)]
    assert min(spec.accepted) == 0 and max(spec.accepted) == span - 1
    want = torch.bincount(torch.tensor(spec.tokens), minlength=V)
    assert torch.equal(spec.head.counts.cpu().long(), want)


def test_choices_of_a_pass_against_64_bits():
    glue, w, bias, stream = _make(4, 64, 5)
    s = stream()
    tokens, drafts = [1, 2, 2, 5, 9], [2, 11, 11, 30]
    s.head.accept(tokens)
    out = torch.randn(5, w.inner, device="cuda")
    logits = out.double().cpu() @ values64(w).t()
    ids = s.head.choose(out, tokens, drafts)
    counts = torch.bincount(torch.tensor(tokens), minlength=V).double()
    for r in range(5):
        if r:
            counts[drafts[r - 1]] += 1
        x = logits[r]
        y = torch.where(counts > 0, torch.where(x > 0, x / 1.2, x * 1.2) - 0.5 * counts - 1.0, x) + bias.double().cpu()
        t = torch.arange(V)
        y = torch.where((t + len(tokens) + r) % 3 != 0, y, -torch.inf)
        top = y.topk(2).values
        if top[0] - top[1] > 1e-3:                                             # far from a tie in either precision
            assert ids[r] == int(y.argmax()), r


def test_a_grammar_that_allows_nothing_is_an_error():
    nothing = lambda tokens, drafts: torch.zeros(1, device="cuda", dtype=torch.int32)
    glue, w, bias, stream = _make(5, 64, 5, allowed=nothing)
    s = stream()
    s.feed([1, 2])
    with pytest.raises(ValueError):
        s.decode_one()

"""Penalties, biases, grammar masks and the choice of a token (cr_logits_choose, cr_token_count) against the formula in 64 bits.

Tolerance of the processed logits: five roundings (quotient or product, n * frequency, two differences, the sum with the bias), each
half a step, 2^-24, of a number no larger than |l| max(rep, 1 / rep) + n |frequency| + |presence| + |bias|; six are allowed for the
second order.  The choice is compared with the processed logits' own: exactly."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def layers():
    from crucible_strix_halo_b200 import layers
    return layers


def formula(sp):
    """(processed logits, limit of their error, allowed) in 64 bits."""
    l = sp["logits"].double().cpu().clone()
    R, V = l.shape
    rep, freq, pres = (torch.tensor(sp.get(k, d), dtype=torch.float32).double().item() for k, d in (("repetition", 1.0), ("frequency", 0.0), ("presence", 0.0)))
    counts = sp["counts"].cpu().clone() if sp.get("counts") is not None else torch.zeros(V, dtype=torch.int32)
    bias = sp["bias"].double().cpu() if sp.get("bias") is not None else torch.zeros(V, dtype=torch.float64)
    allowed = torch.ones(R, V, dtype=torch.bool)
    if sp.get("mask") is not None:
        words = sp["mask"].cpu().long()
        words = words.expand(R, -1) if words.dim() == 1 else words
        v = torch.arange(V)
        allowed = (words[:, v // 32] >> (v % 32)) & 1 == 1
    limit = torch.zeros_like(l)
    for r in range(R):
        if r and sp.get("drafts") is not None:
            d = int(sp["drafts"][r - 1])
            if 0 <= d < V:
                counts[d] += 1
        n = counts.double()
        x = l[r]
        y = torch.where(n > 0, torch.where(x > 0, x / rep, x * rep) - n * freq - pres, x) + bias
        limit[r] = 6 * 2.0 ** -24 * (x.abs() * max(rep, 1 / rep) + n * abs(freq) + abs(pres) + bias.abs())
        l[r] = torch.where(allowed[r], y, -math.inf)
    return l, limit, allowed


def lowest_best(row, allowed):
    """The lowest index among the largest allowed values, a NaN above all; -1 without any."""
    at = torch.nonzero(allowed).flatten()
    if not len(at):
        return -1
    v = row[at]
    best = v.isnan() if v.isnan().any() else v == v.max()
    return int(at[torch.nonzero(best).flatten()[0]])


def check(spans, outs=None):
    L = layers()
    wants = [formula(sp) for sp in spans]                    # before the call: it may work in place
    choices = L.logits_choose(spans, outs)
    torch.cuda.synchronize()
    for sp, choice, (want, limit, allowed) in zip(spans, choices, wants):
        got = sp["out"].cpu()
        fine = torch.isfinite(want)
        assert torch.equal(torch.isfinite(got), fine) and torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got[~fine & ~want.isnan()].double(), want[~fine & ~want.isnan()])
        over = ((got.double() - want).abs() - limit)[fine]
        assert not len(over) or over.max() <= 0
        assert choice.tolist() == [lowest_best(got[r], allowed[r]) for r in range(len(got))]
    # the choices alone
    kept = [(sp, c) for sp, c in zip(spans, choices) if sp["out"].data_ptr() != sp["logits"].data_ptr()]
    if kept:
        assert all(torch.equal(a, c) for a, (_, c) in zip(L.logits_choose([dict(sp, out=None) for sp, _ in kept]), kept))
    return choices


def span(R, V, seed, dtype=torch.float32, drafts=True, mask=None, **kw):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    said = (V * torch.rand(200, device="cuda", generator=gen) ** 3).long().clamp_(max=V - 1)
    sp = dict(logits=(3 * torch.randn(R, V, device="cuda", generator=gen)).to(dtype), out=torch.full((R, V), 7.0, device="cuda"),
              counts=torch.zeros(V, device="cuda", dtype=torch.int32).scatter_add_(0, said, torch.ones_like(said, dtype=torch.int32)),
              bias=torch.randn(V, device="cuda", generator=gen), repetition=1.3, frequency=0.25, presence=0.5)
    if drafts and R > 1:
        sp["drafts"] = torch.randint(0, V, (R - 1,), device="cuda", generator=gen, dtype=torch.int32)
    if mask:
        words = (V + 31) // 32
        sp["mask"] = torch.randint(-2 ** 31, 2 ** 31, (R, words) if mask == "rows" else (words,), device="cuda", generator=gen).to(torch.int32)
    return dict(sp, **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,mask", [(1, 1, None), (1, 31, "one"), (2, 33, "rows"), (1, 1000, None), (9, 4097, "rows"), (13, 32000, "one"),
                                      (3, 131072, None), (1, 131071, "rows"), (40, 777, "rows")])
def test_processed_logits_and_choice(R, V, mask, dtype):
    check([span(R, V, R + V, dtype, mask=mask)])


@pytest.mark.parametrize("without", ["counts", "drafts", "bias", "mask", "all"])
def test_parts_that_are_left_out(without):
    sp = span(5, 1003, 3, mask="rows")
    if without == "all":
        sp = dict(logits=sp["logits"], out=sp["out"])
    else:
        sp.pop(without)
    check([sp])


def test_many_spans_of_different_sizes():
    check([span(1 + i % 13, 500 + 37 * i, i, TYPES[i % 3], mask=[None, "one", "rows"][i % 3]) for i in range(70)])


def test_repeated_drafts_and_drafts_outside_the_vocabulary():
    V = 300
    sp = span(7, V, 1, drafts=False)
    sp["drafts"] = torch.tensor([5, 5, V, -1, 5, 299], device="cuda", dtype=torch.int32)
    check([sp])


def test_the_penalties_move_the_choice_from_row_to_row():
    """A row whose best token was drafted before takes the second best: 10 and 9 for all rows, each draft takes 2 off."""
    V = 1000
    logits = torch.zeros(4, V, device="cuda")
    logits[:, 700], logits[:, 20] = 10, 9
    sp = dict(logits=logits, out=torch.empty(4, V, device="cuda"), drafts=torch.tensor([700, 20, 700], device="cuda", dtype=torch.int32), frequency=2.0)
    assert [c.tolist() for c in check([sp])] == [[700, 20, 700, 20]]


def test_ties_take_the_lowest_index():
    V = 50000
    logits = torch.zeros(3, V, device="cuda")
    logits[0, [49999, 31, 12345]] = 4.0
    logits[1] = -0.0
    logits[1, 17:] = 0.0                                     # both zeros are as large
    logits[2] = -math.inf
    assert [c.tolist() for c in check([dict(logits=logits, out=torch.empty_like(logits))])] == [[31, 0, 0]]


@pytest.mark.parametrize("V", [64, 5000, 100003])
def test_masks_that_leave_one_token_or_none(V):
    words = (V + 31) // 32
    mask = torch.zeros(4, words, device="cuda", dtype=torch.int32)
    mask[1, (V - 1) // 32] = 1 << ((V - 1) % 32) if (V - 1) % 32 < 31 else -2 ** 31
    mask[2, 0] = 1
    mask[3, (V - 1) // 32] = -1                               # bits past the vocabulary are set too
    sp = span(4, V, 2, drafts=False)
    sp["mask"] = mask
    sp["logits"][:, 1:V - 1] = math.nan                       # what is not allowed may hold anything
    sp["logits"][0] = math.inf
    sp["logits"][3] = -5.0
    c = check([sp])[0].tolist()
    assert c[:3] == [-1, V - 1, 0] and c[3] >= V // 32 * 32 - 32


def test_infinities_and_nans_in_allowed_places():
    V = 2000
    logits = torch.randn(5, V, device="cuda")
    logits[0, 1500] = math.nan
    logits[1, 1999] = math.inf
    logits[2, :] = -math.inf
    logits[3, 7], logits[3, 8] = math.inf, math.nan
    logits[4, :1990] = -math.inf
    bias = torch.zeros(V, device="cuda")
    bias[7] = -math.inf                                       # a banned token; infinity less infinity is NaN
    sp = dict(logits=logits, out=torch.empty_like(logits), bias=bias, counts=torch.ones(V, device="cuda", dtype=torch.int32), repetition=1.5)
    c = check([sp])[0].tolist()
    assert c[:4] == [1500, 1999, 0, 7]


@pytest.mark.parametrize("dtype,bits", [(torch.float32, -1), (torch.float32, -0x400000), (torch.bfloat16, -1), (torch.float16, -1)])
def test_a_nan_of_either_sign_is_the_largest(dtype, bits):
    logits = torch.randn(1, 900, device="cuda").to(dtype)
    view = logits.view(torch.int32 if dtype == torch.float32 else torch.int16)
    view[0, 500] = bits
    logits[0, 600] = math.nan
    logits[0, 700] = math.inf
    assert check([dict(logits=logits, out=torch.empty(1, 900, device="cuda"))])[0].tolist() == [500]


def test_logits_of_the_types_lowest_value():
    V = 3000
    for dtype in TYPES:
        logits = torch.full((2, V), torch.finfo(dtype).min, device="cuda", dtype=dtype)
        logits[1, 2999] = torch.finfo(dtype).max
        assert [c.tolist() for c in check([dict(logits=logits, out=torch.empty(2, V, device="cuda"))])] == [[0, 2999]]


@pytest.mark.parametrize("V", [1000, 70001])
def test_in_place(V):
    sp = span(6, V, 5, mask="rows")
    sp["out"] = sp["logits"]
    check([sp])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset,pitch", [(0, 1200), (1, 1003), (3, 1001)])
def test_rows_at_any_pitch_and_address(offset, pitch, dtype):
    V = 1001
    sp = span(5, V, 6, dtype, mask="rows")
    buf, out = torch.zeros(5 * pitch + offset, device="cuda", dtype=dtype), torch.full((5 * pitch + offset,), 7.0, device="cuda")
    rows = buf[offset:].view(5, pitch)
    rows[:, :V] = sp["logits"]
    sp["logits"], sp["out"] = rows[:, :V], out[offset:].view(5, pitch)[:, :V]
    check([sp])
    out[offset:].view(5, pitch)[:, :V] = 7
    assert (out == 7).all()


@pytest.mark.parametrize("what", ["counts", "bias", "out", "logits"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_buffer_off_the_others_alignment(what, dtype):
    V = 4100
    sp = span(3, V, 8, dtype, mask="rows")
    if what in ("counts", "bias"):
        off = torch.zeros(V + 1, device="cuda", dtype=sp[what].dtype)
        off[1:] = sp[what]
        sp[what] = off[1:]
    else:
        off = torch.zeros(3 * V + 1, device="cuda", dtype=sp[what].dtype)
        off[1:] = sp[what].flatten()
        sp[what] = off[1:].view(3, V)
    check([sp])


def test_more_drafts_than_a_warp_has_lanes():
    V = 600
    sp = span(75, V, 9, drafts=False)
    sp["drafts"] = torch.tensor([5, 255, 256, 599] * 18 + [5, 5], device="cuda", dtype=torch.int32)
    check([sp])


def test_counts_are_kept():
    L = layers()
    V = 1000
    gen = torch.Generator(device="cuda").manual_seed(0)
    tokens = torch.randint(-5, V + 5, (20000,), device="cuda", generator=gen, dtype=torch.int32)
    counts = torch.zeros(V, device="cuda", dtype=torch.int32)
    L.token_count(counts, tokens)
    inside = tokens[(tokens >= 0) & (tokens < V)].long()
    assert torch.equal(counts.long(), torch.bincount(inside, minlength=V))
    L.token_count(counts, tokens[5000:], -1)
    head = tokens[:5000]
    assert torch.equal(counts.long(), torch.bincount(head[(head >= 0) & (head < V)].long(), minlength=V))
    L.token_count(counts, tokens[:0])


def test_captured_calls_replay_on_new_inputs():
    L = layers()
    V = 5003
    sp = span(9, V, 1, mask="rows")
    outs = [torch.empty(9, device="cuda", dtype=torch.int32)]
    L.logits_choose([sp], outs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        L.logits_choose([sp], outs)
        L.token_count(sp["counts"], outs[0][:1])
    for seed in (2, 3):
        new = span(9, V, seed, mask="rows")
        for k in ("logits", "bias", "mask", "drafts", "counts"):
            sp[k].copy_(new[k])
        want = check([dict(sp, out=torch.empty(9, V, device="cuda"))])[0]
        before = sp["counts"].clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want)
        before[want[0].long()] += 1
        assert torch.equal(sp["counts"], before)


def test_calls_on_two_streams_do_not_disturb_each_other():
    L = layers()
    spans = [span(9, 30000, i, mask="rows") for i in range(2)]
    want = [L.logits_choose([sp])[0] for sp in spans]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(20):
        for s, sp in zip(streams, spans):
            with torch.cuda.stream(s):
                got.append(L.logits_choose([sp])[0])
    torch.cuda.synchronize()
    assert all(torch.equal(c, want[i % 2]) for i, c in enumerate(got))


@pytest.mark.parametrize("change,error", [
    (dict(logits=torch.zeros(2, 64)), ValueError), (dict(counts="cuda64"), TypeError), (dict(counts="short"), ValueError), (dict(drafts="short"), ValueError),
    (dict(bias="short"), ValueError), (dict(mask="short"), ValueError), (dict(out="half"), TypeError), (dict(out="shape"), ValueError),
    (dict(repetition=0.0), RuntimeError), (dict(repetition=math.nan), RuntimeError), (dict(frequency=math.inf), RuntimeError), (dict(presence="x"), TypeError),
])
def test_refusals(change, error):
    L = layers()
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)
    named = {"cuda64": z(64, dtype=torch.int64), "short": None, "half": z(2, 64).half(), "shape": z(2, 63), "x": "x"}
    short = dict(counts=z(63, dtype=torch.int32), drafts=z(0, dtype=torch.int32), bias=z(63), mask=z(1, dtype=torch.int32))
    (key, value), = change.items()
    value = short[key] if isinstance(value, str) and value == "short" else named[value] if isinstance(value, str) else value
    with pytest.raises(error):
        L.logits_choose([dict(dict(logits=z(2, 64)), **{key: value})])
    with pytest.raises(RuntimeError):
        L.logits_choose([])
    torch.cuda.synchronize()

"""Performance cases of the operators between the attention core's rows and the tokens: 4-bit projections and the choice
of a token from logits, through crucible_strix_halo_b200.layers.

Kinds of case
  quant    rows to microscaled 4-bit floats and back (layers.mx4_quant, layers.mx4_dequant)
  gemm     the product of two 4-bit matrices (layers.mx4_gemm)
  linear   a projection of a prompt's rows: quantised, then multiplied with 4-bit weights (mx4_quant, mx4_gemm)
  rows     a projection of decode or verify rows as they are with 4-bit weights (layers.mx4_rows)
  choose   penalties, bias and grammar mask on logits, and the choice of a token (layers.logits_choose)
  head     output rows to tokens: the 4-bit head product, then the choice (mx4_rows, logits_choose)

A 4-bit matrix [rows][inner] is codes, uint8 [rows][inner / 2] (e2m1, the even element in the low nibble), and scales, one
e8m0 byte per 32 elements in tiles of 128 rows x 4 blocks: byte (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4 of tile
(r // 128, b // 4).
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def listed():
    return [
        # A verify span's rows into 4 bits: the smallest call, launches decide.
        dict(name="quant_13x2048", kind="quant", rows=13, inner=2048, type="bf16"),
        # The fp32 output rows of a long prompt's attention (24 heads of 256), a ragged number of them.
        dict(name="quant_16001x6144", kind="quant", rows=16001, inner=6144, type="f32"),
        # The output projection of a short chat turn, both operands in hand.
        dict(name="gemm_333x4096x2048", kind="gemm", rows=333, inner=4096, columns=2048, out="f32"),
        # The input projection of a Gated DeltaNet layer over a 32K prompt: the largest.
        dict(name="gemm_32768x2048x12352", kind="gemm", rows=32768, inner=2048, columns=12352, out="bf16"),
        # The input projection of a QSA layer for a chat turn of 117 tokens at the engine's geometry, fp32 rows for the core.
        dict(name="linear_117x2560x13952", kind="linear", rows=117, inner=2560, columns=13952, type="bf16", out="f32"),
        # The same for one whole part of a prompt at the benchmark geometry.
        dict(name="linear_2048x2048x9856", kind="linear", rows=2048, inner=2048, columns=9856, type="bf16", out="f32"),
        # One user's output projection in a decode step.
        dict(name="rows_1x4096x2048", kind="rows", rows=1, inner=4096, columns=2048, type="f32", out="f32"),
        # The input projection of a Gated DeltaNet layer for a decode step of four sessions.
        dict(name="rows_4x2048x12352", kind="rows", rows=4, inner=2048, columns=12352, type="bf16", out="bf16"),
        # The head over a verify span of one certain row and eight drafts.
        dict(name="rows_9x2048x131072", kind="rows", rows=9, inner=2048, columns=131072, type="bf16", out="f32"),
        # One user's next token: every penalty, a bias, no grammar; only the token is wanted.
        dict(name="choose_1x1x131071", kind="choose", sessions=1, rows=1, vocabulary=131071, type="f32", grammar=False, processed=False),
        # Eight sessions verify eight drafts each under a grammar, the processed logits wanted.
        dict(name="choose_8x9x100352", kind="choose", sessions=8, rows=9, vocabulary=100352, type="bf16", grammar=True, processed=True),
        # Four sessions' decode step from output rows to tokens.
        dict(name="head_4x1x2560x65536", kind="head", sessions=4, rows=1, inner=2560, vocabulary=65536, type="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quant", "gemm", "gemm", "linear", "rows", "rows", "choose", "choose", "head"])
    inner = 64 * rng.choice([rng.randint(1, 96), 32, 40, 64, 96])
    if kind == "quant":
        return dict(kind=kind, rows=_log(rng, 1, 16001 * 6144 // max(inner, 2048)), inner=inner, type=rng.choice(["f32", "bf16", "f16"]))
    if kind in ("gemm", "linear"):
        case = dict(kind=kind, rows=_log(rng, 1, 16384), inner=inner, columns=32 * _log(rng, 1, 400), out=rng.choice(["f32", "bf16"]))
        return dict(case, type=rng.choice(["f32", "bf16", "f16"])) if kind == "linear" else case
    if kind == "rows":
        return dict(kind=kind, rows=rng.choice([1, 2, 4, 9, 13, _log(rng, 1, 72)]), inner=inner, columns=32 * _log(rng, 1, 4096),
                    type=rng.choice(["f32", "bf16", "f16"]), out=rng.choice(["f32", "bf16"]))
    vocabulary = _log(rng, 2000, 160000)
    sessions, rows = rng.choice([1, 1, 2, 4, 8, 16]), rng.choice([1, 1, 2, 5, 9, 13])
    if kind == "choose":
        return dict(kind=kind, sessions=sessions, rows=rows, vocabulary=vocabulary, type=rng.choice(["f32", "bf16", "f16"]), grammar=rng.random() < 0.5,
                    processed=rng.random() < 0.5)
    return dict(kind=kind, sessions=min(sessions, 8), rows=rows, inner=inner, vocabulary=32 * (vocabulary // 32), type=rng.choice(["f32", "bf16", "f16"]))


# ---- inputs ------------------------------------------------------------------------------------------------------

def _activations(gen, rows, inner, dtype):
    """Rows as they leave a norm: channels of different sizes, a few large ones, and some dead blocks of 32."""
    x = torch.randn(rows, inner, device="cuda", generator=gen)
    x.mul_(torch.exp(0.7 * torch.randn(inner, device="cuda", generator=gen)))
    x.view(rows, -1, 32).mul_(torch.rand(rows, inner // 32, 1, device="cuda", generator=gen) > 0.005)
    return x.to(dtype)


def _weights(gen, columns, inner):
    """A 4-bit weight matrix in hand: codes and tiled scales."""
    codes = torch.randint(0, 256, (columns, inner // 2), device="cuda", generator=gen, dtype=torch.uint8)
    byte = (126 - int(math.log2(inner)) // 2 - torch.randint(0, 3, (columns, inner // 32), device="cuda", generator=gen)).to(torch.uint8)
    return {"codes": codes, "scales": _tiled(byte)}


def _tiled(byte):
    rows, blocks = byte.shape
    full = torch.zeros(-(-rows // 128) * 128, -(-blocks // 4) * 4, device=byte.device, dtype=torch.uint8)
    full[:rows, :blocks] = byte
    return full.view(-1, 4, 32, full.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).reshape(-1).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, state = case["kind"], dict(case)
    sessions, rows = case.get("sessions", 1), case["rows"]
    if kind in ("quant", "linear", "rows", "head"):
        state["x"] = _activations(gen, sessions * rows, case["inner"], TYPES[case["type"]])
    if kind == "gemm":
        state["xq"] = _weights(gen, rows, case["inner"])
    if kind in ("gemm", "linear", "rows"):
        state["w"] = _weights(gen, case["columns"], case["inner"])
    if kind in ("choose", "head"):
        V = case["vocabulary"]
        if kind == "head":
            state["w"] = _weights(gen, V, case["inner"])
        else:
            state["logits"] = (3 * torch.randn(sessions, rows, V, device="cuda", generator=gen)).to(TYPES[case["type"]])
        # a conversation of a thousand tokens, frequent ones more often
        said = (V * torch.rand(sessions, 1000, device="cuda", generator=gen) ** 4).long().clamp_(max=V - 1)
        state["counts"] = torch.zeros(sessions, V, device="cuda", dtype=torch.int32).scatter_add_(1, said, torch.ones_like(said, dtype=torch.int32))
        state["drafts"] = torch.randint(0, V, (sessions, max(rows - 1, 1)), device="cuda", generator=gen, dtype=torch.int32)
        state["bias"] = torch.randn(V, device="cuda", generator=gen) * (torch.rand(V, device="cuda", generator=gen) < 0.01)
        state["penalties"] = [(1.0 + 0.05 * (i % 5), 0.1 * (i % 3), 0.25 * (i % 4)) for i in range(1, sessions + 1)]
        state["penalty_rows"] = torch.tensor(state["penalties"], device="cuda", dtype=torch.float32)
        if case.get("grammar"):
            words = (V + 31) // 32
            mask = torch.randint(-2 ** 31, 2 ** 31, (sessions, rows, words), device="cuda", generator=gen).to(torch.int32)
            few = torch.rand(sessions, rows, 1, device="cuda", generator=gen) < 0.5           # half the rows are in a narrow place
            mask[(few & (torch.rand(sessions, rows, words, device="cuda", generator=gen) > 0.003))] = 0
            mask[-1, -1] = 0                                                                   # and one allows nothing
            state["mask"] = mask
    return state


# ---- plain forms ---------------------------------------------------------------------------------------------------

def _quantised(x):
    """(codes 0..15 [rows][inner], scale bytes [rows][inner / 32]) of rows."""
    b = x.float().view(x.shape[0], -1, 32)
    top = b.abs().amax(-1)
    s = ((top.view(torch.int32) >> 23) - 129).clamp(-127, 127)
    y = (b * ((127 - s) << 23).view(torch.float32)[..., None]).abs()         # times 2^-s: -s lies in -126..127
    code = (y > 0.25).int() + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5)
    bad = ~torch.isfinite(top)
    code = torch.where(bad[..., None], 0, code + 8 * torch.signbit(b))
    return code.view(x.shape), torch.where(bad, 255, s + 127)


def _scale(byte):
    byte = byte.int()
    f = (byte << 23).view(torch.float32)
    return torch.where(byte == 0, torch.full_like(f, 2.0 ** -127), torch.where(byte == 255, torch.full_like(f, math.nan), f))


def _values_of(code, byte):
    table = torch.tensor(E2M1 + [-v for v in E2M1], device=code.device)
    return (table[code.long()].view(code.shape[0], -1, 32) * _scale(byte)[..., None]).view(code.shape)


def _values(m):
    """The numbers a 4-bit matrix in hand stands for."""
    codes = m["codes"]
    rows, inner = codes.shape[0], codes.shape[1] * 2
    blocks = inner // 32
    byte = m["scales"].view(-1, -(-blocks // 4), 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-(-rows // 128) * 128, -1)[:rows, :blocks]
    return _values_of(torch.stack([codes & 15, codes >> 4], -1).view(rows, inner), byte)


def _chosen(state, logits):
    """(choice, processed logits) of logits [sessions][rows][vocabulary] in their own precision."""
    S, R, V = logits.shape
    count = torch.zeros(S, R, V, device=logits.device, dtype=torch.int32)
    if R > 1:
        at = state["drafts"][:, None, :R - 1].long().transpose(1, 2)
        count[:, 1:].scatter_(2, at, 1)
        count = count.cumsum(1, dtype=torch.int32)
    count += state["counts"][:, None]
    rep, freq, pres = state["penalty_rows"].to(logits.dtype).view(S, 1, 1, 3).unbind(-1)
    said = count > 0
    l = torch.where(said, torch.where(logits > 0, logits / rep, logits * rep), logits)
    l = l - count.to(l.dtype) * freq
    l = torch.where(said, l - pres, l) + state["bias"].to(l.dtype)
    allowed = torch.ones_like(said)
    if "mask" in state:
        v = torch.arange(V, device=l.device)
        allowed = (state["mask"][..., v // 32] >> (v % 32)) & 1 == 1
        l = torch.where(allowed, l, -math.inf)
    best = (l == l.amax(-1, keepdim=True)) & allowed
    choice = torch.where(allowed.any(-1), best.int().argmax(-1), -1).to(torch.int32)
    return choice, l


def _plain(state):
    kind = state["kind"]
    if kind == "quant":
        return {"values": _values_of(*_quantised(state["x"])).to(state["x"].dtype)}
    if kind == "gemm":
        return {"y": (_values(state["xq"]) @ _values(state["w"]).t()).to(TYPES[state["out"]])}
    if kind == "linear":
        return {"y": (_values_of(*_quantised(state["x"])) @ _values(state["w"]).t()).to(TYPES[state["out"]])}
    if kind == "rows":
        return {"y": (state["x"].float() @ _values(state["w"]).t()).to(TYPES[state["out"]])}
    if kind == "head":
        logits = (state["x"].float() @ _values(state["w"]).t()).view(state["sessions"], state["rows"], -1)
    else:
        logits = state["logits"].float()
    choice, processed = _chosen(state, logits)
    return {"choice": choice, "logits": processed} if state.get("processed") or kind == "head" else {"choice": choice}


# ---- the framework's calls -------------------------------------------------------------------------------------------

def _own(state):
    from crucible_strix_halo_b200 import layers
    kind = state["kind"]
    hand = lambda m: layers.Mx4(m["codes"], m["scales"], m["codes"].shape[0], m["codes"].shape[1] * 2)
    if kind == "quant":
        return {"values": layers.mx4_dequant(layers.mx4_quant(state["x"]), state["x"].dtype)}
    if kind in ("gemm", "linear", "rows"):
        y = torch.empty(state["rows"], state["columns"], device="cuda", dtype=TYPES[state["out"]])
        if kind == "rows":
            layers.mx4_rows(state["x"], hand(state["w"]), [y])
        else:
            layers.mx4_gemm(hand(state["xq"]) if kind == "gemm" else layers.mx4_quant(state["x"]), hand(state["w"]), [y])
        return {"y": y}
    S, R, V = state["sessions"], state["rows"], state["vocabulary"]
    if kind == "head":
        logits = torch.empty(S, R, V, device="cuda")
        layers.mx4_rows(state["x"], hand(state["w"]), [logits.view(S * R, V)])
        processed = logits                                               # in place
    else:
        logits = state["logits"]
        processed = torch.empty(S, R, V, device="cuda") if state["processed"] else None
    choice = torch.empty(S, R, device="cuda", dtype=torch.int32)
    spans = []
    for i in range(S):
        rep, freq, pres = state["penalties"][i]
        spans.append(dict(logits=logits[i], counts=state["counts"][i], drafts=state["drafts"][i], bias=state["bias"],
                          mask=state["mask"][i] if "mask" in state else None, repetition=rep, frequency=freq, presence=pres,
                          out=None if processed is None else processed[i]))
    layers.logits_choose(spans, outs=[choice[i] for i in range(S)])
    return {"choice": choice} if processed is None else {"choice": choice, "logits": processed}


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------

def work(case):
    kind, R = case["kind"], case.get("sessions", 1) * case["rows"]
    four = lambda rows, inner: rows * inner * 17 // 32
    if kind == "quant":
        n = R * case["inner"]
        return {"bytes": 2 * n * BYTES[case["type"]], "flops": 3 * n}
    V = case.get("vocabulary", 0)
    choose = V * (case.get("sessions", 1) * 4 + 4) + R * 4 + (R * V // 8 if case.get("grammar") else 0)
    if kind == "choose":
        return {"bytes": choose + R * V * (BYTES[case["type"]] + (4 if case["processed"] else 0)), "flops": 6 * R * V}
    if kind == "head":
        return {"bytes": choose + R * V * 4 + four(V, case["inner"]) + R * case["inner"] * BYTES[case["type"]], "flops": R * V * (2 * case["inner"] + 6)}
    N, K = case["columns"], case["inner"]
    x = four(R, K) if kind == "gemm" else R * K * BYTES[case["type"]]
    return {"bytes": x + four(N, K) + R * N * BYTES[case["out"]], "flops": 2 * R * N * K}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------

def _grid64(x):
    """The 4-bit numbers nearest to rows, by the definition: the nearest point of the grid, ties to the even code."""
    b = x.double().reshape(x.shape[0], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    exponent = torch.frexp(top)[1].double() - 3                              # top = m 2^e, 1/2 <= m < 1: floor(log2 top) = e - 1
    unit = torch.exp2(torch.where(top > 0, exponent, -127.0).clamp(-127, 127))
    y = b / unit
    size = y.abs().clamp(max=6.0)
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0)).double()
    return (torch.copysign(torch.round(size / step) * step, y) * unit).reshape(x.shape)


def _matrix64(m):
    codes = m["codes"].long()
    rows, half = codes.shape
    nibble = torch.empty(rows, half * 2, device=codes.device, dtype=torch.long)
    nibble[:, 0::2], nibble[:, 1::2] = codes % 16, codes // 16
    e, f = (nibble % 8) // 2, nibble % 2
    size = torch.where(e == 0, 0.5 * f, (1 + 0.5 * f) * torch.exp2(e.double() - 1))
    r = torch.arange(rows, device=codes.device)[:, None]
    b = torch.arange(half // 16, device=codes.device)[None]
    at = (r // 128 * -(-(half // 16) // 4) + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4
    unit = torch.exp2(m["scales"][at].double() - 127)
    return torch.where(nibble >= 8, -size, size) * unit.repeat_interleave(32, 1)


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "quant":
        return {"values": _grid64(state["x"])}
    if kind == "choose":
        logits = state["logits"].double()
    else:
        x = _matrix64(state["xq"]) if kind == "gemm" else _grid64(state["x"]) if kind == "linear" else state["x"].double()
        y = x @ _matrix64(state["w"]).t()
        if kind != "head":
            return {"y": y}
        logits = y.view(state["sessions"], state["rows"], -1)
    S, R, V = logits.shape
    choice = torch.empty(S, R, device=logits.device, dtype=torch.int32)
    for s in range(S):
        rep, freq, pres = (torch.tensor(p, dtype=torch.float32).double().item() for p in state["penalties"][s])
        count = state["counts"][s].double()
        for r in range(R):
            if r:
                count = count.clone()
                count[state["drafts"][s, r - 1].long()] += 1
            l, said = logits[s, r], (count > 0).double()
            l = l * (1 - said) + said * (l.clamp(min=0) / rep + l.clamp(max=0) * rep)
            l = l - freq * count - pres * said + state["bias"].double()
            choice[s, r] = l.argmax()
            if "mask" in state:
                bits = (state["mask"][s, r].long()[:, None] // 2 ** torch.arange(32, device=l.device).long()[None]) % 2
                l = l.masked_fill(bits.flatten()[:V] == 0, -math.inf)
                choice[s, r] = torch.where(l.max() == -math.inf, -1, l.argmax())
            logits[s, r] = l
    return {"choice": choice, "logits": logits} if case.get("processed") or kind == "head" else {"choice": choice}

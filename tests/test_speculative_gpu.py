"""verify_drafts against a plain implementation in 64 bits: tokens, counts and
states exactly, log-probabilities within the rounding of 32-bit arithmetic."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def tables(S: int, V: int, seed: int, share=(0.03, 0.4, 0.9, 1.0)):
    """A random automaton: its bundle on the device and its table on the host."""
    from bpdecode_b200.ops import FsaTensors

    g = torch.Generator().manual_seed(seed)
    keep = torch.tensor(share)[torch.arange(S) % len(share)]
    tn = torch.where(torch.rand(S, V, generator=g) < keep[:, None],
                     torch.randint(0, S, (S, V), generator=g), -1).to(torch.int32)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    fsa = FsaTensors(trans=zero.repeat(S), accept=zero.repeat(S).to(torch.uint8),
                     live=zero.repeat(S).to(torch.uint8), num_symbols=1, dead=-1,
                     offsets=zero.repeat(V + 1), symbols=zero, eos_id=-1, tok_next=tn.cuda())
    return fsa, tn


def plain(src, drafts, uniforms, noise, lens, probs, heats, tn, states, first, pfirst):
    """The definition, request by request, in 64 bits on the host."""
    B, K = drafts.shape
    V = noise.shape[1] if noise is not None else src.shape[1]
    tokens = torch.full((B, K + 1), -1, dtype=torch.int64)
    logprobs = torch.zeros(B, K + 1, dtype=torch.float64)
    counts, nxt = torch.zeros(B, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        n = int(lens[b])
        state = int(states[b]) if states is not None else None
        nxt[b] = state if state is not None else 0
        if (n < 0 or n > K or first[b] < 0 or first[b] + n >= src.shape[0]
                or (probs is not None and n and (pfirst[b] < 0 or pfirst[b] + n > probs.shape[0]))):
            continue
        heat = float(heats[b])
        for i in range(n + 1):
            x = src[int(first[b]) + i, :V].double()
            x = torch.where(torch.isnan(x), -math.inf, x)
            if tn is not None:
                ok = tn[state] >= 0 if 0 <= state < tn.shape[0] else torch.zeros(V, dtype=bool)
                x = torch.where(ok, x, -math.inf)
            m = x.max()
            token = -1
            if m > -math.inf:
                w = torch.where(x == m, 1.0, torch.exp((x - m) / (heat if heat > 0 else 1.0)))
                p = w / w.sum()
                best = int((x == m).nonzero()[0, 0])
                d = int(drafts[b, i]) if i < n else None
                inside = d is not None and 0 <= d < V
                if heat > 0:
                    q = torch.zeros(V, dtype=torch.float64)
                    if d is not None and probs is not None:
                        q = probs[int(pfirst[b]) + i, :V].double()
                    elif inside:
                        q[d] = 1.0
                    if inside and float(uniforms[b, i]) * float(q[d]) < float(p[d]):
                        token = d
                    else:
                        left = torch.clamp(p - q, min=0)
                        left = left if (left > 0).any() else p
                        score = left / noise[b, :V].double()
                        score = torch.where(left > 0, score, -1.0)
                        token = int((score == score.max()).nonzero()[0, 0])
                        d = None
                else:
                    token = best
                    d = d if d == best else None
                tokens[b, i] = token
                if x[token] != m:
                    logprobs[b, i] = (x[token] - m) / (heat if heat > 0 else 1.0)
                logprobs[b, i] -= torch.log(w.sum())
                counts[b] += 1
            if state is not None:
                state = int(tn[state, token]) if token >= 0 else -1
            if token < 0 or d is None or i == n:
                break
        if state is not None:
            nxt[b] = state
    return tokens, counts, logprobs, nxt


def check(got, want, dtype=None) -> None:
    tokens, counts, logprobs, nxt = want
    assert torch.equal(got.tokens.cpu(), tokens)
    assert torch.equal(got.counts.cpu(), counts)
    # Z: terms of weight up to exp(-25) with arguments rounded to 2^-24 each, 2^-22 of the
    # exponential; the quotient and the logarithm add a few roundings of the result
    bound = 25 * 2.0**-23 + 2.0**-21 + 6 * 2.0**-24 * logprobs.abs()
    assert bool(((got.logprobs.cpu().double() - logprobs).abs() <= bound).all())
    if got.states is not None:
        assert torch.equal(got.states.cpu(), nxt)


def make(B, K, V, dtype, seed, probs=None, heats="mixed", pad=0, ragged=True, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, K + 1, (B,), generator=g) if ragged else torch.full((B,), K)
    first = torch.cumsum(lens + 1, 0) - (lens + 1)
    rows = int((lens + 1).sum())
    src = (torch.randn(rows, V + pad, generator=g) * scale).to(dtype)
    pfirst = torch.cumsum(lens, 0) - lens
    z = torch.randn(max(int(lens.sum()), 1), V + pad, generator=g) * scale
    for b in range(B):
        for i in range(int(lens[b])):
            z[int(pfirst[b]) + i] = src[int(first[b]) + i].float() + 0.7 * torch.randn(
                V + pad, generator=g)
    q = torch.softmax(z[:, :V], -1)
    drafts = torch.zeros(B, K, dtype=torch.int64)
    for b in range(B):
        for i in range(int(lens[b])):
            drafts[b, i] = torch.multinomial(q[int(pfirst[b]) + i], 1, generator=g)
    wide = torch.zeros(q.shape[0], V + pad)
    wide[:, :V] = q
    heat = {"mixed": torch.tensor([0.0, 0.6, 1.0, 1.7])[torch.randint(0, 4, (B,), generator=g)],
            "one": torch.ones(B), "zero": torch.zeros(B)}[heats]
    return dict(src=src, drafts=drafts, uniforms=torch.rand(B, K, generator=g),
                noise=torch.empty(B, V).exponential_(generator=g).clamp_(min=1e-20), lens=lens,
                probs=wide.to(probs) if probs is not None else None, heats=heat, first=first,
                pfirst=pfirst)


def run(c, fsa=None, tn=None, states=None, int64=False, **over):
    from bpdecode_b200.speculative import verify_drafts

    c = {**c, **over}
    want = plain(c["src"], c["drafts"], c["uniforms"], c["noise"], c["lens"], c["probs"],
                 c["heats"], tn, states, c["first"], c["pfirst"])

    def up(t, dtype=None):
        return None if t is None else t.to("cuda") if dtype is None else t.to("cuda", dtype)

    got = verify_drafts(
        up(c["src"]), up(c["drafts"], torch.int64 if int64 else torch.int32), up(c["uniforms"]),
        up(c["noise"]), draft_lens=up(c["lens"], torch.int32), draft_probs=up(c["probs"]),
        temperature=up(c["heats"]), fsa=fsa, states=up(states), src_rows=up(c["first"]),
        prob_rows=up(c["pfirst"]) if c["probs"] is not None else None)
    check(got, want)
    return got, want


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("probs", [None, F32, BF16, F16])
@pytest.mark.parametrize("B,K,V,pad", [(1, 4, 1000, 0), (5, 3, 4099, 0), (37, 7, 517, 5),
                                       (9, 1, 32000, 8), (3, 31, 64, 0), (4, 2, 1, 0),
                                       (6, 0, 5003, 3), (700, 2, 131, 0)])
def test_against_the_definition(dtype, probs, B, K, V, pad) -> None:
    c = make(B, K, V, dtype, seed=B * 1000 + K, probs=probs, pad=pad)
    # the padding columns are not part of the vocabulary
    if pad:
        fsa, tn = tables(7, V, seed=V)
        states = torch.randint(0, 7, (B,), generator=torch.Generator().manual_seed(5)).int()
        run(c, fsa, tn, states)
    else:
        run(c)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("probs", [None, F32])
@pytest.mark.parametrize("V", [33, 1024, 50257])
def test_grammar(dtype, probs, V) -> None:
    fsa, tn = tables(12, V, seed=V)
    c = make(24, 4, V, dtype, seed=V + 1, probs=probs)
    g = torch.Generator().manual_seed(3)
    states = torch.randint(0, 12, (24,), generator=g).int()
    states[3], states[4], states[5] = -1, -2, 12  # broken, free, outside the table
    got, want = run(c, fsa, tn, states, int64=True)
    assert int(got.counts[3]) == int(got.counts[4]) == int(got.counts[5]) == 0
    assert got.states[3:6].tolist() == [-1, -1, -1]


def test_rows_of_nan_infinities_and_nothing() -> None:
    V = 300
    c = make(10, 2, V, F32, seed=4, ragged=False, heats="mixed")
    x = c["src"].view(10, 3, V)
    x[0, 0, 7] = float("nan")
    x[1, 0] = -math.inf  # nothing at all
    x[2, 0, 5], x[2, 0, 9] = math.inf, math.inf  # share everything
    x[3, 0] = float("nan")
    x[4, 1] = -math.inf
    x[4, 0, 11] = 100.0
    c["drafts"][4, 0] = 11  # accepted, then a row of nothing
    x[5, 0, 200:] = torch.finfo(F32).min
    c["drafts"][6, 0] = 10**6  # no token of the vocabulary
    c["drafts"][7, 0] = -5
    c["heats"] = torch.tensor([0.7, 1.0, 1.0, 0.0, 1.0, 1.0, 0.9, 0.0, 1e-3, math.inf])
    for probs in (None, torch.softmax(torch.randn(20, V, generator=torch.Generator().manual_seed(1)), -1)):
        got, _ = run({**c, "probs": probs})
        assert got.counts[1] == 0 and got.counts[3] == 0 and got.counts[4] == 1


def test_nan_and_infinities_in_rejected_places_change_nothing() -> None:
    V = 700
    fsa, tn = tables(4, V, seed=2)
    c = make(8, 2, V, BF16, seed=9, probs=F32)
    states = torch.tensor([0, 1, 2, 0, 1, 2, 0, 1], dtype=torch.int32)
    got, _ = run(c, fsa, tn, states)
    dirty = c["src"].clone()
    g = torch.Generator().manual_seed(0)
    for b in range(8):
        s = int(states[b])
        for i in range(int(c["lens"][b]) + 1):
            row = dirty[int(c["first"][b]) + i]
            off = (tn[s] < 0) if s >= 0 else torch.ones(V, dtype=bool)
            bad = torch.tensor([float("nan"), math.inf, -math.inf, 3e38])[
                torch.randint(0, 4, (V,), generator=g)].to(BF16)
            row[off] = bad[off]
            if i < int(c["lens"][b]) and s >= 0:
                s = int(tn[s, int(c["drafts"][b, i])])
    again, _ = run({**c, "src": dirty}, fsa, tn, states)
    for x, y in zip(got, again):
        assert torch.equal(x, y)


def test_ties_go_to_the_lowest_index() -> None:
    V, B = 5000, 6
    c = make(B, 1, V, BF16, seed=8, ragged=False, heats="one")
    c["noise"] = torch.ones(B, V)
    c["src"][:] = 1.0
    c["src"][:, 4090:4100] = 3.0
    c["drafts"][:] = torch.tensor([4090, 4091, 4095, 17, 4090, 0])[:, None]
    c["uniforms"][:] = 0.999
    got, _ = run(c)
    assert got.tokens[:, 0].tolist() == [4091, 4090, 4090, 4090, 4091, 4090]
    c["heats"] = torch.zeros(B)
    got, _ = run(c)
    assert got.tokens[0].tolist() == [4090, 4090] and got.tokens[1].tolist() == [4090, -1]


def test_probabilities_equal_to_the_target_leave_the_target() -> None:
    """max(p - q, 0) with nothing left falls back to p."""
    V, B = 257, 4
    c = make(B, 1, V, F32, seed=11, ragged=False, heats="one", probs=F32)
    c["probs"] = torch.ones(B, V)  # above p everywhere
    c["uniforms"][:] = 1.0 - 2.0**-24
    run(c)


def test_idle_requests() -> None:
    V = 400
    fsa, tn = tables(5, V, seed=1)
    c = make(6, 2, V, F32, seed=2, ragged=False, probs=BF16)
    states = torch.tensor([0, 1, 2, 3, 4, 1], dtype=torch.int32)
    c["lens"] = torch.tensor([-1, 3, 2, 2, 2, 2])
    c["first"][2] = -1
    c["first"][3] = c["src"].shape[0] - 2
    c["pfirst"][4] = c["probs"].shape[0] - 1
    got, _ = run(c, fsa, tn, states)
    assert got.counts[:5].tolist() == [0] * 5 and got.states[:5].tolist() == [0, 1, 2, 3, 4]
    assert (got.tokens[:5] == -1).all() and int(got.counts[5]) > 0


def test_padded_layout_strides_and_defaults() -> None:
    from bpdecode_b200.speculative import verify_drafts

    B, K, V = 7, 3, 1003
    c = make(B, K, V, F16, seed=21, ragged=False, heats="one", probs=F16)
    want = plain(c["src"], c["drafts"], c["uniforms"], c["noise"], c["lens"], c["probs"],
                 c["heats"], None, None, c["first"], c["pfirst"])

    def strided(t, pad):
        wide = torch.full((t.shape[0], t.shape[1] + pad), 7, dtype=t.dtype, device="cuda")
        wide[:, pad // 2:pad // 2 + t.shape[1]] = t.cuda()
        return wide[:, pad // 2:pad // 2 + t.shape[1]]

    got = verify_drafts(strided(c["src"], 6), strided(c["drafts"], 4), strided(c["uniforms"], 2),
                        strided(c["noise"], 10), draft_probs=strided(c["probs"], 14))
    check(got, want)


def test_sampling_alone_and_greedy_without_random_numbers() -> None:
    from bpdecode_b200.speculative import verify_drafts

    c = make(40, 0, 3001, BF16, seed=31, heats="one")
    got = verify_drafts(c["src"].cuda(), noise=c["noise"].cuda(), temperature=0.8)
    check(got, plain(c["src"], c["drafts"], c["uniforms"], c["noise"], c["lens"], None,
                     torch.full((40,), 0.8, dtype=torch.float32), None, None, c["first"],
                     c["pfirst"]))
    got = verify_drafts(c["src"].cuda(), temperature=0.0)
    assert torch.equal(got.tokens[:, 0].cpu(), c["src"].float().argmax(-1))
    empty = verify_drafts(c["src"][:0].cuda(), temperature=0.0)
    assert empty.tokens.shape == (0, 1)


@pytest.mark.parametrize("given", [True, False])
def test_tokens_are_distributed_as_the_target(given) -> None:
    """Over many requests with the same rows, the first token's frequencies are
    the target's probabilities, whatever the drafts (six standard deviations)."""
    from bpdecode_b200.speculative import verify_drafts

    B, V = 60000, 6
    g = torch.Generator().manual_seed(77)
    x = torch.randn(2, V, generator=g)
    p = torch.softmax(x[0].double(), -1)
    q = torch.softmax(x[1], -1)
    if given:
        draft = torch.multinomial(q.expand(B, V), 1, generator=g)
    else:
        draft = torch.full((B, 1), int(p.argmax()))
    got = verify_drafts(
        x[:1].repeat(2 * B, 1).cuda(), draft.cuda(), torch.rand(B, 1, generator=g).cuda(),
        torch.empty(B, V).exponential_(generator=g).cuda(),
        draft_probs=q.expand(B, V).contiguous().cuda() if given else None)
    freq = torch.bincount(got.tokens[:, 0].cpu(), minlength=V).double() / B
    assert bool(((freq - p).abs() <= 6 * (p * (1 - p) / B).sqrt()).all())
    assert int(got.counts.min()) >= 1 and int(got.counts.max()) == 2


def test_another_stream_and_repeated_calls_give_the_same_bits() -> None:
    from bpdecode_b200.speculative import verify_drafts

    c = make(33, 3, 9001, BF16, seed=5, probs=F32)
    args = (c["src"].cuda(), c["drafts"].cuda(), c["uniforms"].cuda(), c["noise"].cuda())
    more = dict(draft_lens=c["lens"].int().cuda(), draft_probs=c["probs"].cuda(),
                temperature=c["heats"].cuda(), src_rows=c["first"].cuda(),
                prob_rows=c["pfirst"].cuda())
    one = verify_drafts(*args, **more)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        two = verify_drafts(*args, **more)
    side.synchronize()
    for x, y in zip(one, two):
        assert x is y or torch.equal(x, y)


def test_refusals() -> None:
    from bpdecode_b200.speculative import MAX_DRAFTS, verify_drafts

    src = torch.randn(6, 50, device="cuda")
    drafts = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    u, e = torch.rand(2, 2, device="cuda"), torch.ones(2, 50, device="cuda")
    ok = dict(src=src, drafts=drafts, uniforms=u, noise=e)
    verify_drafts(**ok)
    fsa, _ = tables(3, 50, seed=0)
    states = torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (dict(src=src.cpu()), dict(src=src[:5]), dict(src=src.double()),
                dict(src=src.t()), dict(drafts=drafts.float()), dict(drafts=drafts.cpu()),
                dict(uniforms=None), dict(noise=None), dict(noise=e[:1]), dict(noise=e.half()),
                dict(noise=e[:, :40]), dict(temperature=-1.0), dict(temperature=float("nan")),
                dict(temperature=torch.ones(3, device="cuda")),
                dict(draft_lens=torch.zeros(2, device="cuda")), dict(fsa=fsa),
                dict(states=states), dict(fsa=fsa, states=states[:1]),
                dict(src_rows=torch.zeros(2, dtype=torch.int32, device="cuda")),
                dict(draft_probs=e[:1]), dict(draft_probs=e[:, :40].repeat(4, 1)),
                dict(prob_rows=torch.zeros(2, dtype=torch.int64, device="cuda")),
                dict(drafts=torch.zeros(2, MAX_DRAFTS + 1, dtype=torch.int32, device="cuda"),
                     src=src.repeat(20, 1), uniforms=torch.rand(2, 40, device="cuda"))):
        with pytest.raises((RuntimeError, ValueError)):
            verify_drafts(**{**ok, **bad})

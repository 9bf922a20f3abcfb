"""The measured cases of two operators that sit on either side of a model's logits.

``project``: hidden rows times a weight that all requests share, plus each row's own low-rank adapter
(``y[t] = W x[t] + scale[a] * B[a] (A[a] x[t])`` with ``a = ids[t]``, none where ``ids[t] < 0``).

``verify``: drafted tokens are verified against the target's probabilities, from random numbers that the
caller gives, under each request's grammar. A request brings ``n`` drafts and ``n + 1`` rows of logits. Row ``i``
is masked by the grammar state that the first ``i`` drafts lead to. With ``p = softmax(row / temperature)`` and
the draft's own distribution ``q`` (all of it on the drafted token where no probabilities are given), draft
``d`` is accepted when ``u * q[d] < p[d]``. The first one that is not accepted is replaced by
``argmax(max(p - q, 0) / e)`` with exponential noise ``e``; after the last one the next token is
``argmax(p / e)``. At temperature 0 both are the argmax. No drafts at all is plain sampling of one token.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}

# shares of the vocabulary that the states of the synthetic automaton allow: a number or a date, an identifier,
# the inside of a string (twice)
SHARES = (0.02, 0.3, 0.95, 0.95)

# about the share of drafts that these inputs have accepted
KEEP = {"none": 0.5, "float32": 0.75, "bfloat16": 0.75}


def listed():
    return [
        # one user, one token: the logits of a 32,000-token vocabulary; latency is all of it
        {"name": "project 1 row", "op": "project", "rows": 1, "inner": 2048, "outer": 32000, "adapters": 4, "rank": 16, "dtype": "bfloat16", "out": "bfloat16", "order": "mixed"},
        # a served batch, an adapter for two rows in three: the logits of a large vocabulary, in 32 bits for the sampler
        {"name": "project 64 rows, logits", "op": "project", "rows": 64, "inner": 4096, "outer": 128256, "adapters": 24, "rank": 16, "dtype": "bfloat16", "out": "float32", "order": "mixed"},
        # the same batch at a projection inside a layer
        {"name": "project 64 rows, square", "op": "project", "rows": 64, "inner": 4096, "outer": 4096, "adapters": 24, "rank": 16, "dtype": "bfloat16", "out": "bfloat16", "order": "mixed"},
        # drafts to be verified: more rows than requests, odd counts, an odd vocabulary, a small rank, halves
        {"name": "project 215 rows, odd", "op": "project", "rows": 215, "inner": 1608, "outer": 50257, "adapters": 43, "rank": 12, "dtype": "float16", "out": "float16", "order": "runs"},
        # prompts of several requests, one after the other: bound by the products
        {"name": "project 4096 rows", "op": "project", "rows": 4096, "inner": 4096, "outer": 8192, "adapters": 8, "rank": 64, "dtype": "bfloat16", "out": "bfloat16", "order": "runs"},
        # one user with four drafts
        {"name": "verify 1 request", "op": "verify", "requests": 1, "drafts": 4, "vocab": 32000, "dtype": "bfloat16", "probs": "float32", "states": 16, "temperature": "one", "ragged": False},
        # a served batch of grammar-bound requests with a small draft model
        {"name": "verify 64 x 4", "op": "verify", "requests": 64, "drafts": 4, "vocab": 128256, "dtype": "bfloat16", "probs": "float32", "states": 48, "temperature": "mixed", "ragged": True},
        # the largest: a full batch, logits in 32 bits, drafts looked up in the text (no probabilities)
        {"name": "verify 256 x 3, looked up", "op": "verify", "requests": 256, "drafts": 3, "vocab": 128256, "dtype": "float32", "probs": "none", "states": 48, "temperature": "mixed", "ragged": True},
        # no drafts: one token sampled for each row of a full batch
        {"name": "sample 1024", "op": "verify", "requests": 1024, "drafts": 0, "vocab": 128256, "dtype": "bfloat16", "probs": "none", "states": 48, "temperature": "one", "ragged": False},
        # an odd vocabulary, long drafts, halves, no grammar, the draft's probabilities in 16 bits
        {"name": "verify 37 x 7, odd", "op": "verify", "requests": 37, "drafts": 7, "vocab": 50257, "dtype": "float16", "probs": "bfloat16", "states": 0, "temperature": "one", "ragged": True},
        # greedy verification: needs no random numbers
        {"name": "verify 128 x 2, greedy", "op": "verify", "requests": 128, "drafts": 2, "vocab": 151936, "dtype": "bfloat16", "probs": "none", "states": 48, "temperature": "zero", "ragged": False},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.5:
        while True:
            dtype = rng.choice(("bfloat16", "bfloat16", "float16"))
            c = {"op": "project", "rows": _log(rng, 1, 4096), "inner": 8 * _log(rng, 64, 1024), "outer": _log(rng, 1000, 151936), "adapters": _log(rng, 1, 96),
                 "rank": rng.choice((4, 8, 12, 16, 16, 24, 32, 64)), "dtype": dtype, "out": rng.choice((dtype, dtype, "float32")), "order": rng.choice(("mixed", "runs"))}
            large = c["inner"] * c["outer"] <= 4096 * 128256 and c["adapters"] * c["rank"] * (c["inner"] + c["outer"]) <= 24 * 16 * 132352
            if large and c["rows"] * c["inner"] * c["outer"] <= 4096 * 4096 * 8192 and 3072 not in c.values():
                return c
    while True:
        c = {"op": "verify", "requests": _log(rng, 1, 1024), "drafts": rng.randint(0, 8), "vocab": _log(rng, 1000, 151936), "dtype": rng.choice(("bfloat16", "bfloat16", "float16", "float32")),
             "probs": rng.choice(("none", "float32", "bfloat16")), "states": rng.choice((0, 16, 48)), "temperature": rng.choice(("one", "mixed", "mixed", "zero")), "ragged": rng.random() < 0.5}
        if c["temperature"] == "zero" or c["drafts"] == 0:
            c["probs"] = "none"
        if c["requests"] * (c["drafts"] + 1) * c["vocab"] <= 1024 * 128256 and 3072 not in c.values():
            return c


# --- inputs ----------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return _prepare_project(case, g) if case["op"] == "project" else _prepare_verify(case, g)


def _prepare_project(c, g):
    dt, n, r = DTYPES[c["dtype"]], c["adapters"], c["rank"]
    T, K, N = c["rows"], c["inner"], c["outer"]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dt).mul_(std)

    if c["order"] == "runs":  # the rows of one request stand together, one adapter each
        ids = torch.sort(torch.randint(0, n, (T,), generator=g, device="cuda")).values
        ids = torch.randperm(n, generator=g, device="cuda")[ids]
    else:  # one row for each request, two in three of them with an adapter
        ids = torch.randint(0, n, (T,), generator=g, device="cuda")
        ids = torch.where(torch.rand(T, generator=g, device="cuda") < 2 / 3, ids, -1)
        ids[0] = 0
    s = {"case": c, "x": normal(T, K), "weight": normal(N, K, std=K**-0.5), "a": normal(n, r, K, std=K**-0.5), "b": normal(n, N, r, std=0.5 * r**-0.5),
         "scale": torch.rand(n, generator=g, device="cuda") + 0.5, "ids": ids.to(torch.int32)}
    if own:
        from bpdecode_b200.adapters import AdapterBank

        bank = AdapterBank(K, N, max_adapters=n, max_rank=r, dtype=dt, device="cuda")
        for i, scale in enumerate(s["scale"].tolist()):
            bank.load(i, s["a"][i], s["b"][i], scaling=scale)
        s["bank"] = bank
    return s


def _prepare_verify(c, g):
    B, K, V, S = c["requests"], c["drafts"], c["vocab"], c["states"]

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    def randint(high, *shape):
        return torch.randint(0, high, shape, generator=g, device="cuda")

    lens = randint(K + 1, B) if c["ragged"] else torch.full((B,), K, device="cuda")
    lens[0] = K
    first = torch.cumsum(lens + 1, 0) - (lens + 1)
    rows = int((lens + 1).sum())
    # a model's rows: most tokens unlikely, a few of them far above the rest
    logits = torch.randn(rows, V, generator=g, device="cuda").mul_(2.0)
    logits.scatter_reduce_(1, randint(V, rows, 24), 6.0 + 14.0 * rand(rows, 24), "amax")
    src = logits.to(DTYPES[c["dtype"]])
    temperature = {"one": torch.ones(B, device="cuda"), "mixed": torch.tensor((0.0, 0.7, 1.0, 1.3), device="cuda")[randint(4, B)], "zero": torch.zeros(B, device="cuda")}[c["temperature"]]
    heat = torch.where(temperature > 0, temperature, 1.0)[:, None]
    s = {"case": c, "src": src, "first": first, "lens": lens.to(torch.int32), "temperature": temperature if c["temperature"] != "zero" else 0.0, "tok_next": None, "states": None, "probs": None,
         "prob_first": None, "uniforms": None, "noise": None}
    state = None
    if S:
        share = torch.tensor(SHARES, device="cuda")[torch.arange(S, device="cuda") % len(SHARES)]
        s["tok_next"] = torch.where(rand(S, V) < share[:, None], randint(S, S, V), -1).to(torch.int32)
        state = randint(S, B)
        s["states"] = state.to(torch.int32)
    draft = torch.zeros(B, K, dtype=torch.int64, device="cuda")
    given = c["probs"] != "none"
    if given:  # rows of all requests' drafts, one after the other
        s["prob_first"] = torch.cumsum(lens, 0) - lens
        s["probs"] = torch.zeros(max(int(lens.sum()), 1), V, dtype=DTYPES[c["probs"]], device="cuda")
    for i in range(K):  # the draft model: it is near the target, and keeps to the grammar
        have = lens > i
        z = logits[(first + i).clamp(max=rows - 1)]
        z = z + 0.6 * torch.randn(B, V, generator=g, device="cuda")
        if S:
            z = torch.where(s["tok_next"][state] >= 0, z, -math.inf)
        if given:
            q = torch.softmax(z / heat, -1).to(DTYPES[c["probs"]])
            draft[:, i] = torch.argmax(q.float() / torch.empty_like(z).exponential_(generator=g), -1)
            s["probs"][(s["prob_first"] + i)[have]] = q[have]
        else:  # what the text says next: the likeliest token, or some other
            draft[:, i] = torch.where(rand(B) < 0.8, z.argmax(-1), randint(V, B))
        if S:
            state = s["tok_next"][state, draft[:, i]].long().clamp(min=0)
    s["drafts"] = draft.to(torch.int32)
    if c["temperature"] != "zero":
        s["uniforms"] = rand(B, K)
        s["noise"] = torch.empty(B, V, device="cuda").exponential_(generator=g).clamp_(min=1e-30)
    if own and S:
        from bpdecode_b200.ops import FsaTensors

        zero = torch.zeros(1, dtype=torch.int32, device="cuda")
        s["fsa"] = FsaTensors(trans=zero.repeat(S), accept=zero.repeat(S).to(torch.uint8), live=zero.repeat(S).to(torch.uint8), num_symbols=1, dead=-1,
                              offsets=zero.repeat(V + 1), symbols=zero, eos_id=-1, tok_next=s["tok_next"])
        s["fsa"].dense_tables()
    return s


# --- one pass --------------------------------------------------------------------


def run(state):
    if state["case"]["op"] == "project":
        return _own_project(state) if own else _plain_project(state)
    return _own_verify(state) if own else _plain_verify(state)


def _own_project(s):
    from bpdecode_b200.adapters import project

    return project(s["x"], s["weight"], s["bank"], s["ids"], out_dtype=DTYPES[s["case"]["out"]])


def _own_verify(s):
    from bpdecode_b200.speculative import verify_drafts

    r = verify_drafts(s["src"], s["drafts"], s["uniforms"], s["noise"], draft_lens=s["lens"], draft_probs=s["probs"], temperature=s["temperature"], fsa=s.get("fsa"), states=s["states"],
                      src_rows=s["first"], prob_rows=s["prob_first"])
    return {"tokens": r.tokens, "counts": r.counts, "logprobs": r.logprobs, **({"states": r.states} if s["states"] is not None else {})}


def _plain_project(s):
    x, n, r = s["x"].float(), s["a"].shape[0], s["a"].shape[1]
    low = (x @ s["a"].float().reshape(n * r, -1).T).view(-1, n, r)
    mine = s["ids"].long()[:, None] == torch.arange(n, device=x.device)
    low = torch.where(mine[:, :, None], low * s["scale"][:, None], 0.0)
    y = x @ s["weight"].float().T
    y += low.view(-1, n * r) @ s["b"].float().transpose(1, 2).reshape(n * r, -1)
    return y.to(DTYPES[s["case"]["out"]])


def _plain_verify(s):
    c = s["case"]
    B, K, V = c["requests"], c["drafts"], c["vocab"]
    dev = s["src"].device
    lens, drafts = s["lens"].long(), s["drafts"].long()
    place = torch.arange(K + 1, device=dev)
    here = place[None, :] <= lens[:, None]
    rows = torch.where(here, s["first"][:, None] + place, 0)
    x = s["src"][rows].float()
    path = None
    if s["states"] is not None:
        path = [s["states"].long()]
        for i in range(K):
            path.append(torch.where(path[-1] >= 0, s["tok_next"][path[-1].clamp(min=0), drafts[:, i]].long(), -1))
        path = torch.stack(path, 1)
        x = torch.where((s["tok_next"][path.clamp(min=0)] >= 0) & (path >= 0)[:, :, None], x, -math.inf)
    x = torch.where(x == x, x, -math.inf)
    temperature = torch.full((B,), s["temperature"], device=dev) if isinstance(s["temperature"], float) else s["temperature"]
    greedy = temperature <= 0
    heat = torch.where(greedy, 1.0, temperature)[:, None, None]
    top, best = x.max(-1)
    w = torch.where(x > -math.inf, torch.where(x == top[:, :, None], 1.0, torch.exp((x - top[:, :, None]) / heat)), 0.0)
    z = w.sum(-1)
    some = top > -math.inf
    p = w / torch.where(some, z, 1.0)[:, :, None]
    at = drafts[:, :, None]
    pd = p[:, :K].gather(2, at)[:, :, 0]
    qd = torch.ones(B, K, device=dev)
    if s["probs"] is not None:
        qrows = torch.where(here[:, 1:], s["prob_first"][:, None] + place[:K], 0)
        qd = s["probs"][qrows[:, :, None], at][:, :, 0].float()
    kept = torch.where(greedy[:, None], (drafts == best[:, :K]) & some[:, :K], (0.0 if s["uniforms"] is None else s["uniforms"]) * qd < pd)
    n = torch.cumprod((kept & here[:, 1:]).long(), 1).sum(1)
    each = torch.arange(B, device=dev)
    refused = n < lens
    last = p[each, n]
    token = best[each, n]
    if s["noise"] is not None:
        left = last
        if K:
            ni = n.clamp(max=K - 1)
            if s["probs"] is not None:
                q = s["probs"][torch.where(refused, s["prob_first"] + ni, 0)].float()
                left = torch.where(refused[:, None], last - q, last)
            else:
                left = torch.where(refused[:, None] & (torch.arange(V, device=dev) == drafts[each, ni][:, None]), 0.0, last)
            left = torch.where(left > 0, left, 0.0)
            left = torch.where((left > 0).any(-1, keepdim=True), left, last)
        token = torch.where(greedy, token, torch.argmax(left / s["noise"], -1))
    token = torch.where(some[each, n], token, -1)
    padded = torch.cat([drafts, torch.full((B, 1), -1, device=dev)], 1)
    tokens = torch.where(place < n[:, None], padded, torch.where(place == n[:, None], token[:, None], -1))
    picked = x.gather(2, tokens.clamp(min=0)[:, :, None])[:, :, 0]
    logprobs = torch.where(tokens >= 0, torch.where(picked == top, 0.0, (picked - top) / heat[:, :, 0]) - torch.log(z), 0.0)
    out = {"tokens": tokens, "counts": (n + (token >= 0)).to(torch.int32), "logprobs": logprobs}
    if path is not None:
        state = path[each, n]
        out["states"] = torch.where((token >= 0) & (state >= 0), s["tok_next"][state.clamp(min=0), token.clamp(min=0)], -1).to(torch.int32)
    return out


# --- the definition, in 64 bits --------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_project(s) if case["op"] == "project" else _exact_verify(s)


def _exact_project(s):
    x, w = s["x"].double(), s["weight"]
    y = torch.empty(x.shape[0], w.shape[0], dtype=torch.float64, device=x.device)
    for k in range(0, w.shape[0], 16384):
        y[:, k : k + 16384] = x @ w[k : k + 16384].double().T
    for i in torch.unique(s["ids"]).tolist():
        if i >= 0:
            mine = (s["ids"] == i).nonzero()[:, 0]
            y[mine] += s["scale"][i].double() * (x[mine] @ s["a"][i].double().T @ s["b"][i].double().T)
    return y


def _exact_verify(s):
    c = s["case"]
    B, K = c["requests"], c["drafts"]
    lens, drafts, first = s["lens"].tolist(), s["drafts"].tolist(), s["first"].tolist()
    heats = [s["temperature"]] * B if isinstance(s["temperature"], float) else s["temperature"].tolist()
    uniforms = None if s["uniforms"] is None else s["uniforms"].tolist()
    starts = None if s["states"] is None else s["states"].tolist()
    logprobs = torch.zeros(B, K + 1, dtype=torch.float64)
    for b in range(B):
        state = None if starts is None else starts[b]
        for i in range(lens[b] + 1):
            x = s["src"][first[b] + i].double()
            allowed = torch.ones_like(x, dtype=torch.bool) if state is None else s["tok_next"][state] >= 0
            if not bool(allowed.any()):
                break
            logp = torch.log_softmax(torch.where(allowed, x, -math.inf) / (heats[b] or 1.0), -1)
            p, q = logp.exp(), None
            if i < lens[b]:
                d = drafts[b][i]
                if s["probs"] is not None:
                    q = s["probs"][int(s["prob_first"][b]) + i].double()
                else:
                    q = torch.zeros_like(p)
                    q[d] = 1.0
                if (d == int(logp.argmax())) if heats[b] == 0 else (uniforms[b][i] * float(q[d]) < float(p[d])):
                    logprobs[b, i] = logp[d]
                    state = None if state is None else int(s["tok_next"][state, d])
                    continue
            if heats[b] == 0:
                token = int(logp.argmax())
            else:
                left = p if q is None else (p - q).clamp(min=0)
                left = left if bool((left > 0).any()) else p
                token = int((left / s["noise"][b].double()).argmax())
            logprobs[b, i] = logp[token]
            break
    out = {"tokens": None, "counts": None, "logprobs": logprobs}
    if starts is not None:
        out["states"] = None
    return out


# --- what a pass cannot do without -----------------------------------------------


def work(case):
    c = case
    size = {"float32": 4, "bfloat16": 2, "float16": 2, "none": 0}
    if c["op"] == "project":
        T, K, N, n, r = c["rows"], c["inner"], c["outer"], c["adapters"], c["rank"]
        share = 1.0 if c["order"] == "runs" else 2 / 3
        met = n * (1 - (1 - 1 / n) ** (share * T)) if n > 1 else 1.0  # adapters that some row has
        two = size[c["dtype"]]
        moved = two * (T * K + N * K + met * r * (K + N)) + size[c["out"]] * T * N + 4 * T
        return {"bytes": moved, "flops": 2.0 * T * N * K + 2.0 * share * T * r * (K + N)}
    B, K, V = c["requests"], c["drafts"], c["vocab"]
    share = sum(SHARES) / len(SHARES) if c["states"] else 1.0
    mean = K / 2 if c["ragged"] else float(K)
    keep = KEEP[c["probs"]]
    kept = sum(keep ** (i + 1) * (1 - i / (K + 1) if c["ragged"] else 1.0) for i in range(K))
    rows = B * (1 + min(kept, mean))  # the row of the first draft that is refused is the last one needed
    refused = B * min(1.0, mean * (1 - keep)) if K else 0.0
    moved = share * V * (rows * size[c["dtype"]] + (0 if c["temperature"] == "zero" else 4 * B) + refused * size[c["probs"]])
    moved += (rows * V / 8 if c["states"] else 0) + 28.0 * B * (K + 1)
    return {"bytes": moved, "flops": 4.0 * share * V * (rows + B)}

"""The products and the selection around the sampler in a decode step: beam
search's selection over beams and vocabulary, the reordering of the beams'
states, products with 4-bit weights, and products grouped by expert.

A case is a dict of plain values.  `prepare` makes what a program holds before
the call, `run` makes one pass (plain torch operations in 32 bits, or the
framework's kernels where `own` is set), `exact` computes the same from the
definitions in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda"


def listed():
    return [
        # One request decoded with 4 beams: latency of one selection.
        {"name": "beam_one_request", "kind": "beam", "batch": 1, "beams": 4, "vocab": 151936, "dtype": "f32",
         "n_out": 8, "mask": False, "finished": 0.0},
        # A translation or summarisation server's step: bf16 logits straight
        # from the model, some beams finished, twice as many candidates as
        # beams (those that end leave enough to go on).
        {"name": "beam_batch", "kind": "beam", "batch": 64, "beams": 8, "vocab": 151936, "dtype": "bf16",
         "n_out": 16, "mask": False, "finished": 0.2},
        # Constrained beams over an odd vocabulary: a grammar's mask.
        {"name": "beam_grammar", "kind": "beam", "batch": 24, "beams": 5, "vocab": 50257, "dtype": "f32",
         "n_out": 5, "mask": True, "finished": 0.1},
        # The caches of one request's beams follow their parents.
        {"name": "reorder_one_request", "kind": "reorder", "outer": 16, "batch": 1, "beams": 4, "heads": 2,
         "max_len": 512, "len_lo": 300, "len_hi": 420, "head_dim": 128},
        # A batch's caches, requests of different lengths.
        {"name": "reorder_batch", "kind": "reorder", "outer": 8, "batch": 8, "beams": 8, "heads": 4,
         "max_len": 2048, "len_lo": 1000, "len_hi": 2048, "head_dim": 128},
        # The output head of a quantised model for one request: f32 logits
        # for the sampler.
        {"name": "w4_head_one_row", "kind": "w4", "rows": 1, "k": 4096, "n": 151936, "group": 32, "zeros": False,
         "scales": "bf16", "out": "f32"},
        # A projection inside the model for a batch of requests, asymmetric
        # weights with long groups.
        {"name": "w4_batch", "kind": "w4", "rows": 32, "k": 4096, "n": 16384, "group": 128, "zeros": True,
         "scales": "bf16", "out": "bf16"},
        # A small projection of odd sizes, a few rows (a draft being verified).
        {"name": "w4_small_odd", "kind": "w4", "rows": 5, "k": 1184, "n": 1000, "group": 32, "zeros": True,
         "scales": "f32", "out": "f32"},
        # A decode step's gate and up products: 8 tokens meet some 60 of 256
        # experts, nearly each alone with its own.
        {"name": "grouped_decode", "kind": "grouped", "tokens": 8, "top_k": 8, "experts": 256, "k": 2048, "n": 1536,
         "swiglu": True, "out": "bf16"},
        # A prefill chunk's product over fewer, larger experts.
        {"name": "grouped_prefill", "kind": "grouped", "tokens": 4096, "top_k": 8, "experts": 64, "k": 2048,
         "n": 2048, "swiglu": False, "out": "bf16"},
        # The whole expert layer (grouping, gate and up, down, combination) of
        # a large decode batch, sizes that are no multiple of a tile.
        {"name": "experts_batch", "kind": "experts", "tokens": 200, "top_k": 4, "experts": 60, "hidden": 1448,
         "inter": 712},
        # The same for a prefill chunk over many small experts.
        {"name": "experts_prefill", "kind": "experts", "tokens": 2048, "top_k": 8, "experts": 128, "hidden": 2048,
         "inter": 768},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["beam", "beam", "reorder", "w4", "w4", "grouped", "grouped", "experts"])
    if kind == "beam":
        vocab, beams = _log_int(rng, 4000, 256000), rng.randrange(1, 17)
        vocab = (vocab + 63) // 64 * 64 if rng.random() < 0.5 else vocab
        batch = _log_int(rng, 1, max(1, min(128, 64 * 8 * 151936 // (2 * vocab * beams))))
        return {"kind": kind, "batch": batch, "beams": beams, "vocab": vocab, "dtype": rng.choice(["f32", "bf16"]),
                "n_out": min(64, beams * rng.choice([1, 2, 2])), "mask": rng.random() < 0.3,
                "finished": rng.choice([0.0, 0.1, 0.3])}
    if kind == "reorder":
        beams, head_dim, heads = rng.randrange(1, 17), rng.choice([64, 72, 128]), rng.randrange(1, 9)
        batch, max_len = _log_int(rng, 1, 16), _log_int(rng, 16, 2048)
        row = batch * beams * heads * max_len * head_dim * 2
        outer = _log_int(rng, 1, max(1, min(64, 700 * 1000 * 1000 // row)))
        hi = rng.randrange(max_len // 2, max_len + 1)
        return {"kind": kind, "outer": outer, "batch": batch, "beams": beams, "heads": heads, "max_len": max_len,
                "len_lo": hi // 2, "len_hi": hi, "head_dim": head_dim}
    if kind == "w4":
        group = rng.choice([32, 64, 128])
        k = group * max(1, _log_int(rng, 512, 8192) // group)
        n = _log_int(rng, 512, min(151936, 4096 * 151936 // k))
        n = n // 64 * 64 if rng.random() < 0.5 else n
        return {"kind": kind, "rows": rng.choice([1, 1, _log_int(rng, 2, 64)]), "k": k, "n": n, "group": group,
                "zeros": rng.random() < 0.5, "scales": rng.choice(["bf16", "f32"]),
                "out": rng.choice(["f32", "bf16"])}
    if kind == "grouped":
        experts, top_k = rng.choice([8, 16, 60, 64, 128, 160, 256]), rng.choice([1, 2, 4, 6, 8])
        k, n = 8 * rng.randrange(64, 257), 16 * rng.randrange(24, 97 if experts > 128 else 129)
        return {"kind": kind, "tokens": _log_int(rng, 1, min(4096, 4096 * 8 // top_k)), "top_k": min(top_k, experts),
                "experts": experts, "k": k, "n": n, "swiglu": rng.random() < 0.5, "out": rng.choice(["f32", "bf16"])}
    experts = rng.choice([8, 16, 60, 64, 128])
    return {"kind": kind, "tokens": _log_int(rng, 1, 2048), "top_k": rng.choice([1, 2, 4, 6, 8]), "experts": experts,
            "hidden": 8 * rng.randrange(64, 257), "inter": 8 * rng.randrange(32, 97)}


# ---- inputs ----------------------------------------------------------------

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, shape, scale, dtype):
    """N(0, scale), a block of rows at a time (the f32 form of a large weight is twice its size)."""
    out = torch.empty(shape, dtype=dtype, device=DEV)
    flat = out.view(shape[0], -1)
    step = max(1, (1 << 27) // flat.shape[1])
    for a in range(0, shape[0], step):
        part = flat[a:a + step]
        part.copy_(torch.randn(part.shape, generator=g, device=DEV).mul_(scale))
    return out


def _beam_inputs(c, seed):
    g = _gen(seed)
    B, K, V = c["batch"], c["beams"], c["vocab"]
    rows = B * K
    x = torch.randn(rows, V, generator=g, device=DEV).mul_(2.5)
    at = torch.randint(0, V, (rows, 16), generator=g, device=DEV)  # the few likely tokens of each beam
    x.scatter_(1, at, x.gather(1, at) + 8.0)
    mask = None
    if c["mask"]:  # a fifth of the vocabulary allowed
        words = (V + 31) // 32
        bits = torch.rand(rows, words * 32, generator=g, device=DEV).lt_(0.2).to(torch.int64).view(rows, words, 32)
        w = (bits << torch.arange(32, device=DEV)).sum(2)
        mask = torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)
    # beams of one request lie a few nats apart
    scores = (-20.0 - 4.0 * torch.rand(rows, generator=g, device=DEV)).float()
    finished = (torch.rand(rows, generator=g, device=DEV) < c["finished"]).to(torch.uint8)
    finished.view(B, K)[:, 0] = 0
    return {"logits": x.to(_TYPES[c["dtype"]]), "scores": scores, "finished": finished, "mask": mask, "eos": V - 1}


def _reorder_inputs(c, seed):
    g = _gen(seed)
    B, K = c["batch"], c["beams"]
    shape = (c["outer"], B * K, c["heads"], c["max_len"], c["head_dim"])
    # most beams go on from one of the better parents
    parents = (torch.rand(B, K, generator=g, device=DEV).pow_(1.5) * K).int().clamp_(max=K - 1)
    lengths = torch.randint(c["len_lo"], c["len_hi"] + 1, (B,), generator=g, device=DEV).int()
    return {"src": _normal(g, shape, 1.0, torch.bfloat16), "parents": parents, "lengths": lengths}


def _w4_inputs(c, seed):
    g = _gen(seed)
    M, K, N, G = c["rows"], c["k"], c["n"], c["group"]
    t = _TYPES[c["scales"]]
    s = torch.rand(N, K // G, generator=g, device=DEV).add_(0.5).mul_(1.0 / (4.6 * K ** 0.5)).to(t)
    z = torch.randint(4, 12, (N, K // G), generator=g, device=DEV).to(t) if c["zeros"] else None
    return {"x": torch.randn(M, K, generator=g, device=DEV).bfloat16(),
            "q": torch.randint(0, 256, (N, K // 2), generator=g, device=DEV, dtype=torch.uint8), "s": s, "z": z}


def _routes(g, tokens, experts, top_k):
    """A router's choice: some experts are liked more than others."""
    like = torch.randn(experts, generator=g, device=DEV).mul_(0.5)
    w, ids = torch.softmax(torch.randn(tokens, experts, generator=g, device=DEV) + like, 1).topk(top_k, 1)
    return ids.int(), (w / w.sum(1, keepdim=True)).float()


def _grouped_inputs(c, seed):
    g = _gen(seed)
    ids, w = _routes(g, c["tokens"], c["experts"], c["top_k"])
    s = {"x": torch.randn(c["tokens"], c.get("k", c.get("hidden")), generator=g, device=DEV).bfloat16(), "ids": ids,
         "weights": w}
    if c["kind"] == "grouped":
        s["w"] = _normal(g, (c["experts"], c["n"], c["k"]), c["k"] ** -0.5, torch.bfloat16)
    else:
        H, I = c["hidden"], c["inter"]
        s["up"] = _normal(g, (c["experts"], 2 * I, H), H ** -0.5, torch.bfloat16)
        s["down"] = _normal(g, (c["experts"], H, I), I ** -0.5, torch.bfloat16)
    return s


_INPUTS = {"beam": _beam_inputs, "reorder": _reorder_inputs, "w4": _w4_inputs, "grouped": _grouped_inputs,
           "experts": _grouped_inputs}


def prepare(case, seed):
    c, k = case, case["kind"]
    s = _INPUTS[k](c, seed)
    s["case"] = c
    if k == "reorder":
        s["dst"] = torch.zeros_like(s["src"])  # the caches' second buffer
    if k in ("grouped", "experts"):
        s["counts"] = torch.bincount(s["ids"].view(-1).long(), minlength=c["experts"]).tolist()
    if own:
        _PLAN[k](s, c)
    return s


# What a program that uses the framework keeps from call to call: workspaces,
# outputs, weights laid out once.

def _plan_beam(s, c):
    from hi_amd.beam import BeamSearch
    s["plan"] = BeamSearch(c["batch"], c["beams"], c["vocab"], c["n_out"], device=DEV)
    s["out"] = s["plan"].outputs(c["batch"])


def _plan_reorder(s, c):
    pass


def _plan_w4(s, c):
    from hi_amd.w4 import W4Linear
    s["plan"] = W4Linear(s["q"], s["s"], s["z"])
    s["y"] = torch.empty(c["rows"], c["n"], dtype=_TYPES[c["out"]], device=DEV)


def _plan_grouped(s, c):
    from hi_amd import moe
    s["plan"] = moe.RowGroups(c["tokens"], c["top_k"], c["experts"], device=DEV)
    s["y"] = torch.empty(c["tokens"] * c["top_k"], c["n"] // 2 if c["swiglu"] else c["n"], dtype=_TYPES[c["out"]],
                         device=DEV)


def _plan_experts(s, c):
    from hi_amd.moe import MoeExperts
    s["plan"] = MoeExperts(s["up"], s["down"], max_tokens=c["tokens"], top_k=c["top_k"])
    s["y"] = torch.empty_like(s["x"])


_PLAN = {"beam": _plan_beam, "reorder": _plan_reorder, "w4": _plan_w4, "grouped": _plan_grouped,
         "experts": _plan_experts}


# ---- one pass --------------------------------------------------------------

def _allowed(mask, V):
    bits = (mask[:, :, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
    return bits.view(mask.shape[0], -1)[:, :V] != 0


def _run_beam(s):
    c = s["case"]
    if own:
        return s["plan"].select(s["logits"], s["scores"], finished=s["finished"], eos_id=s["eos"],
                                mask_words=s["mask"], out=s["out"])
    B, K, V, n = c["batch"], c["beams"], c["vocab"], c["n_out"]
    x = s["logits"].float()
    if s["mask"] is not None:
        x = torch.where(_allowed(s["mask"], V), x, torch.full_like(x, -math.inf))
    m = x.max(1, keepdim=True).values
    lse = m + torch.log(torch.exp(x - m).sum(1, keepdim=True))
    top, tok = torch.sort(x, dim=1, descending=True, stable=True)
    top, tok = top[:, :n], tok[:, :n]
    score = s["scores"][:, None] + (top - lse)
    done = s["finished"].bool()[:, None]
    first = torch.arange(score.shape[1], device=DEV)[None] == 0
    score = torch.where(done, torch.where(first, s["scores"][:, None], torch.full_like(score, -math.inf)), score)
    tok = torch.where(done, torch.full_like(tok, s["eos"]), tok)
    score, at = torch.sort(score.view(B, -1), dim=1, descending=True, stable=True)
    score, at = score[:, :n], at[:, :n]
    parents = at // top.shape[1]
    tok = tok.view(B, -1).gather(1, at)
    return {"scores": score, "tokens": tok.int(), "parents": parents.int(),
            "finished": (done.view(B, K).gather(1, parents) | (tok == s["eos"])).to(torch.uint8)}


def _run_reorder(s):
    c = s["case"]
    if own:
        from hi_amd.beam import reorder_states
        reorder_states(s["src"], s["parents"], dst=s["dst"], row_dim=1, length_dim=3, lengths=s["lengths"])
        return {"state": s["dst"]}
    B, K = c["batch"], c["beams"]
    rows = (torch.arange(B, device=DEV)[:, None] * K + s["parents"]).view(-1)
    keep = torch.arange(c["max_len"], device=DEV)[None] < s["lengths"].repeat_interleave(K)[:, None]
    return {"state": torch.where(keep[None, :, None, :, None], s["src"].index_select(1, rows), s["dst"])}


def _run_w4(s):
    c = s["case"]
    if own:
        return {"y": s["plan"](s["x"], out=s["y"])}
    q, K, G = s["q"], c["k"], c["group"]
    x = s["x"].float()
    parts = []
    for a in range(0, c["n"], 16384):
        part = q[a:a + 16384]
        w = torch.stack((part & 15, part >> 4), 2).float().view(part.shape[0], K // G, G)
        z = s["z"][a:a + 16384].float()[:, :, None] if s["z"] is not None else 8.0
        w = (w - z) * s["s"][a:a + 16384].float()[:, :, None]
        parts.append(x @ w.view(part.shape[0], K).t())
    return {"y": torch.cat(parts, 1).to(_TYPES[c["out"]])}


def _plain_order(s):
    """The (token, slot) pairs sorted by expert, and each expert's range."""
    ids = s["ids"].view(-1)
    order = torch.sort(ids, stable=True).indices
    e = torch.arange(s["case"]["experts"] + 1, device=DEV, dtype=torch.int32)
    offsets = (ids[None] < e[:, None]).sum(1)
    return order, offsets.int()


def _plain_grouped(x, w, counts, swiglu):
    """x [pairs][k] in the experts' order times each expert's w [n][k]."""
    parts, a = [], 0
    for e, n in enumerate(counts):
        if n:
            parts.append(x[a:a + n] @ w[e].float().t())
            a += n
    y = torch.cat(parts)
    if swiglu:
        gate, up = y.chunk(2, 1)
        y = gate / (1.0 + torch.exp(-gate)) * up
    return y


def _run_grouped(s):
    c = s["case"]
    if own:
        from hi_amd import moe
        groups = moe.group_rows(s["ids"], c["experts"], out=s["plan"])
        moe.grouped_product(s["x"], s["w"], groups, gather=True, swiglu=c["swiglu"], out=s["y"])
        return {"order": groups.order, "offsets": groups.offsets, "y": s["y"]}
    order, offsets = _plain_order(s)
    y = _plain_grouped(s["x"].float().index_select(0, order // c["top_k"]), s["w"], s["counts"], c["swiglu"])
    return {"order": order.int(), "offsets": offsets, "y": y.to(_TYPES[c["out"]])}


def _run_experts(s):
    c = s["case"]
    if own:
        return {"y": s["plan"](s["x"], s["ids"], s["weights"], out=s["y"])}
    order, _ = _plain_order(s)
    h = _plain_grouped(s["x"].float().index_select(0, order // c["top_k"]), s["up"], s["counts"], True)
    y = _plain_grouped(h, s["down"], s["counts"], False) * s["weights"].view(-1).index_select(0, order)[:, None]
    back = torch.empty_like(y).index_copy_(0, order, y)
    return {"y": back.view(c["tokens"], c["top_k"], -1).sum(1).bfloat16()}


_RUN = {"beam": _run_beam, "reorder": _run_reorder, "w4": _run_w4, "grouped": _run_grouped, "experts": _run_experts}


def run(state):
    return _RUN[state["case"]["kind"]](state)


# ---- what a pass cannot do without -----------------------------------------

def _met(c):
    """Experts that some token meets, about."""
    return c["experts"] * (1.0 - (1.0 - c["top_k"] / c["experts"]) ** c["tokens"])


def work(case):
    c, k = case, case["kind"]
    if k == "beam":
        rows, V = c["batch"] * c["beams"], c["vocab"]
        going = rows * (1.0 - c["finished"])  # a finished beam's logits are not needed
        n = going * V * (2 if c["dtype"] == "bf16" else 4) + (going * V / 8 if c["mask"] else 0)
        return {"bytes": n + rows * 5 + c["batch"] * c["n_out"] * 13, "flops": 0}
    if k == "reorder":
        K = c["beams"]
        row = c["outer"] * c["batch"] * c["heads"] * (c["len_lo"] + c["len_hi"]) / 2 * c["head_dim"] * 2
        # distinct parents of K draws of the law in _reorder_inputs
        p = [((j + 1) / K) ** (1 / 1.5) - (j / K) ** (1 / 1.5) for j in range(K)]
        return {"bytes": row * (K + sum(1.0 - (1.0 - q) ** K for q in p)), "flops": 0}
    if k == "w4":
        M, K, N, G = c["rows"], c["k"], c["n"], c["group"]
        per = 2 if c["scales"] == "bf16" else 4
        n = N * K / 2 + N * (K // G) * per * (2 if c["zeros"] else 1)
        return {"bytes": n + 2 * M * K + M * N * (4 if c["out"] == "f32" else 2), "flops": 2 * M * K * N}
    T, P = c["tokens"], c["tokens"] * c["top_k"]
    if k == "grouped":
        out = P * (c["n"] // 2 if c["swiglu"] else c["n"]) * (4 if c["out"] == "f32" else 2)
        return {"bytes": 2 * T * c["k"] + 2 * _met(c) * c["n"] * c["k"] + out + 8 * P, "flops": 2 * P * c["n"] * c["k"]}
    H, I = c["hidden"], c["inter"]
    return {"bytes": 4 * T * H + 6 * _met(c) * H * I + 8 * P, "flops": 6 * P * H * I}


# ---- the definitions in 64 bits --------------------------------------------

def _exact_beam(c, seed):
    s = _beam_inputs(c, seed)
    B, K, V = c["batch"], c["beams"], c["vocab"]
    x = s["logits"].double()
    if s["mask"] is not None:
        x.masked_fill_(~_allowed(s["mask"], V), -math.inf)
    cum = s["scores"].double()[:, None]
    x = torch.log_softmax(x, 1).add_(cum)
    done = s["finished"].bool()
    x[done] = -math.inf
    x[done, s["eos"]] = cum[done, 0]
    # tokens and parents: whole numbers, which two scores a rounding apart may swap
    return {"scores": x.view(B, K * V).topk(c["n_out"], 1).values, "tokens": None, "parents": None, "finished": None}


def _exact_w4(c, seed):
    s = _w4_inputs(c, seed)
    x, q = s["x"].double(), s["q"]
    y = torch.empty(c["rows"], c["n"], dtype=torch.float64, device=DEV)
    at = torch.arange(c["k"], device=DEV) // c["group"]
    for a in range(0, c["n"], 8192):
        b = min(c["n"], a + 8192)
        w = torch.empty(b - a, c["k"], dtype=torch.float64, device=DEV)
        w[:, 0::2] = (q[a:b] % 16).double()
        w[:, 1::2] = (q[a:b] // 16).double()
        w -= s["z"][a:b].double()[:, at] if s["z"] is not None else 8.0
        w *= s["s"][a:b].double()[:, at]
        y[:, a:b] = x @ w.t().contiguous()
    return {"y": y}


def _exact_expert(x, w, ids, swiglu):
    """x [pairs][k] of pairs routed to ids [pairs]: each pair's product with its expert."""
    n = w.shape[1] // 2 if swiglu else w.shape[1]
    y = torch.zeros(x.shape[0], n, dtype=torch.float64, device=DEV)
    for e in range(w.shape[0]):
        at = (ids == e).nonzero()[:, 0]
        if at.numel():
            r = x[at] @ w[e].double().t().contiguous()
            y[at] = torch.nn.functional.silu(r[:, :n]) * r[:, n:] if swiglu else r
    return y


def _exact_grouped(c, seed):
    s = _grouped_inputs(c, seed)
    ids = s["ids"].view(-1).long()
    x = s["x"].double().repeat_interleave(c["top_k"], 0)
    if c["kind"] == "grouped":
        order = torch.argsort(ids * ids.numel() + torch.arange(ids.numel(), device=DEV))
        offsets = torch.cat((ids.new_zeros(1), torch.bincount(ids, minlength=c["experts"]).cumsum(0)))
        return {"order": order.int(), "offsets": offsets.int(), "y": _exact_expert(x, s["w"], ids, c["swiglu"])[order]}
    y = _exact_expert(_exact_expert(x, s["up"], ids, True), s["down"], ids, False)
    return {"y": (y.view(c["tokens"], c["top_k"], -1) * s["weights"].double()[:, :, None]).sum(1)}


_EXACT = {"beam": _exact_beam, "w4": _exact_w4, "grouped": _exact_grouped, "experts": _exact_grouped}


def exact(case, seed):
    return _EXACT[case["kind"]](case, seed) if case["kind"] in _EXACT else None

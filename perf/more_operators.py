"""A speculative decode step's verification with sampled drafts, and the
products of its many rows with microscaled 4-bit floating point (blocks of 32
elements E2M1 with a power-of-two scale): quantisation, linear layers, experts.

A case is a dict of plain values.  `prepare` makes what a program holds before
the call, `run` makes one pass (plain torch operations, or the framework's
kernels where `own` is set), `exact` computes the same from the definitions in
64 bits.
"""
import math

import torch

own = False

DEV = "cuda"


def listed():
    return [
        # One request with four drafts: latency of a verification.
        {"name": "verify_one_request", "kind": "verify", "batch": 1, "drafts": 4, "vocab": 151936, "dtype": "f32",
         "draft_probs": True, "ragged": False},
        # A server's step: every request verifies eight drafts of a smaller model.
        {"name": "verify_batch", "kind": "verify", "batch": 64, "drafts": 8, "vocab": 151936, "dtype": "f32",
         "draft_probs": True, "ragged": False},
        # Drafts looked up in the prompt: no draft probabilities, some requests
        # without any draft; an odd vocabulary, probabilities in bf16.
        {"name": "verify_lookup_ragged", "kind": "verify", "batch": 24, "drafts": 5, "vocab": 50257, "dtype": "bf16",
         "draft_probs": False, "ragged": True},
        # The rows of a small step on their way into a 4-bit product.
        {"name": "quantize_few_rows", "kind": "quantize", "rows": 5, "k": 1184, "dtype": "bf16"},
        # A weight quantised as a checkpoint is loaded.
        {"name": "quantize_weight", "kind": "quantize", "rows": 16384, "k": 4096, "dtype": "f32"},
        # The output head of a 4-bit model for one request: f32 logits for the sampler.
        {"name": "linear_head_one_row", "kind": "linear", "rows": 1, "k": 4096, "n": 151936, "bias": False,
         "out": "f32"},
        # A small projection of odd sizes, a few rows (one request's drafts).
        {"name": "linear_small_odd", "kind": "linear", "rows": 5, "k": 1184, "n": 1000, "bias": True, "out": "f32"},
        # A projection for 64 requests that verify four drafts each.
        {"name": "linear_verify_batch", "kind": "linear", "rows": 320, "k": 4096, "n": 16384, "bias": False,
         "out": "bf16"},
        # The same projection for prompts.
        {"name": "linear_prefill", "kind": "linear", "rows": 8192, "k": 4096, "n": 16384, "bias": False,
         "out": "bf16"},
        # The expert layer of a decode step: 8 tokens meet some 60 of 256 experts.
        {"name": "experts_decode", "kind": "experts", "tokens": 8, "top_k": 8, "experts": 256, "hidden": 2048,
         "inter": 768},
        # A step that verifies drafts, sizes that are no multiple of a tile.
        {"name": "experts_verify_batch", "kind": "experts", "tokens": 200, "top_k": 4, "experts": 60, "hidden": 1440,
         "inter": 704},
        # A chunk of prompts over many small experts.
        {"name": "experts_prefill", "kind": "experts", "tokens": 4096, "top_k": 8, "experts": 128, "hidden": 2048,
         "inter": 768},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["verify", "verify", "quantize", "linear", "linear", "linear", "experts", "experts"])
    if kind == "verify":
        vocab, drafts = _log_int(rng, 4000, 256000), rng.randrange(1, 9)
        vocab = (vocab + 63) // 64 * 64 if rng.random() < 0.5 else vocab
        batch = _log_int(rng, 1, max(1, min(128, 64 * 9 * 151936 // (vocab * (drafts + 1)))))
        return {"kind": kind, "batch": batch, "drafts": drafts, "vocab": vocab, "dtype": rng.choice(["f32", "bf16"]),
                "draft_probs": rng.random() < 0.7, "ragged": rng.random() < 0.5}
    if kind == "quantize":
        k = 32 * _log_int(rng, 4, 512)
        return {"kind": kind, "rows": _log_int(rng, 1, min(16384, 16384 * 4096 // k)), "k": k,
                "dtype": rng.choice(["f32", "bf16"])}
    if kind == "linear":
        k = 32 * _log_int(rng, 16, 256)
        n = _log_int(rng, 512, min(151936, 4096 * 151936 // k))
        n = n // 64 * 64 if rng.random() < 0.5 else n
        most = max(1, min(8192, 8192 * 4096 * 16384 // (n * k)))
        rows = rng.choice([1, _log_int(rng, 2, min(64, most)), _log_int(rng, min(64, most), most)])
        return {"kind": kind, "rows": rows, "k": k, "n": n, "bias": rng.random() < 0.3,
                "out": rng.choice(["f32", "bf16"])}
    experts, top_k = rng.choice([8, 16, 60, 64, 128, 256]), rng.choice([1, 2, 4, 6, 8])
    return {"kind": kind, "tokens": _log_int(rng, 1, 4096), "top_k": top_k, "experts": experts,
            "hidden": 32 * rng.randrange(16, 65), "inter": 32 * rng.randrange(8, 25)}


# ---- inputs ----------------------------------------------------------------

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _verify_inputs(c, seed):
    g = _gen(seed)
    B, K, V, t = c["batch"], c["drafts"], c["vocab"], _TYPES[c["dtype"]]
    x = torch.randn(B, K + 1, V, generator=g, device=DEV).mul_(1.5)
    at = torch.randint(0, V, (B, K + 1, 32), generator=g, device=DEV)  # the few likely tokens
    x.scatter_(2, at, x.gather(2, at) + 9.0)
    d = torch.randn(B, K, V, generator=g, device=DEV).mul_(0.5).add_(x[:, :K])  # the draft model is a little off
    target = torch.softmax(x, 2).to(t)
    del x
    if c["draft_probs"]:
        draft = torch.softmax(d, 2)
        race = torch.rand(B, K, V, generator=g, device=DEV).log_().neg_().add_(1e-20)
        tokens = race.div_(draft).argmin(2).int()  # sampled from the draft's probabilities
        draft = draft.to(t)
    else:
        draft, tokens = None, d.argmax(2).int()
    length = torch.randint(0, K + 1, (B,), generator=g, device=DEV).int() if c["ragged"] else None
    return {"target": target, "draft": draft, "tokens": tokens, "length": length,
            "uniforms": torch.rand(B, K + 1, generator=g, device=DEV)}


def _quantize_inputs(c, seed):
    g = _gen(seed)
    x = torch.randn(c["rows"], c["k"], generator=g, device=DEV)
    x *= torch.exp(torch.randn(c["k"], generator=g, device=DEV))  # some inputs are larger than others throughout
    return {"x": x.mul_(0.05).to(_TYPES[c["dtype"]])}


def _weight(g, rows, k):
    """N(0, 1 / k) rounded to blocks: codes [rows][k / 2] and scales [rows][k / 32]."""
    codes = torch.empty(rows, k // 2, dtype=torch.uint8, device=DEV)
    scales = torch.empty(rows, k // 32, dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 25) // k)
    for a in range(0, rows, step):
        n = min(step, rows - a)
        c, s = _plain_codes(torch.randn(n, k, generator=g, device=DEV).mul_(k ** -0.5))
        codes[a:a + n], scales[a:a + n] = c[:, 0::2] | c[:, 1::2] << 4, s
    return codes, scales


def _linear_inputs(c, seed):
    g = _gen(seed)
    s = {"x": torch.randn(c["rows"], c["k"], generator=g, device=DEV).bfloat16(),
         "bias": torch.randn(c["n"], generator=g, device=DEV) if c["bias"] else None}
    s["codes"], s["scales"] = _weight(g, c["n"], c["k"])
    return s


def _experts_inputs(c, seed):
    g = _gen(seed)
    T, E, H, I = c["tokens"], c["experts"], c["hidden"], c["inter"]
    like = torch.randn(E, generator=g, device=DEV).mul_(0.5)  # some experts are liked more than others
    w, ids = torch.softmax(torch.randn(T, E, generator=g, device=DEV) + like, 1).topk(c["top_k"], 1)
    s = {"x": torch.randn(T, H, generator=g, device=DEV).bfloat16(), "ids": ids.int(),
         "weights": (w / w.sum(1, keepdim=True)).float()}
    for name, n, k in (("up", 2 * I, H), ("down", H, I)):
        codes, scales = _weight(g, E * n, k)
        s[name], s[name + "_scales"] = codes.view(E, n, k // 2), scales.view(E, n, k // 32)
    return s


_INPUTS = {"verify": _verify_inputs, "quantize": _quantize_inputs, "linear": _linear_inputs,
           "experts": _experts_inputs}


def prepare(case, seed):
    c, k = case, case["kind"]
    s = _INPUTS[k](c, seed)
    s["case"] = c
    if k == "experts":
        s["counts"] = torch.bincount(s["ids"].view(-1).long(), minlength=c["experts"]).tolist()
    if own:
        _PLAN[k](s, c)
    return s


# What a program that uses the framework keeps from call to call: workspaces,
# outputs, weights laid out once.

def _plan_verify(s, c):
    from hi_amd.speculative import SpecVerifier
    s["plan"] = SpecVerifier(c["batch"], c["drafts"], c["vocab"], device=DEV)
    s["out"] = s["plan"].outputs(c["batch"])


def _plan_quantize(s, c):
    s["codes"] = torch.empty(c["rows"], c["k"] // 2, dtype=torch.uint8, device=DEV)
    s["scales"] = torch.empty(c["rows"], c["k"] // 32, dtype=torch.uint8, device=DEV)
    s["values"] = torch.empty(c["rows"], c["k"], dtype=torch.bfloat16, device=DEV)


def _plan_linear(s, c):
    from hi_amd.mx4 import Mx4Linear
    s["plan"] = Mx4Linear(s["codes"], s["scales"], s["bias"])
    s["y"] = torch.empty(c["rows"], c["n"], dtype=_TYPES[c["out"]], device=DEV)


def _plan_experts(s, c):
    from hi_amd.mx4 import Mx4Experts
    s["plan"] = Mx4Experts(s["up"], s["up_scales"], s["down"], s["down_scales"], max_tokens=c["tokens"],
                           top_k=c["top_k"])
    s["y"] = torch.empty_like(s["x"])


_PLAN = {"verify": _plan_verify, "quantize": _plan_quantize, "linear": _plan_linear, "experts": _plan_experts}


# ---- one pass --------------------------------------------------------------

def _run_verify(s):
    c = s["case"]
    if own:
        return s["plan"](s["target"], s["tokens"], s["uniforms"], draft_probs=s["draft"], draft_len=s["length"],
                         out=s["out"])
    B, K, V = c["batch"], c["drafts"], c["vocab"]
    t = s["tokens"].long()
    p = s["target"][:, :K].gather(2, t[:, :, None])[:, :, 0].double()
    q = s["draft"].gather(2, t[:, :, None])[:, :, 0].double() if s["draft"] is not None else torch.ones_like(p)
    place = torch.arange(K + 1, device=DEV)[None]
    length = s["length"].long() if s["length"] is not None else torch.full((B,), K, device=DEV)
    taken = (s["uniforms"][:, :K].double() * q < p) & (place[:, :K] < length[:, None])
    n = taken.long().cumprod(1).sum(1)
    b = torch.arange(B, device=DEV)
    r = s["target"][b, n].double()
    at, rejected = n.clamp(max=K - 1), (n < length)[:, None]
    if s["draft"] is not None:
        less = s["draft"][b, at].double()
    else:
        less = (torch.arange(V, device=DEV)[None] == t[b, at][:, None]).double()
    rest = torch.where(rejected, r - less, r).clamp(min=0.0)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, r)
    total = rest.cumsum(1)
    drawn = (total <= s["uniforms"][:, K:].double() * total[:, -1:]).sum(1).clamp(max=V - 1)
    tokens = torch.where(place < n[:, None], torch.nn.functional.pad(t, (0, 1)), torch.full_like(place, -1))
    tokens = torch.where(place == n[:, None], drawn[:, None], tokens)
    return {"tokens": tokens.int(), "counts": (n + 1).int()}


def _plain_codes(x):
    """Codes (one a byte) and scales of x [rows][k] f32."""
    b = x.view(x.shape[0], -1, 32)
    a = b.abs().amax(2)
    s = (torch.frexp(a).exponent + 124).clamp(0, 254)  # a = m 2^e, 0.5 <= m < 1: floor(log2 a) - 2 + 127
    s = torch.where(a == 0, torch.zeros_like(s), s).int()
    m = b.abs() * ((254 - s) << 23).view(torch.float32)[:, :, None]  # times 2^(127 - s)
    c = (m > 0.25).byte()
    for edge, tie_up in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        c += m >= edge if tie_up else m > edge
    return (c + (torch.signbit(b).byte() << 3)).view(x.shape), s.byte()


def _plain_values(codes, scales):
    """The f32 values of packed codes [rows][k / 2] with scales [rows][k / 32]."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=DEV)
    table = torch.cat((table, -table))
    v = table[torch.stack((codes & 15, codes >> 4), 2).int()].view(codes.shape[0], -1, 32)
    # (a scale of 0 is 2^-127, the subnormal with only the bit below the first set)
    e = torch.where(scales == 0, torch.full_like(scales, 1, dtype=torch.int32) << 22, scales.int() << 23)
    return (v * e.view(torch.float32)[:, :, None]).view(codes.shape[0], -1)


def _plain_rounded(x):
    c, s = _plain_codes(x)
    return _plain_values(c[:, 0::2] | c[:, 1::2] << 4, s), s


def _run_quantize(s):
    if own:
        from hi_amd.mx4 import dequantize_mx4, quantize_mx4
        codes, scales = quantize_mx4(s["x"], out=(s["codes"], s["scales"]))
        return {"values": dequantize_mx4(codes, scales, out=s["values"]), "scales": scales}
    values, scales = _plain_rounded(s["x"].float())
    return {"values": values.bfloat16(), "scales": scales}


def _run_linear(s):
    c = s["case"]
    if own:
        return {"y": s["plan"](s["x"], out=s["y"])}
    x, _ = _plain_rounded(s["x"].float())
    parts = []
    for a in range(0, c["n"], 16384):
        parts.append(x @ _plain_values(s["codes"][a:a + 16384], s["scales"][a:a + 16384]).t())
    y = torch.cat(parts, 1)
    if s["bias"] is not None:
        y = y + s["bias"]
    return {"y": y.to(_TYPES[c["out"]])}


def _plain_grouped(x, codes, scales, counts):
    """x [pairs][k] in the experts' order times each expert's weight [n][k]."""
    parts, a = [], 0
    for e, n in enumerate(counts):
        if n:
            parts.append(x[a:a + n] @ _plain_values(codes[e], scales[e]).t())
            a += n
    return torch.cat(parts)


def _run_experts(s):
    c = s["case"]
    if own:
        return {"y": s["plan"](s["x"], s["ids"], s["weights"], out=s["y"])}
    order = torch.sort(s["ids"].view(-1), stable=True).indices
    x, _ = _plain_rounded(s["x"].float())
    h = _plain_grouped(x.index_select(0, order // c["top_k"]), s["up"], s["up_scales"], s["counts"])
    gate, up = h.double().chunk(2, 1)  # what is rounded next lies next to borders
    h, _ = _plain_rounded((gate / (1.0 + torch.exp(-gate)) * up).float())
    y = _plain_grouped(h, s["down"], s["down_scales"], s["counts"])
    y = y * s["weights"].view(-1).index_select(0, order)[:, None]
    back = torch.empty_like(y).index_copy_(0, order, y)
    return {"y": back.view(c["tokens"], c["top_k"], -1).sum(1).bfloat16()}


_RUN = {"verify": _run_verify, "quantize": _run_quantize, "linear": _run_linear, "experts": _run_experts}


def run(state):
    return _RUN[state["case"]["kind"]](state)


# ---- what a pass cannot do without -----------------------------------------

_MX4 = 0.5 + 1.0 / 32.0  # bytes an element


def work(case):
    c, k = case, case["kind"]
    if k == "verify":  # one row of the target and one of the draft a request
        size = 4 if c["dtype"] == "f32" else 2
        B, K, V = c["batch"], c["drafts"], c["vocab"]
        rows = 2 if c["draft_probs"] else 1
        return {"bytes": B * (rows * V * size + rows * K * size + 4 * K + 4 * (K + 1) * 2 + 4), "flops": 0}
    if k == "quantize":  # x read, codes and scales written and read, values written
        n = c["rows"] * c["k"]
        return {"bytes": n * ((4 if c["dtype"] == "f32" else 2) + 2 * _MX4 + 2), "flops": 0}
    if k == "linear":
        M, K, N = c["rows"], c["k"], c["n"]
        return {"bytes": _MX4 * N * K + 2 * M * K + M * N * (4 if c["out"] == "f32" else 2) + (4 * N if c["bias"] else 0),
                "flops": 2 * M * N * K}
    T, P, E, H, I = c["tokens"], c["tokens"] * c["top_k"], c["experts"], c["hidden"], c["inter"]
    met = E * (1.0 - (1.0 - c["top_k"] / E) ** T)  # experts that some token meets, about
    return {"bytes": 4 * T * H + _MX4 * 3 * met * H * I + 8 * P, "flops": 6 * P * H * I}


# ---- the definitions in 64 bits --------------------------------------------

def _exact_verify(c, seed):
    s = _verify_inputs(c, seed)
    B, K = c["batch"], c["drafts"]
    out = torch.full((B, K + 1), -1, dtype=torch.int32, device=DEV)
    counts = torch.zeros(B, dtype=torch.int32, device=DEV)
    tokens, u = s["tokens"].tolist(), s["uniforms"].tolist()  # (an f32 as a Python float is itself)
    lengths = s["length"].tolist() if s["length"] is not None else [K] * B
    for b in range(B):
        n = 0
        while n < lengths[b]:
            t = tokens[b][n]
            q = float(s["draft"][b, n, t]) if s["draft"] is not None else 1.0
            if not u[b][n] * q < float(s["target"][b, n, t]):
                break
            out[b, n] = t
            n += 1
        p = s["target"][b, n].double()
        r = p
        if n < lengths[b]:
            q = s["draft"][b, n].double() if s["draft"] is not None else torch.zeros_like(p)
            if s["draft"] is None:
                q[tokens[b][n]] = 1.0
            r = torch.maximum(p - q, torch.zeros_like(p))
            if not float(r.sum()) > 0:
                r = p
        mass = r.cumsum(0)
        out[b, n] = torch.searchsorted(mass, mass[-1:] * u[b][K], right=True)[0].clamp(max=c["vocab"] - 1).int()
        counts[b] = n + 1
    return {"tokens": out, "counts": counts}


def _exact_rounded(x):
    """x [rows][k] in 64 bits rounded to blocks of 32: the values, and the scales' exponents + 127."""
    b = x.view(x.shape[0], -1, 32)
    a = b.abs().amax(2, keepdim=True)
    e = torch.floor(torch.log2(torch.where(a > 0, a, torch.ones_like(a))))
    e = torch.where(torch.ldexp(torch.ones_like(e), e) > a, e - 1, e)  # log2 rounds
    e = torch.where(torch.ldexp(torch.ones_like(e), e + 1) <= a, e + 1, e)
    e = torch.where(a > 0, e - 2, torch.full_like(e, -127)).clamp(min=-127)
    m = torch.ldexp(b, -e)
    half, one, two = torch.round(m * 2) / 2, torch.round(m), torch.round(m / 2) * 2  # round: ties to even
    v = torch.where(m.abs() < 2, half, torch.where(m.abs() < 4, one, two)).clamp(-6.0, 6.0)
    return torch.ldexp(v, e).view(x.shape), (e[:, :, 0] + 127).byte()


def _exact_weight(codes, scales):
    c = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.float64, device=DEV)
    c[:, 0::2], c[:, 1::2] = (codes % 16).double(), (codes // 16).double()
    low = c % 8  # 1 bit of mantissa: 0, 0.5, then (1 + m / 2) 2^(exponent - 1)
    v = torch.where(low < 2, low / 2, torch.ldexp(1 + (low % 2) / 2, torch.floor(low / 2) - 1))
    v = torch.where(c >= 8, -v, v).view(codes.shape[0], -1, 32)
    return torch.ldexp(v, scales.double()[:, :, None] - 127).view(codes.shape[0], -1)


def _exact_quantize(c, seed):
    x = _quantize_inputs(c, seed)["x"]
    values = torch.empty(x.shape, dtype=torch.float64, device=DEV)
    scales = torch.empty(c["rows"], c["k"] // 32, dtype=torch.uint8, device=DEV)
    for a in range(0, c["rows"], 2048):
        values[a:a + 2048], scales[a:a + 2048] = _exact_rounded(x[a:a + 2048].double())
    return {"values": values, "scales": scales}


def _exact_linear(c, seed):
    s = _linear_inputs(c, seed)
    x, _ = _exact_rounded(s["x"].double())
    y = torch.empty(c["rows"], c["n"], dtype=torch.float64, device=DEV)
    for a in range(0, c["n"], 8192):
        w = _exact_weight(s["codes"][a:a + 8192], s["scales"][a:a + 8192])
        y[:, a:a + 8192] = x @ w.t().contiguous()
    if s["bias"] is not None:
        y += s["bias"].double()
    return {"y": y}


def _exact_experts(c, seed):
    s = _experts_inputs(c, seed)
    x, _ = _exact_rounded(s["x"].double())
    y = torch.zeros(c["tokens"], c["hidden"], dtype=torch.float64, device=DEV)
    for e in range(c["experts"]):
        t, slot = (s["ids"] == e).nonzero(as_tuple=True)
        if t.numel() == 0:
            continue
        h = x[t] @ _exact_weight(s["up"][e], s["up_scales"][e]).t().contiguous()
        h = torch.nn.functional.silu(h[:, :c["inter"]]) * h[:, c["inter"]:]
        h, _ = _exact_rounded(h)
        h = h @ _exact_weight(s["down"][e], s["down_scales"][e]).t().contiguous()
        y.index_add_(0, t, h * s["weights"][t, slot].double()[:, None])
    return {"y": y}


_EXACT = {"verify": _exact_verify, "quantize": _exact_quantize, "linear": _exact_linear, "experts": _exact_experts}


def exact(case, seed):
    return _EXACT[case["kind"]](case, seed)

"""The decode step's operators around its products, as cases that can be timed and compared:

    w4        matrix-vector products with 4-bit weights, group scales and zero points
    moe       a whole mixture-of-experts layer for a few tokens: router, choice, experts, weighted sum
    norm      the norms after a block and before the next, with the gate and the scaled residual sum
    logprobs  log probabilities of given tokens, their ranks, the entropy and the top alternatives

    listed()            the cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) inputs and what else a program holds before the call
    run(state)          one pass: the framework's calls where `own`, else the plain form
    work(case)          bytes and operations a pass cannot do without
    exact(case, seed)   what a pass returns, in 64 bits from the definition

Weights and activations are synthetic: 4-bit codes drawn evenly, scales around those of a matrix
of standard deviation k^-1/2, activations N(0, 1) with the few large channels that hidden states
have, logits of a peaked distribution.
"""
from __future__ import annotations

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}
GLUS = ("none", "swiglu", "swiglu_clamp", "geglu")


def listed() -> list[dict]:
    return [
        # One sequence's token through a square projection: what a single small product costs.
        {"name": "w4_t1_bf16", "kind": "w4", "rows": 1, "k": 4096, "n": 4096, "group": 128, "type": "bf16",
         "scales": "bf16", "zeros": False, "glu": "none"},
        # The gate | up product of a feed-forward block with its GLU, four sequences, F32 activations.
        {"name": "w4_glu_t4_f32", "kind": "w4", "rows": 4, "k": 2560, "n": 10240, "group": 64, "type": "f32",
         "scales": "f16", "zeros": True, "glu": "geglu"},
        # The head of a vocabulary of odd size for the most rows a call takes.
        {"name": "w4_head_t16_f16", "kind": "w4", "rows": 16, "k": 4096, "n": 32003, "group": 32, "type": "f16",
         "scales": "f16", "zeros": True, "glu": "none"},
        # A routed block's decode step: one sequence of a model with many small experts.
        {"name": "moe_t1_bf16", "kind": "moe", "tokens": 1, "experts": 128, "used": 8, "hidden": 2048, "inter": 768,
         "group": 128, "type": "bf16", "scales": "bf16", "zeros": False, "router": "f32", "score": "softmax",
         "bias": False, "renormalize": True, "scale": 1.0, "glu": "swiglu"},
        # A few sequences, F32, scores by sigmoid with a selection bias, experts of an odd width.
        {"name": "moe_t5_f32", "kind": "moe", "tokens": 5, "experts": 60, "used": 4, "hidden": 1280, "inter": 416,
         "group": 32, "type": "f32", "scales": "f16", "zeros": True, "router": "f32", "score": "sigmoid",
         "bias": True, "renormalize": True, "scale": 2.5, "glu": "swiglu_clamp"},
        # A small batch of sequences: most experts are named by someone.
        {"name": "moe_t16_bf16", "kind": "moe", "tokens": 16, "experts": 128, "used": 8, "hidden": 2048, "inter": 768,
         "group": 64, "type": "bf16", "scales": "bf16", "zeros": True, "router": "bf16", "score": "softmax",
         "bias": False, "renormalize": True, "scale": 1.0, "glu": "swiglu"},
        # A decode step's norms between two blocks, one sequence.
        {"name": "norm_t1_f32", "kind": "norm", "rows": 1, "width": 2560, "type": "f32", "post": True, "gate": "none",
         "scale": 1.0, "offset": 1.0},
        # A batch of sequences, a gate for each channel, rows of odd length.
        {"name": "norm_t37_f16", "kind": "norm", "rows": 37, "width": 5119, "type": "f16", "post": True,
         "gate": "channel", "scale": 0.25, "offset": 0.0},
        # A long prompt's, with a gate for each token and channel.
        {"name": "norm_t4096_bf16", "kind": "norm", "rows": 4096, "width": 4096, "type": "bf16", "post": True,
         "gate": "token", "scale": 0.5, "offset": 0.0},
        # The chosen token's log probability and twenty alternatives, one sequence.
        {"name": "logprobs_t1_bf16", "kind": "logprobs", "rows": 1, "vocab": 32000, "given": 1, "top": 20, "type": "bf16",
         "temperature": 1.0, "masked": 0.0},
        # A batch of sequences over a large vocabulary, half of it masked by a grammar.
        {"name": "logprobs_t16_f32", "kind": "logprobs", "rows": 16, "vocab": 131072, "given": 3, "top": 8,
         "type": "f32", "temperature": 0.7, "masked": 0.5},
        # A prompt's tokens scored under a vocabulary of odd size.
        {"name": "logprobs_t2048_bf16", "kind": "logprobs", "rows": 2048, "vocab": 32003, "given": 1, "top": 5,
         "type": "bf16", "temperature": 1.0, "masked": 0.0},
    ]


def _log(rng, lo: int, hi: int) -> int:
    """An integer of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng) -> dict:
    kind = rng.choice(["w4", "moe", "norm", "logprobs"])
    kind_type = rng.choice(list(TYPES))
    if kind == "w4":
        group, glu = rng.choice([32, 64, 128]), rng.choice(GLUS)
        k = group * _log(rng, 256 // group, 16384 // group)
        most = 32003 * 4096 // (k * (1 if glu == "none" else 2))
        return {"kind": kind, "rows": rng.randint(1, 16), "k": k, "n": _log(rng, 100, min(most, 40000)), "group": group,
                "type": kind_type, "scales": rng.choice(["bf16", "f16"]), "zeros": rng.random() < 0.5, "glu": glu}
    if kind == "moe":
        group = rng.choice([32, 64, 128])
        experts = _log(rng, 4, 256)
        used = rng.randint(1, min(8, experts))
        hidden = group * _log(rng, 512 // group, 4096 // group)
        inter = group * _log(rng, 128 // group, 1536 // group)
        experts = max(used, min(experts, 128 * 2048 * 768 // (hidden * inter)))
        return {"kind": kind, "tokens": rng.randint(1, 16), "experts": experts, "used": used, "hidden": hidden,
                "inter": inter, "group": group, "type": kind_type, "scales": rng.choice(["bf16", "f16"]),
                "zeros": rng.random() < 0.5, "router": rng.choice(["f32", kind_type]),
                "score": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.5,
                "renormalize": rng.random() < 0.7, "scale": rng.choice([1.0, 2.5]), "glu": rng.choice(GLUS[1:])}
    if kind == "norm":
        width = _log(rng, 128, 16384)
        return {"kind": kind, "rows": _log(rng, 1, min(8192, 4096 * 4096 // width)), "width": width, "type": kind_type,
                "post": rng.random() < 0.7, "gate": rng.choice(["none", "channel", "token"]),
                "scale": rng.choice([1.0, 0.25]), "offset": rng.choice([0.0, 1.0])}
    vocab = _log(rng, 1000, 262144)
    return {"kind": kind, "rows": _log(rng, 1, min(2048, 2048 * 32003 * 2 // (vocab * SIZES[kind_type]))), "vocab": vocab,
            "given": rng.randint(0, 4), "top": rng.randint(0, 20), "type": kind_type,
            "temperature": rng.choice([1.0, 0.7, 1.5]), "masked": rng.choice([0.0, 0.0, 0.5])}


# ------------------------------------------------------------------ inputs
def _rng(case: dict, seed: int):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _hidden(g, rows: int, k: int, dtype) -> torch.Tensor:
    x = torch.randn((rows, k), generator=g, device="cuda")
    loud = torch.rand((k,), generator=g, device="cuda") < 0.005
    return torch.where(loud, x * 8.0, x).to(dtype)


def _w4(g, lead: tuple, n: int, k: int, group: int, scales: str, zeros: bool):
    """Raw 4-bit weights: codes (value 2 i in byte i's low nibble), scales and zero points."""
    codes = torch.randint(0, 256, lead + (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    groups = k // group
    s = torch.rand(lead + (n, groups), generator=g, device="cuda") + 0.5
    s = (s / (4.6 * k ** 0.5)).to(TYPES[scales])
    z = None
    if zeros:       # around the middle of the range
        lo = torch.randint(5, 11, lead + (n, (groups + 1) // 2), generator=g, device="cuda", dtype=torch.uint8)
        hi = torch.randint(5, 11, lead + (n, (groups + 1) // 2), generator=g, device="cuda", dtype=torch.uint8)
        z = lo | (hi << 4)
    return codes, s, z


def _inputs(case: dict, seed: int) -> dict:
    g = _rng(case, seed)
    t = {"case": case}
    dtype = TYPES[case["type"]]
    if case["kind"] == "w4":
        t["x"] = _hidden(g, case["rows"], case["k"], dtype)
        rows = case["n"] if case["glu"] == "none" else 2 * case["n"]      # gate rows, then up rows
        t["w"] = _w4(g, (), rows, case["k"], case["group"], case["scales"], case["zeros"])
    elif case["kind"] == "moe":
        e, h, i = case["experts"], case["hidden"], case["inter"]
        t["x"] = _hidden(g, case["tokens"], h, dtype)
        router = torch.randn((e, h), generator=g, device="cuda") * (1.5 * h ** -0.5)
        t["router"] = router.to(TYPES[case["router"]])
        t["bias"] = torch.randn((e,), generator=g, device="cuda") * 0.1 if case["bias"] else None
        t["gate_up"] = _w4(g, (e,), 2 * i, h, case["group"], case["scales"], case["zeros"])
        t["down"] = _w4(g, (e,), h, i, case["group"], case["scales"], case["zeros"])
    elif case["kind"] == "norm":
        rows, width = case["rows"], case["width"]
        t["block"] = _hidden(g, rows, width, dtype)
        t["residual"] = (_hidden(g, rows, width, torch.float32) * 3.0).to(dtype)

        def weight():
            return torch.rand((width,), generator=g, device="cuda") + (0.5 - case["offset"])
        t["post"] = weight().to(dtype) if case["post"] else None
        t["pre"] = weight().to(dtype)
        shape = {"none": None, "channel": (width,), "token": (rows, width)}[case["gate"]]
        t["gate"] = None if shape is None else torch.rand(shape, generator=g, device="cuda").to(dtype)
    else:
        rows, vocab = case["rows"], case["vocab"]
        logits = torch.randn((rows, vocab), generator=g, device="cuda") * 2.5
        peaks = torch.randint(0, vocab, (rows, 8), generator=g, device="cuda")
        logits.scatter_add_(1, peaks, torch.rand((rows, 8), generator=g, device="cuda") * 12.0)
        t["tokens"] = torch.cat([peaks, torch.randint(0, vocab, (rows, 8), generator=g, device="cuda")], 1)[
            :, torch.randperm(16, generator=g, device="cuda")[:case["given"]]].to(torch.int32).contiguous()
        if case["masked"]:
            mask = torch.rand((rows, vocab), generator=g, device="cuda") < case["masked"]
            logits.masked_fill_(mask, float("-inf"))
        t["logits"] = logits.to(dtype)
    return t


def prepare(case: dict, seed: int) -> dict:
    t = _inputs(case, seed)
    if own:
        import llmp_b200 as ops
        if case["kind"] == "w4":     # the weights as a program lays them out once at load time
            t["matrix"] = ops.w4_relayout(*t["w"], glu=case["glu"] != "none")
        elif case["kind"] == "moe":
            t["gate_up_matrix"] = ops.w4_relayout(*t["gate_up"], glu=True)
            t["down_matrix"] = ops.w4_relayout(*t["down"])
    return t


# ------------------------------------------------------------------ one pass
def run(t: dict):
    case = t["case"]
    if not own:
        return {"w4": _plain_w4, "moe": _plain_moe, "norm": _plain_norm, "logprobs": _plain_logprobs}[case["kind"]](t)
    import llmp_b200 as ops
    glus = {"none": ops.GLU_NONE, "swiglu": ops.GLU_SWIGLU, "swiglu_clamp": ops.GLU_SWIGLU_CLAMP, "geglu": ops.GLU_GEGLU}
    if case["kind"] == "w4":
        return ops.w4_vector(t["matrix"], t["x"], glu=glus[case["glu"]], limit=_limit(case))
    if case["kind"] == "moe":
        return ops.moe_layer(t["x"], t["router"], t["gate_up_matrix"], t["down_matrix"], case["used"], bias=t["bias"],
                             score=ops.SCORE_SIGMOID if case["score"] == "sigmoid" else ops.SCORE_SOFTMAX,
                             renormalize=case["renormalize"], scale=case["scale"], glu=glus[case["glu"]],
                             limit=_limit(case))
    if case["kind"] == "norm":
        return ops.block_norm(t["block"], t["residual"], pre=t["pre"], post=t["post"], gate=t["gate"],
                              scale=case["scale"], offset=case["offset"], eps=1e-6)
    return ops.logprobs(t["logits"], t["tokens"], top=case["top"], temperature=case["temperature"])


def _limit(case: dict) -> float:
    return 1.5 if case["glu"] == "swiglu_clamp" else 0.0


def _glu(name: str, gate: torch.Tensor, up: torch.Tensor, limit: float) -> torch.Tensor:
    if name == "geglu":
        return 0.5 * gate * (1.0 + torch.tanh(0.7978845608028654 * gate * (1.0 + 0.044715 * gate * gate))) * up
    if name == "swiglu_clamp":
        gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
    return gate / (1.0 + torch.exp(-gate)) * up


def _values(codes: torch.Tensor, scales: torch.Tensor, zeros, dtype) -> torch.Tensor:
    """[..., n, k] of scale * (code - zero point)."""
    groups = scales.shape[-1]
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (groups, -1)).to(dtype)
    if zeros is None:
        q = q - 8.0
    else:
        q = q - torch.stack([zeros & 15, zeros >> 4], -1).flatten(-2)[..., :groups, None].to(dtype)
    return (q * scales[..., None].to(dtype)).flatten(-2)


def _plain_w4(t: dict) -> torch.Tensor:
    case, x = t["case"], t["x"]
    y = x.float() @ _values(*t["w"], torch.float32).T
    if case["glu"] != "none":
        y = _glu(case["glu"], y[:, :case["n"]], y[:, case["n"]:], _limit(case))
    return y.to(x.dtype)


def _choose(case: dict, logits: torch.Tensor, bias):
    """The experts of a token, best first (ties to the lowest index), and their weights."""
    p = torch.softmax(logits, -1) if case["score"] == "softmax" else torch.sigmoid(logits)
    by = logits if bias is None else p + bias.to(p.dtype)
    ids = torch.sort(by, dim=-1, descending=True, stable=True).indices[:, :case["used"]]
    weights = torch.gather(p, 1, ids)
    if case["renormalize"]:
        weights = weights / weights.sum(-1, keepdim=True)
    return ids, weights * case["scale"]


def _plain_moe(t: dict):
    case, x = t["case"], t["x"]
    # 64 bits: the choice of an expert is a comparison of values that may lie next to each other
    ids, weights = _choose(case, x.double() @ t["router"].double().T, t["bias"])
    weights = weights.float()
    y = torch.zeros((case["tokens"], case["hidden"]), device=x.device)
    for j in range(case["used"]):           # a slot of every token at a time
        def named(w):
            return _values(w[0][ids[:, j]], w[1][ids[:, j]], None if w[2] is None else w[2][ids[:, j]], torch.float32)
        gate_up = torch.matmul(named(t["gate_up"]), x.float()[:, :, None])[..., 0]
        h = _glu(case["glu"], gate_up[:, :case["inter"]], gate_up[:, case["inter"]:], _limit(case))
        y = y + torch.matmul(named(t["down"]), h[:, :, None])[..., 0] * weights[:, j:j + 1]
    return y.to(x.dtype), ids.int(), weights


def _plain_norm(t: dict):
    case, dtype = t["case"], t["block"].dtype
    u = t["block"].float()
    if t["post"] is not None:
        u = u * torch.rsqrt((u * u).mean(-1, keepdim=True) + 1e-6) * (t["post"].float() + case["offset"])
    if t["gate"] is not None:
        u = u * t["gate"].float()
    r = t["residual"].float() + case["scale"] * u
    h = r * torch.rsqrt((r * r).mean(-1, keepdim=True) + 1e-6) * (t["pre"].float() + case["offset"])
    return r.to(dtype), h.to(dtype)


def _plain_logprobs(t: dict):
    case = t["case"]
    x = t["logits"].float()
    ids = t["tokens"].long()
    given = torch.gather(x, 1, ids)
    ranks = torch.stack([(x > given[:, j:j + 1]).sum(-1) for j in range(case["given"])], 1) + 1 \
        if case["given"] else ids
    top_values, top_ids = torch.sort(x, dim=-1, descending=True, stable=True)
    top_values, top_ids = top_values[:, :case["top"]], top_ids[:, :case["top"]]
    m = x.max(-1, keepdim=True).values
    d = (x - m) / case["temperature"]
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    entropy = torch.log(total) - torch.where(e > 0, d * e, 0.0).sum(-1, keepdim=True) / total

    def lp(v):
        return (v - m) / case["temperature"] - torch.log(total)
    return lp(given), ranks.int(), entropy[:, 0], top_ids.int(), lp(top_values)


# ------------------------------------------------------------------ what a pass needs, what it returns
def _w4_bytes(n: int, k: int, group: int, zeros: bool) -> float:
    return n * k * (0.5 + (2.0 + (0.5 if zeros else 0.0)) / group)


def work(case: dict) -> dict:
    size = SIZES[case["type"]]
    if case["kind"] == "w4":
        rows = case["n"] * (1 if case["glu"] == "none" else 2)
        return {"bytes": _w4_bytes(rows, case["k"], case["group"], case["zeros"])
                + case["rows"] * (case["k"] + case["n"]) * size,
                "flops": 2.0 * case["rows"] * rows * case["k"]}
    if case["kind"] == "moe":
        e, u, t, h, i = (case[n] for n in ("experts", "used", "tokens", "hidden", "inter"))
        named = e * (1.0 - (1.0 - u / e) ** t)      # the experts that someone names, for tokens that choose evenly
        expert = _w4_bytes(2 * i, h, case["group"], case["zeros"]) + _w4_bytes(h, i, case["group"], case["zeros"])
        return {"bytes": named * expert + e * h * SIZES[case["router"]] + 2 * t * h * size + t * u * 8,
                "flops": 2.0 * t * (e * h + u * 3 * h * i)}
    if case["kind"] == "norm":
        n = case["rows"] * case["width"]
        gates = {"none": 0, "channel": case["width"], "token": n}[case["gate"]]
        return {"bytes": (4 * n + gates + (2 if case["post"] else 1) * case["width"]) * size, "flops": 12.0 * n}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * size + case["rows"] * (12 * case["given"] + 8 * case["top"] + 4),
            "flops": n * (6.0 + case["given"])}


def exact(case: dict, seed: int):
    t = _inputs(case, seed)
    if case["kind"] == "w4":
        return _exact_rows(case, t["x"], t["w"], case["n"])
    if case["kind"] == "moe":
        return _exact_moe(case, t)
    if case["kind"] == "norm":
        return _exact_norm(case, t)
    return _exact_logprobs(case, t)


def _exact_matrix(codes, scales, zeros, group: int) -> torch.Tensor:
    n, half = codes.shape
    w = torch.empty((n, 2 * half), dtype=torch.float64, device=codes.device)
    w[:, 0::2] = torch.remainder(codes, 16).double()
    w[:, 1::2] = torch.div(codes, 16, rounding_mode="floor").double()
    for i in range(2 * half // group):
        z = 8.0
        if zeros is not None:
            pair = zeros[:, i // 2]
            z = (torch.div(pair, 16, rounding_mode="floor") if i % 2 else torch.remainder(pair, 16)).double()[:, None]
        part = w[:, i * group:(i + 1) * group]
        part -= z
        part *= scales[:, i].double()[:, None]
    return w


def _exact_glu(name: str, a: torch.Tensor, b: torch.Tensor, limit: float) -> torch.Tensor:
    if name == "geglu":
        inner = (2.0 / torch.pi) ** 0.5 * (a + 0.044715 * a ** 3)
        return a * b * (1.0 + torch.tanh(inner)) / 2.0
    if name == "swiglu_clamp":
        a = torch.where(a > limit, torch.full_like(a, limit), a)
        b = torch.where(b > limit, torch.full_like(b, limit), torch.where(b < -limit, torch.full_like(b, -limit), b))
    return a * b * torch.sigmoid(a)


def _exact_rows(case: dict, x, w, n: int) -> torch.Tensor:
    y = torch.einsum("tk,nk->tn", x.double(), _exact_matrix(*w, case["group"]))
    return y if case["glu"] == "none" else _exact_glu(case["glu"], y[:, :n], y[:, n:], _limit(case))


def _exact_moe(case: dict, t: dict):
    x = t["x"].double()
    ids, weights, out = [], [], []
    for row in x:
        logits = (t["router"].double() * row).sum(1)
        p = 1.0 / (1.0 + torch.exp(-logits))
        if case["score"] == "softmax":
            p = torch.exp(logits - logits.max())
            p = p / p.sum()
        by = logits.clone() if t["bias"] is None else p + t["bias"].double()
        chosen = []
        for _ in range(case["used"]):
            best = int((by == by.max()).nonzero()[0, 0])
            chosen.append(best)
            by[best] = float("-inf")
        w = p[chosen]
        w = (w / w.sum() if case["renormalize"] else w) * case["scale"]
        y = torch.zeros_like(row)
        for e, share in zip(chosen, w):
            def expert(m):
                return _exact_matrix(m[0][e], m[1][e], None if m[2] is None else m[2][e], case["group"])
            both = expert(t["gate_up"]) @ row
            h = _exact_glu(case["glu"], both[:case["inter"]], both[case["inter"]:], _limit(case))
            y = y + share * (expert(t["down"]) @ h)
        ids.append(chosen)
        weights.append(w)
        out.append(y)
    return torch.stack(out), torch.tensor(ids, dtype=torch.int32, device=x.device), torch.stack(weights)


def _exact_norm(case: dict, t: dict):
    def rms(v, weight):
        return v / (v.square().sum(-1, keepdim=True) / v.shape[-1] + 1e-6).sqrt() * (weight.double() + case["offset"])
    u = t["block"].double()
    u = u if t["post"] is None else rms(u, t["post"])
    u = u if t["gate"] is None else u * t["gate"].double()
    r = t["residual"].double() + u * case["scale"]
    return r, rms(r, t["pre"])


def _exact_logprobs(case: dict, t: dict):
    x = t["logits"].double()
    lp = torch.log_softmax(x / case["temperature"], -1)
    entropy = -(torch.where(torch.isinf(lp), 0.0, lp) * lp.exp()).sum(-1)
    ids = t["tokens"].long()
    given = torch.gather(lp, 1, ids)
    ranks = 1 + (x[:, None, :] > torch.gather(x, 1, ids)[:, :, None]).sum(-1) if case["rows"] <= 64 else \
        1 + torch.stack([(row[None] > row[i][:, None]).sum(-1) for row, i in zip(x, ids)])
    order = torch.argsort(x, dim=-1, descending=True, stable=True)[:, :case["top"]]
    return given, ranks.int(), entropy, order.int(), torch.gather(lp, 1, order)

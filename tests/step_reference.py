"""The decode step's operators in 64 bits by plain torch, with bounds on what F32 may add to each
result: `slack` arrays are sums of magnitudes times unit roundings, worked out below."""
import torch

U = 2.0 ** -24                                     # half a step of F32
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
GLUS = {"none": 0, "swiglu": 1, "swiglu_clamp": 2, "geglu": 3}


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def assert_within(got, want, slack, what=""):
    """|got - want| <= slack + the rounding of `want` (and what slack adds to it) to got's type; a value
    below the type's normal range rounds in steps of its own."""
    got64 = got.double()
    rounding = half_step(got.dtype) * (want.abs() + slack) + torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    assert got.shape == want.shape, (what, got.shape, want.shape)
    err, most = (got64 - want).abs(), slack + rounding
    same = (got64 == want) | (got64.isnan() & want.isnan())
    ok = same | (err <= most)
    assert bool(ok.all()), (what, int((~ok).sum()), float((err / most)[~ok].max()))


def w4_source(g, lead, n, k, group, scales, zeros, device="cuda"):
    codes = torch.randint(0, 256, lead + (n, k // 2), generator=g, dtype=torch.uint8).to(device)
    s = ((torch.rand(lead + (n, k // group), generator=g) + 0.25) * k ** -0.5 / 4).to(TYPES[scales]).to(device)
    s = torch.where(torch.rand(s.shape, generator=g).to(device) < 0.1, -s, s)
    z = torch.randint(0, 256, lead + (n, (k // group + 1) // 2), generator=g, dtype=torch.uint8).to(device) if zeros else None
    return codes, s, z


def w4_values(codes, scales, zeros):
    groups = scales.shape[-1]
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (groups, -1)).double()
    z = 8.0 if zeros is None else torch.stack([zeros & 15, zeros >> 4], -1).flatten(-2)[..., :groups, None].double()
    return ((q - z) * scales[..., None].double()).flatten(-2)


def w4_rows(x, values, group):
    """x values^T and a bound on F32's share of the error.  Products of codes and pieces of x are exact; a
    group's sum is a chain of group / 16 MMAs, each adding 16 products to the sum with at most a
    unit of 2^-23 of the magnitudes lost an addition; then k / group multiply-adds, up to 32 partial
    sums of the split over warps and CTAs, and the three pieces' sums."""
    y = x.double() @ values.T
    magnitude = x.double().abs() @ values.abs().T
    additions = group + values.shape[-1] / group + 32 + 3
    return y, magnitude * additions * 2 * U


def glu(name, gate, up, limit):
    """The GLU, and how far its result moves for one unit of error in gate and in up (both activations'
    derivatives lie within 1.13)."""
    if name == "geglu":
        act = 0.5 * gate * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (gate + 0.044715 * gate ** 3)))
    else:
        if name == "swiglu_clamp":
            gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
        act = gate * torch.sigmoid(gate)
    return act * up, 1.13 * up.abs(), act.abs()


def glu_rows(name, gate, gate_slack, up, up_slack, limit):
    """... of F32 sums; the activation itself: expf or tanhf (2 and 4 units), a division or a polynomial, products; tanh near
    -1 loses what 1 + tanh cancels, at most a unit of |gate| / 2."""
    h, by_gate, by_up = glu(name, gate, up, limit)
    g = gate.clamp(max=limit) if name == "swiglu_clamp" else gate
    return h, by_gate * gate_slack + by_up * up_slack + 1.13 * gate_slack * up_slack + 24 * U * h.abs() + \
        8 * U * (g * up).abs()


def choose(logits, used, score, bias, renormalize, scale):
    p = torch.softmax(logits, -1) if score == "softmax" else torch.sigmoid(logits)
    by = logits if bias is None else p + bias.double()
    by = torch.where(by.isnan(), -torch.inf, by)
    ids = torch.sort(by, dim=-1, descending=True, stable=True).indices[:, :used]
    w = torch.gather(p, 1, ids)
    return ids, (w / w.sum(-1, keepdim=True) if renormalize else w) * scale


def moe(x, router, bias, gate_up, down, used, score, renormalize, scale, glu_name, limit, group_up, group_down):
    """(y, its slack, ids, weights, their slack)."""
    logits = x.double() @ router.double().T
    # up to 128 values' products are added in F32 for each pair of pieces, these sums in 64 bits
    logit_slack = (x.double().abs() @ router.double().abs().T).amax() * 130 * 2 * U
    ids, weights = choose(logits, used, score, bias, renormalize, scale)
    # p moves by exp of twice the logits' error, expf and the sums' roundings; renormalizing doubles that
    weight_slack = weights.abs() * (4 * logit_slack + 2 * (router.shape[0] / 32 + 24) * U)
    inter = down[0].shape[-1] * 2
    y, slack = torch.zeros_like(x, dtype=torch.float64), torch.zeros_like(x, dtype=torch.float64)
    pieces = 24 if x.dtype == torch.float32 else 16
    for t in range(x.shape[0]):
        for j in range(used):
            e = int(ids[t, j])
            both, both_slack = w4_rows(x[t:t + 1], w4_values(*(None if a is None else a[e] for a in gate_up)), group_up)
            h, h_slack = glu_rows(glu_name, both[:, :inter], both_slack[:, :inter], both[:, inter:], both_slack[:, inter:], limit)
            h_slack = h_slack + h.abs() * 2.0 ** (1 - pieces)     # pieces are truncations
            values = w4_values(*(None if a is None else a[e] for a in down))
            z, z_slack = w4_rows(h, values, group_down)
            z_slack = z_slack + h_slack @ values.abs().T
            w = weights[t, j].abs()
            y[t] += weights[t, j] * z[0]
            slack[t] += w * z_slack[0] + weight_slack[t, j] * z[0].abs() + (used + 2) * U * w * z[0].abs()
    return y, slack, ids, weights, weight_slack


def norm(block, residual, gate, post, pre, scale, offset, eps):
    """(r, slack, h or None, slack).  Sums of squares: 32 values a thread, then 10 levels of a tree, half of
    whose relative error reaches the inverse root."""
    def rms(v, v_slack, weight):
        inverse = 1 / ((v * v).mean(-1, keepdim=True) + eps).sqrt()
        w = weight.double() + offset
        lost = (v.abs() * v_slack).mean(-1, keepdim=True) * inverse ** 2     # of the inverse, relative
        out = v * inverse * w
        return out, out.abs() * (lost + 30 * U) + v_slack * inverse * w.abs() + (v * inverse).abs() * U * w.abs() * 2 + \
            (v * inverse).abs() * U * (weight.double().abs() + abs(offset))
    u = block.double()
    slack = torch.zeros_like(u)
    if post is not None:
        u, slack = rms(u, slack, post)
    factor = scale * (1.0 if gate is None else gate.double())
    r = u * factor
    slack = slack * abs(factor) + r.abs() * 3 * U
    if residual is not None:
        r = r + residual.double()
        slack = slack + r.abs() * U
    h = rms(r, slack, pre) if pre is not None else (None, None)
    return r, slack, h[0], h[1]


def logprobs(logits, tokens, top, temperature):
    """(log p, ranks, entropy, top ids, top log p, all log p)."""
    x = logits.double()
    bad = (x.isnan() | (x == torch.inf)).any(-1)
    nothing = (x == -torch.inf).all(-1)
    lp = torch.log_softmax(x / temperature, -1)
    lp = torch.where(bad[:, None], torch.nan, torch.where(nothing[:, None], -torch.inf, lp))
    entropy = -(torch.where(lp == -torch.inf, 0.0, lp) * lp.exp()).sum(-1)
    inside = (tokens >= 0) & (tokens < x.shape[1])
    ids = torch.where(inside, tokens, 0).long()
    given = torch.where(inside, torch.gather(lp, 1, ids), torch.nan)
    own = torch.gather(x, 1, ids)
    ranks = torch.stack([(x > own[:, j:j + 1]).sum(-1) + 1 for j in range(ids.shape[1])], 1) if ids.shape[1] else ids
    order_by = torch.where(x.isnan(), -torch.inf, x)
    # NaN below -inf: a stable sort by value, NaN last among its equals
    last = torch.sort(x.isnan().int(), dim=-1, stable=True).indices
    order = torch.gather(last, 1, torch.sort(torch.gather(order_by, 1, last), dim=-1, descending=True, stable=True).indices)[:, :top]
    return given, torch.where(inside, ranks, 0), entropy, order, torch.gather(lp, 1, order), lp

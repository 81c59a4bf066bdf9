"""The whole mixture-of-experts layer against 64 bits: choice, weights and result."""
import pytest

import step_reference as ref

pytestmark = pytest.mark.gpu


def _case(torch, seed, tokens, experts, hidden, inter, group_up=64, group_down=32, kind="bf16", router="f32", zeros=True,
          scales="bf16", bias=False):
    g = torch.Generator().manual_seed(seed)
    c = {"x": torch.randn((tokens, hidden), generator=g).to(ref.TYPES[kind]).cuda(),
         "router": (torch.randn((experts, hidden), generator=g) * 1.5 * hidden ** -0.5).to(ref.TYPES[router]).cuda(),
         "bias": (torch.randn((experts,), generator=g) * 0.2).cuda() if bias else None,
         "gate_up": ref.w4_source(g, (experts,), 2 * inter, hidden, group_up, scales, zeros),
         "down": ref.w4_source(g, (experts,), hidden, inter, group_down, scales, zeros),
         "groups": (group_up, group_down)}
    return c


def _check(torch, ops, c, used, score="softmax", renormalize=True, scale=1.0, glu="swiglu", limit=0.0):
    gate_up, down = ops.w4_relayout(*c["gate_up"], glu=True), ops.w4_relayout(*c["down"])
    got = ops.moe_layer(c["x"], c["router"], gate_up, down, used, bias=c["bias"],
                        score=ops.SCORE_SIGMOID if score == "sigmoid" else ops.SCORE_SOFTMAX, renormalize=renormalize,
                        scale=scale, glu=ref.GLUS[glu], limit=limit)
    y, slack, ids, weights, weight_slack = ref.moe(c["x"], c["router"], c["bias"], c["gate_up"], c["down"], used, score,
                                                   renormalize, scale, glu, limit, *c["groups"])
    assert torch.equal(got[1].long(), ids)
    ref.assert_within(got[2], weights, weight_slack, "weights")
    ref.assert_within(got[0], y, slack, "output")
    return (gate_up, down), got


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tokens", [1, 2, 5, 9, 16])
def test_types_and_tokens(cuda, kind, tokens):
    import llmp_b200 as ops
    c = _case(cuda, tokens, tokens, 24, 512, 192, kind=kind)
    _check(cuda, ops, c, 4)


@pytest.mark.parametrize("experts,used", [(1, 1), (3, 3), (16, 1), (17, 5), (60, 16), (130, 8), (512, 10)])
def test_experts(cuda, experts, used):
    import llmp_b200 as ops
    c = _case(cuda, experts, 6, experts, 256, 64)
    _check(cuda, ops, c, used)


@pytest.mark.parametrize("hidden,inter,group_up,group_down", [(32, 32, 32, 32), (160, 96, 32, 32), (1088, 416, 64, 32),
                                                             (2176, 128, 128, 128), (4096, 320, 128, 64)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_sizes(cuda, hidden, inter, group_up, group_down, kind):
    import llmp_b200 as ops
    c = _case(cuda, hidden, 7, 9, hidden, inter, group_up, group_down, kind=kind, scales="f16")
    _check(cuda, ops, c, 3)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("router", ["f32", "bf16", "f16"])
def test_choices(cuda, score, bias, renormalize, router):
    import llmp_b200 as ops
    c = _case(cuda, 5, 8, 40, 384, 128, group_up=128, kind="f32", router=router, bias=bias, zeros=False)
    _check(cuda, ops, c, 6, score, renormalize, 2.5, "geglu")


@pytest.mark.parametrize("glu", ["swiglu", "swiglu_clamp", "geglu"])
def test_glus(cuda, glu):
    import llmp_b200 as ops
    c = _case(cuda, 6, 3, 8, 256, 96, kind="f16")
    c["x"] = c["x"] * 3
    _check(cuda, ops, c, 2, glu=glu, limit=0.5 if glu == "swiglu_clamp" else 0.0)


def test_more_tokens_than_are_staged_at_once(cuda):
    """F32 rows of 8192 take shared memory two tokens at a time; all name the same experts."""
    import llmp_b200 as ops
    c = _case(cuda, 7, 11, 4, 8192, 64, 128, 64, kind="f32")
    _check(cuda, ops, c, 3)
    c = _case(cuda, 8, 16, 2, 16384, 32, 128, 32, kind="bf16")
    _check(cuda, ops, c, 2)


def test_the_largest_shapes_that_are_taken(cuda):
    """One F32 token of 16384 values a pass, 512 experts, groups of 32: all of a CTA's shared memory."""
    import llmp_b200 as ops
    c = _case(cuda, 14, 16, 512, 16384, 32, 32, 32, kind="f32")
    _check(cuda, ops, c, 2)


def test_ties_go_to_the_lowest_index(cuda):
    torch = cuda
    import llmp_b200 as ops
    c = _case(torch, 9, 4, 70, 256, 64)
    c["router"] = c["router"][:1].expand(70, 256).contiguous()
    _, got = _check(torch, ops, c, 5)
    assert torch.equal(got[1], torch.arange(5, device="cuda", dtype=torch.int32).expand(4, 5))
    c["router"] = torch.zeros_like(c["router"])
    c["router"][1::2] = -0.0
    _check(torch, ops, c, 5)


def test_values_that_are_not_finite(cuda):
    torch = cuda
    import llmp_b200 as ops
    c = _case(torch, 10, 4, 12, 256, 64, kind="f32")
    (gate_up, down), want = _check(torch, ops, c, 3)
    x = c["x"].clone()
    x[1, 5], x[2, 9] = float("nan"), float("inf")
    y, ids, weights = ops.moe_layer(x, c["router"], gate_up, down, 3)
    assert torch.equal(y[0], want[0][0]) and torch.equal(y[3], want[0][3])       # the other tokens' results stand
    assert bool(y[1].isnan().all() and weights[1].isnan().all() and y[2].isnan().any())
    assert bool((ids >= 0).all() and (ids < 12).all())
    assert ids[1].tolist() == [0, 1, 2]
    router = c["router"].clone()
    router[4] = float("nan")                                                  # an expert without a logit comes last
    y, ids, _ = ops.moe_layer(c["x"], router, gate_up, down, 12, score=ops.SCORE_SIGMOID)
    assert bool((ids[:, -1] == 4).all())


def test_a_token_does_not_depend_on_its_company(cuda):
    torch = cuda
    import llmp_b200 as ops
    c = _case(torch, 11, 16, 32, 512, 128)
    (gate_up, down), (y, ids, weights) = _check(torch, ops, c, 4)
    for t in (0, 7, 15):
        one = ops.moe_layer(c["x"][t:t + 1], c["router"], gate_up, down, 4)
        assert torch.equal(one[0][0], y[t]) and torch.equal(one[1][0], ids[t]) and torch.equal(one[2][0], weights[t])


def test_strides_outputs_and_no_tokens(cuda):
    torch = cuda
    import llmp_b200 as ops
    c = _case(torch, 12, 5, 10, 320, 96, kind="f32")
    (gate_up, down), (y, ids, _) = _check(torch, ops, c, 2)
    wide = torch.zeros((5, 331), device="cuda")
    wide[:, 3:323] = c["x"]
    router = torch.zeros((10, 323), device="cuda")
    router[:, 1:321] = c["router"]
    out = torch.full((5, 330), 5.0, device="cuda")
    got = ops.moe_layer(wide[:, 3:323], router[:, 1:321], gate_up, down, 2, out=out[:, 2:322])
    assert torch.equal(out[:, 2:322], y) and torch.equal(got[1], ids)
    assert bool((out[:, :2] == 5).all() and (out[:, 322:] == 5).all())
    half = torch.empty((5, 320), dtype=torch.bfloat16, device="cuda")
    ops.moe_layer(c["x"], c["router"], gate_up, down, 2, out=half)
    assert torch.equal(half, y.bfloat16())
    empty = ops.moe_layer(c["x"][:0], c["router"], gate_up, down, 2)
    assert empty[0].shape == (0, 320) and empty[1].shape == (0, 2)


def test_two_streams_at_once_and_a_graph(cuda):
    torch = cuda
    import llmp_b200 as ops
    c = _case(torch, 13, 6, 20, 1024, 256)
    (gate_up, down), want = _check(torch, ops, c, 4)
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            results.append(ops.moe_layer(c["x"], c["router"], gate_up, down, 4))
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(r, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.moe_layer(c["x"], c["router"], gate_up, down, 4)
    c["x"].copy_(c["x"].flip(0))
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b.flip(0)) for a, b in zip(held, want))


@pytest.mark.parametrize("glu", ["swiglu", "swiglu_clamp", "geglu"])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_a_nan_of_an_expert_reaches_the_tokens_that_name_it(cuda, glu, kind):
    torch = cuda
    import llmp_b200 as ops
    c = _case(torch, 15, 9, 12, 256, 64, kind=kind)
    c["gate_up"][1][3, 7, 1] = float("nan")         # a scale of expert 3's gate row 7
    c["gate_up"][1][8, 64 + 20, 0] = float("nan")   # of expert 8's up row 20
    y, ids, weights = ops.moe_layer(c["x"], c["router"], ops.w4_relayout(*c["gate_up"], glu=True), ops.w4_relayout(*c["down"]), 3,
                                    glu=ref.GLUS[glu], limit=0.5 if glu == "swiglu_clamp" else 0.0)
    named = ((ids == 3) | (ids == 8)).any(-1)
    assert bool(named.any() and not named.all() and weights.isfinite().all())
    assert torch.equal(y.isnan(), named[:, None].expand_as(y))


@pytest.mark.parametrize("out", ["f16", "f32"])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tokens", [1, 7])
def test_how_wide_the_glu_rows_are(cuda, tokens, kind, out):
    """Down is the identity and one expert has all the weight, so the result is the GLU row: rounded to F16 from within
    2^-17 of it, and whole where activations or output are F32.  Each token has one value that is not zero, so gate and
    up are single products of 8 bits, 4 bits and the activation's 11: exact, and what is lost is the GLU's."""
    torch = cuda
    import llmp_b200 as ops
    size, group = 512, 64
    c = _case(torch, 16, tokens, 1, size, size, group, group, kind=kind)
    x = c["x"].to(torch.bfloat16 if kind == "bf16" else torch.float16).to(ref.TYPES[kind]) * 8
    c["x"] = torch.where(torch.arange(size, device="cuda") == (torch.arange(tokens, device="cuda") * 67 + 5)[:, None], x, 0.0)
    codes = torch.full((1, size, size // 2), 0x88, dtype=torch.uint8)      # the zero point: weights of nothing
    at = torch.arange(size)
    codes[0, at, at // 2] = torch.where(at % 2 == 0, 0x89, 0x98).to(torch.uint8)
    down = ops.w4_relayout(codes.cuda(), torch.ones((1, size, size // group), dtype=torch.float16).cuda())
    y = torch.empty((tokens, size), dtype=ref.TYPES[out], device="cuda")
    ops.moe_layer(c["x"], c["router"], ops.w4_relayout(*c["gate_up"], glu=True), down, 1, out=y)
    both = c["x"].double() @ ref.w4_values(*(a[0] for a in c["gate_up"])).T
    none = torch.zeros_like(both)
    h, h_slack = ref.glu_rows("swiglu", both[:, :size], none[:, :size], both[:, size:], none[:, size:], 0.0)
    lost = 2.0 ** -23 if "f32" in (kind, out) else 2.0 ** -17
    ref.assert_within(y, h, h_slack + h.abs() * lost)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("tokens,experts,used", [(1, 24, 4), (16, 24, 4), (16, 3, 2)])
def test_an_f32_output_of_16_bit_activations(cuda, kind, group, tokens, experts, used):
    """The same values' bounds in F32."""
    torch = cuda
    import llmp_b200 as ops
    c = _case(torch, 17, tokens, experts, 384, 256, 64, group, kind=kind)
    y = torch.empty((tokens, 384), device="cuda")
    ops.moe_layer(c["x"], c["router"], ops.w4_relayout(*c["gate_up"], glu=True), ops.w4_relayout(*c["down"]), used, out=y)
    want, slack, *_ = ref.moe(c["x"].float(), c["router"], None, c["gate_up"], c["down"], used, "softmax", True, 1.0, "swiglu",
                              0.0, 64, group)
    ref.assert_within(y, want, slack)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("router", ["f32", "bf16", "f16"])
def test_infinities_in_the_router_s_product(cuda, kind, router):
    """An infinite activation, or an infinite router value, makes a logit an infinity of its sign, no NaN."""
    torch = cuda
    import llmp_b200 as ops
    c = _case(torch, 18, 11, 16, 512, 64, kind=kind, router=router)
    gate_up, down = ops.w4_relayout(*c["gate_up"], glu=True), ops.w4_relayout(*c["down"])
    for change in ("x", "router"):
        x, weights = c["x"].clone(), c["router"].clone()
        if change == "x":
            x[3, 100], x[4, 7], x[10, 500] = float("inf"), -float("inf"), float("nan")
        else:
            weights[6, 33], weights[13, 400] = float("inf"), -float("inf")
        logits = x.double() @ weights.double().T
        assert bool(logits[:, 6].isinf().any())
        _, ids, got = ops.moe_layer(x, weights, gate_up, down, 16, score=ops.SCORE_SIGMOID, renormalize=False)
        finite = logits.isfinite().all(-1)
        want, w = ref.choose(torch.where(logits.isnan(), -torch.inf, logits), 16, "sigmoid", None, False, 1.0)
        plain = ~logits.isnan().any(-1)
        assert torch.equal(ids[plain].long(), want[plain])
        # (a logit's error, up to 130 unit roundings of its products' magnitudes, moves a sigmoid by a quarter of it)
        slack = (x.double().abs().nan_to_num(posinf=0.0) @ weights.double().abs().nan_to_num(posinf=0.0).T).amax() * 130 * ref.U + 8 * ref.U
        ref.assert_within(got[plain], w[plain], slack.expand_as(w)[plain])
        if change == "x":
            assert ids[10].tolist() == list(range(16)) and bool(got[10].isnan().all())
            assert finite.sum() == 8


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("router", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("experts,used,hidden,inter,out", [(32, 4, 512, 128, None), (3, 2, 512, 96, None), (32, 4, 512, 128, "f32"),
                                                          (2, 1, 8192, 64, None), (100, 6, 288, 160, "bf16")])
def test_company_of_every_type_and_size(cuda, kind, router, experts, used, hidden, inter, out):
    """A token's results are the same bits alone and among others: where tokens name the same experts and their groups are cut,
    where not all of a call's tokens are staged at once, for every type of activations, router and output."""
    torch = cuda
    import llmp_b200 as ops
    c = _case(torch, 19, 16, experts, hidden, inter, 32, 32, kind=kind, router=router)
    gate_up, down = ops.w4_relayout(*c["gate_up"], glu=True), ops.w4_relayout(*c["down"])
    out = ref.TYPES[out or kind]

    def layer(x):
        y = torch.empty(x.shape, dtype=out, device="cuda")
        return ops.moe_layer(x, c["router"], gate_up, down, used, out=y)
    y, ids, weights = layer(c["x"])
    for chosen in ([0], [15], [3, 9], [1, 2, 4, 8, 13], list(range(15, -1, -1))):
        some = layer(c["x"][chosen].contiguous())
        assert torch.equal(some[1], ids[chosen]) and torch.equal(some[2], weights[chosen])
        assert torch.equal(some[0], y[chosen])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("experts", [16, 40, 512])
def test_the_most_pairs(cuda, kind, experts):
    """Sixteen experts for each of sixteen tokens: all of the lists' 256 places, named by all tokens or by one."""
    import llmp_b200 as ops
    c = _case(cuda, 20, 16, experts, 128, 64, 64, 32, kind=kind)
    _check(cuda, ops, c, 16)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("hidden,inter", [(64, 65536), (32, 20000)])
def test_long_inter(cuda, kind, hidden, inter):
    import llmp_b200 as ops
    c = _case(cuda, 21, 3, 2, hidden, inter, 32, 32, kind=kind)
    _check(cuda, ops, c, 1)

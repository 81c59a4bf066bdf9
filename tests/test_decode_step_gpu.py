"""A decode step of a routed model with 4-bit weights by the framework's calls, one after the other:
norms between the blocks, projections, the mixture-of-experts layer, the head, log probabilities;
queued as they come, on another stream, captured and replayed; and the norm's Q8_1 rows through
a Q4_K product."""
import numpy as np
import pytest

import step_reference as ref

pytestmark = pytest.mark.gpu

HIDDEN, INTER, EXPERTS, USED, VOCAB, LAYERS = 512, 192, 12, 3, 1003, 3


def _model(torch, kind):
    g = torch.Generator().manual_seed(21)

    def weight(width):
        return (torch.rand((width,), generator=g) + 0.5).to(ref.TYPES[kind]).cuda()
    layers = [{"post": weight(HIDDEN), "pre": weight(HIDDEN), "post_moe": weight(HIDDEN), "pre_next": weight(HIDDEN),
               "proj": ref.w4_source(g, (), HIDDEN, HIDDEN, 64, "bf16", True),
               "router": (torch.randn((EXPERTS, HIDDEN), generator=g) * 0.1).cuda(),
               "gate_up": ref.w4_source(g, (EXPERTS,), 2 * INTER, HIDDEN, 128, "bf16", False),
               "down": ref.w4_source(g, (EXPERTS,), HIDDEN, INTER, 32, "f16", True)} for _ in range(LAYERS)]
    return {"layers": layers, "first": weight(HIDDEN), "head": ref.w4_source(g, (), VOCAB, HIDDEN, 64, "bf16", True)}


def _step(ops, m, x, tokens):
    r, h = ops.block_norm(x, pre=m["first"])
    for layer in m["layers"]:
        y = ops.w4_vector(layer["proj"], h)
        r, h = ops.block_norm(y, r, post=layer["post"], pre=layer["pre"], scale=0.5)
        y, _, _ = ops.moe_layer(h, layer["router"], layer["gate_up"], layer["down"], USED)
        r, h = ops.block_norm(y, r, post=layer["post_moe"], pre=layer["pre_next"], scale=0.5)
    logits = ops.w4_vector(m["head"], h, out=x.new_empty((x.shape[0], VOCAB), dtype=__import__("torch").float32))
    return logits, ops.logprobs(logits, tokens, top=4, temperature=0.9)


def _loaded(ops, m):
    return {"first": m["first"], "head": ops.w4_relayout(*m["head"]),
            "layers": [{**layer, "proj": ops.w4_relayout(*layer["proj"]), "gate_up": ops.w4_relayout(*layer["gate_up"], glu=True),
                        "down": ops.w4_relayout(*layer["down"])} for layer in m["layers"]]}


def _step64(torch, m, x):
    def rms(v, w):
        return v / ((v * v).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    r = x.double()
    h = rms(r, m["first"])
    for layer in m["layers"]:
        y = h @ ref.w4_values(*layer["proj"]).T
        r = r + 0.5 * rms(y, layer["post"])
        h = rms(r, layer["pre"])
        ids, weights = ref.choose(h @ layer["router"].double().T, USED, "softmax", None, True, 1.0)
        out = torch.zeros_like(r)
        for t in range(x.shape[0]):
            for j in range(USED):
                e = int(ids[t, j])
                both = ref.w4_values(*(None if a is None else a[e] for a in layer["gate_up"])) @ h[t]
                out[t] += weights[t, j] * (ref.w4_values(*(a[e] for a in layer["down"])) @
                                           ref.glu("swiglu", both[:INTER], both[INTER:], 0.0)[0])
        r = r + 0.5 * rms(out, layer["post_moe"])
        h = rms(r, layer["pre_next"])
    return h @ ref.w4_values(*m["head"]).T


@pytest.mark.parametrize("rows", [1, 6])
def test_a_step_against_64_bits(cuda, rows):
    """F32: each of the six operators between x and the logits adds at most about 1e-5 of its values' size
    (their own tests' bounds), norms keep the size: 2e-4 covers 3 layers of 4 with the head."""
    torch = cuda
    import llmp_b200 as ops
    m = _model(torch, "f32")
    x = torch.randn((rows, HIDDEN), generator=torch.Generator().manual_seed(3)).cuda()
    tokens = torch.zeros((rows, 1), dtype=torch.int32, device="cuda")
    logits, lp = _step(ops, _loaded(ops, m), x, tokens)
    want = _step64(torch, m, x)
    assert float((logits.double() - want).norm() / want.norm()) <= 2e-4
    again = ops.logprobs(logits, tokens, top=4, temperature=0.9)
    assert all(torch.equal(a, b) for a, b in zip(lp, again))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_streams_and_graphs_give_the_same_bits(cuda, kind):
    torch = cuda
    import llmp_b200 as ops
    m = _loaded(ops, _model(torch, kind))
    g = torch.Generator().manual_seed(4)
    inputs = [torch.randn((5, HIDDEN), generator=g).to(ref.TYPES[kind]).cuda() for _ in range(4)]
    tokens = torch.randint(0, VOCAB, (5, 2), generator=g, dtype=torch.int32).cuda()
    want = [_step(ops, m, x, tokens) for x in inputs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [_step(ops, m, x, tokens) for x in inputs]
    both = [_step(ops, m, x, tokens) for x in inputs]           # two streams at once
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, both):
        assert torch.equal(a[0], b[0]) and torch.equal(a[0], c[0])
        assert all(torch.equal(p, q) and torch.equal(p, r) for p, q, r in zip(a[1], b[1], c[1]))
    held = inputs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = _step(ops, m, held, tokens)
    for x, (logits, lp) in zip(inputs, want):
        held.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(result[0], logits) and all(torch.equal(a, b) for a, b in zip(result[1], lp))
    assert ops.device_faults() == 0


def test_the_norm_s_q8_1_rows_feed_a_q4_k_product(cuda):
    torch = cuda
    import llmp_b200 as ops
    from llmp_b200 import synth
    rng = np.random.default_rng(5)
    w = torch.from_numpy(synth.q4_k_weights(rng, 300, 1024)).cuda()
    g = torch.Generator().manual_seed(6)
    block, residual = torch.randn((4, 1024), generator=g).cuda(), torch.randn((4, 1024), generator=g).cuda()
    weight = torch.rand((1024,), generator=g).cuda()
    _, h, q8 = ops.block_norm(block, residual, post=weight, pre=weight, q8=True)
    assert torch.equal(ops.vecq(w, ops.TYPE_Q4_K, 1024, 300, q8, 4), ops.vecq(w, ops.TYPE_Q4_K, 1024, 300, ops.quantize_q8(h), 4))

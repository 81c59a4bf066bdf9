"""Log probabilities, ranks, entropy and top alternatives against 64 bits."""
import pytest

import step_reference as ref

pytestmark = pytest.mark.gpu


def _logits(torch, seed, rows, vocab, kind, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, vocab), generator=g) * spread).to(ref.TYPES[kind]).cuda(), g


def _check(torch, ops, logits, tokens, top, temperature=1.0):
    got = ops.logprobs(logits, tokens, top=top, temperature=temperature)
    if tokens is None:
        tokens = torch.empty((logits.shape[0], 0), dtype=torch.int32, device="cuda")
    lp, ranks, entropy, ids, top_lp, everything = ref.logprobs(logits, tokens, top, temperature)
    assert torch.equal(got.top_ids.long(), ids), "top ids"
    assert torch.equal(got.ranks.long(), ranks.long()), "ranks"
    # S: every e^d has its exponential's 2 units and, as d = (x - m) / T has up to 3 roundings, 3 |d| e^d <= 1.2
    # more; terms are added in chains of up to vocab / 256 with a rescaling (4 roundings) a link, then a tree
    links = logits.shape[1] / 256 + 40
    s_slack = (5 * links) * ref.U + 4 * ref.U

    def slack(v):
        return torch.where(v.isfinite(), v.abs(), 0.0) * 4 * ref.U + s_slack + 4 * ref.U * torch.log(torch.tensor(logits.shape[1] + 1.0))
    ref.assert_within(got.logprobs, lp, slack(lp), "logprobs")
    ref.assert_within(got.top_logprobs, top_lp, slack(top_lp), "top logprobs")
    # U / S moves by the relative errors of both, U's terms having d's too
    finite = torch.where(everything.isfinite(), everything, 0.0)
    mean = (finite.abs() * torch.where(everything.isfinite(), everything.exp(), 0.0)).sum(-1)
    ref.assert_within(got.entropy, entropy, (mean + 1) * 3 * s_slack + 4 * ref.U * entropy.nan_to_num().abs(), "entropy")
    return got


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 31, 500, 1024, 4097, 32003, 131072, 262147])
def test_sizes_and_types(cuda, kind, vocab):
    import llmp_b200 as ops
    logits, g = _logits(cuda, vocab, 3, vocab, kind)
    tokens = cuda.randint(0, vocab, (3, 2), generator=g, dtype=cuda.int32).cuda()
    _check(cuda, ops, logits, tokens, min(vocab, 20), 0.8)


@pytest.mark.parametrize("rows", [1, 2, 17, 150, 700])
@pytest.mark.parametrize("given,top", [(0, 0), (1, 0), (0, 5), (16, 32)])
def test_rows_and_counts(cuda, rows, given, top):
    import llmp_b200 as ops
    logits, g = _logits(cuda, rows, rows, 3001, "bf16")
    tokens = cuda.randint(0, 3001, (rows, given), generator=g, dtype=cuda.int32).cuda()
    _check(cuda, ops, logits, tokens if given else None, top, 1.3)


@pytest.mark.parametrize("vocab", [40, 5000, 70001])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_ties_and_orders(cuda, vocab, kind):
    """Equal rows, rising and falling ones, a few distinct values, all the large ones in one stretch."""
    torch = cuda
    import llmp_b200 as ops
    g = torch.Generator().manual_seed(1)
    rows = [torch.zeros(vocab), -torch.zeros(vocab), torch.arange(vocab) / vocab, -torch.arange(vocab) / vocab,
            torch.randint(0, 3, (vocab,), generator=g).float(), torch.randn(vocab, generator=g),
            torch.where(torch.arange(vocab) % 8 == 3, 5.0, 0.0) + torch.randn(vocab, generator=g),
            torch.where(torch.arange(vocab) % 512 < 9, 9.0, 0.0) + torch.randn(vocab, generator=g) * 0.1,
            torch.where(torch.arange(vocab) // 64 == 3, 50.0, 0.0)]
    rows[0][1::3] = -0.0
    logits = torch.stack(rows).to(ref.TYPES[kind]).cuda()
    tokens = torch.tensor([[0, vocab - 1, vocab // 2]] * len(rows), dtype=torch.int32).cuda()
    _check(torch, ops, logits, tokens, 32)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [100, 9001])
def test_masks_and_values_that_are_not_finite(cuda, kind, vocab):
    torch = cuda
    import llmp_b200 as ops
    logits, g = _logits(torch, 2, 9, vocab, kind)
    lowest = torch.finfo(ref.TYPES[kind]).min
    inf, nan = float("inf"), float("nan")
    logits[0, torch.rand(vocab, generator=g).cuda() < 0.5] = -inf
    logits[1] = -inf                        # nothing is left
    logits[2, 1:] = -inf                    # one is
    logits[2, 0] = 4.0
    logits[3, 5:] = lowest                  # masked by the type's lowest value
    logits[4] = lowest
    logits[5, 11] = nan
    logits[6, 3] = inf
    logits[7, :] = nan
    logits[8, 40:] = -inf
    logits[8, 7] = nan
    tokens = torch.tensor([[0, 11, 3, 50]] * 9, dtype=torch.int32).cuda()
    got = _check(torch, ops, logits, tokens, 30)
    assert bool((got.logprobs[1] == -inf).all() and got.entropy[1] == 0 and got.logprobs[2, 0] == 0 and got.entropy[2] == 0)
    assert got.top_ids[1].tolist() == list(range(30))


def test_tokens_outside_the_vocabulary(cuda):
    torch = cuda
    import llmp_b200 as ops
    logits, _ = _logits(torch, 3, 2, 1000, "f32")
    tokens = torch.tensor([[-1, 5, 1000], [999, 2 ** 31 - 1, -2 ** 31]], dtype=torch.int32).cuda()
    got = _check(torch, ops, logits, tokens, 3)
    assert got.ranks[0, 0] == 0 and bool(got.logprobs[0, 0].isnan())


@pytest.mark.parametrize("temperature", [1e-3, 0.1, 1.0, 50.0])
def test_temperatures_and_spread(cuda, temperature):
    import llmp_b200 as ops
    logits, g = _logits(cuda, 4, 4, 2000, "f32", 20.0)
    tokens = cuda.randint(0, 2000, (4, 3), generator=g, dtype=cuda.int32).cuda()
    _check(cuda, ops, logits, tokens, 6, temperature)


def test_strides_and_alignment(cuda):
    torch = cuda
    import llmp_b200 as ops
    for kind in ("f32", "bf16"):
        logits, g = _logits(torch, 5, 5, 6000, kind)
        tokens = torch.randint(0, 6000, (5, 1), generator=g, dtype=torch.int32).cuda()
        for offset, extra in ((1, 3), (8, 64)):
            wide = torch.full((5, 6000 + extra + offset), 90.0, dtype=logits.dtype, device="cuda")
            view = wide[:, offset:offset + 6000]
            view.copy_(logits)
            _check(torch, ops, view, tokens, 10)
        _check(torch, ops, logits[:1].expand(5, 6000), tokens, 4)
    assert ops.logprobs(logits[:0], tokens[:0], top=3).top_ids.shape == (0, 3)


def test_graph_and_stream(cuda):
    torch = cuda
    import llmp_b200 as ops
    logits, g = _logits(torch, 6, 4, 50000, "bf16")
    tokens = torch.randint(0, 50000, (4, 1), generator=g, dtype=torch.int32).cuda()
    want = _check(torch, ops, logits, tokens, 8)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for i in range(4):
        with torch.cuda.stream(streams[i % 2]):
            results.append(ops.logprobs(logits, tokens, top=8))
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(r, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.logprobs(logits, tokens, top=8)
    logits.copy_(logits.flip(0))
    tokens.copy_(tokens.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b.flip(0)) for a, b in zip(held, want))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("temperature", [1e-6, 1e6])
@pytest.mark.parametrize("rows", [2, 600])
def test_the_first_and_the_last_temperature(cuda, kind, temperature, rows):
    import llmp_b200 as ops
    logits, g = _logits(cuda, 7, rows, 3000, kind)
    tokens = cuda.randint(0, 3000, (rows, 2), generator=g, dtype=cuda.int32).cuda()
    tokens[:, 1] = tokens[:, 0]                       # the same token twice
    got = _check(cuda, ops, logits, tokens, 3, temperature)
    assert cuda.equal(got.logprobs[:, 0], got.logprobs[:, 1]) and cuda.equal(got.ranks[:, 0], got.ranks[:, 1])

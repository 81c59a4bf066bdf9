"""The norms between two blocks against 64 bits."""
import pytest

import step_reference as ref

pytestmark = pytest.mark.gpu


def _case(torch, seed, rows, width, kind, weights=None):
    g = torch.Generator().manual_seed(seed)

    def make(*shape):
        return torch.randn(shape, generator=g).to(ref.TYPES[kind]).cuda()

    def weight():
        return (torch.rand((width,), generator=g) + 0.5).to(ref.TYPES[weights or kind]).cuda()
    return {"block": make(rows, width), "residual": make(rows, width) * 2, "channel": make(width), "token": make(rows, width),
            "post": weight(), "pre": weight()}


def _check(ops, block, residual, gate, post, pre, scale=1.0, offset=0.0, eps=1e-6, **kw):
    got = ops.block_norm(block, residual, gate=gate, post=post, pre=pre, scale=scale, offset=offset, eps=eps, **kw)
    r, r_slack, h, h_slack = ref.norm(block, residual, gate, post, pre, scale, offset, eps)
    ref.assert_within(got[0], r, r_slack, "r")
    if pre is None:
        assert got[1] is None
    else:
        ref.assert_within(got[1], h, h_slack, "h")
    return got


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("width", [1, 3, 8, 33, 255, 512, 1000, 2560, 4096, 5119, 8192, 16384, 20001, 32768])
def test_widths_and_types(cuda, kind, width):
    import llmp_b200 as ops
    c = _case(cuda, width, 5, width, kind)
    _check(ops, c["block"], c["residual"], c["token"], c["post"], c["pre"], 0.5, 1.0)


@pytest.mark.parametrize("gate", [None, "channel", "token"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("pre", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("weights", ["f32", "bf16"])
def test_parts(cuda, gate, post, pre, residual, weights):
    import llmp_b200 as ops
    c = _case(cuda, 3, 4, 640, "bf16", weights)
    _check(ops, c["block"], c["residual"] if residual else None, c[gate] if gate else None, c["post"] if post else None,
           c["pre"] if pre else None, 0.25)


@pytest.mark.parametrize("rows", [1, 2, 300, 5000])
def test_rows(cuda, rows):
    import llmp_b200 as ops
    c = _case(cuda, rows, rows, 768, "bf16")
    _check(ops, c["block"], c["residual"], c["channel"], c["post"], c["pre"])


@pytest.mark.parametrize("width", [1, 31, 32, 100, 512, 513, 2560, 4099, 32768])
def test_q8_1_rows_are_the_quantizer_s(cuda, width):
    torch = cuda
    import llmp_b200 as ops
    c = _case(torch, width, 6, width, "f32")
    _, h, q8 = _check(ops, c["block"], c["residual"], None, c["post"], c["pre"], q8=True)
    assert torch.equal(q8, ops.quantize_q8(h))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_strides_alignment_and_places(cuda, kind):
    torch = cuda
    import llmp_b200 as ops
    c = _case(torch, 4, 7, 520, kind)
    want = _check(ops, c["block"], c["residual"], c["token"], c["post"], c["pre"])

    def moved(t, offset, extra):
        wide = torch.full((t.shape[0], t.shape[1] + extra), 3.0, dtype=t.dtype, device="cuda")
        view = wide[:, offset:offset + t.shape[1]]
        view.copy_(t)
        return wide, view
    for offset, extra in ((1, 3), (8, 16)):
        _, b = moved(c["block"], offset, extra)
        _, r = moved(c["residual"], offset, extra)
        _, gate = moved(c["token"], offset, extra)
        wide_h, h = moved(c["block"], offset, extra)
        got = ops.block_norm(b, r, gate=gate, post=c["post"], pre=c["pre"], out_residual=r, out=h)
        assert got[0] is r and got[1] is h
        # another path may add the squares in another order: within the same bounds
        r64, r_slack, h64, h_slack = ref.norm(c["block"], c["residual"], c["token"], c["post"], c["pre"], 1.0, 0.0, 1e-6)
        ref.assert_within(r, r64, r_slack)
        ref.assert_within(h, h64, h_slack)
        assert bool((wide_h[:, :offset] == 3).all() and (wide_h[:, offset + 520:] == 3).all())
    same = c["block"].clone()
    ops.block_norm(same, c["residual"], gate=c["token"], post=c["post"], pre=c["pre"], out=same)
    assert torch.equal(same, want[1])
    row = ops.block_norm(c["block"][:1].expand(7, 520), c["residual"], post=c["post"], pre=c["pre"])
    repeated = ops.block_norm(c["block"][:1].expand(7, 520).contiguous(), c["residual"], post=c["post"], pre=c["pre"])
    assert torch.equal(row[0], repeated[0]) and torch.equal(row[1], repeated[1])
    assert ops.block_norm(c["block"][:0], c["residual"][:0], pre=c["pre"])[1].shape == (0, 520)


def test_zero_rows_tiny_and_not_finite_values(cuda):
    torch = cuda
    import llmp_b200 as ops
    c = _case(torch, 5, 6, 300, "f32")
    b, r = c["block"], c["residual"]
    b[0], r[0] = 0.0, 0.0
    b[1], r[1] = b[1] * 1e-12, r[1] * 1e-12
    b[2] = b[2] * 1e12
    b[3, 7] = float("nan")
    r[4, 9] = float("inf")
    got = ops.block_norm(b, r, post=c["post"], pre=c["pre"], eps=1e-5)
    r64, r_slack, h64, h_slack = ref.norm(b, r, None, c["post"], c["pre"], 1.0, 0.0, 1e-5)
    keep = [0, 1, 2, 5]
    ref.assert_within(got[0][keep], r64[keep], r_slack[keep])
    ref.assert_within(got[1][keep], h64[keep], h_slack[keep])
    assert bool((got[1][0] == 0).all() and got[0][3].isnan().all() and got[1][3].isnan().all())
    assert bool(got[1][4, 9].isnan() and (got[1][4, :9] == 0).all())      # inf / inf, and finite / inf
    assert torch.equal(got[0][4].isinf(), r64[4].isinf())


def test_graph_and_stream(cuda):
    torch = cuda
    import llmp_b200 as ops
    c = _case(torch, 6, 3, 1280, "f32")
    want = _check(ops, c["block"], c["residual"], None, c["post"], c["pre"])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.block_norm(c["block"], c["residual"], post=c["post"], pre=c["pre"])
    side.synchronize()
    assert torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.block_norm(c["block"], c["residual"], post=c["post"], pre=c["pre"])
    c["block"].copy_(c["block"].flip(0))
    c["residual"].copy_(c["residual"].flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held[1], want[1].flip(0))

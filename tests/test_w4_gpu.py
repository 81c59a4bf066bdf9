"""4-bit products with group scales against 64 bits: types, groups, odd sizes, strides, row counts,
GLUs, alignment, streams, graphs, values that are not finite."""
import pytest

import step_reference as ref

pytestmark = pytest.mark.gpu


def _case(torch, seed, rows, n, k, group, scales="bf16", zeros=True, kind="bf16", glu=False):
    g = torch.Generator().manual_seed(seed)
    source = ref.w4_source(g, (), 2 * n if glu else n, k, group, scales, zeros)
    x = torch.randn((rows, k), generator=g).to(ref.TYPES[kind]).cuda()
    return source, x


def _check(torch, ops, source, x, n, group, glu="none", limit=0.0, out=None):
    m = ops.w4_relayout(*source, glu=glu != "none")
    got = ops.w4_vector(m, x, glu=ref.GLUS[glu], limit=limit, out=out)
    y, slack = ref.w4_rows(x, ref.w4_values(*source), group)
    if glu != "none":
        y, slack = ref.glu_rows(glu, y[:, :n], slack[:, :n], y[:, n:], slack[:, n:], limit)
    ref.assert_within(got, y, slack, (glu, x.dtype, x.shape))
    return m, got


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 2, 3, 5, 8, 9, 16])
def test_types_groups_and_rows(cuda, kind, group, rows):
    import llmp_b200 as ops
    n, k = 75, group * 11
    source, x = _case(cuda, rows, rows, n, k, group, "f16" if rows % 2 else "bf16", rows % 3 != 0, kind)
    _check(cuda, ops, source, x, n, group)


@pytest.mark.parametrize("n", [1, 7, 16, 17, 128, 300])
@pytest.mark.parametrize("k", [32, 96, 128, 160, 1024, 1056, 2560, 8224])
def test_sizes(cuda, n, k):
    import llmp_b200 as ops
    source, x = _case(cuda, n + k, 3, n, k, 32)
    _check(cuda, ops, source, x, n, 32)


@pytest.mark.parametrize("glu", ["swiglu", "swiglu_clamp", "geglu"])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [1, 8, 77, 512])
def test_glu(cuda, glu, kind, n):
    import llmp_b200 as ops
    source, x = _case(cuda, n, 4, n, 640, 64, kind=kind, glu=True)
    _check(cuda, ops, source, x * 4, n, 64, glu, 0.75 if glu == "swiglu_clamp" else 0.0)


def test_many_rows_of_weights_and_a_long_k(cuda):
    import llmp_b200 as ops
    source, x = _case(cuda, 1, 2, 20011, 256, 128, kind="f16")
    _check(cuda, ops, source, x, 20011, 128)
    source, x = _case(cuda, 2, 16, 40, 40960, 64, kind="f32")
    _check(cuda, ops, source, x, 40, 64)


@pytest.mark.parametrize("kind,rows,k", [("bf16", 16, 4096), ("bf16", 16, 8192), ("f16", 9, 16384), ("f32", 16, 4096),
                                         ("f32", 7, 12288), ("f32", 16, 16384), ("f32", 1, 131072)])
@pytest.mark.parametrize("n,glu", [(40, "none"), (300, "none"), (133, "swiglu")])
def test_activations_that_fill_shared_memory_or_a_cluster_s(cuda, kind, rows, k, n, glu):
    import llmp_b200 as ops
    source, x = _case(cuda, rows + n, rows, n, k, 128, kind=kind, glu=glu != "none")
    _check(cuda, ops, source, x, n, 128, glu)


def test_strides_alignment_and_outputs(cuda):
    torch = cuda
    import llmp_b200 as ops
    n, k, group = 50, 320, 64
    source, x = _case(torch, 3, 5, n, k, group, kind="f32")
    _, base = _check(torch, ops, source, x, n, group)
    # arrays that begin at odd places and have rows of other lengths
    codes = torch.zeros((n, k // 2 + 3), dtype=torch.uint8, device="cuda")[:, 1:1 + k // 2]
    codes.copy_(source[0])
    scales = torch.zeros((n, k // group + 2), dtype=source[1].dtype, device="cuda")[:, 1:1 + k // group]
    scales.copy_(source[1])
    zeros = torch.zeros((n, source[2].shape[1] + 1), dtype=torch.uint8, device="cuda")[:, 1:]
    zeros.copy_(source[2])
    m = ops.w4_relayout(codes, scales, zeros)
    assert torch.equal(ops.w4_vector(m, x), base)
    for offset, width in ((1, k + 5), (4, k + 12)):
        wide = torch.zeros((5, width), device="cuda")
        wide[:, offset:offset + k] = x
        assert torch.equal(ops.w4_vector(m, wide[:, offset:offset + k]), base)
    out = torch.full((5, n + 9), 7.0, device="cuda")
    ops.w4_vector(m, x, out=out[:, 3:3 + n])
    assert torch.equal(out[:, 3:3 + n], base) and bool((out[:, :3] == 7).all() and (out[:, 3 + n:] == 7).all())
    for dtype in (torch.bfloat16, torch.float16):
        other = ops.w4_vector(m, x, out=torch.empty((5, n), dtype=dtype, device="cuda"))
        assert torch.equal(other, base.to(dtype))
    assert ops.w4_vector(m, x[:0]).shape == (0, n)


def test_a_row_does_not_depend_on_its_company_of_the_same_call_size(cuda):
    torch = cuda
    import llmp_b200 as ops
    source, x = _case(torch, 4, 8, 333, 1536, 128)
    m = ops.w4_relayout(*source)
    y = ops.w4_vector(m, x)
    order = torch.tensor([3, 1, 7, 0, 2, 6, 5, 4], device="cuda")
    assert torch.equal(ops.w4_vector(m, x[order].contiguous()), y[order])


def test_values_that_are_not_finite(cuda):
    torch = cuda
    import llmp_b200 as ops
    for kind in ("f32", "bf16", "f16"):
        source, x = _case(torch, 5, 3, 64, 256, 32, kind=kind)
        x[1, 17] = float("inf")
        x[2, 200] = float("nan")
        m = ops.w4_relayout(*source)
        y = ops.w4_vector(m, x)
        values = ref.w4_values(*source)
        want = x.double() @ values.T
        finite, slack = ref.w4_rows(x[:1], values, 32)
        ref.assert_within(y[:1], finite, slack)
        assert bool(y[2].isnan().all())
        # inf times a code that equals its zero point is NaN, else an infinity of the weight's sign
        assert torch.equal(y[1].isnan(), want[1].isnan())
        assert torch.equal(y[1][~y[1].isnan()].double(), want[1][~want[1].isnan()])


def test_large_and_tiny_activations(cuda):
    torch = cuda
    import llmp_b200 as ops
    source, x = _case(torch, 6, 4, 40, 512, 64, kind="f32")
    scale = torch.tensor([1e30, 3e36, 1e-30, 1.0], device="cuda")[:, None]
    x = x * scale
    m = ops.w4_relayout(*source)
    y, slack = ref.w4_rows(x, ref.w4_values(*source), 64)
    ref.assert_within(ops.w4_vector(m, x), y, slack)


def test_other_stream_and_graph(cuda):
    torch = cuda
    import llmp_b200 as ops
    source, x = _case(torch, 7, 4, 200, 1024, 128)
    m = ops.w4_relayout(*source)
    want = ops.w4_vector(m, x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.w4_vector(m, x)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.w4_vector(m, x, out=out)
    x.mul_(2.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ops.w4_vector(m, x))


def test_relayout_and_product_back_to_back(cuda):
    torch = cuda
    import llmp_b200 as ops
    slabs = []
    source, x = _case(torch, 8, 2, 4096, 2048, 128)
    want = ops.w4_vector(ops.w4_relayout(*source), x)
    for _ in range(8):     # a product right behind its relayout sees all of the slab
        m = ops.w4_relayout(*source)
        slabs.append(m)
        assert torch.equal(ops.w4_vector(m, x), want)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [4, 6, 7, 10, 11, 12, 13, 14, 15])
def test_the_other_row_counts(cuda, kind, rows):
    """With those above every count from 1 to 16: rows that do and do not fill the MMAs' columns."""
    import llmp_b200 as ops
    source, x = _case(cuda, 40 + rows, rows, 77, 704, 64, kind=kind)
    _check(cuda, ops, source, x, 77, 64)


@pytest.mark.parametrize("kind,rows,k", [("f32", 12, 2048), ("f32", 12, 4096), ("f32", 12, 8192), ("f32", 12, 16384),
                                         ("f32", 13, 4096), ("f16", 12, 8192), ("bf16", 15, 16384)])
@pytest.mark.parametrize("group", [32, 128])
def test_rows_that_leave_columns_spare_beside_full_shared_memory(cuda, kind, rows, k, group):
    import llmp_b200 as ops
    source, x = _case(cuda, rows + k, rows, 133, k, group, kind=kind)
    _check(cuda, ops, source, x, 133, group)


@pytest.mark.parametrize("glu", ["swiglu", "swiglu_clamp", "geglu"])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_a_nan_survives_the_glu(cuda, glu, kind):
    """In an activation, in a gate row's scale, in an up row's: silu(limit) * limit is no answer to any of them."""
    torch = cuda
    import llmp_b200 as ops
    n, k, group = 40, 256, 64
    source, x = _case(torch, 9, 3, n, k, group, kind=kind, glu=True)
    x[1, 31] = float("nan")
    source[1][5, 2] = float("nan")              # a group of gate row 5
    source[1][n + 17, 0] = float("nan")         # of up row 17
    limit = 0.5 if glu == "swiglu_clamp" else 0.0
    y = ops.w4_vector(ops.w4_relayout(*source, glu=True), x, glu=ref.GLUS[glu], limit=limit)
    want = torch.zeros((3, n), dtype=torch.bool, device="cuda")
    want[1], want[:, 5], want[:, 17] = True, True, True
    assert torch.equal(y.isnan(), want)


@pytest.mark.parametrize("glu", ["none", "geglu"])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_arrays_of_experts_with_strides(cuda, glu, group):
    """Experts and rows further apart than they are long, arrays that begin at odd bytes, plain and GLU slabs: the slab is
    that of the packed arrays."""
    torch = cuda
    import llmp_b200 as ops
    g = torch.Generator().manual_seed(11)
    experts, n, k = 5, 38, group * 3
    packed = ref.w4_source(g, (experts,), n, k, group, "f16", True)

    def apart(t, rows, before, behind):
        wide = torch.randint(0, 200, (experts, n + rows, t.shape[-1] + before + behind), generator=g).to(t.dtype).cuda()
        view = wide[:, rows // 2:rows // 2 + n, before:before + t.shape[-1]]
        view.copy_(t)
        return view
    want = ops.w4_relayout(*packed, glu=glu != "none").slab
    for rows, before, behind in ((0, 0, 0), (3, 1, 2), (2, 4, 4), (0, 3, 0)):
        moved = [apart(t, rows, before, behind) for t in packed]
        got = ops.w4_relayout(*moved, glu=glu != "none")
        assert torch.equal(got.slab, want)
    order = [2, 0, 4, 1, 3]                       # experts in an order of their own: one array, transposed places
    turned = [t[order].transpose(0, 1).contiguous().transpose(0, 1) for t in packed]
    got = ops.w4_relayout(*turned, glu=glu != "none").slab.view(experts, -1)
    assert torch.equal(got, want.view(experts, -1)[order])
    # what the slab's experts multiply to, one by one
    x = torch.randn((3, k), generator=g).cuda()
    for e in range(experts):
        _check(torch, ops, [t[e] for t in moved], x, n // 2 if glu != "none" else n, group, glu)


@pytest.mark.parametrize("glu", ["swiglu", "geglu"])
def test_a_glu_slab_from_strided_rows(cuda, glu):
    torch = cuda
    import llmp_b200 as ops
    n, k, group = 45, 320, 32
    source, x = _case(torch, 12, 6, n, k, group, kind="f16", glu=True)
    _, want = _check(torch, ops, source, x, n, group, glu)
    for before, behind in ((1, 2), (4, 8), (3, 0)):
        moved = []
        for t in source:
            wide = torch.zeros((2 * n, t.shape[1] + before + behind), dtype=t.dtype, device="cuda")
            wide[:, before:before + t.shape[1]] = t
            moved.append(wide[:, before:before + t.shape[1]])
        assert torch.equal(ops.w4_vector(ops.w4_relayout(*moved, glu=True), x, glu=ref.GLUS[glu]), want)

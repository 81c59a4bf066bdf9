"""The decode step's operators refuse what they do not take before anything is queued, with a message;
what they take reaches the device check.  No GPU: addresses are made up and never read."""
import ctypes as C

import pytest

from llmp_b200 import _native as N

P = 1 << 20                         # an aligned address
pytestmark = pytest.mark.skipif(__import__("torch").cuda.is_available(), reason="needs a machine without a GPU")


def matrix(**kw):
    d = dict(slab=P, n=64, k=256, group=64, experts=1, scale_type=N.TYPE_BF16, glu=0)
    d.update(kw)
    return N.W4MatrixDesc(*[d[f] for f, _ in N.W4MatrixDesc._fields_])


def product(w=None, **kw):
    d = dict(x=P, x_stride=256, y=P, y_stride=64, rows=2, x_type=N.TYPE_BF16, y_type=N.TYPE_F32, glu=0, limit=0.0)
    d.update(kw)
    return N.W4Product(w or matrix(), *[d[f] for f, _ in N.W4Product._fields_[1:]])


def source(**kw):
    d = dict(codes=P, code_row=128, code_expert=0, scales=P, scale_row=4, scale_expert=0, zeros=P, zero_row=2, zero_expert=0)
    d.update(kw)
    return N.W4Source(*[d[f] for f, _ in N.W4Source._fields_])


def layer(gate_up=None, down=None, **kw):
    d = dict(x=P, x_stride=256, router=P, router_stride=256, bias=None, gate_up=gate_up or matrix(n=128, experts=8, glu=1),
             down=down or matrix(n=256, k=64, experts=8), y=P, y_stride=256, ids=P, weights=P, scratch=P, x_type=N.TYPE_BF16,
             router_type=N.TYPE_F32, y_type=N.TYPE_BF16, tokens=2, used=2, score=0, renormalize=1, scale=1.0, glu=1, limit=0.0)
    d.update(kw)
    return N.MoeLayerDesc(*[d[f] for f, _ in N.MoeLayerDesc._fields_])


def norm(**kw):
    d = dict(block=P, block_stride=64, residual=P, residual_stride=64, gate=None, gate_stride=0, post=P, pre=P, out_residual=P,
             out_residual_stride=64, out=P, out_stride=64, q8=None, rows=2, width=64, type=N.TYPE_F32, weight_type=N.TYPE_F32,
             scale=1.0, offset=0.0, eps=1e-6)
    d.update(kw)
    return N.BlockNormDesc(*[d[f] for f, _ in N.BlockNormDesc._fields_])


def logits(**kw):
    d = dict(logits=P, stride=100, tokens=P, logprobs=P, ranks=P, entropy=P, top_ids=P, top_logprobs=P, rows=2, type=N.TYPE_F32,
             vocab=100, given=1, top=5, temperature=1.0)
    d.update(kw)
    return N.LogprobsDesc(*[d[f] for f, _ in N.LogprobsDesc._fields_])


def status(name, *descs):
    return getattr(N.lib(), name)(*[C.byref(d) if d is not None else None for d in descs], None)


TAKEN = [("llmp_b200_w4_vector", (product(),)), ("llmp_b200_w4_vector", (product(rows=1, x_stride=0, y_stride=0),)),
         ("llmp_b200_w4_vector", (product(matrix(n=128, glu=1), glu=1),)),
         ("llmp_b200_w4_relayout", (source(), matrix())),
         ("llmp_b200_w4_relayout", (source(codes=P + 1, zeros=P + 3, code_row=131), matrix(group=128))),
         ("llmp_b200_moe_layer", (layer(),)), ("llmp_b200_moe_layer", (layer(bias=P, score=1, tokens=16, used=8),)),
         ("llmp_b200_block_norm", (norm(),)), ("llmp_b200_block_norm", (norm(q8=P, out=None),)),
         ("llmp_b200_block_norm", (norm(pre=None, out=None, post=None, residual=None),)),
         ("llmp_b200_logprobs", (logits(),)), ("llmp_b200_logprobs", (logits(given=0, tokens=None, logprobs=None, ranks=None),))]
NOTHING = [("llmp_b200_w4_vector", (product(rows=0, x=None),)), ("llmp_b200_moe_layer", (layer(tokens=0, x=None),)),
           ("llmp_b200_block_norm", (norm(rows=0, block=None),)), ("llmp_b200_logprobs", (logits(rows=0, logits=None),))]
REFUSED = (
    [("llmp_b200_w4_vector", (d,)) for d in (
        None, product(matrix(slab=None)), product(matrix(slab=P + 16)), product(matrix(group=16)), product(matrix(k=200)),
        product(matrix(n=0)), product(matrix(k=0)), product(matrix(n=1 << 29)), product(matrix(k=1 << 25)),
        product(matrix(experts=0)), product(matrix(experts=2)), product(matrix(scale_type=N.TYPE_F32)),
        product(matrix(glu=2)), product(matrix(n=65, glu=1), glu=1), product(matrix(n=128, glu=1)), product(glu=1),
        product(matrix(n=128, glu=1), glu=4), product(rows=17), product(rows=-1), product(x=None), product(y=None),
        product(x_type=2), product(y_type=31), product(x=P + 1), product(y=P + 2), product(x_stride=255),
        product(y_stride=63))] +
    [("llmp_b200_w4_relayout", d) for d in (
        (None, matrix()), (source(), None), (source(codes=None), matrix()), (source(scales=None), matrix()),
        (source(scales=P + 1), matrix()), (source(code_row=127), matrix()), (source(scale_row=3), matrix()),
        (source(zero_row=1), matrix()), (source(code_expert=-1), matrix()), (source(), matrix(slab=P + 128)))] +
    [("llmp_b200_moe_layer", (d,)) for d in (
        None, layer(matrix(n=128, experts=8)), layer(down=matrix(n=256, k=64, experts=8, glu=1)),
        layer(down=matrix(n=128, k=64, experts=8)), layer(down=matrix(n=256, k=128, experts=8)),
        layer(down=matrix(n=256, k=64, experts=4)), layer(matrix(n=128, experts=513, glu=1), matrix(n=256, k=64, experts=513)),
        layer(matrix(n=128, k=16448, experts=8, glu=1), matrix(n=16448, k=64, experts=8), x_stride=16448, y_stride=16448,
              router_stride=16448),
        layer(used=0), layer(used=9), layer(tokens=17), layer(tokens=-1), layer(x=None), layer(router=None), layer(y=None),
        layer(ids=None), layer(weights=None), layer(scratch=None), layer(scratch=P + 64), layer(x_type=9), layer(router_type=8),
        layer(y_type=12), layer(glu=0), layer(glu=4), layer(score=2), layer(x_stride=255), layer(y_stride=255),
        layer(router_stride=255), layer(bias=P + 2), layer(router=P + 2))] +
    [("llmp_b200_block_norm", (d,)) for d in (
        None, norm(width=0), norm(width=32769), norm(type=8), norm(type=N.TYPE_BF16, weight_type=N.TYPE_F16), norm(rows=-1),
        norm(rows=1 << 31), norm(block=None), norm(pre=None), norm(out=None), norm(pre=None, out=None, out_residual=None),
        norm(type=N.TYPE_BF16, q8=P), norm(block=P + 2), norm(q8=P + 2), norm(out_stride=63), norm(out_residual_stride=63),
        norm(block_stride=-64), norm(gate=P, gate_stride=-1))] +
    [("llmp_b200_logprobs", (d,)) for d in (
        None, logits(type=12), logits(vocab=0), logits(vocab=(1 << 24) + 1), logits(rows=-1), logits(rows=1 << 31),
        logits(given=17), logits(given=-1), logits(top=33), logits(vocab=4, top=5), logits(top=-1), logits(temperature=0.0),
        logits(temperature=-1.0), logits(temperature=float("nan")), logits(temperature=float("inf")), logits(logits=None),
        logits(tokens=None), logits(ranks=None), logits(entropy=None), logits(top_ids=None), logits(logits=P + 2),
        logits(stride=-1))])


@pytest.mark.parametrize("call", TAKEN, ids=lambda c: c[0])
def test_taken_calls_reach_the_device_check(call):
    assert status(call[0], *call[1]) == N.NO_DEVICE


@pytest.mark.parametrize("call", NOTHING, ids=lambda c: c[0])
def test_no_rows_queue_nothing(call):
    assert status(call[0], *call[1]) == 0


@pytest.mark.parametrize("call", REFUSED, ids=lambda c: c[0])
def test_refusals(call):
    assert status(call[0], *call[1]) == N.REJECTED
    assert call[0][len("llmp_b200_"):].encode() in N.lib().llmp_b200_last_error()


def test_sizes_of_slabs_and_scratch():
    L = N.lib()
    assert L.llmp_b200_w4_slab_bytes(16, 128, 128, 1, 0) == 1024 + 64
    assert L.llmp_b200_w4_slab_bytes(17, 160, 32, 3, 0) == 3 * 2 * 2 * (1024 + 256)
    assert L.llmp_b200_w4_slab_bytes(34, 128, 64, 1, 1) == 3 * (1024 + 128)       # 17 gate and 17 up rows
    assert L.llmp_b200_w4_slab_bytes(1 << 20, 1 << 16, 128, 64, 0) == 64 * (1 << 16) * (1 << 9) * 1088
    assert L.llmp_b200_w4_slab_bytes(16, 128, 16, 1, 0) == 0
    assert L.llmp_b200_moe_layer_scratch(8, 16, 768) >= 8 * 16 * 3 * 768 * 2
    assert L.llmp_b200_moe_layer_scratch(17, 1, 768) == 0


def test_python_refuses_what_the_library_cannot_see():
    import torch

    import llmp_b200 as ops
    cpu = torch.zeros((2, 64))
    for call in (lambda: ops.w4_relayout(torch.zeros((4, 16), dtype=torch.uint8), torch.zeros((4, 1), dtype=torch.float16)),
                 lambda: ops.block_norm(cpu, pre=torch.ones(64)), lambda: ops.logprobs(cpu),
                 lambda: ops.block_norm(cpu.double()), lambda: ops.logprobs(cpu.long())):
        with pytest.raises(ops.Rejected):
            call()

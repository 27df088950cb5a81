"""Microscaled 4-bit matrices without a GPU: their shape, and what their functions refuse."""
import pytest
import torch

from damendaemon_b200 import kernels
from mx4_tools import packed, quantized


def test_shape_and_bytes():
    w = kernels.Mx4Matrix(torch.zeros(5, 128, dtype=torch.uint8), torch.zeros(5, 8, dtype=torch.uint8), 130)
    assert w.shape == (5, 130) and w.dim() == 2 and w.nbytes == 5 * 136
    stack = kernels.Mx4Matrix(torch.zeros(2, 5, 64, dtype=torch.uint8), torch.zeros(2, 5, 4, dtype=torch.uint8), 128)
    assert stack.shape == (2, 5, 128)


@pytest.mark.parametrize("codes,scales,width", [((5, 64), (5, 8), 100), ((5, 64), (5, 4), 129), ((5, 128), (4, 8), 200), ((64,), (4,), 100),
                                                ((5, 64), (5, 4), 0)])
def test_refuses_shapes(codes, scales, width):
    with pytest.raises(kernels.KernelError, match="4-bit matrix"):
        kernels.Mx4Matrix(torch.zeros(codes, dtype=torch.uint8), torch.zeros(scales, dtype=torch.uint8), width)


def test_refuses_types_and_strides():
    codes, scales = torch.zeros(5, 64, dtype=torch.uint8), torch.zeros(5, 4, dtype=torch.uint8)
    with pytest.raises(kernels.KernelError, match="4-bit matrix"):
        kernels.Mx4Matrix(codes.int(), scales, 100)
    with pytest.raises(kernels.KernelError, match="contiguous"):
        kernels.Mx4Matrix(torch.zeros(10, 64, dtype=torch.uint8)[::2], scales, 100)


def test_no_cpu_path():
    x = torch.zeros(2, 64)
    w = kernels.Mx4Matrix(torch.zeros(2, 64, dtype=torch.uint8), torch.zeros(2, 4, dtype=torch.uint8), 64)
    for call in (lambda: kernels.mx4_quantize(x), lambda: kernels.mx4_values(w), lambda: kernels.gemm_mx4(x.bfloat16(), w)):
        with pytest.raises(kernels.KernelError, match="CUDA"):
            call()


def test_product_refusals():
    w = kernels.Mx4Matrix(torch.zeros(2, 64, dtype=torch.uint8), torch.zeros(2, 4, dtype=torch.uint8), 64)
    a = torch.zeros(3, 64, dtype=torch.bfloat16)
    for bad in (lambda: kernels.gemm_mx4(a.float(), w), lambda: kernels.gemm_mx4(a[:, :60], w), lambda: kernels.gemm_mx4(a.t(), w),
                lambda: kernels.gemm_mx4(a, w.codes), lambda: kernels.gemm_mx4(a, w, torch.zeros(3)),
                lambda: kernels.gemm_mx4(a, w, residual=torch.zeros(3, 3)), lambda: kernels.gemm_mx4(a, w, out=torch.zeros(2, 2)),
                lambda: kernels.mx4_quantize(torch.zeros(4, 64).t()), lambda: kernels.mx4_quantize(torch.zeros(64)),
                lambda: kernels.mx4_quantize(torch.zeros(2, 64, dtype=torch.float16))):
        with pytest.raises(kernels.KernelError):
            bad()


def test_plain_quantisation():
    """The tests' own plain form at values that can be checked by eye: 5 and 2.5 are ties, 7 is above the largest number."""
    x = torch.tensor([[7.0, 5.0, -2.5, 0.25, 0.75, -0.2, 1.75, 3.5] + [0.0] * 24 + [0.3, -0.1]])
    values, marks = quantized(x)
    assert values[0, :8].tolist() == [6.0, 4.0, -2.0, 0.0, 1.0, -0.0, 2.0, 4.0]
    assert marks.tolist() == [[127, 123]]
    assert values[0, 32:].tolist() == [0.25, -0.09375]
    codes, scales = packed(values, marks)
    word = int.from_bytes(bytes(codes[0, :4].tolist()), "little")
    assert word & 15 == 7 and word >> 16 & 15 == 6 and word >> 4 & 15 == 8 + 4 and scales[0, :2].tolist() == [127, 123]


# ------------------------------------------------------------------ expert layers

def matrices(E=4, inner=8, width=16, halves=2, dtype=torch.float32):
    return torch.zeros(E, halves * inner, width, dtype=dtype), torch.zeros(E, width, inner, dtype=dtype)


@pytest.mark.parametrize("change,match", [
    (dict(top=5), "experts per token"), (dict(top=0), "experts per token"), (dict(router=None), "a router or a table"),
    (dict(table=torch.zeros(9, 2, dtype=torch.int32)), "a router or a table"), (dict(router=torch.zeros(5, 16)), "router"),
    (dict(router=torch.zeros(4, 16, dtype=torch.bfloat16)), "router"), (dict(router=None, table=torch.zeros(9, 2)), "table"),
    (dict(groups=3), "groups"), (dict(groups=2, keep=3), "groups"), (dict(top=3, groups=2, keep=1), "groups"), (dict(gated=None), "does not fit"),
    (dict(activation="relu2"), "gated"), (dict(weight_input=True), "gated"), (dict(gated=(1.0, 1.0, "other")), "gated"),
    (dict(shared_gate=True, router=torch.zeros(5, 16)), "shared"), (dict(correction=torch.zeros(3)), "correction"),
    (dict(shared=(torch.zeros(12, 16), torch.zeros(16, 8)), shared_gated=(1.0, 1.0, "silu")), "shared"),
    (dict(identity=300, router=torch.zeros(304, 16)), "experts per token")])
def test_expert_layer_refusals(change, match):
    gate_up, down = matrices()
    options = dict(top=2, gated=(7.0, 1.702, "silu"), router=torch.zeros(4, 16))
    options.update(change)
    with pytest.raises(kernels.KernelError, match=match):
        kernels.ExpertLayer(gate_up, down, options.pop("top"), **options)


def test_expert_layer_matrices():
    gate_up, down = matrices()
    good = dict(gated=(7.0, 1.702, "silu"), router=torch.zeros(4, 16))
    for a, b in ((gate_up[:3], down), (gate_up[:, :8], down), (gate_up.bfloat16(), down), (gate_up.half(), down.half()), (gate_up[0], down[0]),
                 (gate_up, down.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(kernels.KernelError, match="expert layer"):
            kernels.ExpertLayer(a, b, 2, **good)
    with pytest.raises(kernels.KernelError, match="CUDA"):
        kernels.ExpertLayer(gate_up, down, 2, **good)

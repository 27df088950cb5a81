"""Products with 4-bit matrices that the kernel before them has just written: the same bits as with the programmatic launch off, where
every kernel starts when the one before it has ended."""
import pytest
import torch

from damendaemon_b200 import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def randn(seed, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def both(run):
    """What run() returns with the early launch, several times, and without it."""
    with kernels.pdl_scope(False):
        want = [t.clone() for t in run()]
        torch.cuda.synchronize()
    for _ in range(4):
        got = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("M,N,K", [(257, 640, 1024), (300, 130, 264), (400, 1600, 6400), (1024, 6400, 1600)])
def test_matrices_of_one_shape_take_turns_in_one_temporary(M, N, K):
    """Beyond MX4_FUSED_ROWS rows every product unpacks its matrix into memory that the one before it has just used."""
    a = randn(M, M, K, dtype=torch.bfloat16)
    stack = [kernels.mx4_quantize(randn(i, N, K)) for i in range(4)]
    both(lambda: [kernels.gemm_mx4(a, w) for w in stack])


@pytest.mark.parametrize("M", [1, 8, 20, 70])
@pytest.mark.parametrize("N,K", [(640, 1024), (130, 264), (6400, 1600)])
def test_a_matrix_is_quantised_just_before_its_product(M, N, K):
    a = randn(M, M, K, dtype=torch.bfloat16)
    matrices = [randn(i, N, K) for i in range(4)]
    both(lambda: [kernels.gemm_mx4(a, kernels.mx4_quantize(w)) for w in matrices])


@pytest.mark.parametrize("M", [1, 8, 70, 300])
def test_codes_are_copied_over_just_before_the_product(M):
    a = randn(M, M, 1600, dtype=torch.bfloat16)
    stack = [kernels.mx4_quantize(randn(i, 1600, 1600)) for i in range(4)]
    place = kernels.Mx4Matrix(torch.empty_like(stack[0].codes), torch.empty_like(stack[0].scales), 1600)

    def run():
        out = []
        for w in stack:
            place.codes.copy_(w.codes)
            place.scales.copy_(w.scales)
            out.append(kernels.gemm_mx4(a, place))
        return out
    both(run)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
def test_a_router_is_written_just_before_its_layer(kind):
    E, width, inner = 16, 520, 104
    gate_up, down, y = randn(1, E, 2 * inner, width, dtype=kind), randn(2, E, width, inner, dtype=kind), randn(3, 4, width, dtype=kind)
    router = torch.empty(E, width, dtype=kind, device=DEV)
    layer = kernels.ExpertLayer(gate_up, down, 2, gated=(0.0, 1.0, "silu"), router=router, settled=False)
    routers = [randn(10 + i, E, width, dtype=kind) for i in range(4)]

    def run():
        out = []
        for r in routers:
            router.copy_(r)
            out.append(kernels.moe_tokens(layer, y))
        return out
    both(run)


def test_settled_matrices_and_layers_have_the_same_bits():
    a, w = randn(1, 8, 1600, dtype=torch.bfloat16), kernels.mx4_quantize(randn(2, 640, 1600))
    want = kernels.gemm_mx4(a, w)
    assert not w.settled and w.settle() is w and w.settled
    both(lambda: [kernels.gemm_mx4(a, w)])
    assert torch.equal(kernels.gemm_mx4(a, w), want)
    E, width, inner = 16, 520, 104
    gate_up, down, y, router = (randn(i, *s, dtype=torch.bfloat16) for i, s in enumerate(((E, 2 * inner, width), (E, width, inner), (4, width), (E, width))))
    layers = [kernels.ExpertLayer(gate_up, down, 2, gated=(0.0, 1.0, "silu"), router=router, settled=s) for s in (True, False)]
    assert [layer._raw.settled for layer in layers] == [1, 0]
    assert torch.equal(*(kernels.moe_tokens(layer, y) for layer in layers))


def test_nothing_settles_in_a_capture():
    w, gate_up, down, router = kernels.mx4_quantize(randn(2, 64, 128)), randn(1, 4, 16, 32), randn(2, 4, 32, 8), randn(3, 4, 32)
    y, caught = randn(4, 2, 32), []
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        try:
            w.settle()
        except kernels.KernelError as e:
            caught.append(str(e))
        layer = kernels.ExpertLayer(gate_up, down, 2, gated=(0.0, 1.0, "silu"), router=router)
        out = kernels.moe_tokens(layer, y)
    graph.replay()
    assert len(caught) == 1 and not w.settled and layer._raw.settled == 0
    assert torch.equal(out, kernels.moe_tokens(layer, y))

"""What 4-bit products and expert layers keep where the general bounds would not show a loss."""
import pytest
import torch

from damendaemon_b200 import kernels
from mx4_tools import activation, gated

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("tile,tiles", [(16, 2), (32, 1), (64, 1), (128, 1), (128, 300)])
@pytest.mark.parametrize("form", ["silu", "clamped_swish"])
def test_float32_units_far_from_zero(tile, tiles, form):
    """Gate and up products that are exact (one element a row), sizes to 60: float32 results keep the exponential's 2 steps of
    2^-23, and half a step each of the addition, the division and the two products: 2^-22 + 4 2^-24, which is below 2^-21."""
    inner, K = 64, 32
    w = torch.zeros(1, 2 * inner, K)
    w[0, :inner, 0], w[0, inner:, 0] = 1.0, 0.5
    a = torch.zeros(tile * tiles, K, dtype=torch.bfloat16)
    a[:, 0] = torch.linspace(-60, 60, tile * tiles)
    q = kernels.mx4_quantize(w.to(DEV))
    got = kernels.gemm_grouped_mx4(a.to(DEV), q, torch.zeros(tiles, dtype=torch.int32, device=DEV), tile, gated=(100.0, 1.0, form),
                                   out_dtype=torch.float32).double().cpu()
    gate = a[:, :1].double()
    want = gated(gate, gate / 2, 100.0, 1.0, form).expand(-1, inner)
    assert ((got - want).abs() <= 2.0 ** -21 * want.abs()).all(), ((got - want).abs() / want.abs()).nan_to_num().max()


def randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


def relative(got, want, mass, K):
    """Sums of K exact products, in chains of at most K, that cut off where they add: K 2^-23 of the sum of their sizes; and the
    smallest float32 number."""
    off = (got.double().cpu() - want).abs() / ((K + 16) * 2.0 ** -23 * mass + 2.0 ** -148)
    assert off.max() <= 1, off.max().item()


@pytest.mark.parametrize("M", [1, 8, 20, 32, 70, 300])
@pytest.mark.parametrize("row,block", [(-100, 0), (-100, 60), (-70, 0), (64, 0), (100, -10), (90, -130), (60, -127), (-120, 100)])
def test_rows_and_blocks_of_every_size(M, row, block):
    """Rows of a around 2^row, blocks of w around 2^block (below 2^-124 the byte of a block's scale is 0)."""
    K = 256
    a, w = (randn(M, M, K).double() * 2.0 ** row).to(torch.bfloat16), (randn(1, 48, K).double() * 2.0 ** block).float()
    q = kernels.mx4_quantize(w.to(DEV))
    values = kernels.mx4_values(q, torch.float32).double().cpu()
    assert (values != 0).any()
    got = kernels.gemm_mx4(a.to(DEV), q, out_dtype=torch.float32)
    relative(got, a.double() @ values.t(), a.double().abs() @ values.abs().t(), K)


@pytest.mark.parametrize("kind", ["bfloat16", "mx4"])
@pytest.mark.parametrize("power", [-45, -30, 36, 44])
def test_hidden_rows_of_every_size(kind, power):
    """Plain units squared: hidden values around 2^(2 power). The down product's terms add up exactly to 24 bits of a hidden value."""
    E, width, inner, T = 4, 96, 64, 5
    matrices = [(randn(1, E, inner, width) * width ** -0.5).bfloat16().to(DEV), (randn(2, E, width, inner) * inner ** -0.5).bfloat16().to(DEV)]
    held = [kernels.mx4_quantize(m) for m in matrices] if kind == "mx4" else matrices
    up, down = ((kernels.mx4_values(m, torch.float32) if kind == "mx4" else m).double().cpu() for m in held)
    table = torch.tensor([[0, 1], [2, 3], [1, 3]], dtype=torch.int32)
    ids = torch.tensor([0, 1, 2, 0, 1], dtype=torch.int32)
    y = (randn(3, T, width).double() * 2.0 ** power).to(torch.bfloat16)
    layer = kernels.ExpertLayer(*held, 2, activation="relu2", table=table.to(DEV))
    got = kernels.moe_tokens(layer, y.to(DEV), ids=ids.to(DEV)).double().cpu()
    for t in range(T):
        want, bound = 0, 0
        for e in table[ids[t]].tolist():
            z, mass = up[e] @ y[t].double(), up[e].abs() @ y[t].double().abs()
            hidden = activation(z, "relu2") / 2
            # up's chain of at most `width` additions, through the square; its and the weight's roundings; the chain of the terms
            error = (width + 16) * 2.0 ** -23 * mass * z.abs() + 4 * 2.0 ** -23 * hidden
            want = want + down[e] @ hidden
            bound = bound + down[e].abs() @ (error + (3 * inner + 16) * 2.0 ** -23 * hidden)
        assert ((got[t] - want).abs() <= bound).all()

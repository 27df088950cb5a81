"""What 4-bit products and expert layers keep where the general bounds would not show a loss."""
import pytest
import torch

from damendaemon_b200 import kernels
from mx4_tools import gated

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

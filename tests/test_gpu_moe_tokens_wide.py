"""Expert layers whose down product runs in blocks of eight and of four warps (widths beyond 16 and 32 times the SMs), against the formula
in float64; and how exact ordinary layers are, beyond what the bounds of test_gpu_moe_tokens would notice."""
import pytest
import torch

from damendaemon_b200 import kernels
from test_gpu_moe_tokens import KINDS, Layer

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("width,inner,experts,top,shared,options", [
    (2376, 72, 6, 2, 40, dict(shared_gate=True)), (2400, 264, 5, 3, 0, dict(softmax=True, identity=3)), (4736, 40, 4, 2, 72, {}),
    (4744, 136, 4, 2, 0, dict(unit="clamped_swish")), (4801, 40, 3, 1, 33, {})])
def test_wide_layers(kind, width, inner, experts, top, shared, options):
    layer = Layer(kind, width, inner, experts, top, shared=shared, seed=width, **options)
    for T in sorted({1, 3, layer.layer.most_tokens}):
        layer.check(T, seed=T)


@pytest.mark.parametrize("kind", ["bfloat16", "mx4"])
@pytest.mark.parametrize("width,inner,shared", [(2048, 2048, 0), (1600, 1600, 1600)])
def test_root_mean_square_error(kind, width, inner, shared):
    """float32 sums whose parts are added rounded, and hidden rows of 24 bits: beside rounding a unit's value (four operations, 2^-24 each) a
    result has the errors of two sums of 32 parts or fewer, each a rounded addition of up to the whole (sqrt(32) 2^-24 / sqrt(3) a sum)
    and of four instructions' cut-off sums (2^-23 of a 32nd part's size each): together below 2^-21.5 of the result's size, 3.4e-7. Hidden rows
    of two bfloat16 terms (2^-18 each at worst, 2e-6), or one chain of additions that cut off over all of K, are above it."""
    layer = Layer(kind, width, inner, 8, 2, shared=shared, seed=3)
    g = torch.Generator().manual_seed(5)
    y = torch.randn((8, width), generator=g).to(torch.bfloat16)
    got = kernels.moe_tokens(layer.layer, y.to(DEV)).double().cpu()
    want, _ = layer.plain(y, torch.zeros(8, width))
    error = ((got - want).square().mean().sqrt() / want.square().mean().sqrt()).item()
    assert error <= 2.0 ** -21.5, error

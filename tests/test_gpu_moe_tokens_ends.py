"""Expert layers where values are infinite or next to float32's largest: an infinity stays one unless the formula has none."""
import pytest
import torch

from damendaemon_b200 import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "mx4": torch.bfloat16}


def plain_layer(kind, up, down, activation):
    """One expert of plain units that every token uses: [inner, width] and [width, inner]."""
    held = [m.unsqueeze(0).to(DTYPES[kind]).to(DEV) for m in (up, down)]
    if kind == "mx4":
        held = [kernels.mx4_quantize(m) for m in held]
    return kernels.ExpertLayer(*held, 1, activation=activation, table=torch.zeros(4, 1, dtype=torch.int32, device=DEV))


def run(layer, kind, y):
    return kernels.moe_tokens(layer, y.to(DTYPES[kind]).to(DEV), ids=torch.zeros(len(y), dtype=torch.int32, device=DEV)).cpu()


@pytest.mark.parametrize("kind", DTYPES)
@pytest.mark.parametrize("T", [1, 2, 4, 8])
def test_an_infinite_hidden_value_is_an_infinite_result(kind, T):
    """The square of a product passes float32: feature 5 of every token is infinite, all others are 4; down's row r has a one or a
    minus one there and ones elsewhere."""
    width, inner = 64, 40
    up, down = torch.zeros(inner, width), torch.ones(width, inner)
    up[:, 0], up[5, 0], up[5, 1] = 1.0, 0.0, 1.0
    down[1::2, 5] = -1.0
    y = torch.zeros(T, width)
    y[:, 0], y[:, 1] = 2.0, 2.0 ** 70
    got = run(plain_layer(kind, up, down, "relu2"), kind, y)
    assert (got[:, ::2] == float("inf")).all() and (got[:, 1::2] == -float("inf")).all()


def test_a_hidden_value_that_rounds_to_no_bfloat16_number():
    """Between bfloat16's largest number and float32's: (2^64 - 2^56 + 2^55 + 2^54)^2 = 2^128 - 2^119 + 2^109 - ... rounds, as a bfloat16
    number, to an infinity."""
    kind = "bfloat16"
    width, inner = 32, 32
    up, down = torch.zeros(inner, width), torch.zeros(width, inner)
    up[0, 0], up[0, 1], down[:, 0] = 1.0, 1.0, 0.25
    y = torch.zeros(3, width)
    y[0, 0], y[0, 1] = 2.0 ** 64 - 2.0 ** 56, 2.0 ** 55 + 2.0 ** 54
    y[1, 0], y[1, 1] = 2.0 ** 64 - 2.0 ** 56, 2.0 ** 55 + 2.0 ** 54 + 2.0 ** 53
    y[2, 0] = 1.0
    z = y.double()[:, 0] + y.double()[:, 1]
    hidden = (z.float() ** 2).double()
    assert hidden[0] > float(torch.finfo(torch.bfloat16).max) and torch.isfinite(hidden).all()
    got = run(plain_layer(kind, up, down, "relu2"), kind, y).double()
    # three terms keep 24 bits; the square is rounded once, the terms' sums twice
    assert ((got - hidden.unsqueeze(1) / 4).abs() <= 2.0 ** -21 * hidden.unsqueeze(1)).all(), got[:, 0] / hidden * 4


@pytest.mark.parametrize("kind", DTYPES)
def test_an_infinite_element_of_a_row(kind):
    """Its own sign decides, whatever large numbers of the other sign stand beside it; a NaN stays with its row."""
    width, inner = 64, 32
    up, down = torch.zeros(inner, width), torch.ones(width, inner)
    up[:, 0], up[:, 1] = 1.0, -1.0
    y = torch.zeros(4, width)
    y[0, 0], y[0, 1] = float("inf"), 2.0 ** 30
    y[1, 0], y[1, 1] = 2.0 ** 100, 2.0 ** 90
    y[2, 0], y[2, 1] = float("nan"), 1.0
    y[3, 0], y[3, 1] = -float("inf"), 2.0 ** 120
    got = run(plain_layer(kind, up, down, "tanh"), kind, y)
    assert (got[0] == inner).all() and (got[1] == inner).all() and got[2].isnan().all() and (got[3] == -inner).all()

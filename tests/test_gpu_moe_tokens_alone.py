"""A token of an expert layer has the same bits alone and beside any others: its sums are cut and joined by the layer alone."""
import pytest
import torch

from damendaemon_b200 import kernels
from test_gpu_moe_tokens import KINDS, Layer

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rows_of(layer, T, seed):
    g = torch.Generator().manual_seed(seed)
    width = layer.down[1].shape[1]
    y = torch.randn((T, width), generator=g).to(layer.dtype).to(DEV)
    residual = torch.randn((T, width), generator=g).to(DEV)
    ids = None if layer.table is None else torch.randint(0, layer.table.shape[0], (T,), generator=g, dtype=torch.int32).to(DEV)
    return y, residual, ids


def check(layer, seed=1):
    T = layer.layer.most_tokens
    y, residual, ids = rows_of(layer, T, seed)
    run = lambda rows: kernels.moe_tokens(layer.layer, y[rows], residual[rows], None if ids is None else ids[rows].contiguous())  # noqa: E731
    alone = torch.cat([run([t]) for t in range(T)])
    assert kernels.read_error_flag(DEV) == 0
    g = torch.Generator().manual_seed(seed)
    sets = [list(range(T)), list(range(T))[::-1]] + [torch.randperm(T, generator=g)[:n].tolist() for n in (2, 3, 4, 5, 6, 7) if n <= T]
    for rows in sets + [[t] * T for t in (0, T - 1)]:
        got = run(rows)
        assert torch.equal(got, alone[rows]), (rows, (got - alone[rows]).abs().max().item())
    assert kernels.read_error_flag(DEV) == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("width,inner,experts,top,shared,options", [
    (96, 64, 8, 2, 0, {}), (264, 200, 16, 2, 64, dict(shared_gate=True, groups=4, keep=2)), (520, 104, 66, 8, 0, dict(softmax=True, identity=2)),
    (1600, 1600, 16, 2, 1600, dict(shared_gate=True)), (2048, 1024, 64, 8, 0, dict(softmax=True, renormalize=True)),
    (260, 44, 16, 16, 12, {}), (64, 1000, 6, 2, 0, {}), (33, 17, 5, 5, 31, dict(unit="clamped_swish"))])
def test_alone_and_beside_others(kind, width, inner, experts, top, shared, options):
    check(Layer(kind, width, inner, experts, top, shared=shared, **options))


@pytest.mark.parametrize("kind", KINDS)
def test_alone_and_beside_others_by_table(kind):
    """Experts by a table, one of them twice for a token, and plain units with weights on their inputs."""
    table = torch.randint(0, 12, (40, 3), generator=torch.Generator().manual_seed(5), dtype=torch.int32)
    table[::7, 1] = table[::7, 0]
    check(Layer(kind, 392, 520, 12, 3, table=table, shared=264, unit="clamped_swish"))
    check(Layer(kind, 392, 520, 12, 3, unit="relu2", weight_input=True))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("width", [2400, 4800])
def test_alone_and_beside_others_in_wide_layers(kind, width):
    """Widths whose down product runs in blocks of eight and of four warps."""
    check(Layer(kind, width, 392, 12, 3, shared=264, softmax=True))

"""The two kernels that choose experts, of a step of any size (kernels.route_by_score) and of a few tokens (kernels.moe_tokens), choose
alike: ties, groups, corrections that are no numbers. Logits are sums of small whole numbers, so both have the same; a layer whose
expert e writes its weight into column e of the result shows what was chosen."""
import pytest
import torch

from damendaemon_b200 import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def both(E, top, T, seed, dtype=torch.float32, correction=None, spread=3, **options):
    g = torch.Generator().manual_seed(seed)
    width = max(64, E)
    up, down = torch.zeros(E, 1, width), torch.zeros(E, width, 1)
    up[:, 0, 0] = 1.0
    down[torch.arange(E), torch.arange(E), 0] = 1.0
    router = torch.randint(-spread, spread + 1, (E, width), generator=g).float() / 8
    router[:, 0] = 0.0
    y = torch.zeros(T, width)
    y[:, 0], y[:, 1:9] = 1.0, torch.randint(-2, 3, (T, 8), generator=g).float()
    y, router = y.to(dtype).to(DEV), router.to(dtype).to(DEV)
    correction = None if correction is None else correction.to(DEV)
    layer = kernels.ExpertLayer(up.to(dtype).to(DEV), down.to(dtype).to(DEV), top, activation="relu2", router=router, correction=correction, **options)
    got = kernels.moe_tokens(layer, y)[:, :E]
    chosen, weight, _ = kernels.route_by_score(y, router, E, top, options.get("groups", 1), options.get("keep", 1), options.get("weight_scale", 1.0),
                                               softmax=options.get("softmax", False), correction=correction, renormalize=options.get("renormalize", False))
    chosen, weight = chosen.view(T, top).long(), weight.view(T, top)
    want = torch.zeros(T, E + 1, device=DEV)
    want.scatter_(1, torch.where(chosen < 0, E, chosen), torch.where(chosen < 0, 0.0, weight))
    kernels.read_error_flag(DEV)                                 # (fewer than `top` may have been eligible)
    assert torch.equal(got, want[:, :E]), (got - want[:, :E]).abs().max()
    return chosen


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("E,top", [(1, 1), (3, 2), (8, 8), (31, 4), (32, 16), (33, 5), (64, 8), (65, 8), (128, 16), (200, 6), (256, 16)])
@pytest.mark.parametrize("options", [dict(), dict(softmax=True), dict(softmax=True, renormalize=True), dict(renormalize=True, weight_scale=2.5)])
def test_ties(E, top, dtype, options):
    for seed in (1, 2):
        both(E, top, 8, seed, dtype, spread=1, **options)


@pytest.mark.parametrize("E,top,groups,keep", [(8, 2, 4, 2), (16, 4, 16, 8), (64, 8, 8, 3), (66, 6, 3, 1), (256, 16, 32, 4), (32, 3, 2, 2)])
@pytest.mark.parametrize("softmax", [False, True])
def test_groups(E, top, groups, keep, softmax):
    for seed in (1, 2, 3):
        both(E, top, 8, seed, groups=groups, keep=keep, softmax=softmax, spread=1)
        both(E, top, 8, seed, groups=groups, keep=keep, softmax=softmax, correction=torch.randint(-2, 3, (E,), generator=torch.Generator().manual_seed(seed)) / 4)


@pytest.mark.parametrize("E,top,groups,keep", [(16, 4, 1, 1), (40, 6, 1, 1), (128, 8, 1, 1), (16, 4, 4, 2), (64, 8, 8, 2)])
@pytest.mark.parametrize("softmax", [False, True])
def test_corrections_that_are_no_numbers(E, top, groups, keep, softmax):
    """A NaN or minus infinity is never chosen, also where too few others are left; in whole groups, and in parts of them."""
    nan, low = float("nan"), -float("inf")
    for bad in (nan, low):
        for where in (slice(0, E // 2), slice(0, E - top + 2), slice(0, E), slice(1, None, 2)):
            correction = torch.zeros(E)
            correction[where] = bad
            chosen = both(E, top, 4, 3, groups=groups, keep=keep, softmax=softmax, correction=correction)
            fine = torch.cat([torch.arange(E)[correction == 0], torch.tensor([-1])]).to(DEV)
            assert torch.isin(chosen, fine).all()

"""How expert layers for a few tokens are cut, asked of the library itself (no GPU is needed for that)."""
import ctypes

import pytest

from damendaemon_b200 import kernels
from damendaemon_b200.csrc import build

KINDS = {"float32": 0, "bfloat16": 1, "mx4": 2}


@pytest.fixture(scope="module")
def core():
    lib = ctypes.CDLL(str(build.build_library("core")))
    for name in ("dd_moe_tokens_most", "dd_moe_tokens_prepare"):
        getattr(lib, name).restype = ctypes.c_int
    return lib


def layer(kind, width, inner, experts, top, shared=0, gated=1):
    raw = kernels._ExpertLayer()
    raw.kind, raw.width, raw.inner, raw.experts, raw.top, raw.gated = KINDS[kind], width, inner, experts, top, gated
    raw.groups = raw.keep = 1
    raw.shared_inner = shared
    return raw


@pytest.mark.parametrize("kind", KINDS)
def test_ordinary_layers_take_eight_tokens(core, kind):
    for sizes in ((1600, 1600, 16, 2, 1600), (2048, 1024, 64, 8, 0), (64, 32, 4, 1, 0)):
        assert core.dd_moe_tokens_most(ctypes.byref(layer(kind, *sizes))) == kernels.MOE_TOKENS


@pytest.mark.parametrize("kind,width,inner,experts,top", [("float32", 64, 40000, 128, 16), ("float32", 64, 70000, 64, 16),
                                                          ("bfloat16", 64, 150000, 128, 16), ("mx4", 64, 150000, 128, 16)])
def test_layers_with_more_tiles_than_are_counted_take_fewer_tokens(core, kind, width, inner, experts, top):
    """Such a layer goes to the kernels of larger steps from there on: a call may not be refused that they can run."""
    raw = layer(kind, width, inner, experts, top)
    most = core.dd_moe_tokens_most(ctypes.byref(raw))
    features = 2 if kind == "float32" else 8
    tiles = lambda T: min(T * top, experts) * -(-inner // features)  # noqa: E731
    assert 0 < most < kernels.MOE_TOKENS and tiles(most) <= 1 << 21 < tiles(most + 1)


def test_layers_whose_rows_pass_32_bits_take_none(core):
    assert core.dd_moe_tokens_most(ctypes.byref(layer("bfloat16", 64, 1 << 23, 256, 1))) == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("sizes", [(1600, 1600, 16, 2, 1600), (2048, 2048, 16, 2, 2048), (2048, 1024, 64, 8, 0), (96, 64, 8, 3, 40), (4800, 392, 12, 3, 264),
                                   (260, 44, 16, 16, 12), (1, 1, 1, 1, 1), (2400, 6400, 200, 16, 6400)])
def test_parts(core, kind, sizes):
    """Every part has a step at least, the parts of gate and up are a power of two of at most sixteen, and the sums of eight tokens fit
    beside the rings."""
    width, inner, experts, top, shared = sizes
    raw, maps = layer(kind, *sizes), ctypes.create_string_buffer(1024)
    at = (ctypes.addressof(maps) + 63) // 64 * 64
    core.dd_moe_tokens_prepare(ctypes.byref(raw), ctypes.c_void_p(at), 148)         # (the maps want a driver; the parts come first)
    step, rows = {"float32": (128, 4), "bfloat16": (64, 16), "mx4": (256, 16)}[kind]
    steps = lambda k: -(-k // step)  # noqa: E731
    assert 1 <= 1 << raw.up_shift <= min(16, steps(width))
    assert 1 <= raw.unit_part <= steps(inner) and 1 <= raw.shared_part <= max(1, steps(shared))
    parts = top * -(-steps(inner) // raw.unit_part) + -(-steps(shared) // raw.shared_part)
    tiles = -(-width // rows)
    assert 8 * parts * rows * 4 <= (64 if tiles <= 148 else 30 if tiles <= 296 else 14) << 10

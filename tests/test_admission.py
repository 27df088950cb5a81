"""What an engine holds against the free memory before it allocates its cache, on the CPU with the device's figures made up."""
import types

import pytest
import torch

from damendaemon_b200 import kernels
from damendaemon_b200.engine import Engine

GIB = 1 << 30


@pytest.fixture
def device_memory(monkeypatch):
    """``free`` bytes by the driver's count; ``held`` more that torch's allocator keeps until it is asked for them."""
    state = types.SimpleNamespace(free=8 * GIB, held=0, emptied=0)

    def empty_cache():
        state.free, state.held, state.emptied = state.free + state.held, 0, state.emptied + 1
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device=None: (state.free, 180 * GIB))
    monkeypatch.setattr(torch.cuda, "empty_cache", empty_cache)
    return state


def engine(cache_bytes, unpacked=0):
    e = object.__new__(Engine)
    e.device, e.dtype, e.max_context, e.kv_tokens, e.weight_bytes = torch.device("cuda:0"), torch.bfloat16, 1024, 4096, 3 * GIB
    e.cache = types.SimpleNamespace(bytes_needed=lambda element: cache_bytes, max_requests=4)
    e.spec = types.SimpleNamespace(layers=[], width=64, vocab_size=128)
    e._plane_width, e._unpacked_bytes = 0, unpacked
    return e


def test_memory_that_the_allocator_keeps_is_free(device_memory):
    """Matrices that were quantised or joined leave their memory with torch's allocator, which the driver counts as used."""
    device_memory.held = 6 * GIB
    engine(10 * GIB)._admit_memory()
    assert device_memory.emptied == 1
    with pytest.raises(MemoryError, match="kv_tokens"):
        engine(20 * GIB)._admit_memory()


def test_nothing_is_given_back_where_the_cache_fits(device_memory):
    device_memory.held = 6 * GIB
    engine(4 * GIB)._admit_memory()
    assert device_memory.emptied == 0


def test_the_matrix_that_a_large_step_unpacks_is_counted(device_memory):
    fits = engine(7 * GIB)
    fits._admit_memory()
    unpacked = engine(7 * GIB, unpacked=GIB)
    with pytest.raises(MemoryError, match="activations"):
        unpacked._admit_memory()
    assert unpacked.workspace_bytes == fits.workspace_bytes + GIB
    small = engine(7 * GIB, unpacked=GIB)
    small.max_context, small.cache.max_requests = kernels.MX4_FUSED_ROWS, 1         # no step of more rows than the fused products take
    small._admit_memory()

"""Two host threads, each on a stream of its own, whose calls want different amounts of shared memory of the same kernels."""
import threading

import pytest
import torch

from damendaemon_b200 import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def randn(seed, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def in_turns(*calls, times=400):
    """Every call over and over in a thread of its own; what each returned the last time, beside what it returns alone."""
    want = [call().clone() for call in calls]
    torch.cuda.synchronize()
    got, errors, start = [None] * len(calls), [], threading.Barrier(len(calls))

    def work(i, call):
        try:
            torch.cuda.set_device(0)
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                for _ in range(times):
                    got[i] = call()
                torch.cuda.current_stream().synchronize()
        except Exception as e:                               # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i, c)) for i, c in enumerate(calls)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def layer(width, experts, kind):
    gate_up, down = randn(1, experts, 64, width, dtype=kind), randn(2, experts, width, 32, dtype=kind)
    return kernels.ExpertLayer(gate_up, down, 2, gated=(0.0, 1.0, "silu"), router=randn(3, experts, width, dtype=kind))


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
def test_expert_layers_of_two_widths(kind):
    small, large = layer(64, 4, kind), layer(2048, 64, kind)
    y, z = randn(4, 1, 64, dtype=kind), randn(5, 8, 2048, dtype=kind)
    in_turns(lambda: kernels.moe_tokens(small, y), lambda: kernels.moe_tokens(large, z))


def test_grouped_products_of_few_and_many_blocks():
    few, many = kernels.mx4_quantize(randn(1, 2, 128, 128)), kernels.mx4_quantize(randn(2, 2, 4096, 128))
    a, b = randn(3, 32, 128), randn(4, 320, 128)
    at, bt = (torch.zeros(n, dtype=torch.int32, device=DEV) for n in (2, 20))
    in_turns(lambda: kernels.gemm_grouped_mx4(a, few, at, 16), lambda: kernels.gemm_grouped_mx4(b, many, bt, 16))

"""What a product over a matrix that the kernel before it has made is told: on the CPU, with the launches recorded instead of made."""
import pytest
import torch

from damendaemon_b200 import kernels


class Recorder:
    """Takes the place of the libraries: every entry point returns 0 and is remembered with its arguments."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def entry(*args):
            self.calls.append((name, args))
            return 0
        return entry


@pytest.fixture
def launches(monkeypatch):
    recorder = Recorder()
    monkeypatch.setattr(kernels, "library", lambda name: recorder)
    monkeypatch.setattr(kernels, "_ptr", lambda t, name="tensor", dtype=None: None if t is None else t.data_ptr())
    monkeypatch.setattr(kernels, "_here", lambda *tensors: None)
    monkeypatch.setattr(kernels, "_stream", lambda: 0)
    monkeypatch.setattr(kernels, "sm_count", lambda device: 148)
    monkeypatch.setattr(kernels, "error_flag", lambda device: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(kernels, "_plans", {})
    return recorder


def matrix(N, K):
    groups = -(-K // 128)
    return kernels.Mx4Matrix(torch.zeros(N, 64 * groups, dtype=torch.uint8), torch.zeros(N, 4 * groups, dtype=torch.uint8), K)


def fresh(args):
    at = kernels._SIGNATURES["tensor"]["dd_gemm_tcgen05"]
    assert len(args) == len(at)
    return args[-3]


def test_a_product_waits_for_the_matrix_that_is_unpacked_for_it(launches):
    a = torch.zeros(kernels.MX4_FUSED_ROWS + 1, 1024, dtype=torch.bfloat16)
    kernels.gemm_mx4(a, matrix(512, 1024))
    names = [name for name, _ in launches.calls]
    assert "dd_mx4_values" in names and names.index("dd_mx4_values") < names.index("dd_gemm_tcgen05")
    assert fresh(dict(launches.calls)["dd_gemm_tcgen05"]) == 1


def test_other_products_ask_for_their_weights_early(launches):
    kernels.gemm_tcgen05(torch.zeros(8, 64, dtype=torch.bfloat16), torch.zeros(16, 64, dtype=torch.bfloat16))
    assert fresh(dict(launches.calls)["dd_gemm_tcgen05"]) == 0
    kernels.gemm_tcgen05(torch.zeros(8, 64, dtype=torch.bfloat16), torch.zeros(16, 64, dtype=torch.bfloat16), fresh_weights=True)
    assert fresh(launches.calls[-1][1]) == 1


@pytest.mark.parametrize("rows,width", [(8, 256), (8, 130), (24, 131)])
def test_a_matrix_is_read_early_only_where_it_is_settled(launches, monkeypatch, rows, width):
    monkeypatch.setattr(kernels, "MX4_SMALL", 0)             # (24 rows of 131 are copied into whole 16-byte pieces first)
    w, a = matrix(64, width), torch.zeros(rows, width, dtype=torch.bfloat16)
    for settled in (False, True):
        w.settled = settled
        kernels.gemm_mx4(a, w)
        args = launches.calls[-1][1]
        assert launches.calls[-1][0] == "dd_gemm_mx4_rows" and len(args) == len(kernels._SIGNATURES["core"]["dd_gemm_mx4_rows"])
        assert args[-2] == int(settled)


def test_limits_of_shared_memory_are_told_once():
    """A launcher that told the driver another limit for every call's size could lower the one that another thread's call has
    just raised. dd_allow_shared tells one constant a kernel."""
    from damendaemon_b200.csrc import build
    for name in ("moe_tokens.cu", "gemm_mx4_tcgen05.cu"):
        source = (build.HERE / name).read_text()
        assert "cudaFuncSetAttribute" not in source and "dd_allow_shared<" in source

"""Every kernel of the products with 4-bit matrices by name: which entry points a call goes through is recorded, so that a rule that moves
cannot leave a kernel untested. Bounds as in test_gpu_mx4."""
import pytest
import torch

from damendaemon_b200 import kernels
from mx4_tools import activation, gated
from test_gpu_mx4 import close, product_bound, randn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ENTRIES = {"rows": ["dd_gemm_mx4_rows"], "tcgen05": ["dd_gemm_mx4"], "unpacked": ["dd_mx4_values", "dd_gemm_tcgen05"]}


@pytest.fixture
def entries(monkeypatch):
    """The entry points that kernels._call has been given, in order."""
    names, call = [], kernels._call
    monkeypatch.setattr(kernels, "_call", lambda lib, fn, *args, **more: (names.append(fn), call(lib, fn, *args, **more))[1])
    return names


@pytest.fixture(params=ENTRIES)
def path(request, monkeypatch, entries):
    """Sends every product through one of the three kernels; returns what has to be called by gemm_mx4(...)."""
    few = 1 << 30 if request.param == "rows" else 0
    for name in ("MX4_UNPADDED_ROWS", "MX4_FEW_ROWS"):
        monkeypatch.setattr(kernels, name, few)
    monkeypatch.setattr(kernels, "MX4_SMALL", 0)
    monkeypatch.setattr(kernels, "MX4_FUSED_ROWS", 1 << 30 if request.param == "tcgen05" else 0)

    def product(*args, **more):
        del entries[:]
        got = kernels.gemm_mx4(*args, **more)
        assert [n for n in entries if n != "dd_mx4_pad_rows"] == ENTRIES[request.param]
        return got
    return product


@pytest.mark.parametrize("M,N,K", [(1, 16, 32), (1, 1, 8), (2, 17, 104), (3, 130, 128), (7, 33, 136), (8, 64, 256), (9, 65, 520), (13, 40, 1000), (16, 48, 1600),
                                   (1, 33, 99), (5, 40, 1601), (33, 96, 2056), (64, 130, 2048), (70, 200, 1030), (130, 200, 1600), (257, 130, 1024)])
def test_sizes(path, M, N, K):
    a, w = randn(M + K, M, K, dtype=torch.bfloat16), randn(N + K, N, K, scale=K ** -0.5)
    q = kernels.mx4_quantize(w.to(DEV))
    values = kernels.mx4_values(q, torch.float32).double().cpu()
    want, bound = a.double() @ values.t(), product_bound(a, values, 1)
    close(path(a.to(DEV), q, out_dtype=torch.float32), want, bound)
    close(path(a.to(DEV), q), want, bound)


@pytest.mark.parametrize("M,N,K", [(1, 33, 104), (8, 64, 256), (12, 50, 200), (40, 130, 2048), (64, 100, 1024), (100, 70, 264), (300, 200, 520)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", [None, "gelu_new", "relu2"])
def test_strides_and_epilogues(path, M, N, K, dtype, act):
    """Rows with a stride and a start of whole 16-byte pieces, which go to the kernels as they are; a strided result whose surroundings
    stay; a strided residual, added in place too."""
    w = kernels.mx4_quantize(randn(N, N, K, scale=K ** -0.5).to(DEV))
    values = kernels.mx4_values(w, torch.float32).double().cpu()
    store = randn(M, M, K + 24, dtype=torch.bfloat16).to(DEV)
    bias, residual = randn(1, N), randn(2, M + 3, N + 7)
    a = store[:, 16:16 + K]
    z = a.double().cpu() @ values.t() + bias.double()
    slope = 2 * z.abs() + 1 if act == "relu2" else 1.13
    want = activation(z, act) + residual[:M, 3:3 + N].double()
    bound = (product_bound(a.cpu(), values, 1) + 2.0 ** -23 * z.abs()) * slope + 2.0 ** -20 * (z.abs() + want.abs() + 1)
    out = torch.full((M + 2, N + 11), 7.0, dtype=dtype, device=DEV)
    part, added = out[:M, 5:5 + N], residual.to(DEV)[:M, 3:3 + N]
    assert path(a, w, bias.to(DEV), added, act, out=part).data_ptr() == part.data_ptr()
    close(part, want, bound)
    assert (out[M:] == 7).all() and (out[:, :5] == 7).all() and (out[:, 5 + N:] == 7).all()
    if dtype == torch.float32:
        stream = residual.to(DEV)
        part = stream[:M, 3:3 + N]
        path(a, w, bias.to(DEV), part, act, out=part)
        close(part, want, bound)
        stream[:M, 3:3 + N] = residual[:M, 3:3 + N].to(DEV)
        assert torch.equal(stream.cpu(), residual)


@pytest.mark.parametrize("M", [1, 2, 16, 70])
def test_not_finite(path, M):
    w, a = randn(1, 40, 160), randn(2, M, 160, dtype=torch.bfloat16)
    w[5, 70] = float("nan")
    a[M - 1, 9] = float("inf")
    got = path(a.to(DEV), kernels.mx4_quantize(w.to(DEV)), out_dtype=torch.float32).cpu()
    fine = torch.ones(M, 40, dtype=torch.bool)
    fine[:, 5], fine[M - 1, :] = False, False
    assert got[fine].isfinite().all() and not got[:, 5].isfinite().any() and not got[M - 1].isfinite().all()


@pytest.mark.parametrize("M", [1, 8, 40, 140])
def test_wide_scales(path, M):
    K = 512
    w = randn(1, 48, K) * torch.exp2(torch.randint(-40, 41, (48, K // 32), generator=torch.Generator().manual_seed(2)).repeat_interleave(32, 1).float())
    a = (randn(3, M, K) * torch.exp2(torch.arange(M) % 7 * 10.0 - 30).unsqueeze(1)).to(torch.bfloat16)
    q = kernels.mx4_quantize(w.to(DEV))
    values = kernels.mx4_values(q, torch.float32).double().cpu()
    close(path(a.to(DEV), q, out_dtype=torch.float32), a.double() @ values.t(), product_bound(a, values, 1))


@pytest.mark.parametrize("M", [2, 16, 64, 256])
def test_rules(entries, M):
    """What the sizes choose, as it is documented: mma.sync up to 32 rows and in small products, the matrix unpacked beyond 256 rows."""
    large, a = kernels.mx4_quantize(randn(1, 1600, 6400).to(DEV)), randn(M, M, 6400, dtype=torch.bfloat16).to(DEV)
    kernels.gemm_mx4(a, large)
    assert entries[-1] == ("dd_gemm_mx4_rows" if M <= 32 else "dd_gemm_mx4")
    kernels.gemm_mx4(torch.cat([a, randn(2, 1, 6400, dtype=torch.bfloat16).to(DEV)]), large)
    assert entries[-1] == ("dd_gemm_mx4_rows" if M < 32 else "dd_gemm_mx4" if M < 256 else "dd_gemm_tcgen05")
    kernels.gemm_mx4(a[:, :64], kernels.mx4_quantize(randn(3, 40, 64).to(DEV)))
    assert entries[-1] == "dd_gemm_mx4_rows"


@pytest.mark.parametrize("inner,K,tiles", [(1300, 200, 10), (65, 72, 90), (640, 1024, 16), (64, 8, 200)])
@pytest.mark.parametrize("form", ["silu", "clamped_swish", "gelu_tanh"])
def test_gated_units_with_more_tiles_than_sms(inner, K, tiles, form):
    """Gate and up of a prompt: tiles of 128 rows that a block takes one after the other, some of them without rows."""
    groups = torch.randint(-1, 3, (tiles,), generator=torch.Generator().manual_seed(inner)).tolist()
    groups[0], groups[-1] = -1, 2
    a, w = randn(inner, 128 * tiles, K, dtype=torch.bfloat16), randn(K, 3, 2 * inner, K, scale=K ** -0.5)
    q = kernels.mx4_quantize(w.to(DEV))
    values = kernels.mx4_values(q, torch.float32).double()
    which = torch.tensor(groups, dtype=torch.int32, device=DEV)
    for dtype in (torch.bfloat16, torch.float32):
        out = torch.full((128 * tiles, inner), 7.0, dtype=dtype, device=DEV)
        kernels.gemm_grouped_mx4(a.to(DEV), q, which, 128, gated=(2.0, 1.702, form), out=out)
        for i, e in enumerate(groups):
            part = slice(128 * i, 128 * (i + 1))
            if e < 0:
                assert (out[part] == 7).all()
                continue
            rows = a[part].to(DEV).double()
            z, mass = rows @ values[e].t(), rows.abs() @ values[e].abs().t()
            bound = (K + 16) * 2.0 ** -23 * mass + 1e-30
            (gate, up), (bg, bu) = z.cpu().chunk(2, 1), bound.cpu().chunk(2, 1)
            want = gated(gate, up, 2.0, 1.702, form)
            close(out[part], want, 1.13 * (up.abs() + 1) * bg + (gate.abs() + 1) * bu + 2.0 ** -18 * (want.abs() + gate.abs()))

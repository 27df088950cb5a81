"""Microscaled 4-bit matrices: quantisation, the values back, and the products that read them, against float64.

Tolerances of the products: the elements' products are exact, their sums float32. With n terms of size |x w| a float32 sum in any
order is within n 2^-23 sum|x w| (the tensor cores cut off where they add: a whole step, not half of one); the tests use 8 chains of
at most K / 8 + 8 terms and 8 more additions that join them, so (K / 8 + 16) 2^-23 sum|x w|, and half a step of the output's
type, eps / 2 of the result, where it is stored."""
import pytest
import torch

from damendaemon_b200 import kernels
from mx4_tools import activation, gated, packed, quantized

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def randn(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g, dtype=torch.float64) * scale).to(dtype)


def close(got, want, bound):
    """bound: an absolute tolerance of every element, before the rounding to got's type."""
    off = (got.double().cpu() - want).abs()
    step = torch.finfo(got.dtype).eps / 2
    allowed = bound * (1 + step) + step * want.abs()
    worst = (off / (allowed + 1e-300)).max().item()
    assert worst <= 1, f"off by {worst} of what is allowed"


def product_bound(a, w, n_chains=8):
    K = a.shape[1]
    mass = a.double().abs() @ w.abs().t()
    return (K / n_chains + 8 + 8) * 2.0 ** -23 * mass + 1e-30


# ------------------------------------------------------------------ quantisation

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 31), (2, 32), (5, 33), (4, 100), (3, 128), (2, 129), (7, 256), (2, 1600)])
def test_quantize(rows, width, dtype):
    x = randn(rows * 1000 + width, rows, width, dtype=dtype) * torch.exp2(torch.arange(rows) * 5.0 - 7).unsqueeze(1).to(dtype)
    q = kernels.mx4_quantize(x.to(DEV))
    want, marks = quantized(x)
    codes, scales = packed(want, marks)
    assert q.shape == (rows, width)
    assert torch.equal(q.scales.cpu(), scales) and torch.equal(q.codes.cpu(), codes)
    for out in (torch.float32, torch.bfloat16):
        assert torch.equal(kernels.mx4_values(q, out).double().cpu(), want)


def test_quantize_ties_and_borders():
    """Middles between two numbers, both signs, beside a largest element that fixes the scale; sizes between 6 and 8."""
    middles = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 6.5, 7.0, 7.96875]
    near = [m * (1 + s * 2.0 ** -7) for m in middles for s in (-1, 0, 1)]
    for power in (-126, -120, -20, 0, 1, 20, 125):
        row = torch.tensor([4.0] + near[:15] + [-v for v in near[:16]] + [4.0] + near[15:] + [-7.96875], dtype=torch.float64)
        x = (row * 2.0 ** power).to(torch.float32).unsqueeze(0)
        want, marks = quantized(x)
        q = kernels.mx4_quantize(x.to(DEV))
        assert torch.equal(q.scales.cpu()[0, :marks.shape[1]].long(), marks[0])
        # (at the largest power the last middle is beyond float32's numbers: an infinity, whose block reads as NaN)
        assert torch.equal(kernels.mx4_values(q, torch.float32).double().cpu().nan_to_num(nan=-1.5), want.nan_to_num(nan=-1.5))


def test_quantize_smallest_largest_and_not_finite():
    top = torch.finfo(torch.float32).max
    x = torch.zeros(6, 64)
    x[1, 3], x[1, 40] = 2.0 ** -149, -2.0 ** -126
    x[2, 0], x[2, 1] = top, -1.0
    x[3, 5], x[3, 45] = float("inf"), 2.0
    x[4, 31], x[4, 32] = 1.0, float("nan")
    x[5, 7] = -0.0
    want, marks = quantized(x)
    q = kernels.mx4_quantize(x.to(DEV))
    assert torch.equal(q.scales.cpu()[:, :2].long(), marks)
    assert torch.equal(kernels.mx4_values(q, torch.float32).double().cpu().nan_to_num(nan=-1.5), want.nan_to_num(nan=-1.5))


def test_quantize_strided_stacked_and_again():
    x = randn(5, 6, 200).to(DEV)
    part = x[::2, 8:168]
    q = kernels.mx4_quantize(part)
    assert torch.equal(q.codes, kernels.mx4_quantize(part.contiguous()).codes)
    odd = x[:, 3:100]                                        # rows that start between 16-byte boundaries
    assert torch.equal(kernels.mx4_quantize(odd).codes, kernels.mx4_quantize(odd.contiguous()).codes)
    stack = randn(6, 3, 5, 96).to(DEV)
    single = stack[:, 0].contiguous().as_strided((3, 1, 96), (96, 1 << 20, 1))      # contiguous: a dimension of one has any stride
    assert torch.equal(kernels.mx4_quantize(single).codes, kernels.mx4_quantize(stack[:, :1].contiguous()).codes)
    q = kernels.mx4_quantize(stack)
    assert q.shape == (3, 5, 96)
    assert torch.equal(q.codes[1], kernels.mx4_quantize(stack[1]).codes)
    values = kernels.mx4_values(q)
    again = kernels.mx4_quantize(values)                     # what is on the grid stays, but for a block's largest power of two
    assert torch.equal(kernels.mx4_values(again), values)


# ------------------------------------------------------------------ the dense product

SHAPES = [(1, 16, 32), (1, 1, 1), (2, 17, 100), (3, 130, 128), (7, 33, 129), (8, 64, 256), (9, 65, 520), (13, 40, 1000), (16, 48, 1600),
          (17, 100, 384), (31, 257, 160), (33, 96, 2056), (61, 103, 1000), (64, 256, 640), (65, 129, 128), (100, 128, 64), (130, 200, 1600),
          (129, 384, 72), (257, 130, 1024), (300, 64, 33)]


@pytest.fixture(params=["rule", "tcgen05", "unpacked"])
def path(request, monkeypatch):
    """The kernel that the sizes choose; tcgen05 wherever it can run; the matrix turned into bfloat16 wherever it can."""
    if request.param != "rule":
        monkeypatch.setattr(kernels, "MX4_SMALL", 0)
        monkeypatch.setattr(kernels, "MX4_FEW_ROWS", 0)
        monkeypatch.setattr(kernels, "MX4_FUSED_ROWS", 1 << 30 if request.param == "tcgen05" else 0)


@pytest.mark.parametrize("M,N,K", SHAPES + [(300, 1100, 520), (64, 1600, 6400), (260, 2048, 1024)])
def test_gemm_mx4(path, M, N, K):
    a, w = randn(M + K, M, K, dtype=torch.bfloat16), randn(N + K, N, K, scale=K ** -0.5)
    q = kernels.mx4_quantize(w.to(DEV))
    values = kernels.mx4_values(q, torch.float32).double().cpu()
    want, bound = a.double() @ values.t(), product_bound(a, values)
    close(kernels.gemm_mx4(a.to(DEV), q, out_dtype=torch.float32), want, bound)
    close(kernels.gemm_mx4(a.to(DEV), q), want, bound)


@pytest.mark.parametrize("M,N,K", [(1, 33, 100), (8, 64, 256), (20, 130, 384), (70, 130, 264), (200, 100, 1000)])
@pytest.mark.parametrize("act", [None, "gelu_new", "gelu", "relu2", "tanh"])
def test_gemm_mx4_epilogue(path, M, N, K, act):
    a, w = randn(M, M, K, dtype=torch.bfloat16), randn(N, N, K, scale=K ** -0.5)
    bias, residual = randn(1, N), randn(2, M, N)
    q = kernels.mx4_quantize(w.to(DEV))
    values = kernels.mx4_values(q, torch.float32).double().cpu()
    z = a.double() @ values.t() + bias.double()
    want = activation(z, act) + residual.double()
    # the activations' slopes are at most 1.13 (relu2: 2 |z|), their own float32 error a few steps of their result
    slope = 2 * z.abs() + 1 if act == "relu2" else 1.13
    bound = (product_bound(a, values) + 2.0 ** -23 * z.abs()) * slope + 2.0 ** -20 * (z.abs() + want.abs() + 1)
    out = residual.to(DEV).clone()
    got = kernels.gemm_mx4(a.to(DEV), q, bias.to(DEV), out, act, torch.float32, out=out)       # added in place
    assert got.data_ptr() == out.data_ptr()
    close(got, want, bound)
    close(kernels.gemm_mx4(a.to(DEV), q, bias.to(DEV), residual.to(DEV), act), want, bound)


def test_gemm_mx4_strides_and_rows_beside(path):
    a, w = randn(3, 12, 600, dtype=torch.bfloat16).to(DEV), randn(4, 50, 200, scale=0.1).to(DEV)
    q = kernels.mx4_quantize(w)
    values = kernels.mx4_values(q, torch.float32).double().cpu()
    for part in (a[:, 200:400], a[:, 3:203], a[1:, 400:], a[::2, :200]):
        store = torch.full((part.shape[0], 70), 7.0, device=DEV)
        got = kernels.gemm_mx4(part, q, out_dtype=torch.float32, out=store[:, 5:55])
        # (rows that are no whole 16-byte pieces go through mma.sync whatever the path: not the same order of summing)
        close(got, part.double().cpu() @ values.t(), product_bound(part.cpu(), values))
        assert (store[:, :5] == 7).all() and (store[:, 55:] == 7).all()
    many = randn(8, 150, 200, dtype=torch.bfloat16).to(DEV)
    store = torch.full((152, 50), 7.0, device=DEV)
    kernels.gemm_mx4(many, q, out_dtype=torch.float32, out=store[:150])
    assert (store[150:] == 7).all()


@pytest.mark.parametrize("M", [1, 8, 40, 140])
def test_gemm_mx4_wide_scales(path, M):
    """Blocks whose scales lie far apart, weights above and below 1, large and small rows of a."""
    K = 512
    w = randn(1, 48, K) * torch.exp2(torch.randint(-40, 41, (48, K // 32), generator=torch.Generator().manual_seed(2)).repeat_interleave(32, 1).float())
    a = (randn(3, M, K) * torch.exp2(torch.arange(M) % 7 * 10.0 - 30).unsqueeze(1)).to(torch.bfloat16)
    q = kernels.mx4_quantize(w.to(DEV))
    values = kernels.mx4_values(q, torch.float32).double().cpu()
    close(kernels.gemm_mx4(a.to(DEV), q, out_dtype=torch.float32), a.double() @ values.t(), product_bound(a, values, 1))


@pytest.mark.parametrize("M,N,K", [(17, 96, 999), (40, 130, 1601), (200, 64, 97), (270, 140, 805), (300, 33, 7)])
def test_gemm_mx4_rows_of_no_whole_pieces(path, M, N, K):
    """More rows than go through mma.sync as they are: widths that are no multiple of 8, a stride or a start between 16-byte boundaries."""
    w = kernels.mx4_quantize(randn(K, N, K, scale=K ** -0.5).to(DEV))
    values = kernels.mx4_values(w, torch.float32).double().cpu()
    store, bias, residual = randn(M, M, K + 11, dtype=torch.bfloat16), randn(1, N), randn(2, M, N)
    for a in (store[:, :K].contiguous(), store[:, 3:K + 3], store[:, 8:K + 8]):
        want, bound = a.double() @ values.t(), product_bound(a, values)
        close(kernels.gemm_mx4(a.to(DEV) if a.is_contiguous() else store.to(DEV)[:, a.storage_offset():a.storage_offset() + K], w,
                               out_dtype=torch.float32), want, bound)
        got = kernels.gemm_mx4(a.to(DEV), w, bias.to(DEV), residual.to(DEV), None, torch.float32)
        close(got, want + bias.double() + residual.double(), bound + 2.0 ** -22 * (want.abs() + bias.abs() + residual.abs() + 1))


@pytest.mark.parametrize("M", [2, 70])
def test_gemm_mx4_not_finite(path, M):
    w, a = randn(1, 40, 160), randn(2, M, 160, dtype=torch.bfloat16)
    w[5, 70] = float("nan")
    a[1, 9] = float("inf")
    got = kernels.gemm_mx4(a.to(DEV), kernels.mx4_quantize(w.to(DEV)), out_dtype=torch.float32).cpu()
    fine = torch.ones(M, 40, dtype=torch.bool)
    fine[:, 5], fine[1, :] = False, False
    assert got[fine].isfinite().all() and not got[:, 5].isfinite().any()
    assert not got[1].isfinite().all()


def test_gemm_mx4_no_rows():
    q = kernels.mx4_quantize(randn(1, 40, 160).to(DEV))
    assert kernels.gemm_mx4(torch.empty((0, 160), dtype=torch.bfloat16, device=DEV), q).shape == (0, 40)


def test_gemm_mx4_replayed(path):
    """Captured once, replayed with other inputs, while the same call runs outside the graph."""
    q = kernels.mx4_quantize(randn(1, 200, 320).to(DEV))
    for M in (4, 90, 300):
        a = randn(M, M, 320, dtype=torch.bfloat16).to(DEV)
        kernels.gemm_mx4(a, q)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = kernels.gemm_mx4(a, q)
        for seed in (5, 6):
            a.copy_(randn(seed, M, 320, dtype=torch.bfloat16))
            graph.replay()
            assert torch.equal(out, kernels.gemm_mx4(a, q))


# ------------------------------------------------------------------ grouped products

@pytest.mark.parametrize("tile", [16, 32, 64, 128])
@pytest.mark.parametrize("N,K", [(1, 8), (100, 64), (128, 72), (130, 136), (257, 520), (64, 1600)])
def test_grouped(tile, N, K):
    groups = [2, 0, -1, 1, 1, 2, -1]
    rows = tile * len(groups)
    a, w = randn(N + K, rows, K, dtype=torch.bfloat16), randn(N + K + 1, 3, N, K, scale=K ** -0.5)
    scale = randn(9, rows).abs()
    q = kernels.mx4_quantize(w.to(DEV))
    values = kernels.mx4_values(q, torch.float32).double().cpu()
    tiles = torch.tensor(groups, dtype=torch.int32, device=DEV)
    for act, row_scale, dtype in ((None, None, torch.bfloat16), (None, scale, torch.float32), ("relu2", scale, torch.float32), ("gelu", None, torch.bfloat16)):
        out = torch.full((rows, N), 7.0, dtype=dtype, device=DEV)
        got = kernels.gemm_grouped_mx4(a.to(DEV), q, tiles, tile, activation=act, out_dtype=dtype, out=out,
                                       row_scale=None if row_scale is None else row_scale.to(DEV))
        assert got is out
        for i, e in enumerate(groups):
            part = slice(i * tile, (i + 1) * tile)
            if e < 0:
                assert (got[part] == 7).all()
                continue
            by = 1.0 if row_scale is None else row_scale[part].double().unsqueeze(1)
            z = a[part].double() @ values[e].t() * by
            want = activation(z, act)
            slope = 2 * z.abs() + 1 if act == "relu2" else 1.13
            close(got[part], want, product_bound(a[part], values[e]) * by * slope + 2.0 ** -20 * (z.abs() + want.abs()))


@pytest.mark.parametrize("tile", [16, 32, 64, 128])
@pytest.mark.parametrize("inner,K", [(1, 8), (100, 64), (130, 200), (128, 520), (65, 1600)])
@pytest.mark.parametrize("form", ["silu", "clamped_swish", "gelu_tanh"])
def test_grouped_gated(tile, inner, K, form):
    groups = [1, -1, 0, 1]
    rows = tile * len(groups)
    a, w = randn(inner + K, rows, K, dtype=torch.bfloat16), randn(inner + K + 1, 2, 2 * inner, K, scale=K ** -0.5)
    q = kernels.mx4_quantize(w.to(DEV))
    values = kernels.mx4_values(q, torch.float32).double().cpu()
    tiles = torch.tensor(groups, dtype=torch.int32, device=DEV)
    for dtype in (torch.bfloat16, torch.float32):
        got = kernels.gemm_grouped_mx4(a.to(DEV), q, tiles, tile, gated=(2.0, 1.702, form), out_dtype=dtype)
        for i, e in enumerate(groups):
            if e < 0:
                continue
            part = slice(i * tile, (i + 1) * tile)
            z, bound = a[part].double() @ values[e].t(), product_bound(a[part], values[e])
            (gate, up), (bg, bu) = z.chunk(2, 1), bound.chunk(2, 1)
            want = gated(gate, up, 2.0, 1.702, form)
            # the unit's slopes: at most 1.13 (|up| + 1) by the gate, |gate| + 1 by up; its exponential is the special-function unit's, 2^-20
            close(got[part], want, 1.13 * (up.abs() + 1) * bg + (gate.abs() + 1) * bu + 2.0 ** -18 * (want.abs() + gate.abs()))


@pytest.mark.parametrize("N,K,tiles", [(2500, 200, 10), (130, 72, 90), (1300, 1024, 16)])
def test_grouped_with_more_tiles_than_sms(N, K, tiles):
    """Tiles of 128 rows that a block takes one after the other, some of them without rows, at either end and in between."""
    g = torch.Generator().manual_seed(N)
    groups = torch.randint(-1, 3, (tiles,), generator=g).tolist()
    groups[0], groups[-1] = -1, 2
    a, w = randn(N, 128 * tiles, K, dtype=torch.bfloat16), randn(K, 3, N, K, scale=K ** -0.5)
    scale = randn(7, 128 * tiles).abs()
    q = kernels.mx4_quantize(w.to(DEV))
    values = kernels.mx4_values(q, torch.float32).double().cpu()
    which = torch.tensor(groups, dtype=torch.int32, device=DEV)
    for dtype, by, act in ((torch.float32, None, None), (torch.bfloat16, scale, "relu2")):
        out = torch.full((128 * tiles, N), 7.0, dtype=dtype, device=DEV)
        kernels.gemm_grouped_mx4(a.to(DEV), q, which, 128, activation=act, row_scale=None if by is None else by.to(DEV), out=out)
        for i, e in enumerate(groups):
            part = slice(128 * i, 128 * (i + 1))
            if e < 0:
                assert (out[part] == 7).all()
                continue
            f = 1.0 if by is None else by[part].double().unsqueeze(1)
            z = a[part].double() @ values[e].t() * f
            want = activation(z, act)
            slope = 2 * z.abs() + 1 if act else 1.0
            close(out[part], want, product_bound(a[part], values[e], 1) * f * slope + 2.0 ** -20 * (z.abs() + want.abs()))


@pytest.mark.parametrize("tile,tiles,gated", [(16, 3, None), (128, 3, None), (128, 200, None), (64, 3, (1.0, 1.0, "silu"))])
def test_grouped_without_such_a_matrix(tile, tiles, gated):
    """A group out of range is an error that the device reports; its rows stay, the others are computed."""
    q = kernels.mx4_quantize(randn(1, 2, 130, 64).to(DEV))
    a = randn(2, tile * tiles, 64, dtype=torch.bfloat16).to(DEV)
    which = torch.ones(tiles, dtype=torch.int32, device=DEV)
    want = kernels.gemm_grouped_mx4(a, q, which, tile, gated)
    assert kernels.read_error_flag(DEV) == 0
    which[1] = 2
    out = torch.full_like(want, 7.0)
    kernels.gemm_grouped_mx4(a, q, which, tile, gated, out=out)
    assert kernels.read_error_flag(DEV) == 1
    assert (out[tile:2 * tile] == 7).all() and torch.equal(out[:tile], want[:tile]) and torch.equal(out[2 * tile:], want[2 * tile:])


def test_grouped_refusals():
    q = kernels.mx4_quantize(randn(1, 2, 32, 64).to(DEV))
    a, tiles = torch.zeros(32, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    for bad in (lambda: kernels.gemm_grouped_mx4(a, q, tiles, 32), lambda: kernels.gemm_grouped_mx4(a, q, tiles, 8),
                lambda: kernels.gemm_grouped_mx4(a[:, :60], q, tiles, 16), lambda: kernels.gemm_grouped_mx4(a.float(), q, tiles, 16),
                lambda: kernels.gemm_grouped_mx4(a, q, tiles, 16, gated=(1.0, 1.0), activation="relu2"),
                lambda: kernels.gemm_grouped_mx4(a, q, tiles.long(), 16), lambda: kernels.gemm_grouped_mx4(a, q, tiles, 16, out=a)):
        with pytest.raises(kernels.KernelError):
            bad()
    odd = kernels.mx4_quantize(randn(1, 2, 32, 60).to(DEV))
    with pytest.raises(kernels.KernelError, match="multiples of 8"):
        kernels.gemm_grouped_mx4(a[:, :60], odd, tiles, 16)

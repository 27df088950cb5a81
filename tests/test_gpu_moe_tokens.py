"""Whole expert layers for one to eight tokens against the formula in float64, and their refusals.

Tolerance: a product's float32 sum of n terms, in chains of at most n / 8 + 16, is within (n / 8 + 16) 2^-23 of the sum of its terms'
sizes (the tensor cores cut off where they add). The hidden rows' own error goes through the down product: with slope 2 at most for the units
at these sizes (|gate|, |up| below 4), relative to the sum of sizes of the up products; the bfloat16 terms of a hidden value
(two would do) keep 2^-17 of it. Every bound below is that sum of sizes, computed beside the result."""
import pytest
import torch

from damendaemon_b200 import kernels
from mx4_tools import activation, gated

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
KINDS = {"float32": torch.float32, "bfloat16": torch.bfloat16, "mx4": torch.bfloat16}


class Layer:
    """Random tensors of one expert layer; ``layer`` for the kernels, ``plain`` in float64."""

    def __init__(self, kind, width, inner, experts, top, unit="silu", shared=0, seed=0, table=None, **options):
        g = torch.Generator().manual_seed(seed)
        randn = lambda *s, scale=1.0: torch.randn(s, generator=g) * scale  # noqa: E731
        self.kind, self.dtype, self.unit, self.top, self.options = kind, KINDS[kind], unit, top, options
        halves = 1 if unit in ("relu2", "gelu_new", "none") else 2
        self.experts, self.identity = experts, options.get("identity", 0)

        def matrix(*shape):
            w = randn(*shape, scale=shape[-1] ** -0.5).to(self.dtype).to(DEV)
            if kind != "mx4":
                return w, w.double().cpu()
            q = kernels.mx4_quantize(w)
            return q, kernels.mx4_values(q, torch.float32).double().cpu()

        self.gate_up = matrix(experts, halves * inner, width)
        self.down = matrix(experts, width, inner)
        self.shared = (matrix(2 * shared, width), matrix(width, shared)) if shared else None
        self.form = (3.0, 1.702, unit) if halves == 2 else None
        shared_form = (2.5, 1.3, "clamped_swish" if unit == "silu" else "silu")
        self.shared_form = shared_form
        self.table = self.router = None
        options = dict(options)
        if table is not None:
            self.table = table if torch.is_tensor(table) else torch.randint(0, experts, (table, top), generator=g, dtype=torch.int32)
            options["table"] = self.table.to(DEV)
        else:
            rows = experts + self.identity + bool(options.get("shared_gate"))
            self.router = randn(rows, width, scale=2 * width ** -0.5).to(self.dtype)
            options["router"] = self.router.to(DEV)
        self.correction = None
        if options.get("correction"):
            self.correction = randn(experts + self.identity, scale=0.1)
            options["correction"] = self.correction.to(DEV)
        else:
            options.pop("correction", None)
        self.layer = kernels.ExpertLayer(self.gate_up[0], self.down[0], top, gated=self.form, activation=None if self.form else unit,
                                         shared=None if not shared else (self.shared[0][0], self.shared[1][0]), shared_gated=shared_form,
                                         **options)

    def unit_of(self, w, y, by=1.0, form=None):
        """(value, a bound of its error) of a unit's product z = W y."""
        n = y.numel()
        z, mass = w @ y, w.abs() @ y.abs()
        err = (n / 8 + 16) * 2.0 ** -23 * mass
        form = form or self.form
        if form is None:
            v = activation(z * by, None if self.unit == "none" else self.unit)
            slope = 2 * (z * by).abs() + 1 if self.unit == "relu2" else 1.13
            return v, err * by * slope + 2.0 ** -20 * (v.abs() + z.abs() * by)
        gate, up = z.chunk(2)
        v = gated(gate, up, *form)
        eg, eu = err.chunk(2)
        return v, 1.5 * (eg * (up.abs() + 1.1) + eu * (gate.abs() + 1)) + 2.0 ** -20 * (v.abs() + gate.abs())

    def route(self, y, ids):
        """Per token [(expert, weight)], the shared unit's gate, and the narrowest gap between a chosen and an unchosen score."""
        o = self.options
        if self.table is not None:
            scale = o.get("weight_scale", 1.0) / self.top
            return [[(int(e), scale) for e in self.table[int(i)]] for i in ids], [1.0] * len(ids), 1.0
        E = self.experts + self.identity
        z = y @ self.router.double().t()
        gates = torch.sigmoid(z[:, E]).tolist() if o.get("shared_gate") else [1.0] * len(y)
        score = torch.softmax(z[:, :E], 1) if o.get("softmax") else torch.sigmoid(z[:, :E])
        order = score + self.correction.double() if self.correction is not None else score
        chosen, gap = [], 1.0
        for t in range(len(y)):
            groups, keep = o.get("groups", 1), o.get("keep", 1)
            per = E // groups
            worth = [sum(sorted(order[t, i * per:(i + 1) * per].tolist())[-2:]) for i in range(groups)]
            kept = sorted(range(groups), key=lambda i: (-worth[i], i))
            if keep < groups:
                gap = min(gap, worth[kept[keep - 1]] - worth[kept[keep]])
            ranked = sorted((e for e in range(E) if e // per in kept[:keep]), key=lambda e: (-float(order[t, e]), e))
            if len(ranked) > self.top:
                gap = min(gap, float(order[t, ranked[self.top - 1]] - order[t, ranked[self.top]]))
            weights = [float(score[t, e]) for e in ranked[:self.top]]
            total = sum(weights) + 1e-20 if o.get("renormalize") else 1.0
            chosen.append([(e, w / total * o.get("weight_scale", 1.0)) for e, w in zip(ranked, weights)])
        return chosen, gates, gap

    def plain(self, y, residual, ids=None):
        y = y.double()
        chosen, gates, gap = self.route(y, ids)
        assert gap > 1e-5, "the case leaves a choice to rounding"
        out, bound = residual.double().clone(), 2.0 ** -23 * residual.double().abs() + 1e-30
        down, down_abs = self.down[1], self.down[1].abs()

        def add(t, value, err, w, w_abs, weight):
            out[t] += weight * (w @ value)
            n = value.numel()
            lost = 0.0 if self.kind == "float32" else 2.0 ** -17
            bound[t] += weight * (w_abs @ (err + (lost + (n * 2 / 8 + 24) * 2.0 ** -23 + 2.0 ** -20) * value.abs()))

        for t in range(len(y)):
            for e, weight in chosen[t]:
                if e >= self.experts:
                    out[t] += weight * y[t]
                    bound[t] += 2.0 ** -18 * weight * y[t].abs()
                    continue
                inside = self.options.get("weight_input")
                value, err = self.unit_of(self.gate_up[1][e], y[t], weight if inside else 1.0)
                add(t, value, err, down[e], down_abs[e], 1.0 if inside else weight)
            if self.shared:
                value, err = self.unit_of(self.shared[0][1], y[t], form=self.shared_form)
                add(t, value, err, self.shared[1][1], self.shared[1][1].abs(), gates[t])
            bound[t] += 2.0 ** -20 * out[t].abs()       # the weights' own float32 error, and the additions of the parts
        return out, bound

    def check(self, T, seed=1, ids=None):
        g = torch.Generator().manual_seed(seed)
        width = self.down[1].shape[1]
        y = torch.randn((T, width), generator=g).to(self.dtype)
        residual = torch.randn((T, width), generator=g)
        if self.table is not None and ids is None:
            ids = torch.randint(0, self.table.shape[0], (T,), generator=g, dtype=torch.int32)
        got = kernels.moe_tokens(self.layer, y.to(DEV), residual.to(DEV), None if ids is None else ids.to(DEV))
        want, bound = self.plain(y, residual, ids)
        assert kernels.read_error_flag(DEV) == 0
        worst = ((got.double().cpu() - want).abs() / bound).max().item()
        assert worst <= 1, f"off by {worst} of what is allowed"
        return y, residual, ids, got


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("options", [dict(top=2, groups=4, keep=2, weight_scale=2.5, shared=40, shared_gate=True),
                                     dict(top=3, unit="clamped_swish", softmax=True, correction=True, renormalize=True, identity=4),
                                     dict(top=2, unit="relu2", weight_input=True),
                                     dict(top=2, unit="clamped_swish", table=50, shared=72),
                                     dict(top=1, unit="gelu_tanh")])
def test_layer(kind, T, options):
    Layer(kind, 96, 64, 8, **options).check(T)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("width,inner,experts,top,shared", [(1, 1, 1, 1, 1), (7, 3, 3, 2, 5), (8, 8, 2, 1, 0), (33, 17, 5, 5, 31), (100, 130, 4, 2, 100),
                                                            (128, 32, 17, 4, 0), (136, 264, 20, 6, 24), (520, 104, 66, 8, 0), (260, 44, 16, 16, 12),
                                                            (1600, 96, 16, 2, 96), (64, 1000, 6, 2, 0), (2048, 40, 130, 6, 0)])
def test_sizes(kind, width, inner, experts, top, shared):
    # (a router of width 1 and 7 leaves near ties: tokens chosen by a table there)
    table = {"table": 30} if width < 30 else {}
    layer = Layer(kind, width, inner, experts, top, shared=shared, seed=width, **table)
    for T in (1, 4, 8):
        layer.check(T, seed=T)


@pytest.mark.parametrize("kind", KINDS)
def test_every_expert_by_every_token_and_one_for_all(kind):
    Layer(kind, 64, 48, 4, 4, softmax=True).check(8)
    table = torch.full((20, 3), 2, dtype=torch.int32)
    table[:, 1], table[:, 2] = 0, 2                     # expert 2 twice: its weights add up
    Layer(kind, 64, 48, 4, 3, table=table).check(8)
    Layer(kind, 64, 48, 2, 1, identity=62, softmax=True, unit="silu").check(8)


def test_all_identity():
    """Where every choice is an identity output no matrix is read."""
    layer = Layer("bfloat16", 64, 48, 1, 1, identity=1, softmax=True, correction=True)
    layer.correction[:] = torch.tensor([-5.0, 5.0])
    layer.layer.tensors[4].copy_(layer.correction)
    layer.check(6)


@pytest.mark.parametrize("kind", KINDS)
def test_in_place_strides_and_nothing_to_add_to(kind):
    layer = Layer(kind, 96, 64, 8, 2, shared=40)
    y, residual, _, got = layer.check(5)
    wide = torch.zeros(5, 300, dtype=y.dtype, device=DEV)
    for at in (0, 8, 101):
        wide[:, at:at + 96] = y.to(DEV)
        assert torch.equal(kernels.moe_tokens(layer.layer, wide[:, at:at + 96], residual.to(DEV)), got)
    stream = torch.full((7, 120), 3.0, device=DEV)
    stream[:5, 10:106] = residual.to(DEV)
    part = stream[:5, 10:106]
    assert kernels.moe_tokens(layer.layer, y.to(DEV), part, out=part).data_ptr() == part.data_ptr()
    assert torch.equal(part, got) and (stream[5:] == 3).all() and (stream[:, :10] == 3).all() and (stream[:, 106:] == 3).all()
    bare = kernels.moe_tokens(layer.layer, y.to(DEV))
    want, bound = layer.plain(y, torch.zeros_like(residual))
    assert ((bare.double().cpu() - want).abs() <= bound).all()
    assert kernels.moe_tokens(layer.layer, y[:0].to(DEV)).shape == (0, 96)


@pytest.mark.parametrize("kind", KINDS)
def test_a_token_has_the_same_bits_alone_and_again(kind):
    """No atomics: the same call gives the same bits, whatever ran in between."""
    layer = Layer(kind, 264, 200, 16, 2, shared=64)
    y, residual, _, got = layer.check(8)
    Layer(kind, 96, 64, 8, 3).check(3)
    for _ in range(3):
        assert torch.equal(kernels.moe_tokens(layer.layer, y.to(DEV), residual.to(DEV)), got)


@pytest.mark.parametrize("kind", KINDS)
def test_a_matrix_that_is_not_finite_stays_with_its_tokens(kind):
    table = torch.tensor([[0, 1], [1, 2]], dtype=torch.int32)
    layer = Layer(kind, 96, 64, 3, 2, table=table, shared=40)
    y, residual, ids, got = layer.check(4, ids=torch.tensor([0, 1, 0, 1], dtype=torch.int32))
    for stack in (layer.gate_up[0], layer.down[0]):
        if kind == "mx4":
            stack.scales[0].fill_(255)
        else:
            stack[0].fill_(float("nan"))
        again = kernels.moe_tokens(layer.layer, y.to(DEV), residual.to(DEV), ids.to(DEV))
        assert torch.equal(again[1::2], got[1::2]) and not again[::2].isfinite().any()


def test_out_of_range_is_reported_and_left_out():
    table = torch.tensor([[0, 1], [1, 9], [-1, 0]], dtype=torch.int32)
    layer = Layer("float32", 32, 16, 2, 2, table=table)
    y = torch.randn(4, 32)
    got = kernels.moe_tokens(layer.layer, y.to(DEV), ids=torch.tensor([0, 1, 2, 7], dtype=torch.int32, device=DEV))
    assert kernels.read_error_flag(DEV) == 1 and kernels.read_error_flag(DEV) == 0
    layer.table = torch.tensor([[0, 1], [1, 1], [0, 0], [0, 0]])
    whole, bound = layer.plain(y, torch.zeros(4, 32), [0, 1, 2, 3])
    assert ((got[:1].double().cpu() - whole[:1]).abs() <= bound[:1]).all()
    assert ((got[1:3].double().cpu() - whole[1:3] / 2).abs() <= bound[1:3]).all() and (got[3] == 0).all()
    layer = Layer("bfloat16", 32, 16, 4, 2)
    y = torch.randn(2, 32).bfloat16().to(DEV)
    y[1, 3] = float("nan")
    got = kernels.moe_tokens(layer.layer, y)
    assert kernels.read_error_flag(DEV) == 1 and got[0].isfinite().all()


@pytest.mark.parametrize("kind", KINDS)
def test_replayed_beside_eager_calls_and_another_graph(kind):
    layer, other = Layer(kind, 264, 200, 16, 2, shared=64), Layer(kind, 96, 64, 8, 3, softmax=True)
    graphs = []
    for part, T in ((layer, 6), (other, 3)):
        y, residual, _, _ = part.check(T)
        y, residual = y.to(DEV), residual.to(DEV)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = kernels.moe_tokens(part.layer, y, residual)
        graphs.append((graph, part, y, residual, out))
    side = torch.cuda.Stream()
    for seed in (5, 6):
        for _, part, y, residual, _ in graphs:
            y.copy_(torch.randn(y.shape, generator=torch.Generator().manual_seed(seed)))
        torch.cuda.synchronize()
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
            eager = kernels.moe_tokens(layer.layer, graphs[0][2], graphs[0][3])
        torch.cuda.synchronize()
        assert torch.equal(eager, graphs[0][4])
        for _, part, y, residual, out in graphs:
            assert torch.equal(out, kernels.moe_tokens(part.layer, y, residual))


def test_a_form_of_two_numbers_is_the_clamped_one():
    layer = Layer("bfloat16", 64, 32, 4, 2, unit="clamped_swish")
    y, residual, _, got = layer.check(3)
    short = kernels.ExpertLayer(layer.gate_up[0], layer.down[0], 2, gated=layer.form[:2], router=layer.router.to(DEV))
    assert torch.equal(kernels.moe_tokens(short, y.to(DEV), residual.to(DEV)), got)


def test_refusals():
    layer = Layer("bfloat16", 32, 16, 4, 2)
    y = torch.zeros(3, 32, dtype=torch.bfloat16, device=DEV)
    for bad in (lambda: kernels.moe_tokens(layer.layer, y.float()), lambda: kernels.moe_tokens(layer.layer, y[:, :30]),
                lambda: kernels.moe_tokens(layer.layer, torch.zeros(9, 32, dtype=torch.bfloat16, device=DEV)),
                lambda: kernels.moe_tokens(layer.layer, y, ids=torch.zeros(3, dtype=torch.int32, device=DEV)),
                lambda: kernels.moe_tokens(layer.layer, y, torch.zeros(2, 32, device=DEV)),
                lambda: kernels.moe_tokens(layer.layer, y, out=torch.zeros(3, 32, device=DEV, dtype=torch.bfloat16)),
                lambda: kernels.moe_tokens(layer.layer, y.cpu())):
        with pytest.raises(kernels.KernelError):
            bad()

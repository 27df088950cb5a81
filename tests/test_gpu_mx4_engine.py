"""Models whose feed-forwards are held in 4 bits, through the engine: against the plain implementation with the matrices that the
4-bit numbers stand for, under several ways of cutting the work, so that one token, a few and many go through the products of each; and
the expert parts of a few tokens beside the kernels of larger steps."""
import inspect
import types

import pytest
import torch

import bonatar_tools
import dozetar_tools
import godotar_tools
import plain_bonatar
import plain_dozetar
import plain_godotar
import plain_zokanex
import zokanex_tools
from conftest import TINY_A
from model_tools import make_model, random_requests
from plain_gpt2 import PlainGpt2
from trace_tools import mixed_steps, portion_steps, tail_steps, whole_steps

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FAMILIES = {"bonatar": (bonatar_tools, plain_bonatar, "PRSU"), "zokanex": (zokanex_tools, plain_zokanex, "PRT"),
            "godotar": (godotar_tools, plain_godotar, "ACE"), "dozetar": (dozetar_tools, plain_dozetar, "ACE")}
CASES = [(f, n) for f, (_, _, names) in FAMILIES.items() for n in names]


def feed_forward_matrices(config):
    """The checkpoint names of every matrix that a feed-forward multiplies with (not its router)."""
    from damendaemon_b200.registry import architecture_of
    arch = architecture_of(config)
    names = set()
    for layer in arch.build_spec(arch.parse_config(config)).layers:
        f = layer.feed_forward
        units = list(getattr(f, "experts", ())) + [u for u in (getattr(f, "shared", None), getattr(f, "unit", None)) if u is not None]
        units += [f] if f.kind == "dense" else []
        for u in units:
            names |= {getattr(u, k) for k in ("gate_weight", "up_weight", "down_weight") if getattr(u, k, None)}
    return names


def rounded(tensors, names):
    from damendaemon_b200 import kernels
    out = dict(tensors)
    for n in names:
        out[n] = kernels.mx4_values(kernels.mx4_quantize(tensors[n].to(DEV, torch.bfloat16).contiguous()), torch.float32).cpu()
    return out


@pytest.fixture(scope="module")
def models():
    out = {}
    for family, name in CASES:
        tools, plain, _ = FAMILIES[family]
        config = tools.CONFIGS[name]
        more = {"decided": True} if "decided" in inspect.signature(tools.make_tensors).parameters else {}
        tensors = tools.make_tensors(config, seed=5 + ord(name), dtype=torch.bfloat16, **more)
        held = rounded(tensors, feed_forward_matrices(config))
        requests = tools.random_requests(config, [1, 6, 25, 60, 130], 11)
        reference = tools.plain_tensors(held)
        want = {r: plain.forward(config, reference, t).float() for r, t in requests.items()}
        # a row's root mean square error, against three times what rounding the activations to bfloat16 does to the plain rows
        plain.ROUND = torch.bfloat16
        moved = max((plain.forward(config, reference, t).float() - want[r]).square().mean(-1).sqrt().max().item() for r, t in requests.items())
        plain.ROUND = None
        # what the rounding to 4 bits itself moves: a model that was not rounded would be this far off
        apart = max((plain.forward(config, tools.plain_tensors(tensors), t).float() - want[r]).square().mean(-1).sqrt().max().item()
                    for r, t in requests.items())
        out[family, name] = (config, tensors, requests, want, 3.0 * moved + 5e-3, apart)
    return out


def replay(engine, builder):
    from damendaemon_b200.engine import StepEntry
    got = {}
    for s in builder.steps:
        entries = [StepEntry(e["id"], e["tokens"], e["want"]) for e in s["entries"]]
        if entries:
            logits = engine.step(entries).cpu()
            for (request, position), row in zip(builder.where[s["step"]], logits):
                got.setdefault(request, {})[position] = row
        for r in s["end"]:
            engine.finish(r)
    return got


@pytest.mark.parametrize("family,name", CASES)
def test_every_cutting(models, family, name):
    from damendaemon_b200.engine import Engine
    config, tensors, requests, want, tol, apart = models[family, name]
    builder, peak = mixed_steps(requests, seed=3, max_live=4)
    for steps, graph in ((whole_steps(requests), False), (tail_steps(requests, tail=30), True), (portion_steps(requests), False), (builder, True)):
        engine = Engine(config=config, tensors=tensors, dtype="bfloat16", kv_tokens=max(320, peak), max_requests=4, use_graph=graph, feed_forward="mx4")
        got = replay(engine, steps)
        for r in want:
            for p, row in got[r].items():
                off = (row - want[r][p]).square().mean().sqrt().item()
                assert off < tol, f"request {r} position {p}: {off} (allowed {tol}; the rounding to 4 bits alone moves {apart})"


@pytest.mark.parametrize("family,name", [("zokanex", "R"), ("bonatar", "S")])
def test_held_bytes(models, family, name):
    from damendaemon_b200.engine import Engine
    config, tensors, *_ = models[family, name]
    whole, held = (Engine(config=config, tensors=tensors, kv_tokens=64, max_requests=2, feed_forward=f).weight_bytes for f in ("auto", "mx4"))
    matrices = sum(tensors[n].numel() for n in feed_forward_matrices(config))
    assert whole - held > matrices * (2 - 17 / 32) * 0.5          # (rows are padded to 128 elements)


def test_gpt2_generates_the_same_from_a_folder_and_the_command_line(tmp_path):
    """Greedy tokens of a 4-bit engine beside the plain model with the rounded matrices; where they part, the plain logits nearly tie."""
    import json
    import subprocess
    import sys
    from pathlib import Path
    from damendaemon_b200.runtime import Runtime, generate
    folder = make_model(tmp_path / "A", TINY_A, 0, "bfloat16")
    plain = PlainGpt2(folder)
    from damendaemon_b200 import kernels
    for name, w in list(plain.w.items()):
        if ".mlp." in name and w.dim() == 2:                       # stored [in, out]: the engine holds the transpose
            q = kernels.mx4_quantize(w.t().to(DEV, torch.bfloat16).contiguous())
            plain.w[name] = kernels.mx4_values(q, torch.float32).cpu().to(w.dtype).t()
    prompts = list(random_requests(TINY_A, [5, 17, 33], 7).values())
    got = Runtime(folder, max_batch=4, feed_forward="mx4").generate_batch(prompts, 12, ignore_eos=True)
    for p, tokens in zip(prompts, got):
        want = plain.greedy(p, 12)
        if tokens != want:
            i = next(i for i in range(12) if tokens[i] != want[i])
            row = plain.logits(p + want[:i])[-1]
            assert abs(float(row[tokens[i]] - row[want[i]])) < 4e-2
    assert generate(folder, prompts[:1], 4, feed_forward="mx4") == [got[0][:4]]
    run = subprocess.run([sys.executable, "-m", "damendaemon_b200", "run", str(folder), "--prompt-ids", ",".join(map(str, prompts[0])), "--max-tokens", "4",
                          "--ignore-eos", "--context", "64", "--feed-forward", "mx4"], capture_output=True, text=True, timeout=300,
                         cwd=Path(__file__).resolve().parent.parent)
    assert run.returncode == 0, run.stderr
    assert [int(t) for t in run.stdout.split()] == got[0][:4]
    assert json.loads(run.stderr.strip().splitlines()[-1])["finish_reason"] == "length"


def test_refused():
    from damendaemon_b200.engine import Engine
    config = bonatar_tools.CONFIGS["P"]
    tensors = bonatar_tools.make_tensors(config, 1)
    for more in (dict(dtype="float32"), dict(gemm="simt"), dict(feed_forward="int4")):
        with pytest.raises(ValueError):
            Engine(config=config, tensors=tensors, **{"kv_tokens": 64, "feed_forward": "mx4", **more})
    odd = bonatar_tools.CONFIGS["T"]                               # experts of 30 features: no whole 16-byte rows
    with pytest.raises(ValueError, match="multiples of 8"):
        Engine(config=odd, tensors=bonatar_tools.make_tensors(odd, 1), kv_tokens=64, feed_forward="mx4")


# ------------------------------------------------------------------ few tokens beside many

def part(dtype, kind, mx4=False, width=1024, inner=1024):
    """An expert part with random weights."""
    from damendaemon_b200.parts.feed_forward import ScoreRoutedExperts, TableRoutedExperts
    from damendaemon_b200.parts.interfaces import Runtime
    from damendaemon_b200.parts.spec import GatedUnitSpec, PlainUnitSpec, ScoreRoutedExpertsSpec, TableRoutedExpertsSpec
    g = torch.Generator().manual_seed(3)
    weights = {}

    def matrix(name, *shape):
        weights[name] = (torch.randn(shape, generator=g) * shape[-1] ** -0.5).to(DEV, dtype)
        return name
    unit = lambda p, n: GatedUnitSpec(n, 3.0, matrix(p + "g", n, width), matrix(p + "u", n, width), matrix(p + "d", width, n))  # noqa: E731
    if kind == "input":
        units = tuple(PlainUnitSpec(inner, matrix(f"{i}u", inner, width), matrix(f"{i}d", width, inner), "relu2") for i in range(6))
    else:
        units = tuple(unit(f"e{i}", inner) for i in range(6))
    runtime = Runtime(dtype=dtype, device=torch.device(DEV), feed_forward="mx4" if mx4 else "auto")
    if kind == "table":
        weights["table"] = torch.randint(0, 6, (40, 2), generator=g, dtype=torch.int32).to(DEV)
        return TableRoutedExperts(TableRoutedExpertsSpec("experts_by_table", width, 40, 2, "table", units, unit("s", 256)), weights, runtime)
    options = dict(groups=dict(groups=3, keep_groups=2, weight_scale=1.5, shared=unit("s", 256), shared_gate="sg") if kind == "groups" else {},
                   identity=dict(score="softmax", correction="c", renormalize=True, identity=2), input=dict(weight_input=True))[kind if kind != "groups" else "groups"]
    spec = ScoreRoutedExpertsSpec("experts_by_score", width, 2, "r", units, **options)
    rows = 6 + spec.identity
    weights["r"] = (2 * torch.randn((rows, width), generator=g) * width ** -0.5).to(DEV, dtype)
    if kind == "groups":
        weights["r+sg"] = torch.cat([weights["r"], torch.randn((1, width), generator=g).to(DEV, dtype) * width ** -0.5])
    if kind == "identity":
        weights["c"] = (0.05 * torch.randn(rows, generator=g)).to(DEV)
    return ScoreRoutedExperts(spec, weights, runtime)


@pytest.mark.parametrize("kind", ["table", "groups", "identity", "input"])
@pytest.mark.parametrize("dtype,mx4", [(torch.float32, False), (torch.bfloat16, False), (torch.bfloat16, True)])
def test_few_tokens_beside_the_kernels_of_larger_steps(kind, dtype, mx4):
    """The same part with and without its two-kernel form. The other kernels round hidden rows to bfloat16: 2^-9 of their size on
    average, which a sum over 1,024 features of random signs keeps relative to the sum's size; four times that is allowed, and in
    float32 the two orders of summing."""
    from damendaemon_b200 import kernels
    feed = part(dtype, kind, mx4)
    assert feed.few is not None
    g = torch.Generator().manual_seed(4)
    for n in (1, 3, 8):
        y, x = torch.randn((n, 1024), generator=g).to(DEV, dtype), torch.randn((n, 1024), generator=g).to(DEV)
        ctx = types.SimpleNamespace(token_ids=torch.randint(0, 40, (n,), generator=g, dtype=torch.int32).to(DEV))
        before = kernels.launches
        got = feed.forward(y, x.clone(), ctx)
        assert kernels.launches - before == 2
        few, feed.few = feed.few, None
        want = feed.forward(y, x.clone(), ctx)
        feed.few = few
        added, off = (want - x).square().mean().sqrt().item(), (got - want).square().mean().sqrt().item()
        assert off < added * (2.0 ** -7 if dtype == torch.bfloat16 else 1e-5), (off, added)
        bare = feed.forward(y, None, ctx)
        assert (bare + x - got).abs().max().item() < 1e-5 * (1 + got.abs().max().item())

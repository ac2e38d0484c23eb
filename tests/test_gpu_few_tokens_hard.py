"""GPU tests of moe_few_tokens with hard inputs on shapes of every kernel: the tiles of both products and the sum over the slots
among them, which few of the other tests' inputs reach."""
import numpy as np
import pytest
import torch

from commbench_amd import ops

from . import expert_rules as rules
from . import expert_util as xu
from .test_gpu_few_tokens import call, on_gpu, problem, reference

pytestmark = pytest.mark.gpu

SHAPES = {("tiles", "tiles"): (128, 1024, 8, 528, 144), ("tiles", "few"): (128, 1024, 8, 144, 48), ("many", "many"): (60, 8, 8, 272, 80),
          ("few", "few"): (24, 64, 4, 400, 144)}
KINDS = pytest.mark.parametrize("kind", SHAPES, ids=lambda kind: "-".join(kind))
TYPES = pytest.mark.parametrize("quantised", [True, False])


def make(seed, kind, quantised, **more):
    shape = SHAPES[kind]
    assert rules.few_tokens_kernels(*shape, rules.compute_units()) == kind
    print(f"{kind} {shape} int8 {quantised}", flush=True)
    return problem(seed, *shape, quantised, **more)


@KINDS
@TYPES
def test_masked_duplicate_and_foreign_ids(kind, quantised):
    p = make(41, kind, quantised, mask=0.05)
    T, E, K = SHAPES[kind][:3]
    p["ids"][0] = -1                                     # no route at all
    p["ids"][1] = 2                                      # one expert in every slot: as many routes
    p["ids"][2] = [E, -1, 1 << 40, -(1 << 50), 3, -2, E + 7, E - 1][:K]
    p["ids"][3, :-1], p["ids"][3, -1] = -1, E - 1
    p["ids"][T - 1] = [-1, -1, 0, 0, 1, 1, -1, 1][:K]
    p["gates"][0] = np.nan                               # weights of slots without a route count for nothing
    p["gates"][2, :3] = np.inf
    p["x"][0] = float("nan")                             # nor does the token
    routed = (p["ids"] >= 0) & (p["ids"] < E)
    q = dict(p, gates=np.where(routed, p["gates"], 0).astype(np.float32), x=p["x"].clone())
    q["x"][0] = 0
    want, bound = reference(q)
    out = xu.f64(call(on_gpu(p)))
    xu.check_within(out, want, bound)
    assert not out[0].any()
    p["ids"][:] = -1
    assert not xu.f64(call(on_gpu(p))).any()


@KINDS
@TYPES
def test_every_token_to_one_expert_besides_its_own(kind, quantised):
    """More routes of an expert than a pass over its weights holds."""
    p = make(42, kind, quantised)
    p["ids"][:, 1] = SHAPES[kind][1] - 1
    want, bound = reference(p)
    g = on_gpu(p)
    out = call(g)
    xu.check_within(xu.f64(out), want, bound)
    assert torch.equal(call(g), out)


@KINDS
@TYPES
def test_a_token_of_nan_or_infinity_leaves_the_others_alone(kind, quantised):
    """Its experts' other tokens share its tiles: their results are the same to the bit."""
    p = make(43, kind, quantised)
    g = on_gpu(p)
    clean = call(g)
    for bad in (float("nan"), float("inf"), 3e38):
        g["x"][5, 7::3] = bad
        dirty = call(g)
        rest = torch.arange(clean.shape[0], device=xu.DEV) != 5
        assert torch.equal(dirty[rest], clean[rest])
        if bad != bad:
            assert bool(torch.isnan(dirty[5]).all())


@KINDS
@TYPES
def test_replays_of_two_graphs_follow_the_ids(kind, quantised):
    p = make(44, kind, quantised)
    g = on_gpu(p)
    bias = xu.bf16_round(np.random.default_rng(1).standard_normal(tuple(p["x"].shape))).to(xu.DEV)
    call(g, True, bias)
    torch.cuda.synchronize()
    graphs, held = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(call(g, True, bias))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    T, E, K = SHAPES[kind][:3]
    for seed, mask in ((1, 0.0), (2, 0.4), (3, 0.9), (4, 1.0)):
        rng = np.random.default_rng(seed)
        ids, gates = xu.routing(rng, T, E, K, mask, "zipf")
        g["ids"].copy_(xu.to_gpu(ids))
        g["gates"].copy_(xu.to_gpu(gates))
        g["x"].copy_(xu.bf16_round(rng.standard_normal(tuple(p["x"].shape))))
        eager = call(g, True, bias)
        for h in held:
            h.fill_(9.0)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held[0], eager) and torch.equal(held[1], eager)


class Few:
    """The experts that have weights, for the 64-bit form, among as many as there are."""

    def __init__(self, count, given):
        self.given, self.shape = given, (count, *next(iter(given.values())).shape)

    def __getitem__(self, e):
        return self.given[e]


@TYPES
def test_weights_behind_4_gib_in_tiles(quantised):
    """64 tokens of top 8 over 1024 experts, of which three have weights and routes: both products take the tiles, and both
    weights of the last expert start behind 4 GiB."""
    T, E, K, H, I = 64, 1024, 8, 2048, 2112
    size = 1 if quantised else 2
    assert rules.few_tokens_kernels(T, E, K, H, I, rules.compute_units()) == ("tiles", "tiles") and (E - 1) * H * I * size > 1 << 32
    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip("needs 40 GiB of device memory")
    print(f"behind 4 GiB int8 {quantised}", flush=True)
    rng = np.random.default_rng(45)
    p = problem(45, T, 3, 1, H, I, quantised)
    experts = np.array([0, 500, E - 1])
    ids = np.full((T, K), -1, dtype=np.int64)
    for t in range(0, T, 5):                              # few tokens have routes: the 64-bit form stays small
        ids[t, rng.permutation(K)[:3]] = rng.permutation(experts)
    gates = rng.random((T, K), dtype=np.float32)
    weights, values = {}, {}
    for name, rows in (("w13", (2 * I, H)), ("w2", (H, I)), ("s13", (2 * I,)), ("s2", (H,))):
        if p[name] is None:
            weights[name] = values[name] = None
            continue
        small = p[name] if isinstance(p[name], torch.Tensor) else torch.from_numpy(p[name])
        wide = torch.zeros((E, *rows), dtype=small.dtype, device=xu.DEV)
        wide[torch.from_numpy(experts).to(xu.DEV)] = small.to(xu.DEV)
        weights[name] = wide
        values[name] = Few(E, {int(e): xu.f64(small[i]) for i, e in enumerate(experts)})
    want, bound = xu.few_tokens64(xu.f64(p["x"]), ids, gates, values["w13"], values["w2"], values["s13"], values["s2"])
    out = ops.moe_few_tokens(p["x"].to(xu.DEV), xu.to_gpu(ids), xu.to_gpu(gates), weights["w13"], weights["w2"], weights["s13"], weights["s2"])
    xu.check_within(xu.f64(out), want, bound)

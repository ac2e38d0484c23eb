"""GPU tests of moe_few_tokens against the layer in 64 bits, within bounds that count its roundings."""
import numpy as np
import pytest
import torch

from commbench_amd import _lib, ops

from . import expert_util as xu
from . import gpu_util as gu

pytestmark = pytest.mark.gpu


def problem(seed, T, E, K, H, I, quantised, mask=0.0, kind="uniform"):
    rng = np.random.default_rng(seed)
    ids, gates = xu.routing(rng, T, E, K, mask, kind)
    p = dict(ids=ids, gates=gates, x=xu.bf16_round(rng.standard_normal((T, H))))
    if quantised:
        p["w13"], p["w2"] = xu.int8_codes(rng, E, 2 * I, H), xu.int8_codes(rng, E, H, I)
        p["s13"] = ((0.5 + rng.random((E, 2 * I))) * H ** -0.5 / 30).astype(np.float32)
        p["s2"] = ((0.5 + rng.random((E, H))) * I ** -0.5 / 30).astype(np.float32)
    else:
        p["w13"] = xu.bf16_round(rng.standard_normal((E, 2 * I, H)) * H ** -0.5)
        p["w2"] = xu.bf16_round(rng.standard_normal((E, H, I)) * I ** -0.5)
        p["s13"] = p["s2"] = None
    return p


def on_gpu(p):
    put = lambda v: None if v is None else v.to(xu.DEV) if isinstance(v, torch.Tensor) else xu.to_gpu(v)
    return {key: put(v) for key, v in p.items()}


def call(g, weights=True, bias=None):
    return ops.moe_few_tokens(g["x"], g["ids"], g["gates"] if weights else None, g["w13"], g["w2"], g["s13"], g["s2"], bias)


def values(v):
    return None if v is None else xu.f64(v) if isinstance(v, torch.Tensor) else v.astype(np.float64)


def reference(p, weights=True, biases=()):
    return xu.few_tokens64(values(p["x"]), p["ids"], p["gates"] if weights else None, values(p["w13"]), values(p["w2"]),
                           values(p["s13"]), values(p["s2"]), [values(b) for b in biases])


CASES = [  # tokens, experts, slots, hidden, intermediate, masked share, routing
    (1, 8, 8, 256, 128, 0.0, "uniform"), (1, 8, 1, 16, 16, 0.0, "uniform"), (1, 16, 2, 272, 48, 0.0, "uniform"),
    (2, 64, 6, 528, 80, 0.3, "uniform"), (3, 8, 3, 1040, 272, 0.0, "zipf"), (5, 4, 4, 144, 208, 0.0, "uniform"),
    (17, 8, 2, 512, 256, 0.05, "zipf"), (33, 4, 1, 256, 64, 0.0, "uniform"), (40, 2, 2, 96, 32, 0.0, "uniform"),
    (64, 32, 8, 128, 96, 0.1, "zipf"), (128, 16, 8, 64, 32, 0.0, "uniform"), (200, 3, 3, 48, 16, 0.5, "zipf")]


@pytest.mark.parametrize("T,E,K,H,I,mask,kind", CASES)
@pytest.mark.parametrize("quantised", [True, False])
def test_layer_against_64_bits(T, E, K, H, I, mask, kind, quantised):
    print(f"tokens {T} experts {E} slots {K} hidden {H} intermediate {I} masked {mask} {kind} int8 {quantised}", flush=True)
    p = problem(T * 100 + H, T, E, K, H, I, quantised, mask, kind)
    want, bound = reference(p)
    xu.check_within(xu.f64(call(on_gpu(p))), want, bound)


FOLDS = [  # few routes for each expert, several for one of them; many for one, few for the others
    (12, 64, 2, 160, 64, 0.0, "zipf"), (12, 64, 4, 272, 48, 0.1, "zipf"), (8, 512, 8, 48, 32, 0.0, "zipf"),
    (40, 64, 4, 160, 64, 0.0, "zipf"), (40, 64, 4, 528, 144, 0.2, "zipf"), (128, 1024, 8, 32, 16, 0.0, "uniform")]


TILES = [  # enough experts and columns for the tiles of the first product: two stages and more, ragged columns, several
    # passes, biases, a token without a route
    (128, 1024, 8, 144, 48, 0.0, "uniform"), (128, 1024, 8, 272, 64, 0.1, "zipf"), (64, 512, 4, 400, 272, 0.0, "uniform"),
    (40, 512, 8, 256, 208, 0.3, "uniform"), (128, 300, 8, 160, 224, 0.05, "zipf"), (16, 256, 8, 1040, 528, 0.0, "uniform"),
    (33, 1000, 8, 656, 256, 0.3, "uniform"),
    (128, 1024, 8, 528, 144, 0.0, "uniform"), (127, 1024, 8, 560, 272, 0.1, "zipf")]   # and for those of the second


@pytest.mark.parametrize("T,E,K,H,I,mask,kind", TILES)
@pytest.mark.parametrize("quantised", [True, False])
def test_many_items_of_a_product(T, E, K, H, I, mask, kind, quantised):
    print(f"tokens {T} experts {E} slots {K} hidden {H} intermediate {I} masked {mask} {kind} int8 {quantised}", flush=True)
    assert min(T * K, E) * ((I + 63) // 64) >= 4 * 256
    p = problem(T * 7 + H, T, E, K, H, I, quantised, mask, kind)
    rng = np.random.default_rng(T)
    biases = [xu.bf16_round(rng.standard_normal((T, H))) for _ in range(2)] if T % 2 else []
    p["ids"][T // 2] = -1                                # a token without a route
    want, bound = reference(p, True, biases)
    g = on_gpu(p)
    arg = tuple(b.to(xu.DEV) for b in biases) or None
    out = call(g, True, arg)
    xu.check_within(xu.f64(out), want, bound)
    for _ in range(3):
        assert torch.equal(call(g, True, arg), out)
    plain, plain_bound = reference(p, False)
    xu.check_within(xu.f64(call(g, False)), plain, plain_bound)


@pytest.mark.parametrize("T,E,K,H,I,mask,kind", FOLDS)
@pytest.mark.parametrize("quantised", [True, False])
def test_experts_of_uneven_counts(T, E, K, H, I, mask, kind, quantised):
    print(f"tokens {T} experts {E} slots {K} hidden {H} intermediate {I} masked {mask} {kind} int8 {quantised}", flush=True)
    p = problem(T * 10 + H, T, E, K, H, I, quantised, mask, kind)
    want, bound = reference(p)
    xu.check_within(xu.f64(call(on_gpu(p))), want, bound)


@pytest.mark.parametrize("T,E,expert", [(16, 512, 511), (17, 1024, 1023), (33, 1024, 0), (128, 64, 63)])
@pytest.mark.parametrize("quantised", [True, False])
def test_every_token_to_one_expert(T, E, expert, quantised):
    """More routes than a pass over an expert's weights holds, where the mean of routes to an expert is tiny."""
    p = problem(T + E, T, E, 2, 96, 48, quantised)
    p["ids"][:, 0], p["ids"][:, 1] = expert, -1
    p["ids"][T // 2, 1] = E - 1 - expert
    want, bound = reference(p)
    xu.check_within(xu.f64(call(on_gpu(p))), want, bound)


@pytest.mark.parametrize("quantised", [True, False])
def test_weights_behind_4_gib(quantised):
    """The last expert's weights lie further than 32 bits of bytes from the first's."""
    E, H, I, size = 700 if quantised else 350, 2560, 1280, 1 if quantised else 2
    assert (E - 1) * 2 * I * H * size > 1 << 32
    p = problem(29, 3, 2, 1, H, I, quantised)
    p["ids"][:] = [[1], [0], [1]]
    want, bound = reference(p)
    g = on_gpu(p)
    for name in ("w13", "w2", "s13", "s2"):
        if g[name] is None:
            continue
        small, wide = g[name], torch.zeros((E, *g[name].shape[1:]), dtype=g[name].dtype, device=xu.DEV)
        wide[0], wide[E - 1] = small[0], small[1]
        g[name] = wide
    g["ids"] = torch.where(g["ids"] == 1, E - 1, 0)
    xu.check_within(xu.f64(call(g)), want, bound)


@pytest.mark.parametrize("quantised", [True, False])
def test_masked_ids_duplicates_and_tokens_without_a_route(quantised):
    T, E, K, H, I = 9, 5, 4, 160, 48
    p = problem(21, T, E, K, H, I, quantised)
    p["ids"][0] = -1                                     # no route at all
    p["ids"][1] = [2, 2, 2, 2]                           # one expert four times: four routes
    p["ids"][2] = [-1, E, 3, 1 << 40]                    # ids out of range are no routes
    p["ids"][3] = [-(1 << 50), -1, -1, 0]
    p["ids"][8] = [-1, -1, 4, 4]
    p["gates"][0] = np.nan                               # weights of masked slots count for nothing
    p["gates"][2, :2] = np.inf
    p["x"][0] = float("nan")                             # nor do the tokens themselves
    q = dict(p, gates=np.where((p["ids"] >= 0) & (p["ids"] < E), p["gates"], 0).astype(np.float32), x=p["x"].clone())
    q["x"][0] = 0
    want, bound = reference(q)
    out = xu.f64(call(on_gpu(p)))
    xu.check_within(out, want, bound)
    assert not out[0].any()
    p["ids"][:] = -1
    assert not xu.f64(call(on_gpu(p))).any()


def test_biases_and_plain_sum():
    p = problem(22, 6, 8, 3, 128, 64, True)
    rng = np.random.default_rng(2)
    b0, b1 = xu.bf16_round(rng.standard_normal((6, 128))), xu.bf16_round(rng.standard_normal((6, 128)))
    p["ids"][2] = -1
    g = on_gpu(p)
    for biases in ((b0,), (b0, b1)):
        want, bound = reference(p, True, biases)
        arg = biases[0].to(xu.DEV) if len(biases) == 1 else tuple(b.to(xu.DEV) for b in biases)
        xu.check_within(xu.f64(call(g, True, arg)), want, bound)
    want, bound = reference(p, False, (b1,))
    xu.check_within(xu.f64(call(g, False, (None, b1.to(xu.DEV)))), want, bound)


def test_small_integers_are_exact():
    """Small whole numbers: no sum rounds, so placement errors cannot hide.  The up half is the identity's multiple
    and the gate half large, so silu(gate) = gate."""
    T, E, K, H, I = 4, 4, 2, 64, 32
    rng = np.random.default_rng(5)
    ids, gates = np.array([[0, 1], [1, 2], [3, -1], [2, 2]]), np.ones((T, K), dtype=np.float32)
    x = np.zeros((T, H))
    x[np.arange(T), np.arange(T) * 7] = 1.0
    w13 = np.zeros((E, 2 * I, H), dtype=np.int8)
    w13[:, :I] = 64                                      # silu(64) = 64 in fp32
    w13[:, I:] = rng.integers(-2, 3, (E, I, H))
    w2 = rng.integers(-1, 2, (E, H, I)).astype(np.int8)
    ones13, ones2 = np.ones((E, 2 * I), dtype=np.float32), np.ones((E, H), dtype=np.float32)
    out = xu.f64(ops.moe_few_tokens(xu.bf16_round(x).to(xu.DEV), xu.to_gpu(ids), xu.to_gpu(gates), xu.to_gpu(w13),
                                    xu.to_gpu(w2), xu.to_gpu(ones13), xu.to_gpu(ones2)))
    want = np.zeros((T, H))
    for t in range(T):
        for k in range(K):
            if ids[t, k] >= 0:
                e = ids[t, k]
                want[t] += w2[e].astype(np.float64) @ (64.0 * (w13[e, I:].astype(np.float64) @ x[t]))
    np.testing.assert_array_equal(out, xu.f64(xu.bf16_round(want)))


def test_repeated_calls_are_the_same_to_the_bit():
    p = on_gpu(problem(23, 48, 16, 8, 512, 128, True, 0.05))
    first = call(p)
    for _ in range(5):
        assert torch.equal(call(p), first)


def test_captured_graphs_replay_with_new_inputs_next_to_each_other():
    p = problem(24, 12, 16, 4, 256, 96, True)
    g = on_gpu(p)
    call(g)
    torch.cuda.synchronize()
    graphs, held = [], []
    for _ in range(2):                                    # two graphs over the same inputs
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(call(g))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for seed in (1, 2, 3):
        new = problem(seed, 12, 16, 4, 256, 96, True, 0.2)
        for key in ("x", "ids", "gates"):
            g[key].copy_(on_gpu(new)[key])
        eager = call(g)
        for h in held:
            h.fill_(9.0)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held[0], eager) and torch.equal(held[1], eager)


def test_workspace_size_is_checked_and_no_tokens_is_no_work():
    lib = _lib.load()
    assert lib.mi_ep_moe_few_tokens_workspace_bytes(128, 8, 7168, 2048) == 128 * 8 * (7168 + 2048) * 4
    g = on_gpu(problem(25, 2, 4, 2, 64, 32, False))
    out = torch.full((2, 64), 5.0, dtype=torch.bfloat16, device=xu.DEV)
    work = torch.empty(2 * 2 * (32 + 64) * 4, dtype=torch.uint8, device=xu.DEV)
    args = lambda nbytes: (g["x"].data_ptr(), g["ids"].data_ptr(), g["gates"].data_ptr(), g["w13"].data_ptr(), None,
                           g["w2"].data_ptr(), None, None, None, 2, 2, 4, 64, 32, out.data_ptr(), work.data_ptr(), nbytes,
                           torch.cuda.current_stream().cuda_stream)
    assert lib.mi_ep_moe_few_tokens(*args(work.numel() - 1)) == -28
    torch.cuda.synchronize()
    assert bool((out == 5.0).all())
    assert lib.mi_ep_moe_few_tokens(*args(work.numel())) == 0
    torch.cuda.synchronize()
    np.testing.assert_array_equal(gu.bf16_bits(out), gu.bf16_bits(call(g)))
    none = ops.moe_few_tokens(g["x"][:0], g["ids"][:0], g["gates"][:0], g["w13"], g["w2"])
    assert none.shape == (0, 64)

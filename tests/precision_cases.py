"""Shapes and inputs of the precision tests of moe_few_tokens; every kernel of the layer is among them."""
import numpy as np

from . import expert_util as xu

# tokens, experts, slots, hidden, intermediate
RANDOM = [(64, 32, 8, 256, 96), (12, 64, 4, 1040, 272), (40, 2, 2, 192, 80), (128, 1024, 8, 144, 48), (128, 1024, 8, 528, 144),
          (127, 1024, 8, 560, 272), (128, 300, 8, 160, 224)]
EXACT = [(5, 16, 2, 160, 48), (20, 4, 2, 272, 144), (40, 2, 2, 192, 80), (128, 1024, 8, 144, 48), (128, 1024, 8, 528, 144),
         (127, 1024, 8, 560, 272), (1, 8, 1, 96, 32)]


class Experts:
    """float64 weights by expert, made when they are asked for: 1024 experts' would take gigabytes."""

    def __init__(self, codes):
        self.codes, self.shape = codes, codes.shape

    def __getitem__(self, e):
        return self.codes[e].astype(np.float64)


def random_problem(shape, quantised):
    T, E, K, H, I = shape
    rng = np.random.default_rng(T + H)
    ids, gates = xu.routing(rng, T, E, K)
    p = dict(ids=ids, gates=gates, x=xu.f64(xu.bf16_round(rng.standard_normal((T, H)))))
    if quantised:
        p["w13"], p["w2"] = Experts(xu.int8_codes(rng, E, 2 * I, H)), Experts(xu.int8_codes(rng, E, H, I))
        p["s13"] = ((0.5 + rng.random((E, 2 * I))) * H ** -0.5 / 30).astype(np.float32).astype(np.float64)
        p["s2"] = ((0.5 + rng.random((E, H))) * I ** -0.5 / 30).astype(np.float32).astype(np.float64)
    else:
        bf16 = lambda *of, scale: xu.bf16_round(rng.standard_normal(of, dtype=np.float32) * np.float32(scale)).to(dtype=xu.torch.float32).numpy()
        p["w13"], p["w2"] = Experts(bf16(E, 2 * I, H, scale=H ** -0.5)), Experts(bf16(E, H, I, scale=I ** -0.5))
        p["s13"] = p["s2"] = None
    return p


def exact_problem(shape):
    """Whole numbers all the way: gate 64 (silu(64) = 64 in fp32), up the sum of two products of codes, at most 2 * 127 * 127, so that the
    activation 64 * up has up to 15 significant bits; every sum stays below 2^24 units of 64, so fp32 holds it and only the last
    rounding to bf16 is left."""
    T, E, K, H, I = shape
    rng = np.random.default_rng(T * H)
    ids, _ = xu.routing(rng, T, E, K, 0.1 if T > 1 else 0.0)
    x = np.zeros((T, H))
    at = np.stack([rng.choice(np.arange(1, H), 2, replace=False) for _ in range(T)])
    x[np.arange(T)[:, None], at] = rng.integers(64, 128, (T, 2)) * rng.choice([-1, 1], (T, 2))
    x[:, 0] = 1.0
    w13 = rng.integers(-127, 128, (E, 2 * I, H), dtype=np.int8)
    w13[:, :I] = 0
    w13[:, :I, 0], w13[:, I:, 0] = 64, 0
    w2 = rng.integers(-1, 2, (E, H, I), dtype=np.int8) * (rng.random((E, H, I), dtype=np.float32) < 0.2)
    return dict(ids=ids, x=x, w13=Experts(w13), w2=Experts(w2.astype(np.int8)))


def exact_result(p):
    """In integers; the last rounding to bf16 is the only one."""
    from . import expert_precision as xp
    T, K = p["ids"].shape
    H, I = p["w2"].shape[1:]
    out, size = np.zeros((T, H)), np.zeros((T, H))
    for t in range(T):
        for k in range(K):
            e = p["ids"][t, k]
            if e < 0:
                continue
            up = p["w13"][e][I:] @ p["x"][t]
            out[t] += p["w2"][e] @ up
            size[t] += np.abs(p["w2"][e]) @ np.abs(up)
    assert size.max() < 2 ** 24
    return xp.to_bf16(64.0 * out)

"""Plain 64-bit forms of the quantisation and expert operators, and error bounds derived from the number of
roundings on the way.  U is half a step of fp32 relative to the value, BF16 half a step of bf16."""
import numpy as np
import torch

from commbench_amd import workloads as wl

U = 2.0 ** -24
BF16 = 2.0 ** -8
DEV = "cuda:0"


def to_gpu(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().cpu().to(torch.float64).numpy()


def bf16_round(a: np.ndarray) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).to(torch.bfloat16)


def int8_codes(rng, *shape) -> np.ndarray:
    return np.clip(np.rint(rng.standard_normal(shape) * 30.0), -127, 127).astype(np.int8)


def routing(rng, T, E, K, mask=0.0, kind="uniform"):
    ids = wl.zipf_distinct_topk(rng, T, E, K, 1.2) if kind == "zipf" else wl.uniform_distinct_topk(rng, T, E, K)
    ids[rng.random((T, K)) < mask] = -1
    return np.ascontiguousarray(ids), wl.softmax_gates(rng, T, K)


def silu64(g):
    with np.errstate(over="ignore"):
        return g / (1.0 + np.exp(-g))


def silu_mul_bound(g, u, g_err, u_err):
    """Bound of the error of silu(g) * u computed in fp32 from values off by g_err and u_err: |silu'| <= 1.1; the
    exponential's argument -g log2(e) is rounded (|g| 1.45 U relative in the result), the exponential
    itself, the addition, the division and two products add at most 16 U; results under the smallest
    normal number may be lost whole (2^-126 times |u|)."""
    s = np.abs(silu64(g))
    err = 1.1 * g_err * (np.abs(u) + u_err) + s * u_err
    return err + (np.abs(g) * 1.45 + 16.0) * U * s * np.abs(u) + 2.0 ** -120 * (1.0 + np.abs(u))


def few_tokens64(x, ids, gates, w13, w2, s13, s2, biases=()):
    """(out, bound) of the expert layer in 64 bits.  x, w13, w2 hold the operands' values in float64 (int8
    codes for quantised weights), the scales float64 or None.  The bound counts: n products summed in
    fp32 (n + 8 roundings of at most a whole step, 2 U, of the sum of magnitudes), silu * up, the
    activation's rounding to two bf16 terms, the second sum, the weighted sum over the slots, and the last rounding."""
    T, K = ids.shape
    E, H, I = w2.shape
    out = np.zeros((T, H))
    err = np.zeros((T, H))
    mag = np.zeros((T, H))
    for t in range(T):
        for k in range(K):
            e = ids[t, k]
            if e < 0 or e >= E:
                continue
            a, b = w13[e], w2[e]
            one = np.ones(2 * I) if s13 is None else s13[e]
            two = np.ones(H) if s2 is None else s2[e]
            c = (a @ x[t]) * one
            c_err = (H + 8) * 2 * U * (np.abs(a) @ np.abs(x[t])) * np.abs(one)
            act = silu64(c[:I]) * c[I:]
            act_err = silu_mul_bound(c[:I], c[I:], c_err[:I], c_err[I:])
            act_err = act_err + BF16 ** 2 * (np.abs(act) + act_err) + 2.0 ** -133   # two bf16 terms: half a step of half a step
            y = (b @ act) * two
            y_err = (np.abs(b) @ act_err + (I + 8) * 2 * U * (np.abs(b) @ (np.abs(act) + act_err))) * np.abs(two)
            w = float(gates[t, k]) if gates is not None else 1.0
            out[t] += w * y
            err[t] += abs(w) * y_err
            mag[t] += abs(w) * (np.abs(y) + y_err)
    for b in biases:
        out += b
        mag += np.abs(b)
    err = err + (K + 4) * 2 * U * mag
    return out, err + BF16 * (np.abs(out) + err) + 2.0 ** -133


def check_within(got: np.ndarray, want: np.ndarray, bound: np.ndarray):
    assert got.shape == want.shape
    assert np.isfinite(got).all()
    over = np.abs(got - want) - bound
    worst = int(np.argmax(over)) if over.size else 0
    assert not over.size or over.flat[worst] <= 0, (
        f"off by {np.abs(got - want).flat[worst]:.3g} at {np.unravel_index(worst, over.shape)}, "
        f"bound {bound.flat[worst]:.3g}, value {want.flat[worst]:.6g}")

"""How exact moe_few_tokens is on average, beside the worst case that expert_util bounds.

error_share: the root mean square of the error over that of rounding the 64-bit result to bf16 once.  A form that
keeps 16 bits of the activation and 24 of everything else is at 1 but for a part in a thousand: the activation's two terms
are off by at most 2^-16 of it, 1 / 256 of the result's own rounding, fp32 sums by less.  One bf16 term for the
activation, or a product of a route rounded to bf16 before the slots are added, adds an error of the size of the result's rounding to
every summand: the share of independent summands is sqrt(2).  LIMIT lies between, sampling included: with n results the
share of a right form spreads by about 1 / sqrt(n)."""
import numpy as np
import torch

from . import expert_util as xu

LIMIT = 1.15


def to_bf16(v: np.ndarray) -> np.ndarray:
    """Rounded to bf16 from float64 in one step."""
    wide = v.astype(np.float32)
    # float64 -> fp32 -> bf16 rounds twice; what lies on a bf16 tie in fp32 but not in float64 is put right.
    out = torch.from_numpy(wide).to(torch.bfloat16).to(torch.float64).numpy()
    bits = wide.view(np.uint32)
    tie = (bits & 0xffff) == 0x8000
    down, up = (bits & 0xffff0000).view(np.float32), ((bits & 0xffff0000) + np.uint32(0x10000)).view(np.float32)
    exact = wide.astype(np.float64)
    grow = np.where(np.abs(v) > np.abs(exact), up, down).astype(np.float64)
    return np.where(tie & (v != exact), grow, out)


def error_share(got: np.ndarray, want: np.ndarray) -> float:
    return float(np.sqrt(((got - want) ** 2).sum() / ((to_bf16(want) - want) ** 2).sum()))


def layer(x, ids, gates, w13, w2, s13, s2, activation_bits=64, product_bits=64):
    """few_tokens64's result with the activation (8: one bf16 term, 16: two) or each route's product (8: bf16) held in fewer
    bits: the mistakes that a kernel could make."""
    T, K = ids.shape
    out = np.zeros((T, w2.shape[1]))
    inner = w2.shape[2]
    for t in range(T):
        for k in range(K):
            e = ids[t, k]
            if not 0 <= e < w2.shape[0]:
                continue
            c = (w13[e] @ x[t]) * (1.0 if s13 is None else s13[e])
            act = xu.silu64(c[:inner]) * c[inner:]
            if activation_bits < 64:
                high = to_bf16(act)
                act = high if activation_bits == 8 else high + to_bf16(act - high)
            y = (w2[e] @ act) * (1.0 if s2 is None else s2[e])
            out[t] += float(gates[t, k]) * (to_bf16(y) if product_bits == 8 else y)
    return out

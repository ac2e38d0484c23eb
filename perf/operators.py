"""Measured cases of the operators around dispatch and combine: the norm that makes an 8-bit payload, quantising
rows and reading them back, the experts' int8 products, and the whole layer for a few tokens.

`run` computes an operator's plain form in elementary torch operations, or, where `own` is set, makes the calls of
commbench_amd.ops that a program makes.  8-bit results are returned as the values they stand for.
"""
import math

import torch

own = False

DEV = "cuda:0"
EPS = 1e-6
BLOCK = 128                       # columns that share a scale in the e4m3 payload


# ---- cases ---------------------------------------------------------------------------------------

def listed():
    return [
        # a decode step's norm in front of the router and the int8 dispatch
        dict(name="norm_decode_int8", op="norm", tokens=16, hidden=7168, quant="int8", residual=True),
        # the norm that makes the e4m3 payload of the 8192-token fp8 configuration
        dict(name="norm_prefill_e4m3", op="norm", tokens=8192, hidden=7168, quant="e4m3", residual=True),
        # a ragged prompt through a first layer: no residual yet
        dict(name="norm_ragged_int8", op="norm", tokens=1021, hidden=4096, quant="int8", residual=False),
        # requantising between the two products: the rows of a small batch, and of 8192 tokens in 8 slots each
        dict(name="quantize_small_int8", op="quantize", rows=96, width=2048, quant="int8"),
        dict(name="quantize_target_int8", op="quantize", rows=65536, width=2048, quant="int8"),
        # the first product of the tiny configuration
        dict(name="gate_up_tiny", op="matmul", tokens=128, experts=8, topk=2, inner=256, outer=512, silu=True, routing="uniform",
             mask=0.0),
        # the first product of 8192 tokens over 256 experts: every expert has about 256 rows
        dict(name="gate_up_target", op="matmul", tokens=8192, experts=256, topk=8, inner=7168, outer=4096, silu=True,
             routing="uniform", mask=0.0),
        # the second product under skewed routing with masked slots: from empty experts to thousands of rows
        dict(name="down_skewed", op="matmul", tokens=4096, experts=256, topk=8, inner=2048, outer=7168, silu=False,
             routing="zipf", mask=0.05),
        # the first product of 16384 tokens over 128 experts: about 1024 rows each
        dict(name="gate_up_long", op="matmul", tokens=16384, experts=128, topk=8, inner=4096, outer=2048, silu=True,
             routing="uniform", mask=0.0),
        # one token through its eight experts; a small batch on bf16 weights; a larger one with masked slots
        dict(name="moe_1_int8", op="moe", tokens=1, experts=256, topk=8, hidden=7168, inter=2048, weights="int8", mask=0.0),
        dict(name="moe_16_bf16", op="moe", tokens=16, experts=128, topk=8, hidden=4096, inter=1408, weights="bf16", mask=0.0),
        dict(name="moe_48_int8", op="moe", tokens=48, experts=256, topk=8, hidden=7168, inter=2048, weights="int8", mask=0.05),
    ]


def _log(rng, low, high, step=1):
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(v) // step * step))


def draw(rng):
    op = rng.choice(("norm", "quantize", "matmul", "matmul", "moe", "moe"))
    if op == "norm":
        quant = rng.choice(("int8", "e4m3"))
        return dict(op=op, tokens=_log(rng, 1, 8192), hidden=_log(rng, 256, 7168, 128 if quant == "e4m3" else 8), quant=quant,
                    residual=rng.random() < 0.7)
    if op == "quantize":
        quant = rng.choice(("int8", "e4m3"))
        return dict(op=op, rows=_log(rng, 1, 65536), width=_log(rng, 128, 2048, 128 if quant == "e4m3" else 8), quant=quant)
    topk = rng.choice((1, 2, 4, 6, 8))
    experts = rng.choice((8, 32, 64, 128, 256))
    mask = rng.choice((0.0, 0.0, 0.05, 0.3))
    if op == "matmul":
        routing = rng.choice(("uniform", "zipf"))
        return dict(op=op, tokens=_log(rng, 1, 8192 if routing == "uniform" else 2048), experts=experts, topk=topk,
                    inner=_log(rng, 128, 4096, 16), outer=_log(rng, 256, 4096, 16), silu=rng.random() < 0.5, routing=routing,
                    mask=mask)
    return dict(op=op, tokens=_log(rng, 1, 48), experts=experts, topk=topk, hidden=_log(rng, 256, 7168, 16),
                inter=_log(rng, 128, 2048, 16), weights=rng.choice(("int8", "bf16")), mask=mask)


# ---- inputs --------------------------------------------------------------------------------------

def _normal(gen, *shape, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)


def _weights(gen, experts, rows, cols, kind):
    """[experts, rows, cols] expert weights, made in pieces: int8 codes with a scale for each row, or bf16."""
    out = torch.empty((experts, rows, cols), dtype=torch.int8 if kind == "int8" else torch.bfloat16, device=DEV)
    piece = max(1, (1 << 28) // (rows * cols))
    for e in range(0, experts, piece):
        w = torch.randn(out[e:e + piece].shape, generator=gen, device=DEV, dtype=torch.bfloat16)
        if kind == "int8":
            out[e:e + piece] = w.mul_(30.0).round_().clamp_(-127.0, 127.0).to(torch.int8)
        else:
            out[e:e + piece] = w.mul_(cols ** -0.5)
    if kind != "int8":
        return out, None
    spread = 0.5 + torch.rand((experts, rows), generator=gen, device=DEV)
    return out, spread * (cols ** -0.5 / 30.0)


def _routing(gen, tokens, experts, topk, routing, mask):
    """Distinct experts for each token (uniform, or skewed by draws without replacement), some slots masked."""
    keys = -torch.log(-torch.log(torch.rand((tokens, experts), generator=gen, device=DEV).clamp_(1e-7, 1.0 - 1e-6)))
    if routing == "zipf":
        order = torch.randperm(experts, generator=gen, device=DEV)
        keys = keys - 1.2 * torch.log(1.0 + order)[None, :]
    ids = keys.topk(topk, dim=1).indices
    if mask > 0.0:
        order = torch.randperm(tokens * topk, generator=gen, device=DEV)
        ids = ids.clone()
        ids.view(-1)[order[:int(mask * tokens * topk)]] = -1       # always as many: outputs keep their sizes
    gates = torch.softmax(torch.randn((tokens, topk), generator=gen, device=DEV), dim=1)
    return ids.contiguous(), gates.contiguous()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    op, state = case["op"], dict(case)
    if op == "norm":
        T, H = case["tokens"], case["hidden"]
        x = _normal(gen, T, H)
        x[:, :: 97] *= 8                                  # a few channels are much larger than the rest
        state["x"] = x
        state["gain"] = (1.0 + 0.1 * torch.randn(H, generator=gen, device=DEV)).to(torch.bfloat16)
        state["addend"] = _normal(gen, T, H, scale=2.0) if case["residual"] else None
    elif op == "quantize":
        rows, width = case["rows"], case["width"]
        size = torch.exp(torch.randn((rows, 1), generator=gen, device=DEV))
        state["x"] = (torch.randn((rows, width), generator=gen, device=DEV) * size).to(torch.bfloat16)
    elif op == "matmul":
        ids, _ = _routing(gen, case["tokens"], case["experts"], case["topk"], case["routing"], case["mask"])
        counts = torch.bincount(ids[ids >= 0], minlength=case["experts"])
        offsets = torch.zeros(case["experts"] + 1, dtype=torch.int64, device=DEV)
        offsets[1:] = counts.cumsum(0)
        rows = int(offsets[-1])
        state["counts"], state["offsets"] = counts.to(torch.int32), offsets.to(torch.int32)
        state["longest"] = max(1, int(counts.max()))      # of the plain form's padded batch
        state["a"] = torch.randn((rows, case["inner"]), generator=gen, device=DEV, dtype=torch.bfloat16).mul_(30.0).round_() \
            .clamp_(-127.0, 127.0).to(torch.int8)
        state["a_scales"] = (0.5 + torch.rand((rows, 1), generator=gen, device=DEV)) / 30.0
        state["b"], state["b_scales"] = _weights(gen, case["experts"], case["outer"], case["inner"], "int8")
    else:
        state["x"] = _normal(gen, case["tokens"], case["hidden"])
        state["ids"], state["gates"] = _routing(gen, case["tokens"], case["experts"], case["topk"], "uniform", case["mask"])
        E, H, I = case["experts"], case["hidden"], case["inter"]
        state["w13"], state["w13_scales"] = _weights(gen, E, 2 * I, H, case["weights"])
        state["w2"], state["w2_scales"] = _weights(gen, E, H, I, case["weights"])
    return state


# ---- the plain forms -------------------------------------------------------------------------------

def _quantized(y, quant):
    """What the 8-bit form of the rows `y` stands for, and its scales: one for a row (int8) or for 128 columns (e4m3)."""
    rows, width = y.shape
    y = y.view(rows, -1, width if quant == "int8" else BLOCK)
    amax = y.abs().amax(dim=2, keepdim=True)
    scales = torch.where(amax > 0, amax / (127.0 if quant == "int8" else 448.0), torch.ones_like(amax))
    q = y / scales
    q = q.round().clamp(-127.0, 127.0) if quant == "int8" else q.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float()
    return (q * scales).view(rows, width).to(torch.bfloat16), scales.view(rows, -1)


def _plain_norm(s):
    h = s["x"].float()
    if s["addend"] is not None:
        h = h + s["addend"].float()
    y = h * torch.rsqrt(h.square().mean(dim=1, keepdim=True) + EPS) * s["gain"].float()
    values, scales = _quantized(y, s["quant"])
    return dict(values=values, scales=scales, residual=h.to(torch.bfloat16) if s["addend"] is not None else None)


def _plain_matmul(s):
    rows, longest = s["a"].shape[0], s["longest"]
    offsets = s["offsets"].long()
    at = (offsets[:-1, None] + torch.arange(longest, device=DEV)).clamp_(max=max(rows - 1, 0))
    product = torch.bmm(s["a"].float()[at], s["b"].float().transpose(1, 2))           # [experts, longest, outer]
    row = torch.arange(rows, device=DEV)
    expert = torch.searchsorted(offsets[1:].contiguous(), row, right=True)
    c = product.view(-1, product.shape[2])[expert * longest + row - offsets[expert]]
    c = c * s["a_scales"] * s["b_scales"][expert]
    if s["silu"]:
        gate, up = c.chunk(2, dim=1)
        c = gate / (1.0 + torch.exp(-gate)) * up
    return c.to(torch.bfloat16)


def _plain_moe(s):
    T, K = s["ids"].shape
    I = s["inter"]
    routed = s["ids"] >= 0
    expert = s["ids"].clamp(min=0).view(-1)
    x = s["x"].float().repeat_interleave(K, dim=0)
    c = torch.bmm(s["w13"][expert].float(), x[:, :, None])[:, :, 0]
    if s["w13_scales"] is not None:
        c = c * s["w13_scales"][expert]
    h = c[:, :I] / (1.0 + torch.exp(-c[:, :I])) * c[:, I:]
    y = torch.bmm(s["w2"][expert].float(), h[:, :, None])[:, :, 0]
    if s["w2_scales"] is not None:
        y = y * s["w2_scales"][expert]
    y = torch.where(routed[:, :, None], y.view(T, K, -1) * s["gates"][:, :, None], 0.0)
    return y.sum(dim=1).to(torch.bfloat16)


def run(state):
    s, op = state, state["op"]
    if own:
        from commbench_amd import ops
        if op == "norm":
            got = ops.rms_norm_quantize(s["x"], s["gain"], EPS, residual=s["addend"], quant=s["quant"])
            return dict(values=ops.dequantize_rows(got[0], got[1]), scales=got[1],
                        residual=got[2] if s["addend"] is not None else None)
        if op == "quantize":
            q, scales = ops.quantize_rows(s["x"], quant=s["quant"])
            return dict(values=ops.dequantize_rows(q, scales), scales=scales)
        if op == "matmul":
            return ops.grouped_matmul_int8(s["a"], s["a_scales"], s["b"], s["b_scales"], s["offsets"], s["counts"],
                                           activation="silu_mul" if s["silu"] else None)
        return ops.moe_few_tokens(s["x"], s["ids"], s["gates"], s["w13"], s["w2"], s["w13_scales"], s["w2_scales"])
    if op == "norm":
        return _plain_norm(s)
    if op == "quantize":
        values, scales = _quantized(s["x"].float(), s["quant"])
        return dict(values=values, scales=scales)
    return _plain_matmul(s) if op == "matmul" else _plain_moe(s)


# ---- what a pass cannot do without -------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op in ("norm", "quantize"):
        rows, width = (case["tokens"], case["hidden"]) if op == "norm" else (case["rows"], case["width"])
        groups = 1 if case["quant"] == "int8" else width // BLOCK
        tensors = 2 + (2 if op == "norm" and case["residual"] else 0)     # bf16 rows read and written
        size = rows * width
        return dict(bytes=2 * size * tensors + 4 * rows * groups + (2 * width if op == "norm" else 0),
                    flops=size * (10 if op == "norm" else 5))
    T, E, K = case["tokens"], case["experts"], case["topk"]
    routes = T * K * (1.0 - case["mask"])
    met = E * (1.0 - (1.0 - K * (1.0 - case["mask"]) / E) ** T)             # experts met by T uniform tokens
    if op == "matmul":
        n, k = case["outer"], case["inner"]
        out = n // 2 if case["silu"] else n
        return dict(bytes=routes * (k + 4 + 2 * out) + met * n * (k + 4), flops=2.0 * routes * n * k)
    H, I = case["hidden"], case["inter"]
    size = 1 if case["weights"] == "int8" else 2
    return dict(bytes=met * 3 * H * I * size + 4 * T * H + 12 * T * K, flops=6.0 * routes * H * I)


# ---- the definition in 64 bits -----------------------------------------------------------------------

def _round_to_e4m3(v):
    """Nearest value of 4 exponent and 3 mantissa bits (smallest exponent -6, largest value 448), ties to even."""
    exponent = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -20))).clamp(min=-6.0)
    step = torch.exp2(exponent - 3.0)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def _exact_quantized(y, quant):
    values, scales = torch.empty_like(y), []
    span = y.shape[1] if quant == "int8" else BLOCK
    for c in range(0, y.shape[1], span):
        part = y[:, c:c + span]
        top = part.abs().max(dim=1, keepdim=True).values
        scale = top / (127 if quant == "int8" else 448)
        scale[top == 0] = 1.0
        code = part / scale
        values[:, c:c + span] = (torch.round(code) if quant == "int8" else _round_to_e4m3(code)) * scale
        scales.append(scale)
    return values, torch.cat(scales, dim=1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double()
        if s["addend"] is not None:
            h += s["addend"].double()
        y = s["gain"].double() * h / torch.sqrt((h * h).sum(dim=1, keepdim=True) / case["hidden"] + EPS)
        values, scales = _exact_quantized(y, case["quant"])
        return dict(values=values, scales=scales, residual=h if s["addend"] is not None else None)
    if case["op"] == "quantize":
        values, scales = _exact_quantized(s["x"].double(), case["quant"])
        return dict(values=values, scales=scales)
    if case["op"] == "matmul":
        n = case["outer"]
        out = torch.empty((s["a"].shape[0], n // 2 if case["silu"] else n), dtype=torch.float64, device=DEV)
        bounds = s["offsets"].tolist()
        for e in range(case["experts"]):
            low, high = bounds[e], bounds[e + 1]
            if high > low:
                b = s["b"][e].double() * s["b_scales"][e].double()[:, None]
                c = (s["a"][low:high].double() * s["a_scales"][low:high].double()) @ b.T
                out[low:high] = torch.sigmoid(c[:, :n // 2]) * c[:, :n // 2] * c[:, n // 2:] if case["silu"] else c
        return out
    T, K = s["ids"].shape
    I = case["inter"]
    out = torch.zeros((T, case["hidden"]), dtype=torch.float64, device=DEV)
    ids, gates = s["ids"].tolist(), s["gates"].double()
    for e in sorted({i for row in ids for i in row if i >= 0}):
        w13, w2 = s["w13"][e].double(), s["w2"][e].double()
        if s["w13_scales"] is not None:
            w13 *= s["w13_scales"][e].double()[:, None]
            w2 *= s["w2_scales"][e].double()[:, None]
        for t in range(T):
            for k in range(K):
                if ids[t][k] == e:
                    c = w13 @ s["x"][t].double()
                    out[t] += gates[t, k] * (w2 @ (torch.sigmoid(c[:I]) * c[:I] * c[I:]))
    return out

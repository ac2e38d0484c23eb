"""The operators together as a layer uses them: norm to int8 -> dispatch -> products -> combine, next to the layer for a few
tokens on the same weights, and the e4m3 payload read back after dispatch."""
import numpy as np
import pytest
import torch

from commbench_amd import ops

from . import expert_util as xu
from . import gpu_util as gu

pytestmark = pytest.mark.gpu


def layer_inputs(seed, T, E, K, H, I, mask):
    rng = np.random.default_rng(seed)
    ids, gates = xu.routing(rng, T, E, K, mask)
    return dict(
        x=xu.bf16_round(rng.standard_normal((T, H))).to(xu.DEV), r=xu.bf16_round(rng.standard_normal((T, H))).to(xu.DEV),
        g=xu.bf16_round(1 + 0.1 * rng.standard_normal(H)).to(xu.DEV), ids_np=ids, ids=xu.to_gpu(ids), gates=xu.to_gpu(gates),
        w13=xu.to_gpu(xu.int8_codes(rng, E, 2 * I, H)), w2=xu.to_gpu(xu.int8_codes(rng, E, H, I)),
        s13=xu.to_gpu(((0.5 + rng.random((E, 2 * I))) * H ** -0.5 / 30).astype(np.float32)),
        s2=xu.to_gpu(((0.5 + rng.random((E, H))) * I ** -0.5 / 30).astype(np.float32)))


@pytest.mark.parametrize("T,E,K,H,I,mask,align", [(300, 16, 4, 512, 256, 0.05, 1), (1, 8, 2, 256, 128, 0.0, 1),
                                                  (97, 8, 8, 272, 144, 0.3, 16), (520, 4, 1, 256, 64, 0.0, 128)])
def test_many_token_layer_step_by_step(T, E, K, H, I, mask, align):
    """Every product of the path against 64 bits, from the codes the path itself handed on (an error in one step
    cannot hide behind the tolerance of another), and the whole as one call."""
    print(f"layer {T} tokens {E} experts {K} slots {H} x {I} align {align}", flush=True)
    v = layer_inputs(T + H, T, E, K, H, I, mask)
    buf = ops.Buffer(T, K, E, 2, device=xu.DEV)
    q, s, stream = ops.rms_norm_quantize(v["x"], v["g"], residual=v["r"])
    recv, recv_s, src, h = buf.dispatch(q, s, v["ids"], v["gates"], align)
    act = ops.grouped_matmul_int8(recv, recv_s, v["w13"], v["s13"], h.expert_offsets, h.num_tokens_per_expert, "silu_mul")
    act_q, act_s = ops.quantize_rows(act, row_limit=h.expert_offsets[-1:])
    y = ops.grouped_matmul_int8(act_q, act_s, v["w2"], v["s2"], h.expert_offsets, h.num_tokens_per_expert)
    out = ops.combine(y, h, v["gates"])
    whole = buf.moe_int8(q, s, v["ids"], v["gates"], v["w13"], v["s13"], v["w2"], v["s2"], expert_alignment=align)
    torch.cuda.synchronize()
    buf.status()
    assert torch.equal(out, whole)

    slots = h.slot_map.cpu().numpy()
    qn, sn = q.cpu().numpy().astype(np.float64), xu.f64(s)
    w13, s13, w2, s2 = (xu.f64(v[key]) for key in ("w13", "s13", "w2", "s2"))
    aq, asc, actn, yn = act_q.cpu().numpy().astype(np.float64), xu.f64(act_s), xu.f64(act), xu.f64(y)
    for t in range(0, T, max(1, T // 23)):
        for k in range(K):
            e, row = v["ids_np"][t, k], slots[t, k]
            if e < 0:
                assert row == -1
                continue
            c = (w13[e] @ qn[t]) * sn[t] * s13[e]
            err = 3 * xu.U * np.abs(c) * (1 + 1e-6)
            a = xu.silu64(c[:I]) * c[I:]
            a_err = xu.silu_mul_bound(c[:I], c[I:], err[:I], err[I:])
            xu.check_within(actn[row], a, a_err + xu.BF16 * (np.abs(a) + a_err) + 2.0 ** -133)
            scale = np.abs(actn[row]).max() / 127 if actn[row].any() else 1.0
            xu.check_within(aq[row] * asc[row], actn[row], np.full(I, 0.5 * scale * (1 + 1e-5)))
            z = (w2[e] @ aq[row]) * asc[row] * s2[e]
            xu.check_within(yn[row], z, np.abs(z) * (xu.BF16 + 4 * xu.U) + 2.0 ** -133)


def test_both_layers_agree_within_the_activation_codes():
    """The same weights through both paths.  They differ by what the many-token path quantises on the way: x (half
    a step of its row scale in every column) and the activation (likewise); all else is bounded as in
    the few-token tests."""
    T, E, K, H, I = 24, 8, 4, 512, 256
    v = layer_inputs(3, T, E, K, H, I, 0.1)
    q, s = ops.quantize_rows(v["x"])
    few = ops.moe_few_tokens(ops.dequantize_rows(q, s), v["ids"], v["gates"], v["w13"], v["w2"], v["s13"], v["s2"])
    buf = ops.Buffer(T, K, E, 2, device=xu.DEV)
    many = buf.moe_int8(q, s, v["ids"], v["gates"], v["w13"], v["s13"], v["w2"], v["s2"])
    x = xu.f64(ops.dequantize_rows(q, s))
    w13, s13, w2, s2 = (xu.f64(v[key]) for key in ("w13", "s13", "w2", "s2"))
    gates = v["gates"].cpu().numpy()
    want, few_bound = xu.few_tokens64(x, v["ids_np"], gates, w13, w2, s13, s2)
    xu.check_within(xu.f64(few), want, few_bound)
    many_bound = few_bound.copy()
    for t in range(T):
        for k in range(K):
            e = v["ids_np"][t, k]
            if e < 0:
                continue
            c = (w13[e] @ x[t]) * s13[e]
            c_err = xu.BF16 * (np.abs(w13[e]) @ np.abs(x[t])) * s13[e]   # reading x back rounds it to bf16
            a = xu.silu64(c[:I]) * c[I:]
            a_err = xu.silu_mul_bound(c[:I], c[I:], c_err[:I], c_err[I:])
            step = 0.5 * (np.abs(a).max() + a_err.max()) * (1 + xu.BF16) / 127
            y_err = (np.abs(w2[e]) @ (a_err + step + 2 * xu.BF16 * np.abs(a))) * s2[e]
            y = np.abs((w2[e] @ a) * s2[e])
            many_bound[t] += gates[t, k] * (y_err * (1 + xu.BF16) + xu.BF16 * y)   # y itself is rounded to bf16
    xu.check_within(xu.f64(many), want, many_bound * 1.01)


def test_e4m3_payload_made_dispatched_and_read_back():
    T, E, K, H = 200, 16, 4, 512
    v = layer_inputs(5, T, E, K, H, 64, 0.1)
    buf = ops.Buffer(T, K, E, 4, device=xu.DEV)
    q, s, _ = ops.rms_norm_quantize(v["x"], v["g"], residual=v["r"], quant="e4m3", column_major_scales=True)
    recv, recv_s, src, h = buf.dispatch(q, s, v["ids"], v["gates"], column_major_recv_scales=True)
    rows = h.num_recv_rows()
    got = ops.dequantize_rows(recv[:rows], recv_s[:rows], row_limit=h.expert_offsets[-1:])
    want = ops.dequantize_rows(q, s)[src[:rows].long()]
    np.testing.assert_array_equal(gu.bf16_bits(got), gu.bf16_bits(want))


def test_layer_captured_whole_and_replayed():
    T, E, K, H, I = 64, 8, 2, 256, 128
    v = layer_inputs(7, T, E, K, H, I, 0.1)
    buf = ops.Buffer(T, K, E, 2, device=xu.DEV)

    def layer():
        q, s, stream = ops.rms_norm_quantize(v["x"], v["g"], residual=v["r"])
        return buf.moe_int8(q, s, v["ids"], v["gates"], v["w13"], v["s13"], v["w2"], v["s2"], bias=stream)

    layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = layer()
    for seed in (8, 9, 10):
        new = layer_inputs(seed, T, E, K, H, I, 0.3)
        for key in ("x", "r", "ids", "gates"):
            v[key].copy_(new[key])
        eager = layer()
        held.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, eager)
    buf.status()


def test_layer_of_no_tokens_and_of_masked_ones():
    v = layer_inputs(11, 4, 8, 2, 256, 128, 0.0)
    buf = ops.Buffer(4, 2, 8, 2, device=xu.DEV)
    for align in (1, 16):
        q, s = ops.quantize_rows(v["x"])
        none = buf.moe_int8(q[:0], s[:0], v["ids"][:0], v["gates"][:0], v["w13"], v["s13"], v["w2"], v["s2"], expert_alignment=align)
        assert none.shape == (0, 256)
        masked = buf.moe_int8(q, s, torch.full_like(v["ids"], -1), v["gates"], v["w13"], v["s13"], v["w2"], v["s2"],
                              bias=v["r"][:4].contiguous(), expert_alignment=align)
        assert torch.equal(masked, v["r"][:4])
    buf.status()

"""Refusals of the quantisation and expert operators, on the CPU: the C entries return before any launch."""
import struct

import pytest
import torch

from commbench_amd import _lib, ops

EINVAL, ENOSPC = -22, -28
EPS = struct.unpack("<I", struct.pack("<f", 1e-6))[0]
A = 4096                                                  # an aligned address that is never followed


def lib():
    return _lib.load()


def norm(x=A, xs=64, r=None, rs=64, w=A, eps=EPS, rows=4, h=64, fmt=0, q=A, s=A, srs=1, shs=1, ro=None, n=None):
    return lib().mi_ep_rms_norm_quantize(x, xs, r, rs, w, eps, rows, h, fmt, q, s, srs, shs, ro, n, None)


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(w=None), dict(q=None), dict(s=None), dict(rows=-1), dict(rows=1 << 30), dict(h=0), dict(h=12), dict(h=32776, xs=32776),
    dict(fmt=2), dict(fmt=-1), dict(fmt=1, h=64), dict(xs=56), dict(xs=68), dict(r=A, rs=60), dict(x=A + 8), dict(w=A + 2),
    dict(q=A + 4), dict(r=A + 8), dict(ro=A), dict(r=A, ro=A + 8), dict(n=A + 8), dict(eps=0x7f800000), dict(eps=0x7fc00000),
    dict(eps=0xbf800000), dict(srs=0), dict(srs=-1), dict(fmt=1, h=256, xs=256, srs=1, shs=1), dict(fmt=1, h=256, xs=256, shs=0),
    dict(r=2 * A, rs=72, ro=2 * A), dict(r=2 * A, xs=72, ro=A)])
def test_norm_refuses(bad):
    assert norm(**bad) == EINVAL


def test_nothing_to_do_is_not_an_error():
    assert norm(rows=0) == 0 and norm(rows=0, x=None, w=None, q=None, s=None) == 0
    assert lib().mi_ep_quantize_rows(None, 64, None, 0, 64, 0, None, None, 1, 1, None) == 0
    assert lib().mi_ep_dequantize_rows(None, None, 1, 1, None, 0, 64, 0, None, None) == 0
    assert lib().mi_ep_grouped_matmul_int8(None, None, 1, None, None, None, None, 0, 1, 8, 16, None, 0, None) == 0
    assert lib().mi_ep_moe_few_tokens(None, None, None, None, None, None, None, None, None, 0, 2, 4, 64, 32, None, None, 0,
                                      None) == 0


def test_row_quantisation_refuses():
    def quantize(x=A, xs=64, rows=4, h=64, fmt=0, q=A, s=A, srs=1, shs=1):
        return lib().mi_ep_quantize_rows(x, xs, None, rows, h, fmt, q, s, srs, shs, None)

    def dequantize(q=A, s=A, srs=1, shs=1, rows=4, h=64, fmt=0, out=A):
        return lib().mi_ep_dequantize_rows(q, s, srs, shs, None, rows, h, fmt, out, None)
    for bad in (dict(x=None), dict(xs=8), dict(xs=66), dict(rows=-1), dict(h=4), dict(fmt=3), dict(fmt=1), dict(q=A + 1),
                dict(x=A + 4), dict(s=None), dict(q=None), dict(srs=0)):
        assert quantize(**bad) == EINVAL, bad
    for bad in (dict(q=None), dict(s=None), dict(out=None), dict(out=A + 8), dict(q=A + 2), dict(rows=-3), dict(h=9), dict(fmt=7),
                dict(fmt=1), dict(srs=-1)):
        assert dequantize(**bad) == EINVAL, bad


def test_product_refuses():
    def matmul(a=A, sa=A, sas=1, b=A, sb=A, off=A, cnt=A, rows=4, e=2, n=64, k=64, out=A, flags=0):
        return lib().mi_ep_grouped_matmul_int8(a, sa, sas, b, sb, off, cnt, rows, e, n, k, out, flags, None)
    for bad in (dict(a=None), dict(sa=None), dict(b=None), dict(sb=None), dict(out=None), dict(off=None, cnt=None),
                dict(off=None, e=1), dict(rows=-1), dict(rows=1 << 28), dict(rows=(1 << 28) - 1, n=1 << 20), dict(sas=(1 << 20) + 1), dict(e=0), dict(e=1025), dict(n=0), dict(n=12), dict(n=24, flags=1),
                dict(k=0), dict(k=24), dict(k=131072), dict(flags=2), dict(sas=-1), dict(a=A + 8), dict(b=A + 1), dict(out=A + 8)):
        assert matmul(**bad) == EINVAL, bad


def test_few_tokens_refuses():
    def few(x=A, ids=A, w=A, w13=A, s13=A, w2=A, s2=A, b0=None, b1=None, t=4, k=2, e=8, h=64, i=32, out=A, ws=A, nbytes=1 << 20):
        return lib().mi_ep_moe_few_tokens(x, ids, w, w13, s13, w2, s2, b0, b1, t, k, e, h, i, out, ws, nbytes, None)
    for bad in (dict(x=None), dict(ids=None), dict(w13=None), dict(w2=None), dict(out=None), dict(ws=None), dict(s13=None), dict(s2=None),
                dict(t=-1), dict(k=0), dict(k=9), dict(t=513), dict(e=0), dict(e=1025), dict(h=0), dict(h=24), dict(i=0), dict(i=40),
                dict(h=65552), dict(i=65552), dict(x=A + 2), dict(w13=A + 8), dict(w2=A + 8), dict(b0=A + 2), dict(b1=A + 2), dict(out=A + 8),
                dict(ws=A + 8)):
        assert few(**bad) == EINVAL, bad
    assert few(nbytes=4 * 2 * (32 + 64) * 4 - 1) == ENOSPC
    assert lib().mi_ep_moe_few_tokens_workspace_bytes(4, 2, 64, 32) == 4 * 2 * (32 + 64) * 4
    assert lib().mi_ep_moe_few_tokens_workspace_bytes(129, 8, 64, 32) == 0
    assert lib().mi_ep_moe_few_tokens_workspace_bytes(4, 2, 64, 30) == 0
    assert lib().mi_ep_moe_few_tokens_workspace_bytes(4, 2, 60, 32) == 0


def test_python_surface_refuses_host_tensors_and_wrong_types():
    x = torch.zeros((4, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="x must be a bf16"):
        ops.rms_norm_quantize(x, torch.ones(64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="x must be a bf16"):
        ops.quantize_rows(x)
    with pytest.raises(ValueError, match="q must be a contiguous int8"):
        ops.dequantize_rows(x.to(torch.int8), torch.ones((4, 1)))
    with pytest.raises(ValueError, match="a must be a contiguous int8"):
        ops.grouped_matmul_int8(x.to(torch.int8), torch.ones(4), torch.zeros((1, 8, 64), dtype=torch.int8), torch.ones((1, 8)))
    with pytest.raises(ValueError, match="x must be a contiguous bf16"):
        ops.moe_few_tokens(x, torch.zeros((4, 2), dtype=torch.int64), None, x, x)

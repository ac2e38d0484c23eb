"""The new residual stream may be x or residual themselves, but not lie across their rows: other rows would be read while it is
written.  On the CPU the C entry refuses before any launch; on the GPU what does not meet is accepted."""
import struct

import pytest
import torch

from commbench_amd import _lib, ops

from . import expert_util as xu

EINVAL = -22
EPS = struct.unpack("<I", struct.pack("<f", 1e-6))[0]
X, R, FAR = 1 << 20, 1 << 24, 1 << 28                     # aligned addresses that are never followed
WIDTH = 64                                                # 128 bytes a row


def norm(x=X, xs=WIDTH, r=R, rs=WIDTH, out=FAR, rows=4):
    return _lib.load().mi_ep_rms_norm_quantize(x, xs, r, rs, FAR * 2, EPS, rows, WIDTH, 0, FAR * 4, FAR * 8, 1, 1, out, None, None)


@pytest.mark.parametrize("bad", [
    dict(out=X + 128), dict(out=X - 128), dict(out=X + 3 * 128), dict(out=X - 3 * 128), dict(out=X + 16), dict(out=X - 16),
    dict(out=R + 128), dict(out=R - 16), dict(out=R + 3 * 128 + 112),
    dict(xs=2 * WIDTH, out=X), dict(rs=2 * WIDTH, out=R), dict(xs=2 * WIDTH, out=X + 128), dict(xs=4 * WIDTH, out=X + 128),
    dict(xs=4 * WIDTH, out=X + 3 * 512 + 112), dict(xs=4 * WIDTH, out=X + 512 - 4 * 128 + 16), dict(rs=4 * WIDTH, out=R + 1024 - 16),
    dict(x=R + 128, out=R), dict(x=R - 128, out=R), dict(r=X + 128, out=X)])
def test_a_residual_written_across_input_rows_is_refused(bad):
    assert norm(**bad) == EINVAL


@pytest.mark.gpu
def test_a_residual_between_the_rows_of_x_is_not():
    """Three rows of output in the gap behind the first row of x; and both inputs the same rows, in place."""
    g = torch.Generator().manual_seed(1)
    wide = torch.randn((3, 4 * WIDTH), generator=g).to(torch.bfloat16).to(xu.DEV)
    x, r = wide[:, :WIDTH], torch.randn((3, WIDTH), generator=g).to(torch.bfloat16).to(xu.DEV)
    w = torch.ones(WIDTH, dtype=torch.bfloat16, device=xu.DEV)
    want = ops.rms_norm_quantize(x.contiguous(), w, residual=r)
    out = wide[0, WIDTH:].view(3, WIDTH)
    q, s = torch.empty((3, WIDTH), dtype=torch.int8, device=xu.DEV), torch.empty(3, device=xu.DEV)
    _lib.check(_lib.load().mi_ep_rms_norm_quantize(
        x.data_ptr(), 4 * WIDTH, r.data_ptr(), WIDTH, w.data_ptr(), EPS, 3, WIDTH, 0, q.data_ptr(), s.data_ptr(), 1, 1, out.data_ptr(),
        None, torch.cuda.current_stream().cuda_stream), "norm")
    assert torch.equal(q, want[0]) and torch.equal(s, want[1][:, 0]) and torch.equal(out, want[2])
    twice = ops.rms_norm_quantize(r, w, residual=r)
    same = r.clone()
    got = ops.rms_norm_quantize(same, w, residual=same, update_residual=True)
    assert all(torch.equal(a, b) for a, b in zip(got, twice))
    stream = torch.randn((5, WIDTH), generator=g).to(torch.bfloat16).to(xu.DEV)
    with pytest.raises(_lib.MiEpError):
        ops.rms_norm_quantize(stream[:4], w, residual=stream[1:], update_residual=True)

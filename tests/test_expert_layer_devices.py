"""Buffer.moe_int8 and devices, on the CPU: stand-ins for tensors and for the steps record where they would run."""
import contextlib

import pytest
import torch

from commbench_amd import ops


class Stand:
    """What moe_int8 looks at in a tensor."""

    def __init__(self, shape, dtype, device="cuda:1"):
        self.shape, self.dtype, self.device = torch.Size(shape), dtype, torch.device(device)
        self.is_cuda = self.device.type == "cuda"

    def dim(self):
        return len(self.shape)


class Handle:
    expert_offsets, num_tokens_per_expert = [0, 1], [1]


@pytest.fixture
def layer(monkeypatch):
    """(call(**changes), devices that were current at each step); the current device is 0, the tensors' 1."""
    current, seen = [0], []

    @contextlib.contextmanager
    def device(where):
        before, current[0] = current[0], torch.device(where).index
        yield
        current[0] = before

    def step(result):
        def run(*args, **kwargs):
            seen.append(current[0])
            return result
        return run
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(ops.Buffer, "dispatch", step((None, None, None, Handle())))
    monkeypatch.setattr(ops, "grouped_matmul_int8", step(None))
    monkeypatch.setattr(ops, "quantize_rows", step((None, None)))
    monkeypatch.setattr(ops, "combine", step("out"))
    buf = ops.Buffer.__new__(ops.Buffer)
    buf.num_experts, buf.workspace = 8, Stand((256,), torch.uint8)

    def call(**changes):
        args = dict(
            q=Stand((4, 64), torch.int8), scales=Stand((4, 1), torch.float32), topk_idx=Stand((4, 2), torch.int64),
            topk_weights=Stand((4, 2), torch.float32), w13=Stand((8, 64, 64), torch.int8), w13_scales=Stand((8, 64), torch.float32),
            w2=Stand((8, 64, 32), torch.int8), w2_scales=Stand((8, 64), torch.float32), bias=None)
        return buf.moe_int8(**dict(args, **changes))
    return call, seen


def test_every_step_runs_on_the_tensors_device(layer):
    call, seen = layer
    assert call() == "out"
    assert seen == [1] * 5                                # dispatch, product, codes, product, combine
    assert torch.cuda.current_device() == 0


@pytest.mark.parametrize("other", ["cpu", "cuda:0"])
@pytest.mark.parametrize("name,shape,dtype", [
    ("q", (4, 64), torch.int8), ("scales", (4, 1), torch.float32), ("topk_idx", (4, 2), torch.int64),
    ("topk_weights", (4, 2), torch.float32), ("bias", (4, 64), torch.bfloat16)])
def test_tensors_of_another_device_are_refused_before_any_launch(layer, other, name, shape, dtype):
    call, seen = layer
    with pytest.raises(ValueError, match="device"):
        call(**{name: Stand(shape, dtype, other)})
    if name == "bias":
        for pair in ([None, Stand(shape, dtype, other)], (Stand(shape, dtype), Stand(shape, dtype, other))):
            with pytest.raises(ValueError, match="device"):
                call(bias=pair)
    assert seen == []

"""The tensor-level helpers of the recurrent-block operators, without a GPU:
sizes that the C interface's 32-bit fields cannot hold are refused by the
helper and not cut off.  Tensors on the meta device have shapes only."""
import contextlib
import types

import pytest
import torch

import mamba_b200 as mb

BIG = 2 ** 32 + 16  # cut off to 32 bits: 16


def _meta(*shape, dtype=torch.float16):
    return torch.empty(shape, dtype=dtype, device="meta")


F32, I8 = torch.float32, torch.int8


@pytest.mark.parametrize("call", [
    lambda: mb.quantize_rows(_meta(1, BIG)),
    lambda: mb.linear_i8(_meta(1, BIG, dtype=I8), _meta(1, dtype=F32), _meta(8, BIG, dtype=I8), _meta(8, dtype=F32)),
    lambda: mb.linear_i8(_meta(1, 16, dtype=I8), _meta(1, dtype=F32), _meta(BIG, 16, dtype=I8), _meta(BIG, dtype=F32)),
    lambda: mb.gated_recurrence_step(*[_meta(BIG, 1)] * 3, _meta(1, dtype=F32), _meta(BIG, 1, dtype=F32)),
    lambda: mb.gated_recurrence_step(*[_meta(1, BIG)] * 3, _meta(BIG, dtype=F32), _meta(1, BIG, dtype=F32)),
    lambda: mb.gated_recurrence(*[_meta(1, BIG, 1)] * 3, _meta(1, dtype=F32)),
    lambda: mb.gated_recurrence(*[_meta(BIG, 1, 1)] * 3, _meta(1, dtype=F32)),
    lambda: mb.gated_recurrence_backward(*[_meta(1, BIG, 1)] * 4, _meta(1, dtype=F32), _meta(1, BIG, 1)),
    lambda: mb.block_norm(_meta(1, BIG), _meta(1, BIG, dtype=F32)),
], ids=["quantize cols", "i8 k", "i8 n", "step batch", "step dim", "seqlen", "batch", "backward seqlen", "norm cols"])
def test_sizes_beyond_32_bits(call):
    with pytest.raises(mb.MambaError, match="32 bits"):
        call()



def test_a_stream_of_another_device(monkeypatch):
    """The stream argument has to belong to the tensors' device: entering another
    device's stream would leave the call on the tensors' device's current one."""
    ran = []

    class Tensor:
        is_cuda, device = True, torch.device("cuda", 0)

    class Stream:
        def __init__(self, index):
            self.device = torch.device("cuda", index)

    cuda = types.SimpleNamespace(Stream=Stream, stream=lambda s: contextlib.nullcontext(ran.append(s)))
    monkeypatch.setattr(mb, "_torch_module", types.SimpleNamespace(Tensor=Tensor, cuda=cuda))
    helper = mb._on_stream(lambda t: "ran")
    same = Stream(0)
    assert helper(Tensor(), stream=same) == "ran" and ran == [same]
    with pytest.raises(mb.MambaError, match="device"):
        helper(Tensor(), stream=Stream(1))
    assert ran == [same]

"""Scratch buffers and rows that the operators of the 8-bit cache and of drafts must not be given."""
import pytest
import torch

from dlgo_amd.kernels import ops

DEV = "cuda:0"


class Claimed(torch.Tensor):
    """A host tensor that says it is on the device, for checks that launch nothing."""
    is_cuda = True


def claimed(t):
    return t.as_subclass(Claimed)


@pytest.mark.parametrize("dtype", [torch.float32, torch.uint8])
def test_elements_that_do_not_lie_in_a_row(dtype):
    """A broadcast element counts as many as are asked for and holds one: the kernels would write behind it."""
    beside = claimed(torch.zeros(4))
    good = claimed(torch.empty(100, dtype=dtype))
    assert ops._given_scratch("x", good, dtype, beside) is good
    for bad in (torch.empty(1, dtype=dtype).expand(100), torch.empty(200, dtype=dtype)[::2], torch.empty(100, dtype=torch.float64),
                torch.empty(10, 10, dtype=dtype), torch.empty(100, dtype=dtype, device="meta")):
        with pytest.raises(ops.KernelError, match="x: scratch"):
            ops._given_scratch("x", claimed(bad), dtype, beside)
    with pytest.raises(ops.KernelError, match="on the GPU"):
        ops._given_scratch("x", torch.empty(100, dtype=dtype), dtype, beside)


@pytest.mark.gpu
def test_the_calls_refuse_them():
    from test_q8_gpu import Step
    s = Step([1], [20000], 8, 2, 32)
    q = torch.randn(1, 256, device=DEV).bfloat16()
    asked = []
    s.fill()
    want = s.attend(q, scratch=lambda n: asked.append(n) or torch.empty(n, device=DEV))
    assert asked and torch.isfinite(want).all()
    v = dict(logits=torch.zeros(3, 50, device=DEV), draft_tokens=torch.zeros(2, dtype=torch.int32, device=DEV),
             cu_drafts=torch.tensor([0, 2], dtype=torch.int32, device=DEV), temperature=torch.ones(1, device=DEV), uniform=torch.zeros(3, device=DEV),
             accepted=torch.zeros(1, dtype=torch.int32, device=DEV), token=torch.zeros(1, dtype=torch.int32, device=DEV), max_drafts=2)
    for make in (lambda n, dt: torch.empty(1, dtype=dt, device=DEV).expand(n), lambda n, dt: torch.empty(2 * n, dtype=dt, device=DEV)[::2],
                 lambda n, dt: torch.empty(n, dtype=dt)):
        with pytest.raises(ops.KernelError, match="attention_q8: scratch"):
            s.attend(q, scratch=lambda n: make(n, torch.float32))
        with pytest.raises(ops.KernelError, match="verify_drafts: scratch"):
            ops.verify_drafts(**v, scratch=lambda n: make(n, torch.uint8))


def test_rows_further_apart_than_a_32_bit_number_says():
    """The kernels take a row's stride in 32 bits: its low ones alone would name other rows."""
    far = torch.empty_strided((2, 256), (2 ** 32 + 256, 1), dtype=torch.bfloat16, device="meta")
    near = torch.empty_strided((2, 256), (2 ** 31 - 8, 1), dtype=torch.bfloat16, device="meta")
    assert ops._rows(far, "x") == 2 ** 32 + 256 and ops._rows32(near, "x") == 2 ** 31 - 8
    with pytest.raises(ops.KernelError, match="x: rows 4294967552 elements apart"):
        ops._rows32(far, "x")

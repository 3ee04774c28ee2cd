"""Weights and rows in 8 bits hand their kernels the places of the tensors that they hold, whatever became of an object they were copied
from; no GPU needed."""
import copy
import io

import pytest
import torch

from tiny_llm_infer_b200 import ops


def saved_and_loaded(x):
    file = io.BytesIO()
    torch.save(x, file)
    file.seek(0)
    return torch.load(file, weights_only=False)


def weight():
    return ops.Fp8Weight(torch.ones((272, 144)).to(torch.float8_e4m3fn), torch.arange(8.0).view(4, 2), gated=True)


def rows():
    return ops.Fp8Rows(torch.ones((3, 144)).to(torch.float8_e4m3fn), torch.arange(6.0).view(3, 2))


@pytest.mark.parametrize("make", [weight, rows])
@pytest.mark.parametrize("how", [copy.copy, copy.deepcopy, saved_and_loaded])
def test_a_copy_knows_its_own_tensors(make, how):
    first = make()
    second = how(first)
    assert type(second) is type(first) and second.shape == first.shape and second.index == first.index
    assert second.pointers == (second.q.data_ptr(), second.scales.data_ptr())
    assert torch.equal(second.q.view(torch.uint8), first.q.view(torch.uint8)) and torch.equal(second.scales, first.scales)
    if make is weight:
        assert second.gated is True


@pytest.mark.parametrize("make", [weight, rows])
def test_tensors_moved_behind_its_back_are_refused(make):
    """A tensor given other storage (``.data``, ``resize_``) is not the one that was checked."""
    for name in ("q", "scales"):
        made = make()
        kept = getattr(made, name)
        kept.data = kept.data.clone()
        with pytest.raises(ops.KernelError, match="moved"):
            made.pointers


def test_rows_of_a_kernel_are_copied_with_their_buffer():
    """What a kernel makes lies in one buffer; a copy is a pair of tensors like any other."""
    made = ops.fp8._empty_rows(3, 144, "cpu")
    made.q.view(torch.uint8).fill_(7)
    made.scales.fill_(0.5)
    other = copy.deepcopy(made)
    assert other.pointers == (other.q.data_ptr(), other.scales.data_ptr()) and other.pointers[0] != made.pointers[0]
    assert (other.q.view(torch.uint8) == 7).all() and (other.scales == 0.5).all()


def test_8_bit_rows_take_an_8_bit_weight():
    plain = torch.zeros((16, 144), dtype=torch.bfloat16)
    for call in (ops.linear, ops.linear_swiglu):
        with pytest.raises(ops.KernelError, match="8-bit weight"):
            call(rows(), plain)

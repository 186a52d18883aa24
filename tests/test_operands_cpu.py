"""CPU tests of the native checks behind NativeOps (csrc/operands.cpp): what they refuse here,
where no tensor is on a GPU, and the tensors they make."""
import pytest

torch = pytest.importorskip("torch")

from tinyinfer_amd import _operands  # noqa: E402


def test_what_is_not_a_gpu_tensor_is_refused():
    x = torch.zeros(2, 3, 4, 8, dtype=torch.float16)
    for other in (x, None, 3, [1.0], "x"):
        assert _operands.operand(other, torch.float16, -2, -1, None) is None
        assert _operands.rows(other, torch.float16, -2, None) is None
    assert _operands.operand(x, torch.float16, -1, 4, x.shape) is None  # (a CPU tensor's GPU is number -1)
    assert _operands.operand(x, "float16", -2, 4, None) is None


def test_tensors_of_a_shape():
    like = torch.zeros(2, 3, dtype=torch.int32)
    for shape in ((5,), (2, 3, 4), torch.Size([7, 1]), (0, 4)):
        y = _operands.empty(shape, like)
        assert y.shape == shape and y.dtype == torch.int32 and y.device == like.device and y.is_contiguous() and not y.requires_grad
        assert _operands.empty_as(shape, torch.float32, like).dtype == torch.float32
    assert _operands.empty((3, 2), like.t()).is_contiguous()


@pytest.mark.parametrize("call", [
    lambda x: _operands.operand(x), lambda x: _operands.rows(x, torch.float16), lambda x: _operands.empty([2, 3], x),
    lambda x: _operands.empty((2, 3), None), lambda x: _operands.empty((2, "3"), x), lambda x: _operands.empty_as((2,), "f", x),
    lambda x: _operands.empty_as((2,), torch.float32, 0), lambda x: _operands.record(x, 0, 0), lambda x: _operands.record([3], 0, 0)])
def test_wrong_arguments(call):
    with pytest.raises(TypeError):
        call(torch.zeros(2))


def test_a_negative_extent():
    with pytest.raises(ValueError):
        _operands.empty((2, -3), torch.zeros(2))

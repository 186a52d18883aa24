"""NativeOps under a torch that csrc/operands.cpp was not compiled for, or without it: the checks
are made in Python, with the same answers, and the calls are the same."""
import sys

import pytest

torch = pytest.importorskip("torch")

import tinyinfer_amd  # noqa: E402
from tinyinfer_amd import native_ops  # noqa: E402
from tinyinfer_amd.native_ops import NativeOps  # noqa: E402


def made(monkeypatch, how):
    """NativeOps whose extension is of another torch, or missing."""
    from tinyinfer_amd import _operands
    with monkeypatch.context() as other:
        if how == "other":
            other.setattr(_operands, "torch_version", "1.0")
        else:
            other.delattr(tinyinfer_amd, "_operands", raising=False)
            other.setitem(sys.modules, "tinyinfer_amd._operands", None)
        with pytest.warns(RuntimeWarning, match="tinyinfer_amd.build"):
            return NativeOps()


def test_the_extension_is_of_this_torch():
    from tinyinfer_amd import _operands
    assert _operands.torch_version == torch.__version__
    assert NativeOps().operands is _operands


@pytest.mark.parametrize("how", ["other", "missing"])
def test_made_without_the_extension(monkeypatch, how):
    ops = made(monkeypatch, how)
    assert isinstance(ops.operands, native_ops._PlainOperands)
    with pytest.raises(TypeError):
        ops.gelu_new(torch.zeros(4, dtype=torch.float16))


def test_plain_checks_refuse_what_is_not_a_gpu_tensor():
    plain = native_ops._PlainOperands(torch)
    x = torch.zeros(2, 3, 4, 8, dtype=torch.float16)
    for other in (x, None, 3, [1.0], "x"):
        assert plain.operand(other, torch.float16, -2, -1, None) is None
        assert plain.rows(other, torch.float16, -2, None) is None
    for shape in ((5,), torch.Size([7, 1]), (0, 4)):
        y = plain.empty(shape, x.int())
        assert y.shape == shape and y.dtype == torch.int32 and y.is_contiguous()
        assert plain.empty_as(shape, torch.float32, x).dtype == torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["other", "missing"])
def test_the_same_answers_and_calls(monkeypatch, how):
    from tinyinfer_amd import _operands
    ops, want = made(monkeypatch, how), NativeOps()
    half = torch.randn(2, 6, 4, 64, device="cuda").half()
    large = torch.empty(1, dtype=torch.float16, device="cuda").expand(1 << 16, 1 << 15)
    operands = (half, half.float(), half[:, ::2], half.transpose(1, 2), half[..., ::2], half[..., :1], half[:0], half[0, 0, 0, 0], large,
                half.clone().requires_grad_(), half.cpu(), None)
    for x in operands:
        for dtype in (torch.float16, torch.float32):
            for index in (-2, 0, 1):
                for shape in (None, (2, 6, 4, 64), torch.Size([2, 6, 4, 64]), (2, 6, 4, 63)):
                    assert ops.operands.rows(x, dtype, index, shape) == _operands.rows(x, dtype, index, shape)
                    for rank in (-1, 0, 4):
                        assert ops.operands.operand(x, dtype, index, rank, shape) == _operands.operand(x, dtype, index, rank, shape)
    # A step of several calls on another stream, its inputs freed behind it.
    rotary, cache = ops.rotary(64), ops.kv_cache_paged(4, 6, 32, 64)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")

    def step(o):
        q, k, v = (half * i for i in (1, 2, 3))
        q = o.kv_append_paged(cache, k, v, table, 7, rotary=rotary, q=q)
        y = o.attention_paged(q, cache, table, 11)
        logits = o.gemm(y.view(48, 64), half[0, 0].t().contiguous(), output_dtype=torch.float32)
        return [q, y, logits, *o.logprobs(logits, table.view(-1)[:1].repeat(48), top=2)]

    expected = step(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(ops)
    side.synchronize()
    for x, y in zip(got, expected):
        assert torch.equal(x, y)

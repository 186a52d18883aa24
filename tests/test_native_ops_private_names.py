"""NativeOps does not need torch's private names: a torch without GPU support lacks them,
and they are not part of its interface."""
import pytest

torch = pytest.importorskip("torch")

from tinyinfer_amd.native_ops import NativeOps  # noqa: E402

NAMES = ("_cuda_getCurrentRawStream", "_cuda_getDevice")


def test_made_without_the_private_names(monkeypatch):
    for name in NAMES:
        monkeypatch.delattr(torch._C, name, raising=False)
    ops = NativeOps()
    with pytest.raises(TypeError):
        ops.gelu_new(torch.zeros(4, dtype=torch.float16))


@pytest.mark.gpu
def test_calls_without_the_private_names(monkeypatch):
    x = torch.randn(4, 100, device="cuda").half()
    want = NativeOps().gelu_new(x)
    with monkeypatch.context() as without:
        for name in NAMES:
            without.delattr(torch._C, name)
        ops = NativeOps()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    assert torch.equal(ops.gelu_new(x), want)
    with torch.cuda.stream(side):
        y = ops.gelu_new(x)
    side.synchronize()
    assert torch.equal(y, want)

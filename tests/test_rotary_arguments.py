"""Rotary positions whose frequencies or factor no kernel could use are refused where they are made,
as every other argument is."""
import math

import pytest

torch = pytest.importorskip("torch")

from tinyinfer_amd.native_ops import NativeOps  # noqa: E402


@pytest.mark.parametrize("rotated,args", [
    (64, {"base": 10 ** 400}), (64, {"base": 5e-324}), (4, {"scaling": "base", "factor": 1e200}), (64, {"factor": 1e-320, "scaling": "linear"}),
    (64, {"scaling": "base", "factor": 1e300}), (4, {"frequencies": [1.0, 10 ** 400]}), (64, {"amplitude": 1e39}), (64, {"amplitude": -1e300}),
    (64, {"amplitude": 10 ** 400}), (64, {"scaling": "parts", "factor": 1e-320, "original_length": 100}),
    (64, {"scaling": "parts", "factor": 2.0, "original_length": 100, "fast": 10 ** 400})])
def test_numbers_out_of_range(rotated, args):
    with pytest.raises(ValueError):
        NativeOps().rotary(rotated, **args)


def test_numbers_in_range_reach_the_device():
    """The last check is the device's, so these are not refused for their numbers."""
    for args in ({"base": 1e300}, {"amplitude": 3e38}, {"factor": 1e30, "scaling": "linear"}, {"frequencies": [1e300, 0.0]}):
        with pytest.raises(TypeError, match="device"):
            NativeOps().rotary(4, device="cpu", **args)
    assert math.isfinite(1e300)

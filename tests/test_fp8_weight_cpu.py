"""CPU: Fp8Weight.quantize refuses what no handle can be made of before it works on it."""
import pytest
import torch

from zoomkv_revision_b200 import ops


@pytest.mark.parametrize("shape,parts", [((32, 256), 0), ((48, 256), 3), ((32, 256), -1), ((33, 256), 2), ((48, 256), 2),
                                         ((32, 250), 1), ((0, 256), 1), ((32, 0), 1), ((32,), 1), ((2, 32, 256), 1)])
def test_shapes(shape, parts):
    with pytest.raises(ValueError, match="parts must|multiple of parts|multiples of 16"):
        ops.Fp8Weight.quantize(torch.zeros(shape), parts)
    assert not torch.cuda.is_initialized()


def test_a_weight_on_the_cpu():
    with pytest.raises(ValueError, match="CUDA"):
        ops.Fp8Weight.quantize(torch.zeros(32, 256))

"""The norms' backward pass on both sides of the sizes at which its launches change."""
import pytest

from tests import test_gpu_all_reduce_norm as base

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gate", ["channel", "element"])
@pytest.mark.parametrize("rows,cols,dtype", [(5, 4096, "bf16"), (6, 4096, "bf16"), (4, 8192, "bf16"), (5, 8192, "bf16"), (4, 4097, "bf16"),
                                             (5, 2048, "fp32"), (6, 2047, "fp32"), (4, 4096, "fp32"), (5, 4095, "fp32"),
                                             (2, 8192, "fp32"), (3, 8192, "fp32"), (3, 5001, "fp32")])
def test_one_workgroup_and_several(cuda, rows, cols, dtype, gate):
    base.test_backward(cuda, (rows, cols), dtype, True, gate, 1.0, True)

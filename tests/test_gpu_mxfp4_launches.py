"""The 4-bit product at the ends of what its launches take: results of many rows or columns."""
import pytest
import torch

from tests.test_gpu_mxfp4 import _activations

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,K", [(16, 64), (1, 31), (32, 256), (17, 200)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_a_narrow_result_of_more_rows_than_one_grid_dimension_has_groups(cuda, N, K, out_dtype):
    """65535 groups of 64 rows and some more: the first and last rows are those rows alone (K is one slab:
    one order of its sum, whatever the kernel)."""
    from symm_mem_recipes import mxfp4_matmul, mxfp4_quantize
    M = 65535 * 64 + 70
    a = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    a[:100], a[-200:] = _activations(100, K, torch.bfloat16, 1), _activations(200, K, torch.bfloat16, 2)
    b = mxfp4_quantize(_activations(N, K, torch.bfloat16, 3))
    got = mxfp4_matmul(a, b, out_dtype=out_dtype)
    assert got.shape == (M, N)
    assert torch.equal(got[:100], mxfp4_matmul(a[:100], b, out_dtype=out_dtype))
    assert torch.equal(got[-200:], mxfp4_matmul(a[-200:], b, out_dtype=out_dtype))
    assert not bool(got[100:-200].any())


@pytest.mark.parametrize("M", [1, 16])
def test_a_few_rows_against_more_columns_than_one_launch_of_rows_takes(cuda, M):
    from symm_mem_recipes import MxFp4Tensor, mxfp4_matmul, mxfp4_quantize
    N, K = 2 ** 28 + 100, 32
    tail = mxfp4_quantize(_activations(116, K, torch.bfloat16, 4))              # rows N - 116 .., whole units
    b = MxFp4Tensor.empty(N, K, "cuda")                                         # 36.5 GB; one slab: units of 16 rows in a row
    b.codes.zero_()
    b.scales.zero_()
    b.codes[-8 * 2048:].copy_(tail.codes)
    b.scales[-8 * 128:].copy_(tail.scales)
    a = _activations(M, K, torch.bfloat16, 5)
    got = mxfp4_matmul(a, b)
    assert torch.equal(got[:, -116:], mxfp4_matmul(a, tail))
    assert not bool(got[:, :2 ** 20].any()) and not bool(got[:, 2 ** 27:2 ** 27 + 2 ** 20].any())
    assert torch.equal(mxfp4_matmul(mxfp4_quantize(a), b)[:, -200:], got[:, -200:])

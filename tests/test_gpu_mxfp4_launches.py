"""The 4-bit product at the ends of what its launches take: results of many rows or columns, rows that fill their
share of LDS, and launches that the sizes of test_gpu_mxfp4.py do not reach."""
import pytest
import torch

from tests import mxfp4_oracle as mx
from tests import test_gpu_mxfp4 as base
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


# A few rows still in their own type, in one launch: one, two and four units of columns per workgroup with up to 80 KB
# of LDS (11 rows of 8192, 16 of 5632: the most that go), and just past it in two launches.
ROWS = [(1, 8192, 8192), (8, 8193, 8192), (11, 8195, 8192), (12, 8195, 8192), (16, 4113, 5632), (16, 4113, 5633), (11, 3584, 8192),
        (12, 3001, 8192), (11, 17003, 8192), (12, 17003, 8192), (2, 4097, 45056), (3, 4097, 40000), (1, 5000, 90112), (1, 5000, 90113)]


@pytest.mark.parametrize("M,N,K", ROWS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_rows_up_to_their_share_of_lds_and_past_it(cuda, lib, M, N, K, dtype):
    from symm_mem_recipes import mxfp4_matmul, mxfp4_quantize
    slabs = -(-K // 256)
    assert lib.smr_mxfp4_matmul_rows_limit(K) == min(16, 352 // slabs)
    a, b = _activations(M, K, dtype, M + K), mxfp4_quantize(_activations(N, K, torch.bfloat16, N))
    a64 = mx.values(*mx.quantize(a))[:, :K].cuda()
    b64 = b.dequantize(torch.float32).double()                # (the quantiser and its inverse have tests of their own)
    want, size = a64 @ b64.t(), a64.abs() @ b64.abs().t()
    for out_dtype in (torch.bfloat16, torch.float32):
        got = mxfp4_matmul(a, b, out_dtype=out_dtype)
        bound = want.abs() * torch.finfo(out_dtype).eps / 2 + (K + 16) * 2.0 ** -24 * size * (1 + 2.0 ** -7)
        off = (got.double() - want).abs()
        assert bool((off <= bound).all()), float((off - bound).max())
        assert torch.equal(mxfp4_matmul(a, b, out_dtype=out_dtype), got)


@pytest.mark.parametrize("M,N,K", [(3080, 4865, 700), (4339, 5739, 300), (3094, 4903, 257)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_several_passes_of_256_x_128_tiles(cuda, M, N, K, out_dtype):
    """More tiles than compute units, the next one's first slabs on their way under the stores of the last."""
    base.test_large_product(cuda, M, N, K, out_dtype)

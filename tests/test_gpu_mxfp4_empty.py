"""4-bit operands that contract over nothing: a weight's gradient for an empty batch."""
import pytest
import torch

from tests.test_gpu_mxfp4 import _activations

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_the_products_of_no_tokens(cuda, dtype):
    """Forward and backward products of a linear layer for zero tokens: empty results, and zeros for the weights."""
    from symm_mem_recipes import MxFp4Tensor, mxfp4_matmul, mxfp4_quantize
    x, dy = (_activations(3, n, dtype, 1)[0:0] for n in (64, 48))
    w = _activations(48, 64, dtype, 2)
    assert mxfp4_matmul(x, mxfp4_quantize(w)).shape == (0, 48)
    assert mxfp4_matmul(dy, mxfp4_quantize(w, transpose=True)).shape == (0, 64)
    left, right = mxfp4_quantize(dy, transpose=True), mxfp4_quantize(x, transpose=True)
    assert left.shape == (48, 0) and right.shape == (64, 0) and left.dequantize().shape == (48, 0)
    for out_dtype in (torch.bfloat16, torch.float32):
        dw = mxfp4_matmul(left, right, out_dtype=out_dtype)
        assert dw.shape == (48, 64) and dw.dtype == out_dtype and not bool(dw.any())
    out = torch.full((48, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    assert mxfp4_matmul(left, right, out=out) is out and not bool(out.any())
    for rows in (1, 16, 40):                                       # a left operand still in its own type
        a = torch.empty(rows, 0, dtype=dtype, device="cuda")
        got = mxfp4_matmul(a, right)
        assert got.shape == (rows, 64) and not bool(got.any())
        assert mxfp4_quantize(a).shape == (rows, 0)
    codes, scales = right.to_blocks()
    assert codes.shape == (64, 0) and scales.shape == (64, 0)
    assert MxFp4Tensor.from_blocks(codes, scales).shape == (64, 0)


def test_a_captured_product_of_no_tokens(cuda):
    from symm_mem_recipes import mxfp4_matmul, mxfp4_quantize
    x = mxfp4_quantize(torch.empty(0, 64, dtype=torch.bfloat16, device="cuda"), transpose=True)
    out = torch.empty(64, 64, dtype=torch.bfloat16, device="cuda")
    mxfp4_matmul(x, x, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mxfp4_matmul(x, x, out=out)
    for _ in range(3):
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert not bool(out.any())

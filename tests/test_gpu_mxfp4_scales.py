"""Products of operands whose scales are far apart: the instruction applies both to an exact product, so neither
operand's own range limits the result."""
import pytest
import torch

from tests.test_gpu_mxfp4 import _activations

pytestmark = pytest.mark.gpu


# a few rows in their own launch, units of rows, the ring, each of the tiles
@pytest.mark.parametrize("M,N,K", [(3, 50, 300), (40, 70, 520), (512, 700, 700), (300, 3000, 900), (1100, 3001, 300), (1500, 3500, 300), (1500, 3500, 1100),
                                   (4000, 3584, 257), (4097, 3585, 257)])
@pytest.mark.parametrize("power", [-120, -60, 60, 120])
def test_scales_far_apart(cuda, M, N, K, power):
    """a * 2^power against b * 2^-power is a against b, bit for bit: every scale moves by a power of two."""
    from symm_mem_recipes import mxfp4_matmul, mxfp4_quantize
    a = _activations(M, K, torch.float32, 1).clamp(-7, 7)
    b = _activations(N, K, torch.float32, 2).clamp(-7, 7)
    # magnitudes of at least 2^-4 leave every block's scale a code at both ends
    a, b = (torch.where(t.abs() < 2.0 ** -4, 2.0 ** -4, t) for t in (a, b))
    want = mxfp4_matmul(a, mxfp4_quantize(b), out_dtype=torch.float32)
    far = mxfp4_quantize(torch.ldexp(b, torch.tensor(-power, device="cuda")))
    shifted = torch.ldexp(a, torch.tensor(power, device="cuda"))
    assert bool(torch.isfinite(shifted).all())
    assert torch.equal(mxfp4_matmul(shifted, far, out_dtype=torch.float32), want)
    assert torch.equal(mxfp4_matmul(mxfp4_quantize(shifted), far, out_dtype=torch.float32),
                       mxfp4_matmul(mxfp4_quantize(a), mxfp4_quantize(b), out_dtype=torch.float32))


def test_results_at_the_ends_of_fp32(cuda):
    """Products past fp32's range are infinite; subnormal ones are kept or become zero, never anything else."""
    from symm_mem_recipes import mxfp4_matmul, mxfp4_quantize
    one = torch.ones(20, 32, device="cuda")
    for M in (4, 20):
        a = one[:M] * 2.0 ** 100
        assert bool((mxfp4_matmul(a, mxfp4_quantize(one * 2.0 ** 100), out_dtype=torch.float32) == float("inf")).all())
        assert bool((mxfp4_matmul(a, mxfp4_quantize(one * -2.0 ** 100)) == -float("inf")).all())
        assert bool((mxfp4_matmul(a, mxfp4_quantize(one * 2.0 ** 20), out_dtype=torch.float32) == 32 * 2.0 ** 120).all())
        small = mxfp4_matmul(one[:M] * 2.0 ** -100, mxfp4_quantize(one * 2.0 ** -40), out_dtype=torch.float32)
        assert bool(((small >= 0) & (small <= 32 * 2.0 ** -140)).all())

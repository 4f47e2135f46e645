"""Rows whose values fit their type but whose squares do not fit fp32: the norms hold over the type's range."""
import pytest
import torch

from tests import norm_oracle as oracle
from tests.test_gpu_all_reduce_norm import DTYPES, _cuda, _inputs, _symmetric, _within

pytestmark = pytest.mark.gpu

# a factor for every third row in turn: ordinary rows stand between them
LARGE, LARGEST, SMALL = 1e25, 2.0 ** 125, 1e-28
SHAPES = [((7, 5), 3, "bf16"), ((7, 3), 2, "fp32"), ((9, 200), 8, "bf16"), ((5, 1001), 5, "fp32"), ((4, 1001), 7, "bf16"),
          ((300, 8192), 8, "bf16"), ((261, 8001), 2, "bf16"), ((270, 4096), 4, "fp32"), ((3, 16384), 3, "bf16"),
          ((4, 16381), 2, "fp32"), ((600, 512), 2, "bf16"), ((700, 64), 1, "fp32")]


def _scaled(t, factors, dim):
    """Rows of t times a factor each; kept within what the type holds."""
    shape = [1] * t.dim()
    shape[dim] = -1
    return (t.double().clamp(-3, 3) * factors.double().view(shape)).to(t.dtype)


def _factors(rows, sizes):
    return torch.tensor([1.0 if r % 3 else sizes[r // 3 % len(sizes)] for r in range(rows)], dtype=torch.float64)


@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("gate", ["none", "channel"])
@pytest.mark.parametrize("shape,ranks,dtype", SHAPES)
def test_forward_over_the_range_of_the_type(cuda, shape, ranks, dtype, gate, post):
    """Sums, residuals or both are large or small in every third row; with eps 0 a row's norm does not depend on
    its size at all.  Scaling by a power of two rounds nothing, so the bounds are those of ordinary rows."""
    from symm_mem_recipes import EmulatedSymmetricMemory as SM, one_shot_all_reduce_norm
    dtype = DTYPES[dtype]
    partials, residual, weight, post_weight, g = _inputs(shape, ranks, dtype, post, gate, sum(shape) + 11)
    w, p, gc = _cuda(weight, post_weight, g)
    for sizes, both, eps in (((LARGE, LARGEST / 8), True, 1e-6), ((LARGE, LARGEST / 8), False, 1e-6), ((SMALL, LARGE), True, 0.0)):
        factors = _factors(shape[0], sizes)
        big = _scaled(partials, factors / ranks, 1)
        x = _scaled(residual, factors if both else torch.ones_like(factors), 0)
        t, handle = _symmetric(big, 0)
        got = one_shot_all_reduce_norm(t, x.cuda(), w, post_weight=p, gate=gc, eps=eps, return_sum=True)
        args = (big, x, weight, post_weight, g, 1.0, eps)
        want = oracle.forward(*args)
        assert bool(torch.isfinite(want[0]).all()) and bool((want[0].abs().amax(-1) > 0.1).all())
        for a, b, c in zip(got, want, oracle.forward_bounds(*args)):
            _within(a, b, c, dtype)
        handle.check_status()
        SM.release()


def test_ordinary_rows_beside_large_ones_keep_their_bits(cuda):
    from symm_mem_recipes import EmulatedSymmetricMemory as SM, one_shot_all_reduce_norm
    for shape in ((301, 8192), (9, 1000), (8, 6)):
        partials, residual, weight, post_weight, g = _inputs(shape, 4, torch.bfloat16, True, "element", 4)
        x, w, p, gc = _cuda(residual, weight, post_weight, g)
        t, _ = _symmetric(partials, 0)
        plain = one_shot_all_reduce_norm(t, x, w, post_weight=p, gate=gc, return_sum=True)
        factors = _factors(shape[0], (LARGE, SMALL, LARGEST / 8))
        t, _ = _symmetric((partials.double() * factors.view(1, -1, 1) / 4).to(torch.bfloat16), 0)
        keep = (factors == 1).cuda()
        t.copy_(torch.where(keep[:, None], partials[0].cuda(), t))
        for r in range(1, 4):
            buf = SM.rendezvous(t).get_buffer(r, shape, torch.bfloat16)
            buf.copy_(torch.where(keep[:, None], partials[r].cuda(), buf))
        for got, want in zip(one_shot_all_reduce_norm(t, x, w, post_weight=p, gate=gc, return_sum=True), plain):
            assert torch.equal(got[keep], want[keep])
        SM.release()


BACKWARD_SHAPES = [((7, 5), "bf16"), ((7, 3), "fp32"), ((9, 200), "bf16"), ((4, 1001), "fp32"), ((530, 8192), "bf16"),
                   ((261, 8001), "bf16"), ((270, 4096), "fp32"), ((265, 8191), "fp32"), ((5, 16384), "bf16"), ((4, 9001), "fp32"),
                   ((600, 512), "bf16")]


@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("gate", ["none", "channel", "token", "element"])
@pytest.mark.parametrize("shape,dtype", BACKWARD_SHAPES)
def test_backward_over_the_range_of_the_type(cuda, shape, dtype, gate, post):
    """The forward pass's sums and outputs are large or small in every third row.  The bound on the terms of a
    gradient is that of ordinary rows (at most 128 roundings, and the terms of a column sum): scaling by a power of two
    rounds nothing, a subnormal reciprocal root (rows past 2^126) does not occur."""
    from symm_mem_recipes import one_shot_all_reduce_norm_backward
    from tests.test_gpu_all_reduce_norm import _backward_inputs
    dtype = DTYPES[dtype]
    dy, dh, s, h, w, p, g = _backward_inputs(shape, dtype, post, gate, True, sum(shape) + 5)
    rows = shape[0]
    for sizes, eps in (((LARGE, 2.0 ** 115), 1e-6), ((1e-16, LARGE), 0.0)):
        factors = _factors(rows, sizes)
        # (without the norm behind the block the gate's gradient has the sums as a factor: D times them may pass the type)
        hs, ss = _scaled(h, factors, 0), _scaled(s, factors.flip(0) if post else torch.ones_like(factors), 0)
        args = (dy, dh, ss, hs, w, p, g, 1.0, eps)
        a = _cuda(*args[:7])
        got = one_shot_all_reduce_norm_backward(a[0], a[1], a[2], a[3], a[4], post_weight=a[5], gate=a[6], eps=eps)
        want, size = oracle.backward(*args), oracle.backward(*args, magnitudes=True)
        for name, b in want.items():
            off = size[name] * (128 + rows / 128 + 64) * oracle.U
            _within(getattr(got, name).reshape(b.shape), b, off, dtype)


def test_gradients_of_ordinary_rows_beside_large_ones_keep_their_bits(cuda):
    from symm_mem_recipes import one_shot_all_reduce_norm_backward
    from tests.test_gpu_all_reduce_norm import _backward_inputs
    for shape in ((301, 8192), (9, 1000), (8, 6), (6, 12000)):
        dy, dh, s, h, w, p, g = _cuda(*_backward_inputs(shape, torch.bfloat16, True, "element", True, 9))
        plain = one_shot_all_reduce_norm_backward(dy, dh, s, h, w, post_weight=p, gate=g)
        factors = _factors(shape[0], (LARGE,)).cuda()
        keep = factors == 1
        large = [torch.where(keep[:, None], t, (t.double() * factors[:, None]).bfloat16()) for t in (s, h)]
        got = one_shot_all_reduce_norm_backward(dy, dh, *large, w, post_weight=p, gate=g)
        for name in ("partial", "residual", "gate"):
            assert torch.equal(getattr(got, name)[keep], getattr(plain, name)[keep]), name

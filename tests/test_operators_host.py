"""Refusals and host-side logic of the layer-boundary operators: nothing here touches a GPU."""
import pytest
import torch

from tests import mxfp4_oracle as mx
from tests import norm_oracle


def test_mxfp4_argument_errors(lib):
    p = 0x1000
    q = lib.smr_mxfp4_quantize
    assert q(p, 64, p, p, 1, 64, 2, 0, None) == -1                   # dtype
    assert q(p, 63, p, p, 2, 64, 0, 0, None) == -1                   # overlapping rows
    assert q(p, 64, p, p, -1, 64, 0, 0, None) == -1
    assert q(None, 64, p, p, 1, 64, 0, 0, None) == -1
    assert q(p, 64, None, p, 1, 64, 0, 0, None) == -1
    assert q(p + 1, 64, p, p, 1, 64, 0, 0, None) == -1               # half an element
    assert q(p, 64, p + 8, p, 1, 64, 0, 0, None) == -1               # codes off their boundary
    assert q(p, 64, p, p + 2, 1, 64, 0, 0, None) == -1
    assert q(p, 2 ** 31 - 1, p, p, 2 ** 31 - 1, 2 ** 31 - 1, 0, 0, None) == -2
    assert q(p, 64, p, p, 0, 64, 0, 0, None) == 0                    # nothing to do: no launch
    d = lib.smr_mxfp4_dequantize
    assert d(p, p, p, 1, 64, 7, None) == -1
    assert d(p, p, None, 1, 64, 0, None) == -1
    assert d(p, p, p + 2, 1, 64, 1, None) == -1                      # fp32 off its boundary
    assert d(p, p + 8, p, 1, 64, 0, None) == -1
    assert d(p, p, p, 0, 64, 0, None) == 0
    m = lib.smr_mxfp4_matmul
    assert m(p, p, p, p, p, 1, 16, 0, 0, None) == -1                 # nothing contracted
    assert m(p, p, p, p, p, 1, 16, 32, 2, None) == -1
    assert m(p, None, p, p, p, 1, 16, 32, 0, None) == -1
    assert m(p, p + 4, p, p, p, 1, 16, 32, 0, None) == -1
    assert m(p, p, p, p, p + 1, 1, 16, 32, 0, None) == -1
    assert m(p, p, p, p, p, 2 ** 31, 16, 32, 0, None) == -1
    assert m(p, p, p, p, p, 0, 16, 32, 0, None) == 0
    assert lib.smr_mxfp4_code_bytes(17, 257) == 2 * 2 * 2048 and lib.smr_mxfp4_scale_bytes(17, 257) == 2 * 2 * 128
    assert lib.smr_mxfp4_code_bytes(-1, 1) == -1


def test_norm_argument_errors(lib):
    import ctypes
    p = 0x1000
    bufs = (ctypes.c_uint64 * 8)(*[0x10000 * (r + 1) for r in range(8)])
    pads = (ctypes.c_uint64 * 8)(*[0x900000 + 0x10000 * r for r in range(8)])

    def forward(buf=bufs, pad=pads, residual=p, weight=p, post=None, gate=None, kind=0, normed=p, rows=1, cols=64, dtype=0,
                rank=0, ws=8, mode=1):
        return lib.smr_all_reduce_norm(buf, pad, residual, weight, post, gate, kind, normed, p, None, rows, cols, dtype, 1.0,
                                       1e-6, rank, ws, mode, None, None)

    assert forward(rows=0) == 0
    assert forward(dtype=2) == -1 and forward(cols=0) == -1 and forward(cols=16385) == -2 and forward(rows=-1) == -1
    assert forward(rank=8) == -1 and forward(rank=-1) == -1 and forward(ws=9) == -1 and forward(mode=2) == -1
    assert forward(buf=None) == -1 and forward(pad=None) == -1 and forward(pad=None, mode=0, rows=0) == 0
    assert forward(gate=p) == -1 and forward(kind=1) == -1 and forward(gate=p, kind=4) == -1
    assert forward(residual=None) == -1 and forward(normed=None) == -1 and forward(weight=p + 1) == -1
    bufs[5] = 0
    assert forward() == -1
    bufs[5], pads[2] = 0x60000, 0x900001
    assert forward() == -1
    assert b"signal pad" in lib.smr_last_error_string()

    need = lib.smr_norm_backward_scratch_bytes(1000, 64, 0, 1, 1)
    assert need == 3 * 1000 * 64 * 4 and lib.smr_norm_backward_scratch_bytes(1000, 8192, 0, 0, 0) == 256 * 8192 * 4
    assert lib.smr_norm_backward_scratch_bytes(1, 64, 0, 1, 1) == 0 and lib.smr_norm_backward_scratch_bytes(1000, 3, 1, 1, 1) == 0
    assert lib.smr_norm_backward_scratch_bytes(1000, 16385, 0, 1, 1) == -1

    def backward(dy=p, post=p, gate=p, kind=1, dpost=p, dgate=p, scratch=p, size=need, rows=1000, cols=64):
        return lib.smr_norm_backward(dy, p, p, p, p, post, gate, kind, p, p, p, dpost, dgate, scratch, size, rows, cols, 0, 1.0,
                                     1e-6, None)

    assert backward(size=need - 4) == -1
    assert b"scratch" in lib.smr_last_error_string()
    assert backward(rows=0) == -1 and backward(cols=16385) == -2 and backward(dy=None) == -1 and backward(scratch=None) == -1
    assert backward(dpost=None) == -1 and backward(dgate=None) == -1 and backward(dy=p + 1) == -1


def test_python_refusals():
    from symm_mem_recipes import (MxFp4Tensor, mxfp4_matmul, mxfp4_quantize, one_shot_all_reduce_norm,
                                  one_shot_all_reduce_norm_backward)
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    for bad in (x.half(), x[0], x.t(), x[:, ::2], torch.zeros(1, 64).bfloat16().expand(4, 64), torch.zeros(64, 0).bfloat16(), x):
        with pytest.raises(AssertionError):
            mxfp4_quantize(bad)                                      # the last one: not on a GPU
    b = MxFp4Tensor.from_blocks(torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.uint8))
    for a in (x, x[:, :32], b):
        with pytest.raises(AssertionError):
            mxfp4_matmul(a, b)
    with pytest.raises(AssertionError):
        mxfp4_matmul(x, x)
    with pytest.raises(AssertionError):
        b.dequantize()
    room = torch.zeros(3 * 2176, dtype=torch.uint8)
    assert MxFp4Tensor(room[16:16 + 2176], 16, 256).shape == (16, 256)
    for storage, rows, cols in ((room, 16, 256), (room[:2175], 16, 256), (room[8:8 + 2176], 16, 256), (room[::2][:2176], 16, 256),
                                (room[:2176].view(torch.int8), 16, 256), (room[:2176].view(2, 1088), 16, 256),
                                (room[:2176], 17, 256), (room[:2176], 16, 257), (room[:0], 0, 0), (room[:0], -1, 256)):
        with pytest.raises(AssertionError):
            MxFp4Tensor(storage, rows, cols)
    for codes, scales, cols in (((8, 31), (8, 2), None), ((8, 32), (7, 2), None), ((8, 32), (8, 2), 32), ((8, 32), (8, 2), 65)):
        with pytest.raises(AssertionError):
            MxFp4Tensor.from_blocks(torch.zeros(codes, dtype=torch.uint8), torch.zeros(scales, dtype=torch.uint8), cols)
    w = torch.ones(64, dtype=torch.bfloat16)
    for args, kw in (((x, x, w), {}), ((x, x[:2], w), {}), ((x, x.float(), w), {}), ((x, x, w[:5]), {}),
                     ((x.t(), x.t(), w[:4]), {}), ((x, x, w), {"gate": w[:4]}), ((x, x, w), {"gate": torch.ones(2, 1, 64).bfloat16()}),
                     ((x, x, w), {"post_weight": w.float()}), ((x.half(), x.half(), w.half()), {})):
        with pytest.raises(AssertionError):
            one_shot_all_reduce_norm(*args, **kw)
    with pytest.raises(AssertionError):
        one_shot_all_reduce_norm(torch.zeros(1, 16385).bfloat16(), torch.zeros(1, 16385).bfloat16(), torch.ones(16385).bfloat16())
    with pytest.raises(AssertionError):
        one_shot_all_reduce_norm_backward(x, x, x[:3], x, w)
    with pytest.raises(AssertionError):
        one_shot_all_reduce_norm_backward(x, None, x, x, w)          # not on a GPU


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (16, 256), (17, 257), (40, 1000)])
def test_blocks_round_trip_on_the_host(rows, cols):
    """from_blocks puts every code and scale where the layout in smr.h says it is, and zeros
    elsewhere; to_blocks brings them back."""
    from symm_mem_recipes import MxFp4Tensor
    gen = torch.Generator().manual_seed(rows)
    blocks = -(-cols // 32)
    codes = torch.randint(0, 256, (rows, blocks * 16), generator=gen, dtype=torch.uint8)
    scales = torch.randint(0, 255, (rows, blocks), generator=gen, dtype=torch.uint8)
    q = MxFp4Tensor.from_blocks(codes, scales, cols)
    slabs = -(-cols // 256)
    want_codes = torch.zeros(-(-rows // 16) * slabs * 2048, dtype=torch.uint8)
    want_scales = torch.zeros(-(-rows // 16) * slabs * 128, dtype=torch.uint8)
    for r in range(rows):
        for b in range(blocks):
            unit, step, lane = (b // 8) * -(-rows // 16) + r // 16, (b % 8) // 4, (b % 4) * 16 + r % 16
            want_scales[unit * 128 + lane * 2 + step] = scales[r, b]
            for i in range(16):
                first = b * 32 + 2 * i
                byte = int(codes[r, b * 16 + i])
                byte = 0 if first >= cols else byte & 15 if first + 1 >= cols else byte
                want_codes[unit * 2048 + (step * 64 + lane) * 16 + i] = byte
    assert torch.equal(q.codes, want_codes) and torch.equal(q.scales, want_scales)
    back_codes, back_scales = q.to_blocks()
    assert torch.equal(back_scales, scales)
    assert torch.equal(mx.values(back_codes, back_scales)[:, :cols], mx.values(codes, scales)[:, :cols])


def test_the_oracle_of_the_format():
    """Known answers: borders go to the even code, 6 saturates, the scale's exponent is the
    largest value's less two."""
    x = torch.zeros(2, 32)
    x[0, :16] = torch.tensor([4, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, 7.9, -.25, -.26, -5.01, 0, .5, 1.5, 6])
    x[1, :4] = torch.tensor([4 * 2.0 ** 10, 5 * 2.0 ** 10, 2.0 ** 9, 0])
    codes, scales = mx.quantize(x)
    v = mx.values(codes, scales)
    assert scales.tolist() == [[127], [137]]
    assert v[0, :16].tolist() == [4, 0, 1, 1, 2, 2, 4, 4, 6, 0, -.5, -6, 0, .5, 1.5, 6]
    assert v[1, :4].tolist() == [4096, 4096, 512, 0]


@pytest.mark.parametrize("gate_shape", [None, (6,), (4, 1), (4, 6)])
@pytest.mark.parametrize("post", [True, False])
def test_the_oracle_of_the_gradients(gate_shape, post):
    """The formulas against automatic differentiation of the 64-bit forward pass, and that
    against differences."""
    gen = torch.Generator().manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64, requires_grad=True)  # noqa: E731
    p, x, w = rand(1, 4, 6), rand(4, 6), rand(6)
    pw = rand(6) if post else None
    g = None if gate_shape is None else rand(*gate_shape)
    dy, dh = torch.randn(4, 6, generator=gen, dtype=torch.float64), torch.randn(4, 6, generator=gen, dtype=torch.float64)
    leaves = [t for t in (p, x, w, pw, g) if t is not None]

    def loss(*values):
        values = list(values)
        a = [values.pop(0) if t is not None else None for t in (p, x, w, pw, g)]
        y, h, _ = norm_oracle.forward(*a, 0.7, 1e-3)
        return (y * dy).sum() + (h * dh).sum()

    assert torch.autograd.gradcheck(loss, leaves)
    grads = iter(torch.autograd.grad(loss(*leaves), leaves))
    _, h, s = norm_oracle.forward(p, x, w, pw, g, 0.7, 1e-3)
    got = norm_oracle.backward(dy, dh, s.detach(), h.detach(), w.detach(), None if pw is None else pw.detach(),
                               None if g is None else g.detach(), 0.7, 1e-3)
    for name, leaf in (("partial", p), ("residual", x), ("weight", w), ("post_weight", pw), ("gate", g)):
        if leaf is not None:
            want = next(grads)
            want = want[0] if name == "partial" else want
            assert torch.allclose(got[name].reshape(want.shape), want, rtol=1e-10, atol=1e-12), name


def test_the_columns_of_the_few_rows_product_end_below_2_to_28(lib):
    p, f = 0x1000, lib.smr_mxfp4_matmul_rows
    assert f(p, 32, 0, p, p, p, 1, 2 ** 28 - 63, 32, 0, None) == -2
    assert b"columns" in lib.smr_last_error_string()
    assert f(p, 32, 0, p, p, p, 0, 2 ** 28 - 64, 32, 0, None) == 0               # no rows: no launch


def test_operands_that_contract_over_nothing_on_the_host():
    from symm_mem_recipes import MxFp4Tensor
    none = torch.zeros(8, 0, dtype=torch.uint8)
    q = MxFp4Tensor.from_blocks(none, none)
    assert q.shape == (8, 0) and [t.shape for t in q.to_blocks()] == [(8, 0), (8, 0)]
    assert MxFp4Tensor(torch.zeros(0, dtype=torch.uint8), 8, 0).shape == (8, 0)
    assert MxFp4Tensor.empty(5, 0, "cpu").storage.numel() == 0
    for rows, cols in ((0, 0), (-1, 4), (4, -1), (2 ** 31, 4), (4, 2 ** 31)):
        with pytest.raises(AssertionError):
            MxFp4Tensor.empty(rows, cols, "cpu")
    with pytest.raises(AssertionError):
        MxFp4Tensor.from_blocks(none[:0], none[:0])


def test_rows_that_one_workgroup_takes_depend_on_their_width(lib):
    """Up to how many rows the norms' backward pass needs no scratch array: fewer the more vectors a thread has."""
    def single(cols, dtype):
        return max(r for r in range(1, 65) if lib.smr_norm_backward_scratch_bytes(r, cols, dtype, 1, 1) == 0)

    assert [single(c, 0) for c in (64, 4096, 4097, 8192)] == [5, 5, 4, 4]
    assert [single(c, 1) for c in (64, 2048, 2049, 4096, 4097, 8192)] == [5, 5, 4, 4, 2, 2]

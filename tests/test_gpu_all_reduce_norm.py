"""The all-reduce fused with norms, gate and residual, and its backward pass, on the GPU against
64-bit arithmetic."""
import pytest
import torch

from tests import norm_oracle as oracle

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _gate_shape(kind, shape):
    return {"none": None, "channel": shape[-1:], "token": tuple(shape[:-1]) + (1,), "element": tuple(shape)}[kind]


def _inputs(shape, ranks, dtype, post, gate, seed):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    shape = tuple(shape)
    partials = rand(ranks, *shape).to(dtype)
    residual = (rand(*shape) * torch.exp(0.5 * rand(shape[-1]))).to(dtype)
    weight = (1 + 0.1 * rand(shape[-1])).to(dtype)
    post_weight = (1 + 0.1 * rand(shape[-1])).to(dtype) if post else None
    gate_shape = _gate_shape(gate, shape)
    gate = None if gate_shape is None else (0.5 + 0.3 * rand(*gate_shape)).to(dtype)
    return partials, residual, weight, post_weight, gate


def _symmetric(partials, rank):
    from symm_mem_recipes import EmulatedSymmetricMemory as SM
    ranks, shape = partials.shape[0], tuple(partials.shape[1:])
    strides, step = [], 1
    for n in reversed(shape):
        strides.insert(0, step)
        step *= n
    t = SM.empty_strided_p2p(shape, strides, partials.dtype, "cuda", world_size=ranks, rank=rank)
    for r in range(ranks):
        SM.rendezvous(t).get_buffer(r, shape, partials.dtype).copy_(partials[r])
    return t, SM.rendezvous(t)


def _cuda(*tensors):
    return [None if t is None else t.cuda() for t in tensors]


def _within(got, want, off, dtype):
    """Half a step of the result's type, of the value that is rounded."""
    half = torch.finfo(dtype).eps / 2
    bound = (want.abs() + off) * half + off + torch.finfo(dtype).tiny
    d = (got.cpu().double() - want).abs()
    assert got.dtype == dtype and got.shape == want.shape
    assert bool((d <= bound).all()), (float((d - bound).max()), int((d > bound).sum()))


FORWARD = [
    # shape, ranks, dtype, post, gate, scale
    ((1, 8), 1, "bf16", True, "none", 1.0), ((1, 1), 2, "fp32", True, "channel", 1.0), ((5,), 3, "bf16", True, "channel", 0.5),
    ((1, 8192), 8, "bf16", True, "channel", 1.25), ((2, 3, 64), 8, "bf16", False, "token", 1.0),
    ((3, 1000), 5, "bf16", True, "element", -0.5), ((4, 1001), 7, "bf16", True, "token", 1.0),
    ((7, 1001), 5, "fp32", True, "element", 1.0), ((3, 63), 4, "fp32", False, "none", 0.0),
    ((300, 96), 8, "bf16", True, "channel", 1.0), ((600, 512), 2, "bf16", False, "channel", 1.0),
    ((2, 8200), 8, "bf16", True, "element", 1.0), ((2, 16384), 4, "bf16", True, "none", 1.0),
    ((2, 16383), 3, "bf16", True, "token", 1.0), ((2, 16381), 2, "fp32", True, "channel", 1.0),
    ((1030, 2048), 6, "bf16", True, "token", 1.0), ((5000, 40), 8, "fp32", True, "element", 1.0),
    # more rows than compute units, wide enough that a workgroup loads its next row ahead
    ((300, 8192), 8, "bf16", True, "channel", 1.0), ((530, 8001), 7, "bf16", False, "element", 1.0), ((260, 4096), 1, "bf16", True, "token", 0.5),
    ((777, 2999), 5, "bf16", True, "none", 1.0), ((270, 4096), 4, "fp32", False, "token", 1.0), ((300, 4093), 3, "fp32", True, "element", 1.0),
    ((513, 2048), 6, "fp32", False, "none", 1.0), ((300, 1025), 2, "fp32", True, "channel", 1.0), ((4200, 1100), 2, "bf16", True, "element", 1.0),
    ((300, 9000), 3, "bf16", True, "channel", 1.0), ((300, 9001), 2, "fp32", False, "element", 1.0),
]


@pytest.mark.parametrize("shape,ranks,dtype,post,gate,scale", FORWARD)
def test_forward(cuda, shape, ranks, dtype, post, gate, scale):
    from symm_mem_recipes import EmulatedSymmetricMemory as SM, one_shot_all_reduce_norm
    dtype = DTYPES[dtype]
    partials, residual, weight, post_weight, g = _inputs(shape, ranks, dtype, post, gate, sum(shape) + ranks)
    t, handle = _symmetric(partials, rank=ranks - 1)
    x, w, p, gc = _cuda(residual, weight, post_weight, g)
    kw = dict(post_weight=p, gate=gc, residual_scale=scale, eps=1e-5)
    got = one_shot_all_reduce_norm(t, x, w, return_sum=True, **kw)
    want = oracle.forward(partials, residual, weight, post_weight, g, scale, 1e-5)
    off = oracle.forward_bounds(partials, residual, weight, post_weight, g, scale, 1e-5)
    for a, b, c in zip(got, want, off):
        _within(a, b, c, dtype)
    for _ in range(2):
        again = one_shot_all_reduce_norm(t, x, w, return_sum=True, **kw)
        assert all(torch.equal(a, b) for a, b in zip(got, again))
    without = one_shot_all_reduce_norm(t, x, w, barrier=False, **kw)
    assert len(without) == 2 and all(torch.equal(a, b) for a, b in zip(got, without))
    handle.check_status()
    assert all(int(handle.get_signal_pad(r).abs().sum()) == 0 for r in range(ranks))
    for r in range(ranks):
        assert torch.equal(handle.get_buffer(r, shape, dtype).cpu(), partials[r])        # the inputs stay
    SM.release()


def test_the_sum_is_one_shot_all_reduce(cuda):
    from symm_mem_recipes import EmulatedSymmetricMemory as SM, one_shot_all_reduce, one_shot_all_reduce_norm
    for dtype in DTYPES.values():
        partials, residual, weight, post_weight, _ = _inputs((33, 1024), 8, dtype, True, "none", 9)
        t, _ = _symmetric(partials, 2)
        x, w, p = _cuda(residual, weight, post_weight)
        _, _, s = one_shot_all_reduce_norm(t, x, w, post_weight=p, return_sum=True)
        assert torch.equal(s, one_shot_all_reduce(t))
    SM.release()


def test_another_stream_and_a_residual_updated_in_place(cuda, lib):
    """On a stream of its own, and the C entry with residual_out on top of residual, as it allows: ragged
    rows, with and without the norm and the handshake that would order the waves."""
    from symm_mem_recipes import EmulatedSymmetricMemory as SM, one_shot_all_reduce_norm
    for shape in ((700, 1001), (3, 1001), (600, 2050), (9, 5)):
        partials, residual, weight, post_weight, _ = _inputs(shape, 4, torch.bfloat16, True, "none", 21)
        t, handle = _symmetric(partials, 1)
        x, w, p = _cuda(residual, weight, post_weight)
        side = torch.cuda.Stream()
        for pw in (None, p):
            y, h = one_shot_all_reduce_norm(t, x, w, post_weight=pw)
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                y2, h2 = one_shot_all_reduce_norm(t, x, w, post_weight=pw)
            side.synchronize()
            assert torch.equal(y, y2) and torch.equal(h, h2)
            for mode in (0, 1):
                x2, y3 = x.clone(), torch.empty_like(y)
                rc = lib.smr_all_reduce_norm(handle.buffer_ptrs_host, handle.signal_pad_ptrs_host, x2.data_ptr(), w.data_ptr(),
                                             0 if pw is None else pw.data_ptr(), None, 0, y3.data_ptr(), x2.data_ptr(), None,
                                             shape[0], shape[1], 0, 1.0, 1e-6, 1, 4, mode, handle.status.data_ptr(),
                                             torch.cuda.current_stream().cuda_stream)
                assert rc == 0 and torch.equal(x2, h) and torch.equal(y3, y)
        handle.check_status()
    SM.release()


def test_rows_of_zeros_infinities_and_nan(cuda):
    """A row of zeros divides by sqrt(eps) and stays zero; an infinity or NaN spoils its own row
    and no other."""
    from symm_mem_recipes import EmulatedSymmetricMemory as SM, one_shot_all_reduce_norm
    partials, residual, weight, post_weight, _ = _inputs((6, 200), 3, torch.bfloat16, True, "none", 1)
    partials[:, 0] = 0
    residual[0] = 0
    partials[1, 2, 7] = float("inf")
    residual[4, 199] = float("nan")
    t, _ = _symmetric(partials, 0)
    y, h = one_shot_all_reduce_norm(t, residual.cuda(), weight.cuda(), post_weight=post_weight.cuda())
    assert bool((y[0] == 0).all()) and bool((h[0] == 0).all())
    clean = [1, 3, 5]
    want = oracle.forward(partials, residual, weight, post_weight, None, 1.0, 1e-6)
    off = oracle.forward_bounds(partials, residual, weight, post_weight, None, 1.0, 1e-6)
    for got, b, c in zip((y, h), want, off):
        _within(got[clean], b[clean], c[clean], torch.bfloat16)
    assert bool(y[2].isnan().any()) and bool(y[4].isnan().all())
    SM.release()


def test_large_values_do_not_overflow_before_the_type_does(cuda):
    from symm_mem_recipes import EmulatedSymmetricMemory as SM, one_shot_all_reduce_norm
    partials, residual, weight, post_weight, _ = _inputs((2, 256), 2, torch.float32, True, "none", 3)
    partials, residual = partials * 1e15, residual * 1e15
    t, _ = _symmetric(partials, 0)
    got = one_shot_all_reduce_norm(t, residual.cuda(), weight.cuda(), post_weight=post_weight.cuda())
    args = (partials, residual, weight, post_weight, None, 1.0, 1e-6)
    for a, b, c in zip(got, oracle.forward(*args), oracle.forward_bounds(*args)):
        _within(a, b, c, torch.float32)
    SM.release()


def test_no_tokens(cuda):
    from symm_mem_recipes import EmulatedSymmetricMemory as SM, one_shot_all_reduce_norm, one_shot_all_reduce_norm_backward
    t = SM.empty_strided_p2p((0, 64), (64, 1), torch.bfloat16, "cuda", world_size=4, rank=0)
    x, w = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda"), torch.ones(64, dtype=torch.bfloat16, device="cuda")
    y, h, s = one_shot_all_reduce_norm(t, x, w, return_sum=True)
    assert y.shape == h.shape == s.shape == (0, 64)
    g = one_shot_all_reduce_norm_backward(y, h, s, h, w, post_weight=w, gate=w)
    assert g.partial.shape == (0, 64) and not g.weight.any() and not g.post_weight.any() and not g.gate.any()
    SM.release()


BACKWARD = [
    ((1, 8), "bf16", True, "none", 1.0, True), ((1, 1), "fp32", True, "channel", 1.0, True), ((5,), "bf16", True, "channel", 0.5, True),
    ((5, 4096), "bf16", False, "none", 1.25, True), ((2, 3, 64), "bf16", False, "token", 1.0, True),
    ((3, 1000), "bf16", True, "element", -0.5, False), ((4, 1001), "bf16", True, "token", 1.0, True),
    ((7, 1001), "fp32", True, "element", 1.0, True), ((3, 63), "fp32", False, "channel", 0.0, False),
    ((300, 96), "bf16", True, "channel", 1.0, True), ((600, 512), "fp32", True, "channel", 1.0, True),
    ((2, 8200), "bf16", True, "element", 1.0, True), ((2, 16384), "bf16", True, "channel", 1.0, True),
    ((2, 16383), "bf16", True, "token", 1.0, True), ((2, 16381), "fp32", True, "channel", 1.0, True),
    ((1030, 2048), "bf16", True, "token", 1.0, True), ((5000, 40), "fp32", True, "element", 1.0, True),
    # a few rows more than one workgroup takes: a workgroup each and a second launch for their sums (5 x 1536: one workgroup)
    ((80, 512), "bf16", True, "channel", 1.0, True), ((79, 499), "bf16", True, "token", 1.0, False), ((40, 1000), "bf16", False, "channel", 1.0, True),
    ((33, 777), "bf16", True, "element", 2.0, True), ((20, 2048), "bf16", True, "none", 1.0, True), ((10, 4001), "bf16", True, "channel", 1.0, True),
    ((65, 250), "fp32", True, "channel", 1.0, True), ((17, 300), "fp32", False, "token", 1.0, True), ((9, 2048), "fp32", True, "element", 1.0, False),
    ((6, 8), "bf16", True, "channel", 1.0, True), ((13, 1023), "fp32", True, "token", 1.0, True), ((5, 1536), "bf16", True, "element", 1.0, True),
    # several rows per workgroup: rows ahead of one and of two vectors a thread, rows kept, rows read again
    ((600, 4096), "bf16", False, "channel", 1.0, False), ((520, 8192), "bf16", True, "channel", 1.0, True),
    ((530, 8001), "bf16", True, "element", 1.0, True), ((513, 2999), "bf16", True, "none", -1.0, True),
    ((260, 4096), "fp32", True, "token", 1.0, True), ((300, 4093), "fp32", True, "channel", 1.0, False),
    ((270, 8192), "fp32", True, "channel", 1.0, True), ((265, 8191), "fp32", False, "element", 1.0, True),
    ((300, 9001), "fp32", True, "channel", 1.0, True), ((300, 16384), "bf16", True, "token", 1.0, False),
    ((520, 8201), "bf16", True, "channel", 1.0, True),
]


def _backward_inputs(shape, dtype, post, gate, with_dh, seed):
    _, h, weight, post_weight, g = _inputs(shape, 1, dtype, post, gate, seed)
    gen = torch.Generator().manual_seed(seed + 1)
    s, dy, dh = (torch.randn(*shape, generator=gen).to(dtype) for _ in range(3))
    return dy, dh if with_dh else None, s * 2, h, weight, post_weight, g


# (With up to 2048 workgroups, 5000 x 40, a thread of the summing kernel adds 64 of their sums, not 32: 3 terms in a
# workgroup, 64 and 32 are 99, and the bound has 5000 / 128 + 64 = 103.)
@pytest.mark.parametrize("shape,dtype,post,gate,scale,with_dh", BACKWARD)
def test_backward(cuda, shape, dtype, post, gate, scale, with_dh):
    """Every term of a gradient passes through at most 128 roundings on its way (32 values and 22
    partial sums in each of two row sums, the rest single operations); a column sum adds at most
    rows / 128 terms in a workgroup, 32 workgroups' in a thread and 32 threads'."""
    from symm_mem_recipes import one_shot_all_reduce_norm_backward
    dtype = DTYPES[dtype]
    args = _backward_inputs(shape, dtype, post, gate, with_dh, sum(shape))
    dy, dh, s, h, w, p, g = _cuda(*args)
    got = one_shot_all_reduce_norm_backward(dy, dh, s, h, w, post_weight=p, gate=g, residual_scale=scale, eps=1e-5)
    want = oracle.backward(*args, scale, 1e-5)
    size = oracle.backward(*args, scale, 1e-5, magnitudes=True)
    assert (got.post_weight is None) == (not post) and (got.gate is None) == (gate == "none")
    rows = dy.numel() // dy.shape[-1]
    for name, b in want.items():
        a = getattr(got, name)
        off = size[name] * (128 + rows / 128 + 64) * oracle.U
        _within(a.reshape(b.shape), b, off, dtype)
    again = one_shot_all_reduce_norm_backward(dy, dh, s, h, w, post_weight=p, gate=g, residual_scale=scale, eps=1e-5)
    assert all(a is None and b is None or torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("shape,dtype", [((3, 1001), "fp32"), ((8, 1003), "bf16"), ((3, 13000), "bf16"), ((2, 64), "bf16"), ((3, 5), "bf16")])
def test_an_infinite_gradient_stays_an_infinity_whatever_the_width(cuda, shape, dtype):
    """An infinity near the end of a row, where vectors overlap: its row's gradients are infinite or NaN
    where the formula's are, its channel's sums too, and the other rows and channels are untouched."""
    from symm_mem_recipes import one_shot_all_reduce_norm_backward
    args = _backward_inputs(shape, DTYPES[dtype], True, "channel", True, 3)
    args[0][1, shape[1] - 2] = float("inf")
    dy, dh, s, h, w, p, g = _cuda(*args)
    got = one_shot_all_reduce_norm_backward(dy, dh, s, h, w, post_weight=p, gate=g)
    want = oracle.backward(*args, 1.0, 1e-6)
    assert want["residual"][1].isinf().any()
    for name, b in want.items():
        a = getattr(got, name).cpu().double()
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.isinf(), b.isinf()), name
        assert torch.equal(a[a.isinf()].sign(), b[b.isinf()].sign()), name
    keep = [r for r in range(shape[0]) if r != 1]
    clean, magnitudes = oracle.backward(*args, 1.0, 1e-6), oracle.backward(*args, 1.0, 1e-6, magnitudes=True)
    for name in ("residual", "partial"):
        _within(getattr(got, name)[keep], clean[name][keep], magnitudes[name][keep] * 160 * oracle.U, DTYPES[dtype])


def test_offsets_past_32_bits(cuda):
    """Tensors of more than 4 GiB: the last rows against the oracle, forward and backward."""
    from symm_mem_recipes import EmulatedSymmetricMemory as SM, one_shot_all_reduce_norm, one_shot_all_reduce_norm_backward
    for rows, cols in ((270001, 8192), (2200001, 1000), (135001, 16384)):
        partials, residual, weight, post_weight, g = _inputs((3, cols), 2, torch.bfloat16, True, "element", cols)
        t = SM.empty_strided_p2p((rows, cols), (cols, 1), torch.bfloat16, "cuda", world_size=2, rank=1)
        for r in range(2):
            buf = SM.rendezvous(t).get_buffer(r, (rows, cols), torch.bfloat16)
            buf.fill_(0.5)
            buf[-3:] = partials[r].cuda()
        x, gate = torch.full((rows, cols), 0.25, dtype=torch.bfloat16, device="cuda"), torch.ones(rows, cols, dtype=torch.bfloat16, device="cuda")
        x[-3:], gate[-3:] = residual.cuda(), g.cuda()
        w, p = weight.cuda(), post_weight.cuda()
        y, h, s = one_shot_all_reduce_norm(t, x, w, post_weight=p, gate=gate, return_sum=True)
        args = (partials, residual, weight, post_weight, g, 1.0, 1e-6)
        for a, b, c in zip((y, h, s), oracle.forward(*args), oracle.forward_bounds(*args)):
            _within(a[-3:], b, c, torch.bfloat16)
        assert torch.equal(y[0], y[-4]) and torch.equal(h[1], h[-5]) and bool((s[:-3] == 1).all())
        SM.release()
        del t, buf, x
        got = one_shot_all_reduce_norm_backward(y, None, s, h, w, post_weight=p, gate=gate)
        args = (y[-3:].cpu(), None, s[-3:].cpu(), h[-3:].cpu(), weight, post_weight, g, 1.0, 1e-6)
        want, size = oracle.backward(*args), oracle.backward(*args, magnitudes=True)
        for name in ("residual", "partial", "gate"):
            a = getattr(got, name)
            _within(a[-3:], want[name], size[name] * 160 * oracle.U, torch.bfloat16)
            assert torch.equal(a[0], a[-4])
        del y, h, s, gate, got, a


def test_backward_against_differences(cuda):
    """Every gradient against central differences of the 64-bit forward pass, through fp32
    inputs: the loss is a weighted sum of both outputs."""
    from symm_mem_recipes import one_shot_all_reduce_norm_backward
    gen = torch.Generator().manual_seed(5)
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    T, H, scale, eps = 3, 10, 0.75, 1e-3
    for gate_shape in ((H,), (T, 1), (T, H)):
        leaves = {"partial": rand(T, H), "residual": rand(T, H), "weight": 1 + 0.1 * rand(H), "post_weight": 1 + 0.1 * rand(H),
                  "gate": 0.5 + 0.3 * rand(*gate_shape)}
        dy, dh = rand(T, H), rand(T, H)

        def loss(v):
            y, h, _ = oracle.forward(v["partial"][None], v["residual"], v["weight"], v["post_weight"], v["gate"], scale, eps)
            return float((y * dy.double()).sum() + (h * dh.double()).sum())

        _, h, s = oracle.forward(leaves["partial"][None], leaves["residual"], leaves["weight"], leaves["post_weight"],
                                 leaves["gate"], scale, eps)
        got = one_shot_all_reduce_norm_backward(dy.cuda(), dh.cuda(), s.float().cuda(), h.float().cuda(), leaves["weight"].cuda(),
                                                post_weight=leaves["post_weight"].cuda(), gate=leaves["gate"].cuda(),
                                                residual_scale=scale, eps=eps)
        step = 1e-5           # error of a central difference: step^2 * (third derivative) ~ 1e-9, 64-bit rounding ~ 1e-10
        for name, leaf in leaves.items():
            grad = getattr(got, name).cpu().double()
            for i in range(leaf.numel()):
                up, down = ({k: v.double().clone() for k, v in leaves.items()} for _ in range(2))
                up[name].view(-1)[i] += step
                down[name].view(-1)[i] -= step
                slope = (loss(up) - loss(down)) / (2 * step)
                # fp32 inputs h and s and fp32 arithmetic: 200 roundings of terms of order 10
                assert abs(float(grad.view(-1)[i]) - slope) <= 200 * oracle.U * 10 + 1e-6, (name, i)


def test_graphs_replay_the_forward_and_the_backward_pass(cuda):
    """Two captured graphs on one allocation's signal pads, eager calls and synchronisations in
    between; each replay is checked against the eager result for the inputs of the moment."""
    from symm_mem_recipes import (EmulatedSymmetricMemory as SM, one_shot_all_reduce_norm,
                                  one_shot_all_reduce_norm_backward)
    partials, residual, weight, post_weight, g = _inputs((40, 520), 8, torch.bfloat16, True, "channel", 2)
    t, handle = _symmetric(partials, 3)
    x, w, p, gc = _cuda(residual, weight, post_weight, g)
    kw = dict(post_weight=p, gate=gc)

    def both():
        y, h, s = one_shot_all_reduce_norm(t, x, w, return_sum=True, **kw)
        return (y, h, s) + tuple(one_shot_all_reduce_norm_backward(y, h, s, h, w, **kw))

    both()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both()
        graphs.append((graph, out))
    for turn in range(3):
        for graph, out in graphs:
            x.copy_(torch.randn(40, 520) * (turn + 1))
            graph.replay()
            torch.cuda.synchronize()
            want = both()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    handle.check_status()
    SM.release()


def test_a_layer_boundary(cuda):
    """The operators together as a layer uses them: reduce, norms, gate and residual, then the
    next product in 4 bits - for one token and for a prompt - and the way back."""
    from symm_mem_recipes import (EmulatedSymmetricMemory as SM, mxfp4_matmul, mxfp4_quantize, one_shot_all_reduce_norm,
                                  one_shot_all_reduce_norm_backward)
    from tests import mxfp4_oracle as mx
    for T in (1, 150):
        H, N = 512, 320
        partials, residual, weight, post_weight, g = _inputs((T, H), 8, torch.bfloat16, True, "channel", T)
        w_next = (torch.randn(N, H, generator=torch.Generator().manual_seed(T)) * H ** -0.5).bfloat16()
        t, handle = _symmetric(partials, 0)
        x, w, p, gc, wn = _cuda(residual, weight, post_weight, g, w_next)
        y, h, s = one_shot_all_reduce_norm(t, x, w, post_weight=p, gate=gc, return_sum=True)
        out = mxfp4_matmul(y, mxfp4_quantize(wn))
        y64, w64 = mx.values(*mx.quantize(y)), mx.values(*mx.quantize(w_next))
        want = y64 @ w64.t()
        bound = want.abs() * 2.0 ** -8 + (H + 16) * oracle.U * (y64.abs() @ w64.abs().t()) * 1.01
        assert bool(((out.cpu().double() - want).abs() <= bound).all())
        d_out = torch.randn(T, N, generator=torch.Generator().manual_seed(7)).bfloat16().cuda()
        dy = mxfp4_matmul(d_out, mxfp4_quantize(wn, transpose=True))
        dw = mxfp4_matmul(mxfp4_quantize(d_out, transpose=True), mxfp4_quantize(y, transpose=True))
        assert dy.shape == (T, H) and dw.shape == (N, H)
        got = one_shot_all_reduce_norm_backward(dy, None, s, h, w, post_weight=p, gate=gc)
        args = (dy.cpu(), None, s.cpu(), h.cpu(), weight, post_weight, g, 1.0, 1e-6)
        want, size = oracle.backward(*args), oracle.backward(*args, magnitudes=True)
        for name, b in want.items():
            _within(getattr(got, name).reshape(b.shape), b, size[name] * (128 + 32) * oracle.U, torch.bfloat16)
        handle.check_status()
    SM.release()

"""4-bit microscaled operands on the GPU: quantisation bit for bit against the 64-bit oracle,
products against 64-bit products of the operands' exact values."""
import pytest
import torch

from tests import mxfp4_oracle as mx

pytestmark = pytest.mark.gpu


def _activations(rows, cols, dtype, seed, device="cuda"):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=gen) * torch.exp(torch.randn(cols, generator=gen))
    return x.to(dtype).to(device)


def _same_operand(q, codes, scales):
    got_codes, got_scales = q.to_blocks()
    assert torch.equal(got_scales.cpu(), scales)
    assert torch.equal(got_codes.cpu(), codes)


SIZES = [(1, 1), (1, 32), (1, 8192), (2, 33), (15, 255), (16, 256), (17, 257), (3, 1001), (64, 96), (300, 700), (129, 4100), (300, 1), (45, 2), (289, 3)]


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_quantize_is_the_oracle_bit_for_bit(cuda, rows, cols, dtype):
    from symm_mem_recipes import mxfp4_quantize
    x = _activations(rows, cols, dtype, rows * 7 + cols)
    q = mxfp4_quantize(x)
    assert q.shape == (rows, cols)
    _same_operand(q, *mx.quantize(x))


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_quantize_transposed_is_the_oracle_of_the_transpose(cuda, rows, cols, dtype):
    from symm_mem_recipes import mxfp4_quantize
    x = _activations(rows, cols, dtype, rows * 5 + cols)
    q = mxfp4_quantize(x, transpose=True)
    assert q.shape == (cols, rows)
    _same_operand(q, *mx.quantize(x.t()))


@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_quantize_takes_rows_that_are_apart_and_any_alignment(cuda, dtype, transpose):
    from symm_mem_recipes import mxfp4_quantize
    whole = _activations(40, 333, dtype, 3)
    for x in (whole[:, 1:], whole[:, 5:300], whole[3:, :77], whole[::3, 2:], whole[7:8, 3:]):
        _same_operand(mxfp4_quantize(x, transpose=transpose), *mx.quantize(x.t() if transpose else x))


@pytest.mark.parametrize("rows,cols", [(3, 40), (17, 257), (70, 1001)])
def test_storage_is_written_whole(cuda, rows, cols):
    """A used operand written over holds nothing of what it was, in its padding either."""
    from symm_mem_recipes import MxFp4Tensor, mxfp4_quantize
    x = _activations(rows, cols, torch.bfloat16, 12)
    for transpose in (False, True):
        fresh = mxfp4_quantize(x, transpose=transpose)
        used = MxFp4Tensor(torch.full_like(fresh.storage, 255), fresh.rows, fresh.cols)
        assert mxfp4_quantize(x, transpose=transpose, out=used) is used
        assert torch.equal(used.storage, fresh.storage)
        assert torch.equal(MxFp4Tensor.from_blocks(*fresh.to_blocks(), fresh.cols).storage, fresh.storage)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_product_of_rows_that_are_apart_and_any_alignment(cuda, dtype):
    from symm_mem_recipes import mxfp4_matmul, mxfp4_quantize
    whole = _activations(60, 700, dtype, 14)
    for a in (whole[:16, 1:600], whole[5:6, 3:], whole[::7, 2:34], whole[:, 1:402], whole[3:20, :31]):
        K = a.shape[1]
        b = mxfp4_quantize(_activations(50, K, torch.bfloat16, K))
        assert torch.equal(mxfp4_matmul(a, b), mxfp4_matmul(a.contiguous(), b))
        _check_product(mxfp4_matmul(a, b), mx.values(*mx.quantize(a))[:, :K],
                       b.dequantize(torch.float32).cpu().double(), torch.bfloat16)


def test_quantize_special_values(cuda):
    """Every rounding border and its neighbours, both signs, at scales up to the ends of the
    range; zeros, subnormals, the largest value, infinities and NaN."""
    from symm_mem_recipes import mxfp4_quantize
    sixteenths = torch.arange(-127, 128, dtype=torch.float64) / 16            # |v| < 8: the largest sets the scale
    rows = []
    for power in (-127, -126, -100, -3, 0, 5, 100, 124):
        block = torch.zeros(8, 32, dtype=torch.float64)
        for i in range(8):
            block[i] = torch.cat((sixteenths[i * 31:i * 31 + 31], torch.tensor([7.9375]))) * 2.0 ** power
        rows.append(block.reshape(-1))
    x = torch.stack(rows).float()
    up = torch.nextafter(x, torch.full_like(x, float("inf")))
    down = torch.nextafter(x, torch.full_like(x, -float("inf")))
    odd = torch.zeros(12, 256)
    odd[0, 5] = float("inf")
    odd[1, 40] = -float("inf")
    odd[2, 100] = float("nan")
    odd[3] = -0.0
    odd[4, :] = torch.finfo(torch.float32).max
    odd[5, 3] = torch.finfo(torch.float32).tiny
    odd[6, 3] = 2.0 ** -149
    odd[7, 64:96] = 2.0 ** -140
    odd[8, :] = -torch.finfo(torch.float32).max
    odd[9, 0], odd[9, 1] = 3e38, 1e-38
    odd[10, 33:60] = torch.finfo(torch.bfloat16).min
    odd[11] = torch.linspace(-1, 1, 256)
    for v in (x, up, down, odd):
        for dtype in (torch.float32, torch.bfloat16):
            w = v.to(dtype).cuda()
            _same_operand(mxfp4_quantize(w), *mx.quantize(w))
            _same_operand(mxfp4_quantize(w, transpose=True), *mx.quantize(w.t()))


@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 31), (16, 256), (33, 300), (100, 1001)])
def test_dequantize_and_blocks_round_trip(cuda, rows, cols):
    """Every code with every scale (NaN among them) comes back exactly in both types."""
    from symm_mem_recipes import MxFp4Tensor
    gen = torch.Generator().manual_seed(rows + cols)
    blocks = -(-cols // 32)
    codes = torch.randint(0, 256, (rows, blocks * 16), generator=gen, dtype=torch.uint8)
    scales = torch.randint(0, 256, (rows, blocks), generator=gen, dtype=torch.uint8)
    q = MxFp4Tensor.from_blocks(codes.cuda(), scales.cuda(), cols)
    want = mx.values(codes, scales)[:, :cols]
    for dtype in (torch.float32, torch.bfloat16):
        got = q.dequantize(dtype)
        finite = want.float()                       # 6 * 2^127 is beyond both types: infinite in both
        assert torch.equal(got.cpu().double().nan_to_num(nan=-1.25), finite.to(dtype).double().nan_to_num(nan=-1.25))
    got_codes, got_scales = q.to_blocks()
    keep = mx.values(got_codes, got_scales)[:, :cols]
    assert torch.equal(keep.nan_to_num(nan=-1.25), want.nan_to_num(nan=-1.25))
    assert torch.equal(got_scales.cpu(), scales)


def _check_product(got, a64, b64, out_dtype):
    """fp32 accumulation of K exact products: at most K roundings of 2^-24 relative to the sum of
    the magnitudes; then one rounding to the result's type."""
    want = a64 @ b64.t()
    size = a64.abs() @ b64.abs().t()
    K = a64.shape[1]
    bound = want.abs() * torch.finfo(out_dtype).eps / 2 + (K + 16) * 2.0 ** -24 * size * (1 + 2.0 ** -7)
    assert got.dtype == out_dtype and got.shape == want.shape
    off = (got.cpu().double() - want).abs()
    assert bool((off <= bound).all()), float((off - bound).max())


PRODUCTS = [
    (1, 1, 1), (1, 16, 32), (1, 256, 8192), (2, 17, 33), (7, 100, 300), (16, 16, 256), (16, 64, 128), (17, 48, 257),
    (31, 3584, 96), (33, 65, 1000), (64, 128, 512), (65, 130, 520), (100, 1001, 77), (128, 128, 4096), (129, 257, 640),
    (256, 224, 256), (257, 225, 768), (300, 449, 1024), (511, 700, 1500), (1000, 333, 2304), (2, 5, 20000),
    (16, 16401, 300), (5, 16400, 2100), (33, 16395, 520), (64, 17000, 700), (40, 4100, 600), (50, 4500, 300), (20, 4099, 513),
]


@pytest.mark.parametrize("M,N,K", PRODUCTS)
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_product(cuda, M, N, K, out_dtype):
    from symm_mem_recipes import mxfp4_matmul, mxfp4_quantize
    a, b = _activations(M, K, torch.bfloat16, M + K), _activations(N, K, torch.float32, N + K + 1)
    qa, qb = mxfp4_quantize(a), mxfp4_quantize(b)
    a64, b64 = mx.values(*mx.quantize(a))[:, :K], mx.values(*mx.quantize(b))[:, :K]
    got = mxfp4_matmul(qa, qb, out_dtype=out_dtype)
    _check_product(got, a64, b64, out_dtype)
    direct = mxfp4_matmul(a, qb, out_dtype=out_dtype)                          # quantised on the way
    _check_product(direct, a64, b64, out_dtype)
    if M > 16:
        assert torch.equal(direct, got)
    assert torch.equal(mxfp4_matmul(qa, qb, out_dtype=out_dtype), got)         # and again
    assert torch.equal(mxfp4_matmul(a, qb, out_dtype=out_dtype), direct)


# (each of the matrix-tile kernels, one pass over the chip and several - the 256 x 128 tile one pass, several are in
# test_gpu_mxfp4_launches.py; odd widths, units and tiles that end early)
LARGE = [(300, 3000, 900), (1500, 3500, 1100), (1100, 3001, 700), (2049, 3585, 900), (2000, 3300, 1000), (4097, 3585, 700),
         (4000, 3584, 1100), (4200, 7201, 1000), (4090, 7161, 1300), (5003, 7392, 257),
         (512, 3583, 1500), (700, 2001, 700), (4001, 4090, 1111), (8003, 4081, 700), (8200, 2050, 1300)]


@pytest.mark.parametrize("M,N,K", LARGE)
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_large_product(cuda, M, N, K, out_dtype):
    from symm_mem_recipes import mxfp4_matmul, mxfp4_quantize
    a, b = _activations(M, K, torch.bfloat16, M + K), _activations(N, K, torch.float32, N + K + 1)
    qa, qb = mxfp4_quantize(a), mxfp4_quantize(b)
    room = torch.full((M * N + 512,), 7.0, dtype=out_dtype, device="cuda")
    got = mxfp4_matmul(qa, qb, out=room[256:256 + M * N].view(M, N))
    assert bool((room[:256] == 7).all()) and bool((room[256 + M * N:] == 7).all())
    a64, b64 = (mx.values(*mx.quantize(t))[:, :K].cuda() for t in (a, b))
    want = a64 @ b64.t()
    bound = want.abs() * torch.finfo(out_dtype).eps / 2 + (K + 16) * 2.0 ** -24 * (a64.abs() @ b64.abs().t()) * (1 + 2.0 ** -7)
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off - bound).max())
    for _ in range(2):
        assert torch.equal(mxfp4_matmul(a, qb, out_dtype=out_dtype), got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_large_matrices_are_their_parts(cuda, dtype):
    """Sizes that are streamed past the caches, against the same rows and columns in parts that are not."""
    from symm_mem_recipes import mxfp4_quantize
    x = _activations(4101, 8300, torch.bfloat16, 6).to(dtype)
    whole, columns = mxfp4_quantize(x), mxfp4_quantize(x, transpose=True)
    codes, scales = whole.to_blocks()
    t_codes, t_scales = columns.to_blocks()
    values, t_values = whole.dequantize(dtype), columns.dequantize(dtype)
    for first in range(0, 4101, 1024):
        part = mxfp4_quantize(x[first:first + 1024])
        part_codes, part_scales = part.to_blocks()
        assert torch.equal(codes[first:first + 1024], part_codes) and torch.equal(scales[first:first + 1024], part_scales)
        assert torch.equal(values[first:first + 1024], part.dequantize(dtype))
    for first in range(0, 8300, 2048):
        part = mxfp4_quantize(x[:, first:first + 2048], transpose=True)
        part_codes, part_scales = part.to_blocks()
        assert torch.equal(t_codes[first:first + 2048], part_codes) and torch.equal(t_scales[first:first + 2048], part_scales)
        assert torch.equal(t_values[first:first + 2048], part.dequantize(dtype))


def test_offsets_past_32_bits(cuda):
    """Inputs, results and storage of more than 4 GiB: the last rows are those of the last rows alone."""
    from symm_mem_recipes import mxfp4_matmul, mxfp4_quantize
    tail = _activations(100, 65600, torch.bfloat16, 8)
    x = torch.zeros(66000, 65600, dtype=torch.bfloat16, device="cuda")         # 8.7 GB, codes 2.2 GB
    x[-100:] = tail
    q, part = mxfp4_quantize(x), mxfp4_quantize(tail)
    assert torch.equal(q.dequantize()[-100:], part.dequantize())
    del q
    q, part = mxfp4_quantize(x, transpose=True), mxfp4_quantize(x[:, -64:], transpose=True)
    assert torch.equal(q.dequantize()[-64:], part.dequantize())
    del q, x
    a, b = _activations(70000, 256, torch.bfloat16, 9), mxfp4_quantize(_activations(40001, 256, torch.bfloat16, 10))
    got = mxfp4_matmul(a, b)                                                   # 5.6 GB
    assert torch.equal(got[-50:], mxfp4_matmul(a[-50:], b))                    # (one slab: one order of its sum)
    assert torch.equal(got[34000:34050], mxfp4_matmul(a[34000:34050], b))


def test_product_propagates_nan_blocks_to_their_rows_only(cuda):
    from symm_mem_recipes import mxfp4_matmul, mxfp4_quantize
    for M, N in ((5, 40), (200, 300)):
        a, b = _activations(M, 600, torch.bfloat16, 1), _activations(N, 600, torch.bfloat16, 2)
        a[3, 599] = float("inf")
        b[1, 0] = float("nan")
        got = mxfp4_matmul(a, mxfp4_quantize(b)).float().cpu()
        want = torch.zeros(M, N, dtype=torch.bool)
        want[3, :] = True
        want[:, 1] = True
        assert torch.equal(got.isnan(), want)


def test_product_writes_its_result_and_nothing_else(cuda):
    from symm_mem_recipes import mxfp4_matmul, mxfp4_quantize
    for M, N in ((3, 37), (70, 129), (260, 230)):
        for dtype in (torch.bfloat16, torch.float32):
            a, b = _activations(M, 320, torch.bfloat16, 4), mxfp4_quantize(_activations(N, 320, torch.bfloat16, 5))
            room = torch.full((M * N + 256,), 7.0, dtype=dtype, device="cuda")
            out = room[128:128 + M * N].view(M, N)
            assert mxfp4_matmul(a, b, out=out) is out
            assert bool((room[:128] == 7).all()) and bool((room[128 + M * N:] == 7).all())
            assert torch.equal(out, mxfp4_matmul(a, b, out_dtype=dtype))


def test_an_overlapping_result_is_refused(cuda):
    from symm_mem_recipes import MxFp4Tensor, mxfp4_matmul, mxfp4_quantize
    x = _activations(4, 64, torch.bfloat16, 0)
    b = mxfp4_quantize(_activations(64, 64, torch.bfloat16, 1))
    room = torch.zeros(4 * 64 * 2 + 5 * 2176, dtype=torch.uint8, device="cuda")
    y = room[:512].view(torch.bfloat16).view(4, 64)
    with pytest.raises(AssertionError, match="overlap"):
        mxfp4_matmul(x, b, out=x)
    with pytest.raises(AssertionError, match="overlap"):
        mxfp4_matmul(x, b, out=b.storage[:512].view(torch.bfloat16).view(4, 64))
    with pytest.raises(AssertionError, match="overlap"):
        mxfp4_quantize(y, out=MxFp4Tensor(room[496:496 + 2176], 4, 64))
    with pytest.raises(AssertionError, match="overlap"):
        MxFp4Tensor(room[496:496 + 2176], 4, 64).dequantize(out=y)
    assert torch.equal(mxfp4_matmul(x, b, out=y), mxfp4_matmul(x, b))           # side by side is apart
    assert torch.equal(mxfp4_quantize(y, out=MxFp4Tensor(room[512:512 + 2176], 4, 64)).storage, mxfp4_quantize(y).storage)


def test_empty_operands(cuda):
    from symm_mem_recipes import mxfp4_matmul, mxfp4_quantize
    b = mxfp4_quantize(_activations(10, 64, torch.bfloat16, 0))
    none = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    assert mxfp4_quantize(none).shape == (0, 64)
    assert mxfp4_quantize(none).dequantize().shape == (0, 64)
    assert mxfp4_matmul(none, b).shape == (0, 10)
    assert mxfp4_matmul(b, mxfp4_quantize(none)).shape == (10, 0)


def test_training_products(cuda):
    """The three products of a linear layer, each against its operands' exact values."""
    from symm_mem_recipes import mxfp4_matmul, mxfp4_quantize
    T, K, N = 200, 160, 96
    x, w, dy = (_activations(*s, torch.bfloat16, i) for i, s in enumerate(((T, K), (N, K), (T, N))))
    y = mxfp4_matmul(x, mxfp4_quantize(w))
    dx = mxfp4_matmul(dy, mxfp4_quantize(w, transpose=True))
    dw = mxfp4_matmul(mxfp4_quantize(dy, transpose=True), mxfp4_quantize(x, transpose=True), out_dtype=torch.float32)
    value = lambda t: mx.values(*mx.quantize(t))[:, :t.shape[1]]  # noqa: E731
    _check_product(y, value(x), value(w), torch.bfloat16)
    _check_product(dx, value(dy), value(w.t()), torch.bfloat16)
    _check_product(dw, value(dy.t()), value(x.t()), torch.float32)


def test_streams_and_graphs(cuda):
    """Two captured graphs and eager calls in between, on a stream of their own: each replay
    gives the eager result for the inputs of the moment."""
    from symm_mem_recipes import mxfp4_matmul, mxfp4_quantize
    b = mxfp4_quantize(_activations(300, 512, torch.bfloat16, 1))
    inputs = [_activations(m, 512, torch.bfloat16, m) for m in (1, 130)]
    stream = torch.cuda.Stream()
    graphs = []
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for x in inputs:
            mxfp4_matmul(x, b)
    torch.cuda.synchronize()
    for x in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = mxfp4_matmul(x, b)
        graphs.append((g, y))
    for turn in range(3):
        for x, (g, y) in zip(inputs, graphs):
            x.copy_(_activations(*x.shape, torch.bfloat16, 100 + turn))
            g.replay()
            with torch.cuda.stream(stream):
                stream.wait_stream(torch.cuda.default_stream())
                want = mxfp4_matmul(x, b)
            torch.cuda.synchronize()
            assert torch.equal(y, want)

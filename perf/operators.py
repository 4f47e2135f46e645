"""Cases for measuring the operators at a tensor-parallel layer boundary: the one-shot all-reduce
fused with the norms, gate and residual around the block it ends (forward and backward),
quantisation to 4-bit microscaled floats and the product of such operands.

``run`` computes an operator either in elementary torch operations (``own`` false) or through this
package's entry points (``own`` true) from the same inputs, which ``prepare`` makes from a seed.
``exact`` computes the same from the definition in 64 bits.
"""
import math
import sys
import weakref

import torch

own = False

BLOCK = 32                      # elements that share one scale
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-6


def package():
    """The package under test (its folder is not on the path of a plain checkout)."""
    if "symm-mem-recipes_amd" not in sys.path:
        sys.path.insert(0, "symm-mem-recipes_amd")
    import symm_mem_recipes
    return symm_mem_recipes


# ---------------------------------------------------------------------------- cases
def listed():
    return [
        # the activations of one generated token on their way into a 4-bit product
        {"name": "quantize 1x8192", "op": "quantize", "rows": 1, "cols": 8192, "dtype": "bf16", "transpose": False},
        # a long prompt's activations
        {"name": "quantize 16384x8192", "op": "quantize", "rows": 16384, "cols": 8192, "dtype": "bf16", "transpose": False},
        # training: gradients quantised along the tokens for the weights' gradient; a batch that fills no block
        {"name": "quantize transposed 8191x3584", "op": "quantize", "rows": 8191, "cols": 3584, "dtype": "fp32", "transpose": True},
        # generation, one sequence: bf16 activations against 4-bit weights
        {"name": "product 1x8192x8192", "op": "product", "M": 1, "N": 8192, "K": 8192, "left": "bf16", "out": "bf16"},
        # generation, a ragged batch, activations already in 4 bits
        {"name": "product 37x3584x8192", "op": "product", "M": 37, "N": 3584, "K": 8192, "left": "mxfp4", "out": "bf16"},
        # a short prompt, sizes that fill no tile, fp32 logits
        {"name": "product 1001x1777x4000", "op": "product", "M": 1001, "N": 1777, "K": 4000, "left": "bf16", "out": "fp32"},
        # the benchmark's all-gather matmul shape
        {"name": "product 16384x3584x8192", "op": "product", "M": 16384, "N": 3584, "K": 8192, "left": "mxfp4", "out": "bf16"},
        # generation, one sequence, at the end of a block
        {"name": "norm 1x8192", "op": "norm", "T": 1, "H": 8192, "ranks": 8, "dtype": "bf16", "post": True, "gate": "channel", "sum": False},
        # a prompt; the sum is kept for the backward pass
        {"name": "norm 4096x8192", "op": "norm", "T": 4096, "H": 8192, "ranks": 8, "dtype": "bf16", "post": True, "gate": "channel", "sum": True},
        # an odd width, a group that is no power of two, one gate per token
        {"name": "norm 777x1001", "op": "norm", "T": 777, "H": 1001, "ranks": 5, "dtype": "fp32", "post": True, "gate": "token", "sum": True},
        # fine-tuning on a few tokens, no norm behind the block
        {"name": "norm backward 5x4096", "op": "norm_backward", "T": 5, "H": 4096, "dtype": "bf16", "post": False, "gate": "none"},
        # a training step's tokens, gated per element
        {"name": "norm backward 4096x8192", "op": "norm_backward", "T": 4096, "H": 8192, "dtype": "bf16", "post": True, "gate": "element"},
    ]


def _spread(rng, low, high):
    """A size between low and high, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["quantize", "product", "norm", "norm_backward"])
    if op == "quantize":
        rows = _spread(rng, 1, 16384)
        return {"op": op, "rows": rows, "cols": _spread(rng, 33, 8192), "dtype": rng.choice(["bf16", "bf16", "fp32"]),
                "transpose": rows > 1 and rng.random() < 0.4}
    if op == "product":
        few = rng.random() < 0.4                       # generation, or a prompt
        return {"op": op, "M": _spread(rng, 1, 64) if few else _spread(rng, 65, 8192), "N": _spread(rng, 65, 3584),
                "K": _spread(rng, 64, 8192), "left": rng.choice(["bf16", "mxfp4"]),
                "out": rng.choice(["bf16", "bf16", "bf16", "fp32"])}
    case = {"op": op, "T": _spread(rng, 1, 4096), "H": _spread(rng, 64, 8192), "dtype": rng.choice(["bf16", "bf16", "fp32"]),
            "post": rng.random() < 0.75, "gate": rng.choice(["none", "channel", "token", "element"])}
    if rng.random() < 0.6:
        case["H"] = max(64, case["H"] // 64 * 64)      # widths of models; the others stay odd
    if case["dtype"] == "fp32":
        case["T"] = max(1, case["T"] // 2)
    if op == "norm":
        case["ranks"] = rng.choice([2, 3, 4, 8, 8])
        case["sum"] = rng.random() < 0.5
    return case


# ---------------------------------------------------------------------------- inputs
class _Source:
    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)

    def normal(self, *size, std=1.0):
        return torch.randn(*size, generator=self.gen, device="cuda").mul_(std)

    def activations(self, rows, cols, dtype):
        """Activations with a few loud channels, as a transformer's residual stream has them."""
        loud = torch.exp(self.normal(cols, std=0.7))
        return (self.normal(rows, cols) * loud).to(dtype)


def _gate_shape(case):
    return {"none": None, "channel": (case["H"],), "token": (case["T"], 1), "element": (case["T"], case["H"])}[case["gate"]]


def prepare(case, seed):
    src = _Source(seed)
    state = {"case": case}
    if case["op"] == "quantize":
        state["x"] = src.activations(case["rows"], case["cols"], DTYPES[case["dtype"]])
        return state
    if case["op"] == "product":
        M, N, K = case["M"], case["N"], case["K"]
        # weights are quantised once, when a model is loaded: packed codes and scales in hand
        w_codes, w_scales = _pack(*_to_blocks(src.normal(N, K, std=K ** -0.5)))
        a = src.activations(M, K, torch.bfloat16)
        if case["left"] == "mxfp4":
            a_codes, a_scales = _pack(*_to_blocks(a))
        if own:
            smr = package()
            state["b"] = smr.MxFp4Tensor.from_blocks(w_codes, w_scales, K)
            state["a"] = smr.MxFp4Tensor.from_blocks(a_codes, a_scales, K) if case["left"] == "mxfp4" else a
        else:
            state["b"] = (w_codes, w_scales)
            state["a"] = (a_codes, a_scales) if case["left"] == "mxfp4" else a
        return state
    T, H, dtype = case["T"], case["H"], DTYPES[case["dtype"]]
    state["weight"] = (1 + src.normal(H, std=0.1)).to(dtype)
    state["post_weight"] = (1 + src.normal(H, std=0.1)).to(dtype) if case["post"] else None
    shape = _gate_shape(case)
    state["gate"] = None if shape is None else (0.5 + src.normal(*shape, std=0.2)).to(dtype)
    state["scale"] = 1.25
    if case["op"] == "norm":
        partials = src.normal(case["ranks"], T, H).to(dtype)
        state["residual"] = src.activations(T, H, dtype)
        if own:
            symm = package().EmulatedSymmetricMemory
            tensor = symm.empty_strided_p2p((T, H), (H, 1), dtype, "cuda", world_size=case["ranks"], rank=0)
            handle = symm.rendezvous(tensor)
            handle.all_buffers((T, H), dtype).copy_(partials)
            # the registry of symmetric allocations would keep this one beyond its state
            weakref.finalize(tensor, symm.release, handle.get_buffer(0, (T, H), dtype)).atexit = False
            state["tensor"] = tensor
        else:
            state["partials"] = partials
    else:
        state["summed"] = src.normal(T, H, std=2.5).to(dtype)
        state["residual_out"] = src.activations(T, H, dtype)
        state["grad_normed"] = src.normal(T, H).to(dtype)
        state["grad_residual_out"] = src.normal(T, H).to(dtype)
    return state


# ---------------------------------------------------------------------------- the operators in plain form
def _power(exponent):
    """2 ** exponent in fp32, exactly (exponents of a normal number)."""
    return ((exponent.clamp(min=-126) + 127).to(torch.int32) << 23).view(torch.float32)


def _to_blocks(x):
    """fp32 (grid values [rows, blocks, 32], scale exponents [rows, blocks]) of x's rows."""
    x = x.float()
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    if blocks * BLOCK != cols:
        x = torch.nn.functional.pad(x, (0, blocks * BLOCK - cols))
    x = x.reshape(rows, blocks, BLOCK)
    top = x.abs().amax(dim=2)
    exponent = torch.where(top > 0, torch.frexp(top).exponent - 3, -127).clamp(min=-127)   # floor(log2(top)) - 2
    v = x * _power(-exponent).unsqueeze(2)
    size = v.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    size = torch.clamp(torch.round(size / step) * step, max=6.0)                           # ties to the even code
    return torch.where(v < 0, -size, size), exponent


def _pack(values, exponent):
    """Two codes a byte, the first in the low half; scales as biased exponents."""
    rows, blocks, _ = values.shape
    grid = torch.tensor(GRID, device=values.device)
    codes = torch.searchsorted(grid, values.abs().contiguous()).to(torch.uint8)
    codes = (codes | ((values < 0).to(torch.uint8) << 3)).reshape(rows, blocks * BLOCK // 2, 2)
    return codes[..., 0] | (codes[..., 1] << 4), (exponent + 127).to(torch.uint8)


def _unpack(codes, scales):
    rows, blocks = scales.shape
    table = torch.tensor(GRID + tuple(-g for g in GRID), device=codes.device)
    halves = torch.stack((codes & 15, codes >> 4), dim=2).reshape(rows, blocks, BLOCK)
    return (table[halves.int()] * _power(scales.int() - 127).unsqueeze(2)).reshape(rows, blocks * BLOCK)


def _plain_quantize(state):
    case, x = state["case"], state["x"]
    if case["transpose"]:
        x = x.t()
    values, exponent = _to_blocks(x)
    return (values * _power(exponent).unsqueeze(2)).reshape(x.shape[0], -1)[:, :x.shape[1]].to(torch.bfloat16)


def _plain_product(state):
    a, b = state["a"], _unpack(*state["b"])
    a = _unpack(*(_pack(*_to_blocks(a)) if torch.is_tensor(a) else a))
    return torch.matmul(a, b.t()).to(DTYPES[state["case"]["out"]])


def _norm(x):
    return torch.rsqrt(x.square().mean(dim=1, keepdim=True) + EPS)


def _plain_norm(state):
    dtype = state["residual"].dtype
    s = state["partials"].float().sum(dim=0)
    n = s if state["post_weight"] is None else s * _norm(s) * state["post_weight"].float()
    if state["gate"] is not None:
        n = n * state["gate"].float()
    h = state["scale"] * state["residual"].float() + n
    y = h * _norm(h) * state["weight"].float()
    out = {"normed": y.to(dtype), "residual_out": h.to(dtype)}
    if state["case"]["sum"]:
        out["summed"] = s.to(dtype)
    return out


def _plain_norm_backward(state):
    dtype = state["summed"].dtype
    s, h, dy = state["summed"].float(), state["residual_out"].float(), state["grad_normed"].float()
    w2 = state["weight"].float()
    r2 = _norm(h)
    dyw = dy * w2
    d = state["grad_residual_out"].float() + r2 * (dyw - h * r2.square() * (dyw * h).mean(dim=1, keepdim=True))
    out = {"residual": (state["scale"] * d).to(dtype), "weight": (dy * h * r2).sum(dim=0).to(dtype)}
    n = s
    if state["post_weight"] is not None:
        r1, w1 = _norm(s), state["post_weight"].float()
        n = s * r1 * w1
    dn = d
    if state["gate"] is not None:
        g = state["gate"]
        dg = d * n
        dg = dg.sum(dim=0) if g.dim() == 1 else dg.sum(dim=1, keepdim=True) if g.shape[1] == 1 and dg.shape[1] != 1 else dg
        out["gate"] = dg.to(dtype)
        dn = d * g.float()
    if state["post_weight"] is not None:
        out["post_weight"] = (dn * s * r1).sum(dim=0).to(dtype)
        dnw = dn * w1
        dn = r1 * (dnw - s * r1.square() * (dnw * s).mean(dim=1, keepdim=True))
    out["partial"] = dn.to(dtype)
    return out


# ---------------------------------------------------------------------------- the operators through the package
def _own_run(state):
    smr, case = package(), state["case"]
    if case["op"] == "quantize":
        return smr.mxfp4_quantize(state["x"], transpose=case["transpose"]).dequantize()
    if case["op"] == "product":
        return smr.mxfp4_matmul(state["a"], state["b"], out_dtype=DTYPES[case["out"]])
    more = {"post_weight": state["post_weight"], "gate": state["gate"], "residual_scale": state["scale"], "eps": EPS}
    if case["op"] == "norm":
        got = smr.one_shot_all_reduce_norm(state["tensor"], state["residual"], state["weight"], return_sum=case["sum"], **more)
        return dict(zip(("normed", "residual_out", "summed"), got))
    got = smr.one_shot_all_reduce_norm_backward(state["grad_normed"], state["grad_residual_out"], state["summed"],
                                                state["residual_out"], state["weight"], **more)
    return {k: v for k, v in got._asdict().items() if v is not None}


def run(state):
    if own:
        return _own_run(state)
    return {"quantize": _plain_quantize, "product": _plain_product, "norm": _plain_norm,
            "norm_backward": _plain_norm_backward}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "quantize":
        n = case["rows"] * case["cols"]
        # values in, the rounded values out (bf16); a multiplication, a comparison and a rounding each
        return {"bytes": n * (DTYPES[case["dtype"]].itemsize + 2), "flops": 3 * n}
    if case["op"] == "product":
        M, N, K = case["M"], case["N"], case["K"]
        blocks = -(-K // BLOCK)
        left = M * K * 2 if case["left"] == "bf16" else M * blocks * 17
        return {"bytes": left + N * blocks * 17 + M * N * DTYPES[case["out"]].itemsize, "flops": 2 * M * N * K}
    T, H, size = case["T"], case["H"], DTYPES[case["dtype"]].itemsize
    gate = {"none": 0, "channel": H, "token": T, "element": T * H}[case["gate"]]
    weights = H * (1 + case["post"])
    if case["op"] == "norm":
        return {"bytes": size * (T * H * (case["ranks"] + 3 + case["sum"]) + gate + weights), "flops": T * H * (case["ranks"] + 12)}
    return {"bytes": size * (T * H * 6 + 2 * gate + 2 * weights), "flops": T * H * 30}


# ---------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    global own
    keep, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = keep

    def power_of_two(n):
        return ((n.long() + 1023) << 52).view(torch.float64)

    def nearest(x):
        """What the 4-bit microscaled numbers nearest to x's rows stand for: a block's scale puts its largest
        value into [4, 8), and of two grid values equally near the one with the even code is taken."""
        rows, cols = x.shape
        blocks = -(-cols // BLOCK)
        v = torch.zeros(rows, blocks * BLOCK, dtype=torch.float64, device=x.device)
        v[:, :cols] = x
        v = v.view(rows, blocks, BLOCK)
        top = v.abs().max(dim=2, keepdim=True).values
        scale = power_of_two((torch.floor(torch.log2(top)) - 2).clamp(-127, 127))
        scale = torch.where(scale * 8 <= top, scale * 2, torch.where(scale * 4 > top, scale / 2, scale))   # log2 is rounded
        scale = scale.clamp(min=2.0 ** -127)
        size, out = (v / scale).abs(), torch.zeros_like(v)
        for code in range(1, 8):
            border = (GRID[code - 1] + GRID[code]) / 2
            out[size > border if code % 2 else size >= border] = GRID[code]
        return (torch.sign(v) * out * scale).view(rows, -1)

    if case["op"] == "quantize":
        x = state["x"].t() if case["transpose"] else state["x"]
        return nearest(x)[:, :x.shape[1]]
    if case["op"] == "product":
        def values(operand):
            if torch.is_tensor(operand):
                return nearest(operand)
            codes, scales = operand
            table = torch.tensor(GRID, dtype=torch.float64, device=codes.device)
            table = torch.cat((table, -table))
            v = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.float64, device=codes.device)
            v[:, 0::2], v[:, 1::2] = table[(codes % 16).long()], table[(codes // 16).long()]
            return v * power_of_two(scales.int() - 127).repeat_interleave(BLOCK, dim=1)

        return values(state["a"]) @ values(state["b"]).t()
    w2 = state["weight"].double()
    w1 = None if state["post_weight"] is None else state["post_weight"].double()
    gate = None if state["gate"] is None else state["gate"].double()
    if case["op"] == "norm":
        s = state["partials"].double().sum(0)
        n = s if w1 is None else s / (s.pow(2).mean(1, keepdim=True) + EPS).sqrt() * w1
        h = state["scale"] * state["residual"].double() + (n if gate is None else gate * n)
        out = {"normed": h / (h.pow(2).mean(1, keepdim=True) + EPS).sqrt() * w2, "residual_out": h}
        if case["sum"]:
            out["summed"] = s
        return out
    # the backward pass as the derivative of the forward one, row by row: for u = v / |v| with
    # |v| = sqrt(mean v^2 + eps), dv = (du - u mean(du u)) / |v|
    s, h = state["summed"].double(), state["residual_out"].double()
    dy, dh = state["grad_normed"].double(), state["grad_residual_out"].double()

    def through_norm(v, du):
        size = (v.pow(2).mean(1, keepdim=True) + EPS).sqrt()
        u = v / size
        return u, (du - u * (du * u).mean(1, keepdim=True)) / size

    u2, back = through_norm(h, dy * w2)
    total = dh + back
    out = {"residual": state["scale"] * total, "weight": (dy * u2).sum(0)}
    dn = total if gate is None else total * gate
    if w1 is None:
        n, out["partial"] = s, dn
    else:
        u1, out["partial"] = through_norm(s, dn * w1)
        n = u1 * w1
        out["post_weight"] = (dn * u1).sum(0)
    if gate is not None:
        dg = total * n
        out["gate"] = dg.sum(0) if gate.dim() == 1 else dg.sum(1, keepdim=True) if case["gate"] == "token" else dg
    return out

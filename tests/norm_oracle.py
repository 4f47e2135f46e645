"""The reduce with its norms, gate and residual and its backward pass in plain 64-bit arithmetic
(test infrastructure only), with a bound on what fp32 arithmetic may be off by."""
import torch

U = 2.0 ** -24          # half a step of fp32


def forward(partials, residual, weight, post_weight, gate, scale, eps):
    """(normed, residual_out, summed) in 64 bits; differentiable."""
    s = partials.double().sum(0)
    n = s
    if post_weight is not None:
        n = s * torch.rsqrt(s.square().mean(-1, keepdim=True) + eps) * post_weight.double()
    if gate is not None:
        n = gate.double() * n
    h = scale * residual.double() + n
    return h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps) * weight.double(), h, s


def forward_bounds(partials, residual, weight, post_weight, gate, scale, eps):
    """How far fp32 arithmetic may put (normed, residual_out, summed) off, before their last
    rounding.  A sum of m terms is off by at most m u of the magnitudes' sum; a mean of squares
    here adds at most 32 values per thread, 6 levels in the wave and 16 waves (54 u, half of it
    after the root); every other operation is one u."""
    p = partials.double()
    s = p.sum(0)
    off_s = p.shape[0] * U * p.abs().sum(0)
    mean = lambda v: v.square().mean(-1, keepdim=True)  # noqa: E731
    n, off_n = s, off_s
    if post_weight is not None:
        r1 = torch.rsqrt(mean(s) + eps)
        off_r1 = 32 * U + (mean(off_s).sqrt() * r1)
        n = s * r1 * post_weight.double()
        off_n = off_s * r1 * post_weight.double().abs() + n.abs() * (off_r1 + 4 * U)
    if gate is not None:
        n, off_n = n * gate.double(), off_n * gate.double().abs() + n.abs() * gate.double().abs() * U
    x = scale * residual.double()
    h = x + n
    off_h = off_n + 2 * U * (x.abs() + n.abs()) + U * x.abs()
    r2 = torch.rsqrt(mean(h) + eps)
    y = h * r2 * weight.double()
    off_y = off_h * r2 * weight.double().abs() + y.abs() * (32 * U + mean(off_h).sqrt() * r2 + 4 * U)
    return off_y * 1.01, off_h * 1.01, off_s * 1.01


def backward(dy, dh, s, h, weight, post_weight, gate, scale, eps, magnitudes=False):
    """Gradients by the formulas in 64 bits.  ``magnitudes``: every term replaced by its
    magnitude, which is what the errors of the sums are relative to."""
    size = (lambda t: t.abs()) if magnitudes else (lambda t: t)
    sign = 1.0 if magnitudes else -1.0
    dy, s, h, w2 = (size(t.double()) for t in (dy, s, h, weight))
    dh = torch.zeros_like(dy) if dh is None else size(dh.double())
    cols = dy.shape[-1]
    dy, dh, s, h = (t.reshape(-1, cols) for t in (dy, dh, s, h))
    r2 = torch.rsqrt(h.square().mean(-1, keepdim=True) + eps)
    D = dh + r2 * (dy * w2 + sign * h * r2.square() * (dy * w2 * h).mean(-1, keepdim=True))
    out = {"residual": abs(scale) * D if magnitudes else scale * D, "weight": (dy * h * r2).sum(0)}
    n, dn = s, D
    if post_weight is not None:
        w1 = size(post_weight.double())
        r1 = torch.rsqrt(s.square().mean(-1, keepdim=True) + eps)
        n = s * r1 * w1
    if gate is not None:
        g = size(gate.double())
        kind = "channel" if g.dim() == 1 else "token" if g.shape[-1] == 1 and cols != 1 else "element"
        g = g if kind == "channel" else g.reshape(-1, g.shape[-1])
        dg = D * n
        out["gate"] = {"channel": lambda: dg.sum(0), "token": lambda: dg.sum(-1, keepdim=True), "element": lambda: dg}[kind]()
        dn = D * g
    if post_weight is not None:
        out["post_weight"] = (dn * s * r1).sum(0)
        dn = dn * w1
        dn = r1 * (dn + sign * s * r1.square() * (dn * s).mean(-1, keepdim=True))
    out["partial"] = dn
    return out

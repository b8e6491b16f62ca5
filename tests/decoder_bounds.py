"""Definitions in 64 bits of the operators of a decoder's training step, and how far an implementation may be off, element by element.

``u`` is half a step of the result's type (``eps / 2``); every bound is the rounding of the result, the roundings of what it is computed from in
16 bits, and the errors of fp32 arithmetic, each times the magnitudes it acts on.
"""
import math

import torch

IGNORED = -100
F32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def head_exact(hidden, weight, targets, reduction, grad_loss=None, ignore_index=IGNORED, tokens=None):
    """Loss, gradients and bounds of a cross entropy of ``hidden @ weight.T``.

    A logit is a sum of products that the tensor core adds with truncation, 2^-23 of the sum of magnitudes for each of the K / 16 additions at most:
    ``e`` bounds it.  exp, log and the joining of partial sums err by 2^-20 of one more.  The logits' gradient d has 16 bits (fp16: 2^-25 of
    its largest possible value, times 2^-15, below its normal numbers); its products add up with K / 16 truncated additions again.
    bf16 gradients of a reduced loss are made from exponentials that were rounded to fp16 once (2^-11; the target's entry was not), and an
    upstream gradient that is not a power of two rounds the results once more.  Of 256 tokens or fewer (in the whole call, ``tokens``)
    d has two terms, so that u^2 of it is lost.
    """
    dtype = hidden.dtype
    u = half_step(dtype)
    h, w = hidden.detach().double(), weight.detach().double()
    counted = targets != ignore_index
    number = max(1, int(counted.sum()))
    logits = h @ w.t()
    lse = torch.logsumexp(logits, dim=1)
    at = torch.where(counted, targets, 0).long()
    picked = logits.gather(1, at.unsqueeze(1)).squeeze(1)
    losses = torch.where(counted, lse - picked, 0.0)
    magnitude = h.abs() @ w.abs().t()
    e = (h.shape[1] // 16 + 2) * 2.0 ** -23 * magnitude.max(dim=1).values
    e_loss = torch.where(counted, 2 * e + 2.0 ** -20 * (1 + lse.abs()), 0.0) + F32 * losses.abs()
    factor = {"none": grad_loss.double() if grad_loss is not None else torch.ones_like(losses), "sum": torch.ones_like(losses),
              "mean": torch.full_like(losses, 1.0 / number)}[reduction]
    upstream = 1.0 if reduction == "none" or grad_loss is None else float(grad_loss)
    factor = torch.where(counted, factor * upstream, 0.0).unsqueeze(1)
    p = (logits - lse.unsqueeze(1)).exp()
    d = p.clone()
    d[torch.arange(len(at), device=at.device), at] -= 1.0
    # a probability errs by its logit's and its lse's error, its rounding by u of what is stored
    # (and below 2^-126, the smallest normal fp32 number, it is taken as zero: exp(x) < 2^-126 errs by itself, at most 2^-126)
    with_loss = dtype == torch.bfloat16 and reduction != "none"
    e_d = (p * (2 * e.unsqueeze(1) + 2.0 ** -19 + (2.0 ** -11 if with_loss else 0.0)) + ((u * u if (tokens or len(targets)) <= 256 else u) + 4 * F32) * d.abs() + 2.0 ** -126) * factor.abs()
    if dtype == torch.float16:
        e_d = e_d + 2.0 ** -39 * factor.abs().max()
    if with_loss:      # exponentials are kept as fp16 times 2^15, whose subnormal step is 2^-24: half of one is 2^-40 of the largest of 64 words
        e_d = e_d + 2.0 ** -40 * factor.abs()
    d = d * factor
    d_hidden, d_weight = d @ w, d.t() @ h

    def bound(result, a, e_a, b, k):
        roundings = 2 if with_loss and abs(math.log2(abs(upstream))) % 1 else 1
        return roundings * u * result.abs() + (e_a + (k // 16 + 2) * 2.0 ** -23 * a.abs()) @ b.abs() * (1 + u) + smallest(dtype)

    e_hidden = bound(d_hidden, d, e_d, w, w.shape[0])
    e_weight = bound(d_weight, d.t(), e_d.t(), h, h.shape[0])
    if reduction != "none":
        losses, e_loss = losses.sum(), e_loss.sum()
        if reduction == "mean":
            losses, e_loss = losses / number, e_loss / number
        e_loss = e_loss + F32 * losses.abs()
    return (losses, e_loss), (d_hidden, e_hidden), (d_weight, e_weight)


def smallest(dtype):
    """Half of the smallest subnormal number of a type."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def within(got, exact_and_bound):
    exact, bound = exact_and_bound
    off = (got.detach().double().reshape(exact.shape) - exact).abs()
    assert bool(torch.isfinite(off).all()), "not finite"
    worst = (off / bound.clamp(min=1e-300)).max()
    assert float(worst) <= 1.0, f"{float(worst):.3f} times the bound (off by {float(off.max()):.3e})"


def norm_exact(x, branch, weight, branch_weight, gate, scale, eps, grad_h, grad_y):
    """Results and gradients of ``residual_norm`` with bounds, by name.

    fp32 sums over ``dim`` values in runs, lanes and warps: relative errors of ``c`` half steps with c = 64 + dim / 64 (a thread adds 32 values at
    most one after another up to 32768, the rest is trees).
    """
    u, c = half_step(x.dtype), (64 + x.shape[-1] / 64) * F32
    v = {k: t.detach().double() for k, t in dict(x=x, b=branch, w=weight, wb=branch_weight, g=gate).items() if t is not None}
    one = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device)
    wb, g, w = v.get("wb", one), v.get("g", one), v.get("w", one)
    b = v["b"]
    rb = (b.square().mean(-1, keepdim=True) + eps).rsqrt() if "wb" in v else torch.ones_like(b[:, :1])
    n = b * rb * wb
    h = v["x"] + scale * g * n
    mh = v["x"].abs() + (scale * g * n).abs()           # magnitudes that h is a sum of
    out = {"h": (h, u * h.abs() + c * mh + smallest(x.dtype))}
    gh = grad_h.double() if grad_h is not None else torch.zeros_like(h)
    dh, e_dh = gh, F32 * gh.abs()
    if "w" in v:
        r = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
        # r errs by the sums' rounding and by how far h is off where its terms cancel
        e_r = c * (1 + (mh * h.abs()).mean(-1, keepdim=True) * r * r)
        y = h * r * w
        out["y"] = (y, u * y.abs() + r * w.abs() * (c * mh + (e_r + c) * h.abs()) + smallest(x.dtype))
        gy = grad_y.double() if grad_y is not None else torch.zeros_like(h)
        t = gy * w
        mean, mean_abs = (t * h).mean(-1, keepdim=True), (t.abs() * mh).mean(-1, keepdim=True)
        again = c * mh                                  # h, computed once more
        dh = gh + r * (t - h * r * r * mean)
        e_dh = c * gh.abs() + r * (c + e_r) * t.abs() + r ** 3 * ((4 * c + 3 * e_r) * mh * mean_abs + again * mean_abs
                                                                  + h.abs() * (t.abs() * again).mean(-1, keepdim=True))
        dw = (gy * h * r).sum(0)
        e_sum = (64 + x.shape[0] / 8) * F32             # rows one after another in a block, blocks in eight slices
        out["weight"] = (dw, (u if weight.dtype == x.dtype else F32) * dw.abs()
                         + (gy.abs() * r * (again + (c + e_r + e_sum) * mh)).sum(0) + smallest(weight.dtype))
    out["x"] = (dh, u * dh.abs() + e_dh + smallest(x.dtype))
    dn = scale * g * dh
    e_dn = abs(scale) * g.abs() * (e_dh + 2 * F32 * dh.abs())
    e_sum = (64 + x.shape[0] / 8) * F32
    if "wb" in v:
        t = dn * wb
        e_t = e_dn * wb.abs() + F32 * t.abs()
        mean_abs = (t.abs() * b.abs()).mean(-1, keepdim=True)
        db = rb * (t - b * rb * rb * (t * b).mean(-1, keepdim=True))
        e_db = rb * (e_t + 2 * c * t.abs()) + rb ** 3 * b.abs() * ((e_t * b.abs()).mean(-1, keepdim=True) + 8 * c * mean_abs)
        dwb = (dn * b * rb).sum(0)
        out["branch_weight"] = (dwb, (u if branch_weight.dtype == x.dtype else F32) * dwb.abs()
                                + ((e_dn + (3 * c + e_sum) * dn.abs()) * b.abs() * rb).sum(0) + smallest(branch_weight.dtype))
    else:
        db, e_db = dn, e_dn
    out["branch"] = (db, u * db.abs() + e_db + smallest(x.dtype))
    if "g" in v:
        dg = (scale * dh * n).sum(0)
        out["gate"] = (dg, (u if gate.dtype == x.dtype else F32) * dg.abs()
                       + (abs(scale) * (e_dh + (4 * c + e_sum) * dh.abs()) * n.abs()).sum(0) + smallest(gate.dtype))
    return out

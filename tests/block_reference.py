"""The 8-bit and normalising operators of katago_amd.ops from their formulas, in 64
bits on the CPU, each with a bound on how far a right kernel may be from it: every
rounding to the tensors' type is off by at most half a step, fp32 sums by DEPTH *
2^-24 of the terms' magnitudes, DEPTH being how many additions one after the other a
value goes through. `check` is operator_reference's."""
import numpy as np
import torch

from operator_reference import HALF_STEP, SMALLEST, U32, activate

# Values of a thread (at most 128 of a channel), of the threads of a channel, of a
# group's channels, of a group's parts.
DEPTH = 256


def quantize(x):
    """(int8 rows, scales) bit for bit: the definition's fp32 operations on the CPU."""
    v = x.float().cpu().numpy()
    top = np.abs(v).max(-1)
    bad, none = ~np.isfinite(v).all(-1), ~(top >= np.float32(2.0 ** -120))
    safe = np.where(bad | none, np.float32(1), top).astype(np.float32)
    factor = np.float32(127) / safe
    with np.errstate(all="ignore"):
        q = np.rint(v * factor[..., None])
    q = np.where((bad | none)[..., None], np.float32(0), q)
    scale = np.where(bad, np.float32(np.nan), np.where(none, np.float32(0), safe / np.float32(127)))
    return torch.from_numpy(q.astype(np.int8)), torch.from_numpy(scale.astype(np.float32))


def _form(z, act, t):
    """How far the activations' forms may be off, as in operator_reference."""
    return 0.0 if act in ("identity", "relu") else (2.0 ** -18 if t != torch.float32 else 16 * U32) * z.abs().clamp_min(1.0)


def _rounded(y, off, t):
    return off + HALF_STEP[t] * (y.abs() + off) + SMALLEST[t]


def linear_int8(x, xs, w, ws, dtype, bias=None, act="identity", residual=None):
    """(result, bound): the sum is exact; its conversion, two products and a sum are
    rounded."""
    z = (x.double().cpu() @ w.double().cpu().t()) * xs.double().cpu()[:, None] * ws.double().cpu()
    size = z.abs()
    if bias is not None:
        z, size = z + bias.double().cpu(), size + bias.double().cpu().abs()
    off = 1.2 * 4 * U32 * size + _form(z, act, dtype)
    y = activate(z, act)
    if residual is not None:
        y = y + residual.double().cpu()
        off = off + U32 * y.abs()
    return y, _rounded(y, off, dtype)


def valid(x, lengths=None, mask=None):
    b, p, _ = x.shape
    on = torch.ones(b, p, dtype=torch.bool)
    if lengths is not None:
        on &= torch.arange(p) < lengths.cpu()[:, None]
    if mask is not None:
        on &= mask.cpu() != 0
    return on


def statistics(x, groups, eps=1e-5, lengths=None, mask=None):
    """Mean, 1 / sqrt(variance + eps) [batch, groups], and bounds of them."""
    on = valid(x, lengths, mask)
    v = torch.where(on[..., None], x.double().cpu(), 0.0).unflatten(2, (groups, -1))
    n = (on.sum(1) * v.shape[-1]).clamp_min(1)[:, None].double()
    mean = v.sum((1, 3)) / n
    d = torch.where(on[:, :, None, None], v - mean[:, None, :, None], 0.0)
    var = (d * d).sum((1, 3)) / n
    rstd = (var + eps).rsqrt()
    some = on.any(1)[:, None]
    # The mean is put right by the mean of the differences from a first one, and rounded.
    mean_off = U32 * mean.abs() + 4 * DEPTH * U32 * var.sqrt() + 4 * DEPTH * U32 * U32 * mean.abs()
    # Squares are of differences from a point within 2 deviations of the mean.
    var_off = 5 * (DEPTH + 8) * U32 * var
    rstd_off = rstd * (0.5 * var_off / (var + eps) + 4 * U32)
    return torch.where(some, mean, 0.0), torch.where(some, rstd, 0.0), mean_off, rstd_off


def _normalised(x, weight, bias, mean, rstd, mean_off, rstd_off):
    """h, z = h weight + bias, and bounds of them."""
    g = mean.shape[1]
    ext = lambda s: s[:, None, :, None]
    v = x.double().cpu().unflatten(2, (g, -1))
    h = (v - ext(mean)) * ext(rstd)
    h_off = 3 * U32 * h.abs() + ext(mean_off) * ext(rstd) + (v - ext(mean)).abs() * ext(rstd_off)
    h, h_off = h.flatten(2), h_off.flatten(2)
    w = torch.ones(x.shape[2], dtype=torch.float64) if weight is None else weight.double().cpu()
    z = h * w
    z_off = h_off * w.abs() + U32 * z.abs()
    if bias is not None:
        z = z + bias.double().cpu()
    return h, z, w, h_off, z_off + U32 * z.abs()


def group_norm_values(x, groups, weight=None, bias=None, eps=1e-5, act="identity", lengths=None, mask=None):
    """(result before its rounding, bound)."""
    on = valid(x, lengths, mask)[..., None]
    mean, rstd, mean_off, rstd_off = statistics(x, groups, eps, lengths, mask)
    _, z, _, _, z_off = _normalised(x, weight, bias, mean, rstd, mean_off, rstd_off)
    y = activate(z, act)
    off = 1.2 * z_off + _form(z, act, x.dtype)
    return torch.where(on, y, 0.0), torch.where(on, off, 0.0)


def group_norm(x, groups, **kw):
    y, off = group_norm_values(x, groups, **kw)
    return y, torch.where(y == 0, off, _rounded(y, off, x.dtype))


def check_rows(q, scales, want, what=""):
    """8-bit rows against (values before their rounding, bound): a scale is a 127th of
    the row's largest within its bound, a whole number within half a step of its value."""
    y, off = want
    q, scales = q.double().cpu(), scales.double().cpu()
    top, top_off = y.abs().amax(-1), off.amax(-1)
    assert bool(((scales - top / 127).abs() <= (top_off + 2 * U32 * top) / 127 * 1.01).all()), (what, "scales")
    far = (q * scales[..., None] - y).abs()
    room = scales[..., None] * (0.5 + 127 * 4 * U32) + off * 1.01
    assert bool((far <= room).all()), (what, float((far - room).max()))
    on = top > 2.0 ** -119
    assert torch.equal(q.abs().amax(-1)[on], torch.full_like(top[on], 127.0)), what
    assert not q[~on].any() and not scales[top == 0].any(), what


def slope(z, act):
    if act == "relu":
        return (z > 0).double()
    if act == "identity":
        return torch.ones_like(z)
    z = z.clone().requires_grad_(True)
    with torch.enable_grad():
        return torch.autograd.grad(activate(z, act).sum(), z)[0]


def group_norm_backward(x, grad, stats, groups, weight=None, bias=None, act="identity", lengths=None, mask=None):
    """((grad_x, bound), (grad_weight, bound), (grad_bias, bound)) from the fp32
    statistics as they are. Slopes change by at most 1.2 times their argument's change
    (but relu's, which may be either where its argument is within its bound of 0)."""
    t = x.dtype
    on = valid(x, lengths, mask)[..., None]
    s = stats.double().cpu()
    mean, rstd, zero = s[..., 0], s[..., 1], torch.zeros_like(s[..., 0])
    x = torch.where(on.to(x.device), x, 0)
    h, z, w, h_off, z_off = _normalised(x, weight, bias, mean, rstd, zero, zero)
    dy = torch.where(on, grad.double().cpu(), 0.0)
    u = dy * slope(z, act)
    u_off = dy.abs() * (1.2 * z_off + _form(z, act, t) if act not in ("identity", "relu") else (z.abs() <= z_off).double() * (act == "relu")) + 2 * U32 * u.abs()
    b_grad, b_off = u.sum((0, 1)), u_off.sum((0, 1)) + DEPTH * U32 * u.abs().sum((0, 1))
    uh, uh_off = u * h, u_off * h.abs() + u.abs() * h_off + U32 * (u * h).abs()
    w_grad, w_off = uh.sum((0, 1)), uh_off.sum((0, 1)) + DEPTH * U32 * uh.abs().sum((0, 1))
    per = lambda v: v.unflatten(2, (groups, -1))
    n = (on.sum(1) * (x.shape[2] // groups)).clamp_min(1)[:, :, None, None].double()
    a1, a2 = (per(v * w).sum((1, 3), keepdim=True) / n for v in (u, uh))
    a1_off, a2_off = (per((o + (DEPTH + 4) * U32 * v.abs()) * w.abs()).sum((1, 3), keepdim=True) / n for v, o in ((u, u_off), (uh, uh_off)))
    r = rstd[:, None, :, None]
    y = r * (per(u * w) - a1 - per(h) * a2)
    terms = per((u * w).abs()) + a1.abs() + per(h.abs()) * a2.abs()
    off = r * (per(u_off * w.abs()) + a1_off + per(h.abs()) * a2_off + per(h_off) * a2.abs() + 5 * U32 * terms)
    y, off = torch.where(on, y.flatten(2), 0.0), torch.where(on, off.flatten(2), 0.0)
    return (y, torch.where(on, _rounded(y, off, t), off)), (w_grad, w_off + U32 * w_grad.abs()), (b_grad, b_off + U32 * b_grad.abs())

"""The operators of katago_amd.ops from their formulas, in 64 bits on the CPU,
each with a bound on how far a right kernel may be from it: every rounding to
the tensors' type is off by at most half a step, and fp32 sums of n terms by
n * 2^-24 of the terms' magnitudes."""
import math

import torch

U32 = 2.0 ** -24
HALF_STEP = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float64: 0.0, torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}  # half a step of fp16's subnormals


def activate(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "mish":
        return z * torch.tanh(torch.nn.functional.softplus(z, threshold=100.0))
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * torch.erfc(-z * math.sqrt(0.5))
    return z


def linear(x, w, bias=None, act="identity", residual=None):
    """(result, bound). The activations change by at most 1.2 times their
    argument's change; their fp32 forms are within 2^-18 of max(1, |z|) for
    results in 16 bits and within 8 steps of fp32 for results in fp32."""
    t = x.dtype
    x, w = x.double().cpu(), w.double().cpu()
    z, size = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        b = bias.double().cpu()
        z, size = z + b, size + b.abs()
    form = 0.0 if act in ("identity", "relu") else 2.0 ** -18 if t != torch.float32 else 16 * U32
    off = 1.2 * (x.shape[1] + 2) * U32 * size + form * z.abs().clamp_min(1.0)
    y = activate(z, act)
    if residual is not None:
        y = y + residual.double().cpu()
        off = off + U32 * y.abs()
    return y, off + HALF_STEP[t] * (y.abs() + off) + SMALLEST[t]


def rope(x, positions, freqs, layout="interleaved", inverse=False):
    """(result, bound). Sine and cosine are within 2^-17 where the result is
    rounded to 16 bits (64 times finer than fp16's half step) and within 8 steps
    of fp32 otherwise; two products and a sum follow."""
    t = x.dtype
    x = x.double().cpu()
    tables, pairs, _ = freqs.shape
    group = x.shape[1] // tables
    angle = torch.einsum("ta,hpa->thp", positions.double().cpu(), freqs.double().cpu()).repeat_interleave(group, 1)
    if inverse:
        angle = -angle
    c, s = torch.cos(angle), torch.sin(angle)
    y, size = x.clone(), torch.zeros_like(x)
    i0 = torch.arange(pairs) * 2 if layout == "interleaved" else torch.arange(pairs)
    i1 = i0 + 1 if layout == "interleaved" else i0 + pairs
    y[:, :, i0] = x[:, :, i0] * c - x[:, :, i1] * s
    y[:, :, i1] = x[:, :, i0] * s + x[:, :, i1] * c
    size[:, :, i0] = size[:, :, i1] = x[:, :, i0].abs() + x[:, :, i1].abs()
    off = (2.0 ** -17 if t != torch.float32 else 8 * U32) * size
    turned = torch.zeros(x.shape[2], dtype=torch.bool)
    turned[i0] = turned[i1] = True
    bound = torch.where(turned, off + HALF_STEP[t] * (y.abs() + off) + SMALLEST[t], torch.zeros_like(off))
    return y, bound


def attention(q, k, v, scale=None, lengths=None, mask=None):
    """(result, bound). A score is off by (dq + 2) * 2^-24 of its terms'
    magnitudes, its exponential by that (once in p, once in the sum) and 2^-21;
    p is rounded to the tensors' type for the second product (its largest is at
    least 1, and at most 256), whose sums are fp32."""
    t = q.dtype
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    batch, lq, heads, dq = q.shape
    lk, kv = k.shape[1], k.shape[2]
    scale = dq ** -0.5 if scale is None else scale
    out, bound = torch.zeros(batch, lq, heads, v.shape[3], dtype=torch.float64), None
    bound = torch.zeros_like(out)
    for b in range(batch):
        on = torch.ones(lk, dtype=torch.bool)
        if lengths is not None:
            on[max(0, int(lengths[b])):] = False
        if mask is not None:
            on &= mask[b].cpu() != 0
        if not on.any():
            continue
        for h in range(heads):
            kk, vv, qq = k[b, on, h // (heads // kv)], v[b, on, h // (heads // kv)], q[b, :, h]
            p = torch.softmax(scale * (qq @ kk.t()), -1)
            out[b, :, h] = p @ vv
            terms = scale * (qq.abs() @ kk.abs().t()).amax(-1, keepdim=True)
            rel = HALF_STEP[t] + 2 * (dq + 4) * U32 * terms + 2.0 ** -20 + 2 * (len(kk) + 4) * U32
            off = rel * (p @ vv.abs()) + SMALLEST[t] * vv.abs().sum(0)
            bound[b, :, h] = off + HALF_STEP[t] * (out[b, :, h].abs() + off) + SMALLEST[t]
    return out, bound


def check(got, want, what=""):
    """got within the bound of (result, bound), NaN and infinities alike."""
    y, bound = want
    got = got.double().cpu()
    assert got.shape == y.shape, (what, got.shape, y.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(y)), (what, "NaN")
    off = (got - y).abs()
    off[torch.isnan(y) | (got == y)] = 0.0
    worst = (off - bound).flatten().argmax() if off.numel() else None
    assert off.numel() == 0 or bool((off <= bound).all()), (
        what, "index %d: got %g, want %g, bound %g" % (worst, got.flatten()[worst], y.flatten()[worst], bound.flatten()[worst]))

"""The 8-bit and normalising operators against their formulas in 64 bits, at the
sizes, strides, masks and values where their tiles, tails and sums can go wrong, and
as a program runs them: together, on its own stream, captured and replayed, in place,
without torch. Bounds: block_reference.py."""
import threading

import numpy as np
import pytest
import torch

import block_reference as ref
from katago_amd import nn, ops
from operator_reference import check

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16, torch.float32]
ids = lambda v: str(v).replace("torch.", "").replace(" ", "")


def _seeded(*what):
    return torch.Generator().manual_seed(hash(what) % (1 << 31))


def _laid(values, pad=0, shift=0, fill=float("nan")):
    """values on the GPU, rows of the last axis pad apart, starting shift elements past
    a 16-byte border, `fill` between them."""
    row = values.shape[-1] + pad
    n = values.shape[:-1].numel()
    flat = torch.full((shift + n * row,), 0, dtype=values.dtype, device="cuda")
    flat.fill_(fill if values.dtype.is_floating_point else 77)
    t = flat[shift:].view(*values.shape[:-1], row)[..., :values.shape[-1]]
    t.copy_(values)
    return t


def _rand(*shape, dtype=torch.float16, seed=0, scale=1.0, shift=0.0, **layout):
    return _laid((torch.randn(*shape, generator=_seeded(shape, seed)) * scale + shift).to(dtype), **layout)


def _bytes(*shape, seed=0, **layout):
    return _laid(torch.randint(-128, 128, shape, generator=_seeded(shape, seed)).to(torch.int8), **layout)


def _guarded(*shape, dtype, pad=3, shift=5):
    """An output whose surroundings must stay as they are: (tensor, check)."""
    row = shape[-1] + pad
    n = torch.Size(shape[:-1]).numel()
    flat = torch.full((shift + n * row + 64,), 7, dtype=dtype, device="cuda")
    t = flat[shift:shift + n * row].view(*shape[:-1], row)[..., :shape[-1]]

    def untouched():
        rest = flat.clone()
        rest[shift:shift + n * row].view(*shape[:-1], row)[..., :shape[-1]] = 7
        assert bool((rest == 7).all()), "written outside the output"
    return t, untouched


def _space(need):
    """A workspace of just this size, of bits that mean NaN."""
    return torch.full((need,), 255, dtype=torch.uint8, device="cuda") if need else None


def _linear(x, xs, w, ws, out, **kw):
    return ops.linear_int8(x, xs, w, ws, out, workspace=_space(ops.linear_int8_workspace(x, w)), **kw)


def _norm(x, out, groups, **kw):
    return ops.group_norm(x, out, groups, workspace=_space(ops.group_norm_workspace(x, out, groups)), **kw)


def _backward(x, grad, stats, grad_x, groups, **kw):
    return ops.group_norm_backward(x, grad, stats, grad_x, groups, workspace=_space(ops.group_norm_backward_workspace(x, groups)), **kw)


# -- rows in 8 bits -----------------------------------------------------------

def _check_quantized(x, q, scales):
    want_q, want_s = ref.quantize(x)
    np.testing.assert_array_equal(scales.cpu().numpy(), want_s.numpy())
    assert torch.equal(q.cpu(), want_q)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,channels", [(1, 1), (3, 2), (5, 7), (7, 8), (130, 24), (9, 63), (33, 64), (2, 65), (17, 255), (4, 384), (65, 1024), (3, 1031),
                                           (2, 4096), (5, 8200), (2, 40003), (1, 300001), (20011, 40), (70003, 3)], ids=ids)
def test_quantize_sizes(dtype, rows, channels):
    for pad, shift in ((0, 0), (1, 3)):
        x = _rand(rows, channels, dtype=dtype, pad=pad, shift=0.1)
        q, untouched = _guarded(rows, channels, dtype=torch.int8, pad=pad, shift=shift)
        scales, scales_untouched = _guarded(1, rows, dtype=torch.float32)
        assert ops.quantize_rows(x, q, scales[0]) is q
        _check_quantized(x, q, scales[0])
        untouched()
        scales_untouched()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("channels", [5, 64, 700, 9000])
def test_quantize_rows_of_every_kind(dtype, channels):
    """Zeros, NaN, infinities, the type's largest and smallest numbers, one value alone."""
    x = _rand(14, channels, dtype=dtype)
    big, small = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    x[0] = 0
    x[1, channels - 1] = float("nan")
    x[2, 0] = float("inf")
    x[3, channels // 2], x[3, 0] = float("-inf"), float("nan")
    x[4] = big
    x[5, 1], x[6, channels - 1] = -big, big
    x[7] = 0
    x[7, channels - 2] = -small
    x[8] *= 1e-5
    x[9] = -0.0
    x[10] = small / 4
    x[11], x[12] = 0, 1
    x[11, 0] = 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -119
    x[12, 0] = 127
    x[13] = torch.arange(channels, device="cuda") % 254 - 126.5  # halfway between whole numbers
    x[13, 0] = -127
    q, scales = torch.empty(14, channels, dtype=torch.int8, device="cuda"), torch.empty(14, device="cuda")
    ops.quantize_rows(x, q, scales)
    _check_quantized(x, q, scales)


def test_quantize_far_and_shared_rows():
    far = torch.empty((1 << 32) + (1 << 20), dtype=torch.int8, device="cuda")
    x = far.view(torch.float16).as_strided((3, 100), ((1 << 30) + 1024, 1))
    x.copy_(_rand(3, 100))
    q = far.as_strided((3, 100), ((1 << 31) + 4096, 1), 512)
    scales = torch.empty(3, device="cuda")
    ops.quantize_rows(x, q, scales)
    _check_quantized(x, q, scales)
    x = _rand(1, 100).expand(3, 100)
    ops.quantize_rows(x, q, scales)
    _check_quantized(x, q, scales)
    ops.quantize_rows(x[:0], q[:0], scales[:0])


# -- products of 8-bit rows ---------------------------------------------------

LINEAR_SIZES = [(1, 1, 1), (1, 384, 1024), (3, 40, 8), (1, 4112, 24), (7, 1000, 72), (16, 256, 64), (17, 272, 40), (31, 8, 33),
                (33, 528, 129), (64, 64, 64), (65, 96, 257), (100, 33, 31), (129, 72, 63), (200, 1040, 136), (300, 17, 520), (361, 384, 384),
                (5, 24592, 40), (40, 16384, 24), (64, 8192, 1000), (33, 4096, 200), (17, 8208, 72), (32, 12304, 2100), (33, 4112, 17000), (70, 8208, 72), (66, 4112, 65), (1900, 144, 1990), (1905, 1040, 6408), (2888, 1024, 384), (4100, 2064, 4128)]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("m,k,n", LINEAR_SIZES, ids=ids)
def test_linear_int8_sizes(dtype, m, k, n):
    x, w = _bytes(m, k), _bytes(n, k, seed=1)
    xs, ws = torch.rand(m, device="cuda") + 0.5, (torch.rand(n, device="cuda") + 0.5) * k ** -0.5 / 73
    bias, res = _rand(n, dtype=torch.float32, seed=2), _rand(m, n, dtype=dtype, seed=3, pad=1)
    xs /= 73
    out, untouched = _guarded(m, n, dtype=dtype)
    check(_linear(x, xs, w, ws, out, bias=bias, activation="gelu", residual=res), ref.linear_int8(x, xs, w, ws, dtype, bias, "gelu", res))
    untouched()
    plain = torch.empty(m, n, dtype=dtype, device="cuda")
    check(_linear(x, xs, w, ws, plain), ref.linear_int8(x, xs, w, ws, dtype))
    alone = ops.linear_int8(x, xs, w, ws, torch.empty_like(plain))  # no workspace: no split; the sums are the same
    assert torch.equal(plain, alone), "not the same bits"


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("pad,shift", [(16, 0), (1, 0), (0, 1), (3, 5), (8, 8), (16, 4)])
@pytest.mark.parametrize("m,k,n", [(5, 80, 40), (40, 160, 264), (70, 208, 96), (1800, 150, 1900), (1800, 160, 1900), (3, 15, 20), (90, 11, 70), (90, 131, 70), (9, 149, 40), (9, 24592, 40), (40, 24593, 24)], ids=ids)
def test_linear_int8_strides(dtype, pad, shift, m, k, n):
    x, w = _bytes(m, k, pad=pad, shift=shift), _bytes(n, k, seed=1, pad=pad, shift=shift)
    xs, ws = torch.rand(m, device="cuda"), torch.rand(n, device="cuda") * 1e-3
    out, untouched = _guarded(m, n, dtype=dtype, pad=pad, shift=shift)
    check(_linear(x, xs, w, ws, out), ref.linear_int8(x, xs, w, ws, dtype))
    untouched()
    res = _rand(m, n, dtype=dtype, pad=pad, shift=shift % 4)
    want = ref.linear_int8(x, xs, w, ws, dtype, residual=res)
    check(_linear(x, xs, w, ws, res, residual=res), want)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("act", ops.ACTIVATIONS)
@pytest.mark.parametrize("m,k", [(2, 64), (80, 64), (2, 24592), (1800, 64)])
def test_linear_int8_activations(dtype, act, m, k):
    """Values from the far left tail to the far right one, in every kernel."""
    n = 1900 if m == 1800 else 96
    x, w = _bytes(m, k), _bytes(n, k, seed=1)
    xs, ws = torch.full((m,), 1 / 73, device="cuda"), torch.full((n,), k ** -0.5 / 73, device="cuda")
    bias = torch.linspace(-90, 90, n, device="cuda")
    out = torch.empty(m, n, dtype=dtype, device="cuda")
    check(_linear(x, xs, w, ws, out, bias=bias, activation=act), ref.linear_int8(x, xs, w, ws, dtype, bias, act), act)


@pytest.mark.parametrize("m,n,k", [(1, 3, 131071), (40, 24, 131071), (70, 65, 131071), (130, 1, 131056), (1800, 1900, 16000)])
def test_linear_int8_sums_are_exact(m, n, k):
    """The largest sums there are, and small ones of large parts: one byte too much or
    too little would be seen."""
    x = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
    w = torch.full((n, k), -128, dtype=torch.int8, device="cuda")
    w[n // 2:, 1::2] = 127
    x[m // 2, 3] = 5
    one_m, one_n = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
    out = torch.empty(m, n, dtype=torch.float32, device="cuda")
    _linear(x, one_m, w, one_n, out)
    assert torch.equal(out, (x.double() @ w.double().t().contiguous()).float())


@pytest.mark.parametrize("m", [3, 90, 1800])
def test_linear_int8_scales_that_are_not_numbers(m):
    """A row or a channel with a NaN scale is NaN, and no other; scale 0 leaves the bias."""
    n = 1900 if m == 1800 else 48
    x, w = _bytes(m, 80), _bytes(n, 80, seed=1)
    xs, ws, bias = torch.rand(m, device="cuda"), torch.rand(n, device="cuda"), _rand(n, dtype=torch.float32)
    xs[1], xs[2], ws[3], ws[5] = float("nan"), 0, float("nan"), 0
    out = _linear(x, xs, w, ws, torch.empty(m, n, dtype=torch.bfloat16, device="cuda"), bias=bias)
    bad = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    bad[1], bad[:, 3] = True, True
    assert torch.equal(torch.isnan(out), bad)
    y, off = ref.linear_int8(x, xs, w, ws, torch.bfloat16, bias)
    check(out, (y, off.nan_to_num()))


def test_linear_int8_far_offsets():
    far = torch.empty((1 << 33) + (1 << 20), dtype=torch.int8, device="cuda")
    stride = (1 << 31) + 4096
    x = far.as_strided((3, 64), (stride, 1))
    x.copy_(_bytes(3, 64))
    w = _bytes(32, 64, seed=1)
    xs, ws = torch.rand(3, device="cuda"), torch.rand(32, device="cuda") * 0.01
    out = torch.empty(3, 32, dtype=torch.float16, device="cuda")
    check(_linear(x, xs, w, ws, out), ref.linear_int8(x, xs, w, ws, torch.float16))
    back = torch.empty(32, 3, dtype=torch.float16, device="cuda")
    check(_linear(w, ws, x, xs, back), ref.linear_int8(w, ws, x, xs, torch.float16))
    y = far.view(torch.float16).as_strided((3, 32), (stride // 2, 1), 256)
    check(_linear(x, xs, w, ws, y), ref.linear_int8(x, xs, w, ws, torch.float16))
    many = far.as_strided((130, 64), ((1 << 25) + 64, 1))
    many.copy_(_bytes(130, 64, seed=5))
    xs = torch.rand(130, device="cuda")
    out = torch.empty(130, 32, dtype=torch.float16, device="cuda")
    check(_linear(many, xs, w, ws, out), ref.linear_int8(many, xs, w, ws, torch.float16))
    assert ops.linear_int8(x[:0], xs[:0], w, ws, out[:0]).shape == (0, 32)


# -- group norm ---------------------------------------------------------------

NORM_SIZES = [  # batch, positions, channels, groups
    (1, 1, 1, 1), (1, 1, 384, 1), (5, 1, 24, 3), (300, 1, 1000, 1), (3, 1, 70001, 1), (2, 3, 7, 7), (4, 9, 8, 2), (3, 49, 30, 5), (2, 81, 64, 8),
    (2, 361, 384, 32), (1, 361, 1152, 1), (7, 100, 33, 3), (3, 1531, 190, 19), (2, 700, 40, 1), (1, 5000, 24, 2), (1, 4099, 512, 32), (2, 16384, 80, 5),
    (1, 50021, 16, 2), (1, 20000, 3, 3), (3, 625, 97, 97), (2, 2, 40000, 8), (1, 9000, 640, 1), (40, 36, 256, 1), (513, 4, 48, 4)]


def _masks(kind, b, p, g):
    lengths = mask = None
    if kind in ("lengths", "both"):
        lengths = torch.tensor([[0, p, 1, p // 2, p + 9, -3][i % 6] for i in range(b)], dtype=torch.int32, device="cuda")
    if kind in ("mask", "both", "bool"):
        mask = (torch.rand(b, p + 3, generator=g) < 0.4).to(torch.bool if kind == "bool" else torch.uint8).cuda()[:, :p]
        mask[1, :] = False  # an item without a position
        mask[0, :p - 1] = False  # only the last one
        if kind != "bool":
            mask[2] *= 255  # anything but 0 takes part
    return lengths, mask


def _check_statistics(stats, x, groups, **kw):
    mean, rstd, mean_off, rstd_off = ref.statistics(x, groups, **kw)
    check(stats[..., 0], (mean, mean_off + 1e-300), "mean")
    check(stats[..., 1], (rstd, rstd_off + ref.U32 * rstd), "rstd")


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("size", NORM_SIZES, ids=ids)
def test_group_norm_sizes(dtype, size):
    b, p, c, groups = size
    x = _rand(b, p, c, dtype=dtype, shift=0.7, pad=p % 2)
    w, bias = _rand(c, dtype=torch.float32, seed=1, shift=1.0, scale=0.3), _rand(c, dtype=torch.float32, seed=2)
    kw = dict(weight=w, bias=bias, eps=1e-3)
    out, untouched = _guarded(b, p, c, dtype=dtype)
    stats, stats_untouched = _guarded(1, b * groups * 2, dtype=torch.float32)
    stats = stats[0].view(b, groups, 2)
    assert _norm(x, out, groups, activation="silu", stats=stats, **kw) is out
    check(out, ref.group_norm(x, groups, act="silu", **kw))
    untouched()
    stats_untouched()
    _check_statistics(stats, x, groups, eps=1e-3)
    again = _norm(x, torch.empty(b, p, c, dtype=dtype, device="cuda"), groups, activation="silu", **kw)
    assert torch.equal(out, again), "not the same bits again"
    check(_norm(x, torch.empty_like(again), groups), ref.group_norm(x, groups))
    # In 8 bits.
    q, untouched = _guarded(b, p, c, dtype=torch.int8)
    scales, scales_untouched = _guarded(1, b * p, dtype=torch.float32)
    scales = scales[0].view(b, p)
    assert _norm(x, q, groups, activation="silu", out_scales=scales, stats=stats, **kw) is q
    ref.check_rows(q, scales, ref.group_norm_values(x, groups, act="silu", **kw))
    untouched()
    scales_untouched()
    _check_statistics(stats, x, groups, eps=1e-3)
    same = _norm(x, torch.empty(b, p, c, dtype=torch.int8, device="cuda"), groups, activation="silu", out_scales=torch.empty(b, p, device="cuda"), **kw)
    assert torch.equal(q, same), "not the same bits again"


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("kind", ["lengths", "mask", "both", "bool"])
@pytest.mark.parametrize("p,c,groups", [(1, 40, 2), (49, 24, 3), (361, 96, 8), (5003, 40, 5), (12, 700, 1), (20011, 16, 1)], ids=ids)
def test_group_norm_masks(dtype, kind, p, c, groups):
    """Masks that leave items empty or one position; what lies elsewhere (NaN,
    infinities, the type's lowest value) does not matter."""
    b = 6
    lengths, mask = _masks(kind, b, p, _seeded(p, c))
    x = _rand(b, p, c, dtype=dtype, shift=-0.4)
    on = ref.valid(x, lengths, mask).cuda()
    kw = dict(lengths=lengths, mask=mask, weight=_rand(c, dtype=torch.float32, seed=3), bias=_rand(c, dtype=torch.float32, seed=4))
    want = ref.group_norm(x, groups, act="mish", **kw)
    rows = ref.group_norm_values(x, groups, act="mish", **kw)
    for fill in (float("nan"), float("inf"), torch.finfo(dtype).min):
        x.masked_fill_(~on[..., None], fill)
        out, untouched = _guarded(b, p, c, dtype=dtype)
        stats = torch.empty(b, groups, 2, device="cuda")
        check(_norm(x, out, groups, activation="mish", stats=stats, **kw), want, kind)
        untouched()
        assert not out[~on].any() and not torch.isnan(out).any()
        assert not stats[~on.any(1)].any()
        q, untouched = _guarded(b, p, c, dtype=torch.int8)
        scales = torch.full((b, p), 5.0, device="cuda")
        _norm(x, q, groups, activation="mish", out_scales=scales, **kw)
        ref.check_rows(q, scales, rows, kind)
        untouched()
        assert not q[~on].any() and not scales[~on].any()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("pad,shift", [(8, 0), (1, 0), (0, 1), (3, 5), (64, 8)])
@pytest.mark.parametrize("p,c,groups", [(1, 384, 1), (49, 72, 6), (361, 100, 4), (6007, 48, 4)], ids=ids)
def test_group_norm_strides(dtype, pad, shift, p, c, groups):
    """Positions with gaps and shifts, positions outside items, and in place."""
    x = _laid(torch.randn(3, p, c, generator=_seeded(p, c)).to(dtype), pad=pad, shift=shift)
    want = ref.group_norm(x, groups, act="gelu")
    out, untouched = _guarded(3, p, c, dtype=dtype, pad=pad, shift=shift)
    check(_norm(x, out, groups, activation="gelu"), want)
    untouched()
    turned = x.transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.empty(p, 3, c, dtype=dtype, device="cuda").transpose(0, 1)
    check(_norm(turned, out, groups, activation="gelu"), want)
    q = torch.empty(p, 3, c, dtype=torch.int8, device="cuda").transpose(0, 1)
    scales = torch.empty(3, p, device="cuda")
    _norm(x, q, groups, activation="gelu", out_scales=scales)
    ref.check_rows(q, scales, ref.group_norm_values(x, groups, act="gelu"))
    flat = x.as_strided((3 * p, c + pad), (c + pad, 1), x.storage_offset()) if pad and shift == 0 else None
    check(_norm(x, x, groups, activation="gelu"), want)
    if flat is not None:
        assert bool(torch.isnan(flat[:-1, c:]).all())


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("act", ops.ACTIVATIONS)
@pytest.mark.parametrize("p,c", [(3, 96), (2003, 96), (30011, 24)])
def test_group_norm_activations(dtype, act, p, c):
    """Values from the far left tail to the far right one."""
    x, bias = _rand(2, p, c, dtype=dtype), torch.linspace(-90, 90, c, device="cuda")
    check(_norm(x, torch.empty_like(x), 4, bias=bias, activation=act), ref.group_norm(x, 4, bias=bias, act=act), act)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("p,c,groups", [(1, 500, 1), (300, 24, 2), (9001, 40, 5), (1, 12, 12)], ids=ids)
@pytest.mark.parametrize("mean,dev", [(300.0, 1.0), (-20.0, 0.05), (0.0, 1e-6), (1000.0, 0.0), (0.5, 200.0)])
def test_group_norm_far_means(dtype, p, c, groups, mean, dev):
    """Means far from 0 against the deviation, equal values, values that eps outweighs."""
    x = _rand(2, p, c, dtype=dtype, shift=mean, scale=dev)
    stats = torch.empty(2, groups, 2, device="cuda")
    out = _norm(x, torch.empty_like(x), groups, stats=stats)
    check(out, ref.group_norm(x, groups))
    _check_statistics(stats, x, groups)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("p,c,groups", [(1, 500, 1), (300, 24, 2), (9001, 40, 5)], ids=ids)
def test_group_norm_one_value_far_out(dtype, p, c, groups):
    """The first value, or the last, a thousand times the others."""
    x = _rand(3, p, c, dtype=dtype)
    x[0, 0, 0], x[1, p - 1, c - 1] = 1000, -1000
    check(_norm(x, torch.empty_like(x), groups), ref.group_norm(x, groups))


@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 1e30), (torch.float32, 1e25), (torch.float32, 3e37), (torch.float16, 6e4), (torch.bfloat16, 1e-30),
                                        (torch.float32, 1e-22), (torch.float32, 1e-38)])
@pytest.mark.parametrize("p,c,groups", [(1, 500, 1), (300, 24, 2), (9001, 40, 5)], ids=ids)
def test_group_norm_of_values_of_any_size(dtype, size, p, c, groups):
    """Values whose squares pass the largest float, and values next to nothing."""
    g = _seeded(p, c)
    x = ((torch.rand(2, p, c, generator=g) * 2 - 1) * size).to(dtype).cuda()
    for eps in (1e-5, 2.0 ** -126):
        y, off = ref.group_norm(x, groups, eps=eps)
        # Below the normal numbers an fp32 number has a fixed step, 2^-149: of x - mean
        # and of 1 / sqrt(var) where x is near the largest float.
        off = off + (4 * 2.0 ** -149 * 2.0 ** 63 if size < 1 else 4 * size * 2.0 ** -149)
        check(_norm(x, torch.empty_like(x), groups, eps=eps), (y, off), (size, eps))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("p,c,groups", [(1, 512, 4), (300, 24, 2), (9001, 40, 5)], ids=ids)
def test_group_norm_not_finite_stays_in_its_group(dtype, bad, p, c, groups):
    x = _rand(3, p, c, dtype=dtype)
    x[1, p - 1, c // groups] = bad  # the first channel of group 1
    out = _norm(x, torch.empty_like(x), groups)
    per = c // groups
    want = torch.zeros(3, p, c, dtype=torch.bool, device="cuda")
    want[1, :, per:2 * per] = True
    assert torch.equal(torch.isnan(out), want)
    keep = x.clone()
    keep[1, :, per:2 * per] = 0
    y, off = ref.group_norm(keep, groups)
    y[want.cpu()] = float("nan")
    check(out, (y, off))
    q, scales = torch.empty(3, p, c, dtype=torch.int8, device="cuda"), torch.empty(3, p, device="cuda")
    _norm(x, q, groups, out_scales=scales)
    assert bool(torch.isnan(scales[1]).all()) and not torch.isnan(scales[0]).any() and not torch.isnan(scales[2]).any() and not q[1].any()


def test_group_norm_far_offsets():
    far = torch.empty((1 << 32) + (1 << 20), dtype=torch.float16, device="cuda")
    for shape, strides in (((3, 5, 64), ((1 << 30) + 1024, 64, 1)), ((2, 3, 64), (128, (1 << 30) + 1024, 1)), ((2, 4, 20), ((1 << 31) + 8, (1 << 29) + 64, 1))):
        x = far.as_strided(shape, strides)
        x.copy_(_rand(*shape))
        want = ref.group_norm(x, 4)
        check(_norm(x, torch.empty(shape, dtype=torch.float16, device="cuda"), 4), want)
        check(_norm(x, x, 4), want)
    x = far.as_strided((2, 40000, 64), ((1 << 31) + 64, 1 << 15, 1))  # parts of an item far apart
    x.copy_(_rand(2, 40000, 64))
    check(_norm(x, torch.empty(2, 40000, 64, dtype=torch.float16, device="cuda"), 4), ref.group_norm(x, 4))


def test_norms_of_nothing():
    x, f32 = torch.empty(0, 9, 8, dtype=torch.float16, device="cuda"), dict(dtype=torch.float32, device="cuda")
    assert ops.group_norm(x, x, 2) is x
    x = torch.empty(3, 0, 8, dtype=torch.float16, device="cuda")
    assert ops.group_norm(x, torch.empty_like(x), 2).shape == (3, 0, 8)
    for x in (x, torch.empty(0, 9, 8, dtype=torch.float16, device="cuda")):
        gw, gb = torch.full((8,), 3.0, **f32), torch.full((8,), 3.0, **f32)
        ops.group_norm_backward(x, torch.empty_like(x), torch.empty(x.shape[0], 2, 2, **f32), torch.empty_like(x), 2, grad_weight=gw, grad_bias=gb)
        assert not gw.any() and not gb.any()


# -- its gradient -------------------------------------------------------------

def _forward_statistics(x, groups, **kw):
    stats = torch.empty(x.shape[0], groups, 2, device="cuda")
    _norm(x, torch.empty(x.shape, dtype=x.dtype, device="cuda"), groups, stats=stats, **kw)
    return stats


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("size", NORM_SIZES, ids=ids)
def test_backward_sizes(dtype, size):
    b, p, c, groups = size
    x, dy = _rand(b, p, c, dtype=dtype, shift=0.7, pad=p % 2), _rand(b, p, c, dtype=dtype, seed=5, pad=c % 3)
    w, bias = _rand(c, dtype=torch.float32, seed=1, shift=1.0, scale=0.3), _rand(c, dtype=torch.float32, seed=2)
    stats = _forward_statistics(x, groups, eps=1e-3)
    want = ref.group_norm_backward(x, dy, stats, groups, w, bias, "silu")
    dx, untouched = _guarded(b, p, c, dtype=dtype)
    dw, w_untouched = _guarded(1, c, dtype=torch.float32)
    db, b_untouched = _guarded(1, c, dtype=torch.float32)
    assert _backward(x, dy, stats, dx, groups, weight=w, bias=bias, activation="silu", grad_weight=dw[0], grad_bias=db[0]) is dx
    for got, to, what in zip((dx, dw[0], db[0]), want, ("x", "weight", "bias")):
        check(got, to, what)
    for f in (untouched, w_untouched, b_untouched):
        f()
    dx2, dw2, db2 = torch.empty(b, p, c, dtype=dtype, device="cuda"), torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
    _backward(x, dy, stats, dx2, groups, weight=w, bias=bias, activation="silu", grad_weight=dw2)
    _backward(x, dy, stats, dx2, groups, weight=w, bias=bias, activation="silu", grad_bias=db2)
    assert torch.equal(dx, dx2) and torch.equal(dw[0], dw2) and torch.equal(db[0], db2), "not the same bits again"
    check(_backward(x, dy, stats, dx2, groups), ref.group_norm_backward(x, dy, stats, groups)[0])


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("kind", ["lengths", "mask", "both", "bool"])
@pytest.mark.parametrize("p,c,groups", [(1, 40, 2), (49, 24, 3), (361, 96, 8), (5003, 40, 5), (12, 700, 1), (20011, 16, 1)], ids=ids)
def test_backward_masks(dtype, kind, p, c, groups):
    """What x and the gradient hold where nothing takes part does not matter."""
    b = 6
    lengths, mask = _masks(kind, b, p, _seeded(p, c))
    x, dy = _rand(b, p, c, dtype=dtype, shift=-0.4), _rand(b, p, c, dtype=dtype, seed=7)
    on = ref.valid(x, lengths, mask).cuda()
    w, bias = _rand(c, dtype=torch.float32, seed=3), _rand(c, dtype=torch.float32, seed=4)
    stats = _forward_statistics(x, groups, lengths=lengths, mask=mask)
    want = ref.group_norm_backward(x, dy, stats, groups, w, bias, "mish", lengths, mask)
    for fill in (float("nan"), float("inf"), torch.finfo(dtype).min):
        x.masked_fill_(~on[..., None], fill)
        dy.masked_fill_(~on[..., None], -fill)
        dx, untouched = _guarded(b, p, c, dtype=dtype)
        dw, db = torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
        _backward(x, dy, stats, dx, groups, weight=w, bias=bias, activation="mish", lengths=lengths, mask=mask, grad_weight=dw, grad_bias=db)
        for got, to, what in zip((dx, dw, db), want, ("x", "weight", "bias")):
            check(got, to, (kind, what))
        untouched()
        assert not dx[~on].any()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("act", ops.ACTIVATIONS)
@pytest.mark.parametrize("p,c", [(3, 96), (1003, 96), (30011, 24)])
def test_backward_activations(dtype, act, p, c):
    """Slopes from the far left tail to the far right one."""
    x, dy = _rand(2, p, c, dtype=dtype), _rand(2, p, c, dtype=dtype, seed=1)
    bias = torch.linspace(-40, 40, c, device="cuda")
    stats = _forward_statistics(x, 4)
    want = ref.group_norm_backward(x, dy, stats, 4, None, bias, act)
    dw, db = torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
    dx = _backward(x, dy, stats, torch.empty_like(x), 4, bias=bias, activation=act, grad_weight=dw, grad_bias=db)
    on = (ref._normalised(x, None, bias, *(stats.double().cpu()[..., i] for i in (0, 1)), *(torch.zeros(2, 4, dtype=torch.float64),) * 2)[1].abs() > 1e-4)
    if act != "relu":
        on[:] = True
    for got, (y, off), what in zip((dx.cpu()[on], dw, db), ((want[0][0][on], want[0][1][on]), *want[1:]), ("x", "weight", "bias")):
        check(got, (y, off), (act, what))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("pad,shift", [(8, 0), (1, 0), (0, 1), (3, 5)])
@pytest.mark.parametrize("p,c,groups", [(1, 384, 1), (361, 100, 4), (6007, 48, 4)], ids=ids)
def test_backward_strides(dtype, pad, shift, p, c, groups):
    g = _seeded(p, c)
    x, dy = (_laid(torch.randn(3, p, c, generator=g).to(dtype), pad=pad, shift=shift) for _ in range(2))
    stats = _forward_statistics(x, groups)
    want = ref.group_norm_backward(x, dy, stats, groups, act="gelu")[0]
    dx, untouched = _guarded(3, p, c, dtype=dtype, pad=pad, shift=shift)
    check(_backward(x, dy, stats, dx, groups, activation="gelu"), want)
    untouched()
    x, dy = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (x, dy))
    dx = torch.empty(p, 3, c, dtype=dtype, device="cuda").transpose(0, 1)
    check(_backward(x, dy, stats, dx, groups, activation="gelu"), want)
    one = dy[:1, :1].expand(3, p, c)  # a gradient that is the same everywhere, as of a sum
    check(_backward(x, one, stats, dx, groups, activation="gelu"), ref.group_norm_backward(x, one, stats, groups, act="gelu")[0])


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("kind", ["none", "lengths", "both"])
@pytest.mark.parametrize("b,p,c,groups", [(1024, 1, 384, 1), (5003, 1, 40, 5), (1500, 4, 33, 3), (2000, 3, 1000, 8), (1027, 2, 2048, 1), (70001, 1, 24, 1), (1100, 1, 9000, 3),
                                          (1031, 4, 7, 7), (1030, 1, 4000, 1000), (3, 1, 384, 1), (63, 1, 4096, 2), (300, 1, 50, 5), (3, 1, 8200, 1)], ids=ids)
def test_backward_of_many_items(dtype, kind, b, p, c, groups):
    """Items of a few positions, whose sums a workgroup has for many of them."""
    lengths, mask = _masks(kind, b, p, _seeded(p, c)) if kind != "none" else (None, None)
    x, dy = _rand(b, p, c, dtype=dtype, shift=0.3), _rand(b, p, c, dtype=dtype, seed=5, pad=1)
    w, bias = _rand(c, dtype=torch.float32, seed=1, shift=1.0, scale=0.3), _rand(c, dtype=torch.float32, seed=2)
    stats = _forward_statistics(x, groups, eps=1e-3, lengths=lengths, mask=mask)
    want = ref.group_norm_backward(x, dy, stats, groups, w, bias, "gelu", lengths, mask)
    if kind != "none":
        on = ref.valid(x, lengths, mask).cuda()
        x.masked_fill_(~on[..., None], float("nan"))
        dy.masked_fill_(~on[..., None], float("inf"))
    dx, untouched = _guarded(b, p, c, dtype=dtype)
    dw, db = torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
    kw = dict(weight=w, bias=bias, activation="gelu", lengths=lengths, mask=mask)
    _backward(x, dy, stats, dx, groups, grad_weight=dw, grad_bias=db, **kw)
    for got, to, what in zip((dx, dw, db), want, ("x", "weight", "bias")):
        check(got, to, what)
    untouched()
    again = torch.empty(c, device="cuda")
    _backward(x, dy, stats, dx, groups, grad_weight=again, **kw)
    assert torch.equal(dw, again), "not the same bits again"


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("act", [a for a in ops.ACTIVATIONS if a != "relu"])
@pytest.mark.parametrize("b,p,c", [(3, 120, 96), (2, 6000, 96), (300, 1, 96)], ids=ids)
def test_sums_of_slopes(dtype, act, b, p, c):
    """grad_weight and grad_bias are fp32 whatever x is: 1e-6 of their norm is what rounding
    in fp32 may cost them (16 roundings of 2^-24 of a term, each of random sign), not what
    rounding to 16 bits would (2^-11)."""
    x, dy = _rand(b, p, c, dtype=dtype), _rand(b, p, c, dtype=dtype, seed=5)
    w, bias = _rand(c, dtype=torch.float32, seed=1, shift=1.0, scale=0.2), _rand(c, dtype=torch.float32, seed=2, scale=0.2)
    stats, dx = _forward_statistics(x, 8), torch.empty_like(x)
    dw, db = torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
    _backward(x, dy, stats, dx, 8, weight=w, bias=bias, activation=act, grad_weight=dw, grad_bias=db)
    want = ref.group_norm_backward(x, dy, stats, 8, w, bias, act)
    for got, (to, _) in zip((dw, db), want[1:]):
        to = to.to(got.device).double()
        assert float((got.double() - to).norm() / to.norm()) < 1e-6


@pytest.mark.parametrize("b,p,c,groups", [(3, 20, 24, 3), (2, 9000, 24, 3), (40, 1, 24, 3)], ids=ids)
def test_statistics_anywhere(b, p, c, groups):
    """Statistics at an address that no pair of numbers begins at."""
    x, dy = _rand(b, p, c, dtype=torch.float16, shift=0.3), _rand(b, p, c, dtype=torch.float16, seed=5)
    stats = torch.empty(b * groups * 2 + 1, device="cuda")[1:].view(b, groups, 2)
    _norm(x, torch.empty_like(x), groups, stats=stats)
    there = _forward_statistics(x, groups)
    assert torch.equal(stats, there)
    dx, want = torch.empty_like(x), torch.empty_like(x)
    _backward(x, dy, stats, dx, groups)
    assert torch.equal(dx, _backward(x, dy, there, want, groups))


@pytest.mark.parametrize("act", [a for a in ops.ACTIVATIONS if a != "relu"])
@pytest.mark.parametrize("p,c,groups", [(1, 16, 2), (9, 12, 3), (2100, 8, 2)], ids=ids)
def test_backward_is_the_forwards_difference(act, p, c, groups):
    """The gradients against differences of the forward pass in 64 bits: along a random
    direction, (f(x + s) - f(x - s)) / 2, whose own error is of the step's third power."""
    x, dy = _rand(2, p, c, dtype=torch.float32), _rand(2, p, c, dtype=torch.float32, seed=1)
    w, b = _rand(c, dtype=torch.float32, seed=2, shift=1.0), _rand(c, dtype=torch.float32, seed=3)
    dw, db = torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
    stats = _forward_statistics(x, groups)
    dx = _backward(x, dy, stats, torch.empty_like(x), groups, weight=w, bias=b, activation=act, grad_weight=dw, grad_bias=db)
    t = [v.double().cpu() for v in (x, w, b)]
    f = lambda x, w, b: float((ref.group_norm(x, groups, weight=w, bias=b, act=act)[0] * dy.double().cpu()).sum())
    for i, grad in enumerate((dx, dw, db)):
        step = torch.randn(t[i].shape, generator=_seeded(i), dtype=torch.float64) * 1e-4
        up, down = ([v + (k == i) * s * step for k, v in enumerate(t)] for s in (1, -1))
        moved = (f(*up) - f(*down)) / 2
        size = float((grad.double().cpu() * step).abs().sum())
        assert abs(moved - float((grad.double().cpu() * step).sum())) <= 1e-5 * size, (act, i)


def test_backward_far_offsets():
    far = torch.empty((1 << 32) + (1 << 20), dtype=torch.float16, device="cuda")
    for shape, strides in (((3, 5, 64), ((1 << 30) + 1024, 64, 1)), ((2, 3, 64), (128, (1 << 30) + 1024, 1))):
        x, dx = far.as_strided(shape, strides), far.as_strided(shape, strides, 1 << 12)
        x.copy_(_rand(*shape))
        dy = far.as_strided(shape, strides, 1 << 14)
        dy.copy_(_rand(*shape, seed=1))
        stats = _forward_statistics(x, 4)
        want = ref.group_norm_backward(x, dy, stats, 4)[0]
        check(_backward(x, dy, stats, dx, 4), want)


class GroupNorm(torch.autograd.Function):
    """The calls as a program that trains uses them."""

    @staticmethod
    def forward(ctx, x, weight, bias, groups, activation, mask):
        stats = torch.empty(x.shape[0], groups, 2, device=x.device)
        out = _norm(x, torch.empty_like(x), groups, weight=weight, bias=bias, activation=activation, mask=mask, stats=stats)
        ctx.save_for_backward(x, weight, bias, stats, mask)
        ctx.kind = groups, activation
        return out

    @staticmethod
    def backward(ctx, grad):
        x, weight, bias, stats, mask = ctx.saved_tensors
        groups, activation = ctx.kind
        dw, db = torch.empty_like(weight), torch.empty_like(bias)
        dx = _backward(x, grad, stats, torch.empty_like(x), groups, weight=weight, bias=bias, activation=activation, mask=mask, grad_weight=dw, grad_bias=db)
        return dx, dw, db, None, None, None


def test_in_an_autograd_function():
    x = _rand(4, 81, 64, dtype=torch.float32).requires_grad_(True)
    w, b = (_rand(64, dtype=torch.float32, seed=i).requires_grad_(True) for i in (1, 2))
    mask = torch.rand(4, 81, generator=_seeded(9)).cuda() < 0.7
    out = GroupNorm.apply(x, w, b, 8, "mish", mask)
    dy = _rand(4, 81, 64, dtype=torch.float32, seed=3)
    out.backward(dy)
    with torch.no_grad():
        stats = _forward_statistics(x, 8, mask=mask)
        for t, want in zip((x, w, b), ref.group_norm_backward(x, dy, stats, 8, w, b, "mish", mask=mask)):
            check(t.grad, want)
    with pytest.raises(nn.StringError, match="gradients"):
        ops.group_norm(x, torch.empty_like(x), 8)


# -- together -----------------------------------------------------------------

def _block_inputs(dtype, b=3, p=81, c=96, wide=160, seed=0):
    """A residual block: norm and activation in 8-bit rows, product, norm, product, sum."""
    s = {"x": _rand(b, p, c, dtype=dtype, seed=seed), "mask": torch.rand(b, p, generator=_seeded(seed)).cuda() < 0.8, "groups": 8}
    for i, (n, k) in enumerate(((wide, c), (c, wide))):
        w = _rand(n, k, dtype=dtype, seed=10 + i, scale=k ** -0.5)
        s[f"w{i}"], s[f"ws{i}"] = torch.empty(n, k, dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
        ops.quantize_rows(w, s[f"w{i}"], s[f"ws{i}"])
        s[f"q{i}"], s[f"qs{i}"] = torch.empty(b, p, k, dtype=torch.int8, device="cuda"), torch.empty(b, p, device="cuda")
        s[f"gamma{i}"], s[f"beta{i}"] = _rand(k, dtype=torch.float32, seed=20 + i, shift=1.0, scale=0.2), _rand(k, dtype=torch.float32, seed=30 + i, scale=0.3)
        s[f"b{i}"] = _rand(n, dtype=torch.float32, seed=40 + i)
        s[f"h{i}"] = torch.empty(b, p, n, dtype=dtype, device="cuda")
        src = s["x"] if i == 0 else s["h0"]
        s[f"space{i}"] = _space(max(16, ops.group_norm_workspace(src, s[f"q{i}"], 8)))
        s[f"product{i}"] = _space(max(16, ops.linear_int8_workspace(s[f"q{i}"].flatten(0, 1), s[f"w{i}"])))
    return s


def _block(s, **kw):
    src = s["x"]
    for i in (0, 1):
        ops.group_norm(src, s[f"q{i}"], s["groups"], weight=s[f"gamma{i}"], bias=s[f"beta{i}"], activation="mish", mask=s["mask"], out_scales=s[f"qs{i}"],
                       workspace=s[f"space{i}"], **kw)
        ops.linear_int8(s[f"q{i}"].flatten(0, 1), s[f"qs{i}"].flatten(), s[f"w{i}"], s[f"ws{i}"], s[f"h{i}"].flatten(0, 1), bias=s[f"b{i}"],
                        residual=s["x"].flatten(0, 1) if i else None, workspace=s[f"product{i}"], **kw)
        src = s[f"h{i}"]
    return s["h1"]


def _block_check(s, out):
    """Each call against its formula on the inputs that it had."""
    src = s["x"]
    for i in (0, 1):
        ref.check_rows(s[f"q{i}"], s[f"qs{i}"], ref.group_norm_values(src, s["groups"], weight=s[f"gamma{i}"], bias=s[f"beta{i}"], act="mish", mask=s["mask"]))
        check(s[f"h{i}"].flatten(0, 1), ref.linear_int8(s[f"q{i}"].flatten(0, 1), s[f"qs{i}"].flatten(), s[f"w{i}"], s[f"ws{i}"], out.dtype, s[f"b{i}"],
                                                        residual=s["x"].flatten(0, 1) if i else None))
        src = s[f"h{i}"]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("sizes", [{}, dict(b=1, p=6000, c=48, wide=80), dict(b=20, p=1, c=1040, wide=2000)], ids=ids)
def test_block(dtype, sizes):
    s = _block_inputs(dtype, **sizes)
    _block_check(s, _block(s))


@pytest.mark.parametrize("sizes", [{}, dict(b=1, p=6000, c=48, wide=80), dict(b=20, p=1, c=1040, wide=24592)], ids=ids)
def test_captured_and_replayed(sizes):
    """A block and a gradient in a graph, replayed over new inputs with the program's
    own eager calls between the replays; every replay gives the eager bits."""
    s = _block_inputs(torch.bfloat16, **sizes)
    other = _block_inputs(torch.bfloat16, **sizes, seed=50)
    shape = s["x"].shape
    dy, dx = _rand(*shape, dtype=torch.bfloat16, seed=9), torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    stats, dw = torch.empty(shape[0], 8, 2, device="cuda"), torch.empty(shape[2], device="cuda")
    y = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    fwd, bwd = _space(max(16, ops.group_norm_workspace(s["x"], y, 8))), _space(max(16, ops.group_norm_backward_workspace(s["x"], 8)))

    def step():
        ops.group_norm(s["x"], y, 8, stats=stats, workspace=fwd, mask=s["mask"])
        ops.group_norm_backward(s["x"], dy, stats, dx, 8, grad_weight=dw, workspace=bwd, mask=s["mask"])
        return _block(s)

    inputs = [_rand(*shape, dtype=torch.bfloat16, seed=60 + i) for i in range(4)]
    eager = []
    for x in inputs:
        s["x"].copy_(x)
        out = step()
        eager.append([t.clone() for t in (out, y, dx, dw, stats, s["q1"], s["qs1"])])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step()
        with torch.cuda.graph(graph, stream=side):
            out = step()
    torch.cuda.synchronize()
    for round_ in range(3):
        for i in (0, 1, 2, 3):
            s["x"].copy_(inputs[i])
            out.fill_(3)
            graph.replay()
            _block(other)
            torch.cuda.synchronize()
            for got, want in zip((out, y, dx, dw, stats, s["q1"], s["qs1"]), eager[i]):
                assert torch.equal(got, want), (round_, i)


def test_other_stream_and_null_stream():
    s = _block_inputs(torch.float16)
    want = _block(s).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    s["h1"].zero_()
    side.wait_stream(torch.cuda.current_stream())
    _block(s, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(s["h1"], want)
    s["h1"].zero_()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        _block(s)  # torch's current stream
    side.synchronize()
    assert torch.equal(s["h1"], want)
    s["h1"].zero_()
    torch.cuda.synchronize()
    _block(s, stream=0)
    torch.cuda.synchronize()
    assert torch.equal(s["h1"], want)


def test_two_threads_at_once():
    states = [_block_inputs(torch.bfloat16, seed=100 * i) for i in range(2)]
    want = [_block(s).clone() for s in states]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    _block(states[i])
            stream.synchronize()
            if not torch.equal(states[i]["h1"], want[i]):
                bad.append(i)
        except Exception as e:
            bad.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_without_torch_tensors():
    """DeviceTensor views of the library's own buffers, on the null stream."""
    x = np.random.default_rng(1).standard_normal((5, 40)).astype(np.float32)
    bx, bq, bs, bo, by = nn.DeviceBuffer.from_array(x), *(nn.DeviceBuffer(n) for n in (200, 20, 100, 800))
    q, s = ops.DeviceTensor(bq.ptr, (5, 40), "int8"), ops.DeviceTensor(bs.ptr, (5,), "float32")
    ops.quantize_rows(ops.DeviceTensor(bx.ptr, (5, 40), "float32"), q, s)
    ops.linear_int8(q, s, q, s, ops.DeviceTensor(bo.ptr, (5, 5), "float32"))
    x3 = ops.DeviceTensor(bx.ptr, (1, 5, 40), "float32")
    need = ops.group_norm_workspace(x3, x3, 4)
    space = nn.DeviceBuffer(max(need, 16))
    ops.group_norm(x3, ops.DeviceTensor(by.ptr, (1, 5, 40), "float32"), 4, workspace=ops.DeviceTensor(space.ptr, (need,), "uint8"))
    torch.cuda.synchronize()
    want = ref.quantize(torch.from_numpy(x))
    check(torch.from_numpy(bo.to_array(np.float32, (5, 5))), ref.linear_int8(*want, *want, torch.float32))
    check(torch.from_numpy(by.to_array(np.float32, (1, 5, 40))), ref.group_norm(torch.from_numpy(x)[None], 4))


def test_refusals_leave_no_error_behind():
    x = _rand(3, 70000, 64)
    q, scales = torch.empty(x.shape, dtype=torch.int8, device="cuda"), torch.empty(3, 70000, device="cuda")
    with pytest.raises(nn.StringError, match="workspace"):
        ops.group_norm(x, q, 4, out_scales=scales)
    with pytest.raises(nn.StringError, match="divide"):
        ops.group_norm(x, x, 5)
    with pytest.raises(nn.StringError, match="same device"):
        ops.quantize_rows(x[0], q[0], scales[0].cpu())
    with pytest.raises(nn.StringError, match="not on a GPU"):
        ops.group_norm(x.cpu(), x, 4)
    assert nn.peek_last_error() == 0
    check(_norm(x[:1, :50], torch.empty(1, 50, 64, dtype=torch.float16, device="cuda"), 4), ref.group_norm(x[:1, :50], 4))

"""Edges of the 8-bit and normalising operators: numbers of the types' far ends, bits
that may not depend on the kernel, sums of very many terms."""
import pytest
import torch

import block_reference as ref
from katago_amd import nn, ops
from operator_reference import U32, check
from test_gpu_block_operators import TYPES, _backward, _bytes, _forward_statistics, _laid, _linear, _norm, _rand, ids

pytestmark = pytest.mark.gpu

CURVED = [a for a in ops.ACTIVATIONS if a not in ("identity", "relu")]
LARGEST = torch.finfo(torch.float32).max


def _same_bits(a, b):
    kind = torch.int32 if a.dtype == torch.float32 else torch.int16
    return torch.equal(a.contiguous().view(kind), b.contiguous().view(kind))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("act", CURVED)
@pytest.mark.parametrize("b,p", [(3, 49), (2, 9001), (40, 1), (1100, 3)], ids=ids)
def test_slopes_at_the_far_ends(dtype, act, b, p):
    """A channel that a bias of the largest or lowest number saturates has the slope 1 or 0
    that it has from a bias of a thousand on, and is no NaN to its group."""
    c, groups = 24, 3
    x, dy = _rand(b, p, c, dtype=dtype), _rand(b, p, c, dtype=dtype, seed=5)
    stats = _forward_statistics(x, groups)
    results = []
    for size in (1000.0, 1e20, 8.6e37, LARGEST):
        bias = _rand(c, dtype=torch.float32, seed=2)
        bias[0], bias[9], bias[17] = -size, size, -size
        dx, dw, db = torch.empty_like(x), torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
        _backward(x, dy, stats, dx, groups, bias=bias, activation=act, grad_weight=dw, grad_bias=db)
        results.append((dx, dw, db))
        if size == 1000.0:
            for got, want, what in zip(results[0], ref.group_norm_backward(x, dy, stats, groups, None, bias, act), ("x", "weight", "bias")):
                check(got, want, what)
            assert not db[0] and not db[17] and not dw[0]
        for got, want in zip(results[-1], results[0]):
            assert torch.equal(got, want), size


def _nans():
    """NaN of several bits: fp32 arithmetic hands on the bits below the first."""
    return torch.tensor([0x7FC00001, -1, 0x7F800001, 0x7FC000FF, -0x3FFFFE], dtype=torch.int32, device="cuda").view(torch.float32)


@pytest.mark.parametrize("channels", [5, 64, 700, 9000, 40003])
def test_quantize_nan_of_any_bits(channels):
    x = _rand(12, channels, dtype=torch.float32)
    for i, nan in enumerate(_nans()):
        x[2 * i, [0, channels - 1, channels // 2, 1, 3][i]] = nan
    x[8] = _nans()[1]  # memory filled with ones
    q, scales = torch.full((12, channels), 9, dtype=torch.int8, device="cuda"), torch.empty(12, device="cuda")
    ops.quantize_rows(x, q, scales)
    bad = torch.arange(12, device="cuda") % 2 == 0
    bad[10] = False
    assert torch.equal(torch.isnan(scales), bad)
    assert not q[bad].any()
    want, want_scales = ref.quantize(x[~bad])
    assert torch.equal(q[~bad].cpu(), want) and torch.equal(scales[~bad].cpu(), want_scales)


@pytest.mark.parametrize("p,c,groups", [(1, 512, 4), (300, 24, 2), (9001, 40, 5), (2, 70000, 1)], ids=ids)
def test_group_norm_rows_with_nan_of_any_bits(p, c, groups):
    for act in ("identity", "relu", "gelu"):
        for nan in _nans():
            x = _rand(3, p, c, dtype=torch.float32)
            x[1, p - 1, c // groups - 1] = nan
            q, scales = torch.full((3, p, c), 9, dtype=torch.int8, device="cuda"), torch.empty(3, p, device="cuda")
            _norm(x, q, groups, activation=act, out_scales=scales)
            assert bool(torch.isnan(scales[1]).all()) and not torch.isnan(scales[0]).any() and not torch.isnan(scales[2]).any()
            assert not q[1].any(), act


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("m,k,n", [(5, 24592, 40), (40, 16384, 24), (64, 8192, 1000), (70, 8208, 72), (66, 4112, 65), (128, 4096, 1024), (361, 384, 384),
                                   (2000, 1040, 1990), (4000, 2048, 3800)], ids=ids)
def test_linear_int8_bits_of_every_kernel(dtype, m, k, n):
    """The same bits with a workspace, without one, from rows of any alignment and among
    other rows, whatever follows the sum."""
    x, w = _bytes(m, k), _bytes(n, k, seed=1)
    x_apart, w_apart = _laid(x.cpu(), pad=1, shift=1), _laid(w.cpu(), pad=1, shift=1)
    xs, ws = torch.rand(m, device="cuda") / 73, (torch.rand(n, device="cuda") + 0.5) * k ** -0.5 / 73
    far = torch.linspace(-12, 12, n, device="cuda")
    far[::9] *= 10
    res = _rand(m, n, dtype=dtype, seed=3)
    for act in ops.ACTIVATIONS:
        for bias in (None, far):
            for residual in (None, res):
                kw = dict(bias=bias, activation=act)
                new = lambda rows=m: torch.empty(rows, n, dtype=dtype, device="cuda")
                want = _linear(x, xs, w, ws, new(), residual=residual, **kw)
                others = {"no workspace": ops.linear_int8(x, xs, w, ws, new(), residual=residual, **kw),
                          "apart": _linear(x_apart, xs, w_apart, ws, new(), residual=residual, **kw)}
                for rows in (1, 30, 60, 300, 2000):
                    if rows < m:
                        others[rows] = _linear(x[:rows], xs[:rows], w, ws, new(rows), residual=None if residual is None else residual[:rows], **kw)
                for name, got in others.items():
                    assert _same_bits(got, want[:got.shape[0]]), (act, bias is None, residual is None, name)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("p,c", [(1 << 18, 1024), (1 << 18, 8), (200001, 264)], ids=ids)
def test_backward_sums_of_very_many_terms(dtype, p, c):
    """Every position the same, so that roundings of a sum go one way: a sum over them is
    `p` times a position's. In fp32 a thread adds at most 64 of them, and 8 roundings are
    left for what is done with these sums in 64 bits and for the terms' own."""
    depth = 64 + 8
    one, grad = _rand(1, 1, c, dtype=dtype), _rand(1, 1, c, dtype=dtype, seed=1).abs() + 0.25
    x, dy = one.expand(1, p, c), grad.expand(1, p, c)
    w = _rand(c, dtype=torch.float32, seed=2, shift=1.0, scale=0.3)
    stats = _forward_statistics(one, 1)
    dx, dw, db = torch.empty(1, p, c, dtype=dtype, device="cuda"), torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
    _backward(x, dy, stats, dx, 1, weight=w, grad_weight=dw, grad_bias=db)
    want_x, want_w, want_b = ref.group_norm_backward(one, grad, stats, 1, weight=w)
    for got, (y, off), what in ((dw, want_w, "weight"), (db, want_b, "bias")):
        check(got, (p * y, p * (off + (depth - ref.DEPTH) * U32 * y.abs())), what)  # the reference's own depth is taken out
    assert torch.equal(dx, dx[:, :1].expand_as(dx))
    check(dx[:, :1], want_x)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("act", CURVED)
@pytest.mark.parametrize("p", [1, 5, 9000])
def test_slopes(dtype, act, p):
    """A weight of 0 leaves a channel's bias as the activation's argument, and one position
    its slope as the bias's gradient: to within 2^-20 of 1 in fp32, 2^-18 in 16 bits."""
    c = 1024
    grid = torch.cat([torch.linspace(*r, c) for r in ((-100, 100), (-20, 0), (0, 20), (16, 17.5), (16.55, 16.7), (-17.5, -16), (-6, -3), (-1, 1))])
    x, dy = _rand(1, p, c, dtype=dtype), torch.ones(1, p, c, dtype=dtype, device="cuda")
    lengths = torch.ones(1, dtype=torch.int32, device="cuda")
    stats = _forward_statistics(x, 8, lengths=lengths)
    dx, db = torch.empty_like(x), torch.empty(c, device="cuda")
    for bias in grid.split(c):
        _backward(x, dy, stats, dx, 8, weight=torch.zeros(c, device="cuda"), bias=bias.cuda(), activation=act, lengths=lengths, grad_bias=db)
        off = 2.0 ** (-20 if dtype == torch.float32 else -18)
        check(db, (ref.slope(bias.double(), act), torch.full((c,), off, dtype=torch.float64)), act)


def test_statistics_of_no_positions():
    """No position, no deviation: 0 and 0, as of an item whose mask leaves none."""
    for b in (1, 3, 700):
        x = torch.empty(b, 0, 8, dtype=torch.float16, device="cuda")
        around = torch.full((b * 2 * 2 + 3,), 5.0, device="cuda")
        stats = around[1:1 + b * 4].view(b, 2, 2)
        ops.group_norm(x, torch.empty_like(x), 2, stats=stats)
        assert not stats.any() and around[0] == 5 and bool((around[1 + b * 4:] == 5).all())


def test_tangents_are_refused():
    """By every call, and only of tensors that have one."""
    x, f32 = _rand(2, 8, 16, dtype=torch.float32), dict(dtype=torch.float32, device="cuda")
    q, scales = torch.empty(8, 16, dtype=torch.int8, device="cuda"), torch.empty(8, **f32)
    ops.quantize_rows(x[0], q, scales)
    stats = _forward_statistics(x, 4)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda x: ops.linear(x[0], torch.ones(16, 16, **f32), torch.empty(8, 16, **f32)),
                     lambda x: ops.rope_axes(x, torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.ones(1, 8, 1, **f32), torch.empty(2, 8, 16, **f32)),
                     lambda x: ops.cross_attention(*(x[:, :, None],) * 3, torch.empty(2, 8, 1, 16, **f32)),
                     lambda x: ops.quantize_rows(x[0], q, scales),
                     lambda x: ops.linear_int8(q, scales, q, scales, torch.empty(8, 8, **f32), bias=x[0, 0, :8]),
                     lambda x: ops.group_norm(x, torch.empty_like(x), 4),
                     lambda x: ops.group_norm_backward(_rand(2, 8, 16, dtype=torch.float32), x, stats, torch.empty(2, 8, 16, **f32), 4,
                                                       workspace=torch.empty(1 << 16, dtype=torch.uint8, device="cuda"))):
            call(x)
            with pytest.raises(nn.StringError, match="tangent"):
                call(dual)


def test_backward_sums_of_very_many_items():
    """A thread adds at most 64 items' terms in fp32 however many there are (see
    test_backward_sums_of_very_many_terms)."""
    b, c, depth = 1 << 29, 8, 64 + 8
    one, grad = _rand(1, 1, c, seed=3), _rand(1, 1, c, seed=1).abs() + 0.25
    stats = _forward_statistics(one, 1)
    dx, dw, db = torch.empty(b, 1, c, dtype=one.dtype, device="cuda"), torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
    _backward(one.expand(b, 1, c), grad.expand(b, 1, c), stats.expand(b, 1, 2).contiguous(), dx, 1, grad_weight=dw, grad_bias=db)
    want_x, want_w, want_b = ref.group_norm_backward(one, grad, stats, 1)
    assert all(bool((part == dx[:1]).all()) for part in dx.split(1 << 26))
    check(dx[:1], want_x)
    for got, (y, off), what in ((dw, want_w, "weight"), (db, want_b, "bias")):
        check(got, (b * y, b * (off + (depth - ref.DEPTH) * U32 * y.abs())), what)

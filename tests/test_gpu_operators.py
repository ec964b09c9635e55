"""The operators on the caller's tensors against their formulas in 64 bits, at
the sizes, strides and masks where their tiles, tails and softmax can go wrong,
and as a program runs them: together, on its own stream, captured and replayed,
in place, without torch. Bounds: operator_reference.py."""
import math
import threading

import pytest
import torch

import operator_reference as ref
from katago_amd import nn, ops

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16, torch.float32]
ids = lambda v: str(v).replace("torch.", "").replace(" ", "")


def _rand(*shape, dtype=torch.float16, seed=0, scale=1.0, pad=0, shift=0):
    """Normal values whose rows lie pad apart and start shift elements past a
    16-byte border."""
    g = torch.Generator().manual_seed(hash((shape, seed)) % (1 << 31))
    row = shape[-1] + pad
    flat = torch.empty(shift + (torch.Size(shape[:-1]).numel()) * row, dtype=dtype, device="cuda").fill_(float("nan"))
    t = flat[shift:].view(*shape[:-1], row)[..., :shape[-1]]
    t.copy_((torch.randn(*shape, generator=g) * scale).to(dtype))
    return t


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _guarded(*shape, dtype, pad=3, shift=5):
    """An output whose surroundings must stay as they are: (tensor, check)."""
    row = shape[-1] + pad
    n = torch.Size(shape[:-1]).numel()
    flat = torch.full((shift + n * row + 64,), 7.0, dtype=dtype, device="cuda")
    t = flat[shift:shift + n * row].view(*shape[:-1], row)[..., :shape[-1]]

    def untouched():
        rest = flat.clone()
        rest[shift:shift + n * row].view(*shape[:-1], row)[..., :shape[-1]] = 7.0
        assert bool((rest == 7.0).all()), "written outside the output"
    return t, untouched


def _linear(x, w, out, **kw):
    need = ops.linear_workspace(x, w)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
    return ops.linear(x, w, out, workspace=ws, stream=_stream(), **kw)


def _attention(q, k, v, out, **kw):
    need = ops.cross_attention_workspace(q, k, v)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
    return ops.cross_attention(q, k, v, out, workspace=ws, stream=_stream(), **kw)


# -- linear -------------------------------------------------------------------

LINEAR_SIZES = [(1, 1, 1), (1, 384, 1024), (3, 40, 8), (1, 4104, 24), (7, 1000, 72), (16, 256, 64), (17, 264, 40), (31, 8, 33),
                (33, 520, 129), (64, 64, 64), (65, 96, 257), (100, 33, 31), (129, 72, 63), (200, 1032, 136), (300, 17, 520),
                # K split over workgroups, 128- and 256-row tiles, each with ends inside a tile and a step
                (5, 12296, 40), (40, 8192, 24), (70, 4100, 72), (66, 2056, 65), (1900, 136, 1990), (1905, 1032, 6408)]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("m,k,n", LINEAR_SIZES, ids=ids)
def test_linear_sizes(dtype, m, k, n):
    x, w = _rand(m, k, dtype=dtype), _rand(n, k, dtype=dtype, seed=1, scale=k ** -0.5)
    bias, res = _rand(n, dtype=torch.float32, seed=2), _rand(m, n, dtype=dtype, seed=3, pad=1)
    out, untouched = _guarded(m, n, dtype=dtype)
    ref.check(_linear(x, w, out, bias=bias, activation="gelu", residual=res), ref.linear(x, w, bias, "gelu", res))
    untouched()
    plain = torch.empty(m, n, dtype=dtype, device="cuda")
    ref.check(_linear(x, w, plain), ref.linear(x, w))
    assert torch.equal(plain, _linear(x, w, torch.empty_like(plain))), "not the same bits again"


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("pad,shift", [(8, 0), (1, 0), (0, 1), (3, 5), (7, 8)])
@pytest.mark.parametrize("m,k,n", [(5, 72, 40), (70, 200, 96), (1800, 150, 1900)], ids=ids)
def test_linear_strides(dtype, pad, shift, m, k, n):
    x, w = _rand(m, k, dtype=dtype, pad=pad, shift=shift), _rand(n, k, dtype=dtype, seed=1, scale=k ** -0.5, pad=pad, shift=shift)
    out, untouched = _guarded(m, n, dtype=dtype, pad=pad, shift=shift)
    ref.check(_linear(x, w, out), ref.linear(x, w))
    untouched()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("act", ops.ACTIVATIONS)
@pytest.mark.parametrize("m", [2, 80])
def test_linear_activations(dtype, act, m):
    """Values from the far left tail to the far right one."""
    x, w = _rand(m, 64, dtype=dtype, scale=2.0), _rand(96, 64, dtype=dtype, seed=1)
    bias = torch.linspace(-90, 90, 96, device="cuda")
    out = torch.empty(m, 96, dtype=dtype, device="cuda")
    ref.check(_linear(x, w, out, bias=bias, activation=act), ref.linear(x, w, bias, act), act)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("m", [1, 90])
def test_linear_in_place_residual(dtype, m):
    x, w, res = _rand(m, 136, dtype=dtype), _rand(72, 136, dtype=dtype, seed=1, scale=0.1), _rand(m, 72, dtype=dtype, seed=2)
    want = ref.linear(x, w, None, "silu", res)
    ref.check(_linear(x, w, res, activation="silu", residual=res), want)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("m,k,pad", [(3, 80, 0), (90, 80, 0), (90, 80, 1), (90, 75, 0), (3, 75, 3)])
def test_linear_infinities_stay_in_their_rows(dtype, m, k, pad):
    """An infinite or NaN input reaches its own row only, in a whole step of K and
    in what is left behind it."""
    x, w = _rand(m, k, dtype=dtype, pad=pad), _rand(48, k, dtype=dtype, seed=1, pad=pad)
    x[1, 7 if m == 3 else k - 2], x[2, 9] = float("inf"), float("nan")
    out = torch.empty(m, 48, dtype=dtype, device="cuda")
    _linear(x, w, out)
    want = x.double() @ w.double().t()
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(torch.isinf(out), torch.isinf(want))
    assert torch.equal(out[1], want[1].to(dtype))
    keep = [i for i in range(m) if i not in (1, 2)]
    y, bound = ref.linear(x[keep], w)
    ref.check(out[keep], (y, bound))


@pytest.mark.parametrize("m,pad", [(3, 0), (90, 0), (90, 1)])
def test_linear_fp32_range(m, pad):
    """Factors at both ends of fp32: what rounds to infinity in 16 bits, what is
    too small for three pieces of them, each with sums well inside the range."""
    x, w = _rand(m, 64, dtype=torch.float32, pad=pad), _rand(40, 64, dtype=torch.float32, seed=1, pad=pad)
    out = torch.empty(m, 40, dtype=torch.float32, device="cuda")
    x[1], w[:, :] = x[1].sign() * 3.4e38, w * 1e-3
    x[0] *= 1e-20
    ref.check(_linear(x, w * 1e-2, out), ref.linear(x, w * 1e-2))


def test_linear_shared_rows_and_far_offsets():
    """One row for all (stride 0), and rows more than 2^31 elements apart."""
    x, w = _rand(1, 64).expand(5, 64), _rand(32, 64, seed=1)
    out = torch.empty(5, 32, dtype=torch.float16, device="cuda")
    ref.check(_linear(x, w, out), ref.linear(x, w))
    far = torch.empty((1 << 31) + 4096, dtype=torch.float16, device="cuda")
    stride = (1 << 30) + 1024
    x = far.as_strided((3, 64), (stride, 1))
    x.copy_(_rand(3, 64, seed=4))
    ref.check(_linear(x, w, out[:3]), ref.linear(x, w))
    ref.check(_linear(w, x, torch.empty(32, 3, dtype=torch.float16, device="cuda")), ref.linear(w, x))
    y = far.as_strided((3, 32), (stride, 1), 256)
    ref.check(_linear(x, w, y), ref.linear(x, w))


def test_linear_no_rows():
    out = torch.full((0, 8), 3.0, dtype=torch.float16, device="cuda")
    assert ops.linear(torch.empty(0, 16, dtype=torch.float16, device="cuda"), _rand(8, 16), out, stream=_stream()) is out


# -- rope ---------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("layout", ops.ROPE_LAYOUTS)
@pytest.mark.parametrize("tokens,heads,dim,pairs,axes,tables", [
    (1, 1, 2, 1, 1, 1), (1, 6, 64, 32, 2, 6), (5, 4, 33, 16, 3, 2), (3, 6, 62, 27, 4, 1), (100, 3, 96, 48, 3, 3), (7, 32, 128, 64, 2, 1),
    (2, 5, 80, 8, 1, 5), (11, 8, 17, 5, 2, 4), (361, 12, 64, 32, 2, 6)], ids=ids)
def test_rope(dtype, layout, tokens, heads, dim, pairs, axes, tables):
    x = _rand(tokens, heads, dim, dtype=dtype, pad=dim % 3)
    g = torch.Generator().manual_seed(pairs)
    pos = torch.randint(-30, 4000, (tokens, axes), generator=g, dtype=torch.int32).cuda()
    freqs = torch.randn(tables, pairs, axes, generator=g).cuda()
    for inverse in (False, True):
        out, untouched = _guarded(tokens, heads, dim, dtype=dtype)
        ops.rope_axes(x, pos, freqs, out, layout=layout, inverse=inverse, stream=_stream())
        ref.check(out, ref.rope(x, pos, freqs, layout, inverse))
        untouched()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_rope_far_positions(dtype):
    """Angles of up to 2^31 radians, and positions at the ends of their type."""
    x = _rand(4, 2, 32, dtype=dtype)
    pos = torch.tensor([[2 ** 31 - 1, 0], [-2 ** 31, 5], [2 ** 31 - 1, -2 ** 31], [0, 0]], dtype=torch.int32, device="cuda")
    freqs = torch.rand(1, 16, 2, generator=torch.Generator().manual_seed(2)).cuda()
    out = torch.empty_like(x)
    ops.rope_axes(x, pos, freqs, out, stream=_stream())
    ref.check(out, ref.rope(x, pos, freqs))
    assert torch.equal(out[3], x[3])


@pytest.mark.parametrize("layout", ops.ROPE_LAYOUTS)
def test_rope_in_place_in_a_fused_projection(layout):
    """Query and key heads of [Q|K|V] rows, the values beside them untouched."""
    qkv = _rand(50, 9 * 32, dtype=torch.bfloat16)
    before = qkv.clone()
    qk = qkv[:, :6 * 32].unflatten(1, (6, 32))
    pos = torch.randint(0, 19, (50, 2), dtype=torch.int32, device="cuda")
    freqs = torch.rand(3, 16, 2, device="cuda")
    want = ref.rope(qk, pos, freqs, layout)
    ops.rope_axes(qk, pos, freqs, qk, layout=layout, stream=_stream())
    ref.check(qk, want)
    assert torch.equal(qkv[:, 6 * 32:], before[:, 6 * 32:])


@pytest.mark.parametrize("dtype,layout,tokens,heads,dim,pairs,axes,in_place", [
    (torch.float16, "halves", 35001, 5, 55, 27, 4, True), (torch.bfloat16, "interleaved", 21003, 7, 120, 60, 2, False),
    (torch.float32, "interleaved", 20002, 3, 70, 33, 1, True), (torch.float16, "interleaved", 150001, 1, 64, 29, 3, True),
    (torch.float32, "halves", 41001, 4, 48, 23, 2, False)])
def test_rope_runs_of_tokens(dtype, layout, tokens, heads, dim, pairs, axes, in_place):
    """Every head a table of its own, and tokens enough for runs of them."""
    x = _rand(tokens, heads, dim, dtype=dtype, pad=1)
    g = torch.Generator().manual_seed(pairs)
    pos = torch.randint(-30, 4000, (tokens, axes), generator=g, dtype=torch.int32).cuda()
    freqs = torch.randn(heads, pairs, axes, generator=g).cuda()
    want = ref.rope(x, pos, freqs, layout)
    if in_place:
        flat = x.as_strided((tokens * heads, dim + 1), (dim + 1, 1), x.storage_offset())[:, dim:]
        ops.rope_axes(x, pos, freqs, x, layout=layout, stream=_stream())
        ref.check(x, want)
        assert bool(torch.isnan(flat).all())
        return
    out, untouched = _guarded(tokens, heads, dim, dtype=dtype)
    ops.rope_axes(x, pos, freqs, out, layout=layout, stream=_stream())
    ref.check(out, want)
    untouched()


def test_rope_far_offsets_and_head_major():
    far = torch.empty((1 << 31) + 4096, dtype=torch.float16, device="cuda")
    x = far.as_strided((3, 2, 32), ((1 << 30) + 512, 40, 1))
    x.copy_(_rand(3, 2, 32))
    pos, freqs = torch.arange(6, dtype=torch.int32, device="cuda").view(3, 2), torch.rand(1, 16, 2, device="cuda")
    out = torch.empty(2, 3, 32, dtype=torch.float16, device="cuda").transpose(0, 1)  # tokens inside heads
    want = ref.rope(x, pos, freqs)
    ops.rope_axes(x, pos, freqs, out, stream=_stream())
    ref.check(out, want)
    ops.rope_axes(x, pos, freqs, x, stream=_stream())
    ref.check(x, want)
    ops.rope_axes(x[:0], pos[:0], freqs, out[:0], stream=_stream())


def test_rope_is_the_boards_rotary_embedding():
    """The trunk's fixed rotary embedding (first half of the pairs by one axis,
    second half by the other, theta 100) at a board's positions."""
    pairs, side = 16, 9
    f = 100.0 ** (-torch.arange(pairs // 2) / (pairs // 2))
    freqs = torch.zeros(1, pairs, 2)
    freqs[0, :pairs // 2, 0], freqs[0, pairs // 2:, 1] = f, f
    at = torch.arange(side * side)
    pos = torch.stack((at % side, at // side), 1)
    x = _rand(side * side, 2, 2 * pairs, dtype=torch.float32)
    out = torch.empty_like(x)
    ops.rope_axes(x, pos.int().cuda(), freqs.cuda(), out, stream=_stream())
    ref.check(out, ref.rope(x, pos, freqs))


# -- attention ----------------------------------------------------------------

ATTENTION_SIZES = [  # batch, queries, keys, heads, kv heads, dq, dv
    (1, 1, 1, 1, 1, 1, 1), (1, 1, 361, 6, 6, 64, 64), (2, 3, 31, 4, 4, 32, 32), (1, 5, 32, 8, 2, 64, 64), (2, 7, 33, 4, 1, 48, 80),
    (1, 1, 63, 32, 8, 128, 128), (3, 2, 64, 4, 4, 80, 80), (1, 130, 65, 2, 2, 64, 64), (1, 33, 200, 6, 3, 32, 16), (2, 129, 129, 2, 1, 128, 128),
    (1, 40, 127, 3, 3, 13, 37), (2, 1, 1000, 8, 8, 96, 64), (1, 260, 300, 4, 2, 64, 128), (4, 1, 5000, 4, 1, 128, 128), (1, 9, 0, 2, 2, 64, 64),
    (1, 17, 3000, 2, 2, 64, 64)]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("size", ATTENTION_SIZES, ids=ids)
def test_attention_sizes(dtype, size):
    b, lq, lk, h, kv, dq, dv = size
    q, k, v = _rand(b, lq, h, dq, dtype=dtype, scale=1.5), _rand(b, lk, kv, dq, dtype=dtype, seed=1, scale=1.5), _rand(b, lk, kv, dv, dtype=dtype, seed=2)
    out, untouched = _guarded(b, lq, h, dv, dtype=dtype)
    ref.check(_attention(q, k, v, out), ref.attention(q, k, v))
    untouched()
    alone = ops.cross_attention(q, k, v, torch.empty_like(out), stream=_stream())  # no workspace: no split
    ref.check(alone, ref.attention(q, k, v))
    assert torch.equal(out, _attention(q, k, v, torch.empty_like(out))), "not the same bits again"


def _masks(kind, b, lk, g):
    lengths = mask = None
    if kind in ("lengths", "both"):
        lengths = torch.tensor([[0, lk, 1, lk // 2, lk + 9, -3][i % 6] for i in range(b)], dtype=torch.int32, device="cuda")
    if kind in ("mask", "both", "bool"):
        mask = (torch.rand(b, lk + 3, generator=g) < 0.4).to(torch.bool if kind == "bool" else torch.uint8).cuda()[:, :lk]
        mask[1, :] = False  # a row without a key
        mask[0, :lk - 1] = False  # only the last key
        if kind != "bool":
            mask[2] *= 255  # anything but 0 takes part
    return lengths, mask


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("kind", ["lengths", "mask", "both", "bool"])
@pytest.mark.parametrize("lq,lk,h,kv,d", [(1, 200, 4, 2, 64), (1, 4100, 8, 1, 128), (70, 130, 2, 2, 32), (150, 260, 4, 1, 128), (3, 70, 2, 1, 37)], ids=ids)
def test_attention_masks(dtype, kind, lq, lk, h, kv, d):
    """Masks that leave rows empty or one key; what masked keys hold (NaN,
    infinities, the type's lowest value) does not matter."""
    g = torch.Generator().manual_seed(lk)
    b = 6
    q, k, v = _rand(b, lq, h, d, dtype=dtype), _rand(b, lk, kv, d, dtype=dtype, seed=1), _rand(b, lk, kv, d, dtype=dtype, seed=2)
    lengths, mask = _masks(kind, b, lk, g)
    on = torch.ones(b, lk, dtype=torch.bool, device="cuda")
    if lengths is not None:
        on &= torch.arange(lk, device="cuda") < lengths[:, None]
    if mask is not None:
        on &= mask != 0
    want = ref.attention(q, k, v, lengths=lengths, mask=mask)
    for fill_k, fill_v in ((float("nan"), float("inf")), (torch.finfo(dtype).min, float("nan")), (float("inf"), float("-inf"))):
        k.masked_fill_(~on[:, :, None, None], fill_k)
        v.masked_fill_(~on[:, :, None, None], fill_v)
        out, untouched = _guarded(b, lq, h, d, dtype=dtype)
        ref.check(_attention(q, k, v, out, key_lengths=lengths, key_mask=mask), want, kind)
        untouched()
        assert not out[~on.any(1)].any()
        ref.check(ops.cross_attention(q, k, v, torch.empty_like(out), key_lengths=lengths, key_mask=mask, stream=_stream()), want, kind)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("pad,shift", [(8, 0), (1, 0), (0, 1), (3, 5), (64, 8)])
@pytest.mark.parametrize("lq,d", [(1, 64), (1, 128), (40, 64), (150, 128)])
def test_attention_strides(dtype, pad, shift, lq, d):
    """Heads inside tokens with gaps and shifts, and heads outside tokens."""
    q, k, v = (_rand(2, n, 4, d, dtype=dtype, seed=i, pad=pad, shift=shift) for i, n in enumerate((lq, 90, 90)))
    out, untouched = _guarded(2, lq, 4, d, dtype=dtype, pad=pad, shift=shift)
    want = ref.attention(q, k, v, scale=0.3)
    ref.check(_attention(q, k, v, out, scale=0.3), want)
    untouched()
    turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    out = torch.empty(2, 4, lq, d, dtype=dtype, device="cuda").transpose(1, 2)
    ref.check(_attention(*turned, out, scale=0.3), want)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("lq,lk", [(1, 700), (64, 200)])
def test_attention_scores_that_grow(dtype, lq, lk):
    """Scores of up to hundreds, growing and falling along the keys: the softmax's
    reference point moves, and the last or first key decides."""
    for ramp in (torch.linspace(-1, 1, lk), torch.linspace(1, -1, lk)):
        q = torch.full((1, lq, 2, 32), 4.0, dtype=dtype, device="cuda")
        k = (ramp[None, :, None, None] * 5).expand(1, lk, 2, 32).to(dtype).cuda()
        v = _rand(1, lk, 2, 32, dtype=dtype)
        ref.check(_attention(q, k, v, torch.empty_like(q), scale=1.0), ref.attention(q, k, v, scale=1.0))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("lq", [1, 50])
def test_attention_non_finite_keys_that_take_part(dtype, lq):
    """A NaN key or an infinite score makes its item's rows NaN and no other's;
    a row of scores of minus infinity is zeros."""
    q, k, v = (_rand(4, n, 2, 64, dtype=dtype, seed=i) for i, n in enumerate((lq, 75, 75)))
    q[1:3].abs_()
    k[0, 40, 1, 3] = float("nan")
    k[1, 70, 0] = float("inf")
    k[2] = float("-inf")
    want = ref.attention(q[3:], k[3:], v[3:])
    out = _attention(q, k, v, torch.empty_like(q))
    assert out[0, :, 1].isnan().all() and not out[0, :, 0].isnan().any()
    assert out[1, :, 0].isnan().all() and not out[1, :, 1].isnan().any()
    assert not out[2].any()
    ref.check(out[3:], want)


@pytest.mark.parametrize("b,lq,lk,d,kind", [(90, 40, 70, 64, "none"), (90, 40, 700, 33, "mask"), (44, 130, 97, 32, "lengths"), (44, 129, 33, 20, "none"),
                                            (90, 33, 31, 64, "lengths")])
def test_attention_fp32_of_more_workgroups_than_cus(b, lq, lk, d, kind):
    q, k, v = (_rand(b, n, 3, d, dtype=torch.float32, seed=s, scale=1.5) for n, s in ((lq, 1), (lk, 2), (lk, 3)))
    lengths = mask = None
    if kind == "lengths":
        lengths = (torch.arange(b, dtype=torch.int32, device="cuda") * 7) % (lk + 1)
    if kind == "mask":
        mask = torch.rand(b, lk, device="cuda", generator=torch.Generator("cuda").manual_seed(4)) < 0.5
        mask[1] = False
        mask[2, 64:640] = False
    out = torch.empty_like(q)
    _attention(q, k, v, out, key_lengths=lengths, key_mask=mask)
    ref.check(out, ref.attention(q, k, v, lengths=lengths, mask=mask))


@pytest.mark.parametrize("b,lq,lk,h,d", [(2, 130, 290, 3, 64), (33, 33, 400, 2, 20), (33, 40, 384, 2, 74)])
def test_attention_fp32_keys_split_over_workgroups(b, lq, lk, h, d):
    """Some streams end before the second split's keys, one has none."""
    q, k, v = (_rand(b, n, h, d, dtype=torch.float32, seed=s, scale=1.5, pad=s) for n, s in ((lq, 1), (lk, 2), (lk, 3)))
    lengths = (torch.arange(b, dtype=torch.int32, device="cuda") * 57 + 200) % (lk + 1)
    lengths[-1] = 0
    k[0, int(lengths[0]):] = float("nan")
    v[0, int(lengths[0]):] = float("inf")
    out, untouched = _guarded(b, lq, h, d, dtype=torch.float32)
    assert ops.cross_attention_workspace(q, k, v) > 0
    _attention(q, k, v, out, key_lengths=lengths)
    ref.check(out, ref.attention(q, k, v, lengths=lengths))
    untouched()


@pytest.mark.parametrize("lq", [1, 40, 300])
def test_attention_many_keys_of_little_weight(lq):
    """One key with nearly all of the weight and a value of 0, and 1999 with 2^-24.5
    of its weight each and values of 1: below fp16's smallest numbers, were the
    largest p 1. It is at least 2^7, so a p is off by half of fp16's smallest number
    over 2^7, besides its own rounding; the scores are exact but for the float that
    the product with the scale gives (2^-23 of 24.5)."""
    q, k, v = torch.zeros(1, lq, 2, 64), torch.zeros(1, 2000, 2, 64), torch.ones(1, 2000, 2, 64)
    q[..., 0] = 1.0
    k[:, 700, :, 0] = 16.984375
    v[:, 700] = 0.0
    q, k, v = (t.half().cuda() for t in (q, k, v))
    out = torch.empty_like(q)
    for workspace in (False, True):
        space = torch.empty(ops.cross_attention_workspace(q, k, v) * workspace, dtype=torch.uint8, device="cuda")
        ops.cross_attention(q, k, v, out, scale=1.0, workspace=space if len(space) else None, stream=_stream())
        want = 1999.0 / (1999.0 + math.exp(16.984375))
        bound = 2000 * 2.0 ** -32 + want * (2.0 ** -11 + 2.0 ** -17) + 2.0 ** -25
        assert (out.double() - want).abs().max().item() <= bound


def test_attention_far_offsets():
    """Keys and values more than 2^31 elements from their base."""
    far = torch.empty((1 << 31) + (1 << 16), dtype=torch.float16, device="cuda")
    q = _rand(2, 3, 2, 64)
    k = far.as_strided((2, 70, 1, 64), ((1 << 31) - 4096, 128, 64, 1))
    v = far.as_strided((2, 70, 1, 64), ((1 << 31) - 4096, 128, 64, 1), 64)
    k.copy_(_rand(2, 70, 1, 64, seed=1))
    v.copy_(_rand(2, 70, 1, 64, seed=2))
    ref.check(_attention(q, k, v, torch.empty_like(q)), ref.attention(q, k, v))
    tokens = far.as_strided((1, 3, 1, 64), (0, (1 << 30) + 64, 64, 1))
    tokens.copy_(_rand(1, 3, 1, 64, seed=3))
    ref.check(_attention(q[:1], tokens, tokens, torch.empty_like(q[:1])), ref.attention(q[:1], tokens, tokens))


def test_attention_no_queries():
    e = lambda *s: torch.empty(*s, dtype=torch.float16, device="cuda")
    ops.cross_attention(e(2, 0, 4, 64), e(2, 9, 4, 64), e(2, 9, 4, 64), e(2, 0, 4, 64), stream=_stream())
    ops.cross_attention(e(0, 3, 4, 64), e(0, 9, 4, 64), e(0, 9, 4, 64), e(0, 3, 4, 64), stream=_stream())


# -- together, and as a program calls them ------------------------------------

class Block:
    """A cross-attending block with a feed-forward layer: boards' positions
    attend to an encoder's states."""

    def __init__(self, dtype, boards=3, side=9, states=50, width=64, heads=4, kv=2, d=16):
        t = dict(dtype=dtype)
        self.b, self.l, self.s, self.h, self.kv, self.d = boards, side * side, states, heads, kv, d
        self.x, self.enc = _rand(boards * self.l, width, **t), _rand(boards * states, width, seed=1, **t)
        self.w = {n: _rand(o, i, seed=j, scale=i ** -0.5, **t) for j, (n, o, i) in enumerate(
            (("q", heads * d, width), ("kv", 2 * kv * d, width), ("o", width, heads * d), ("up", 2 * width, width), ("down", width, 2 * width)))}
        self.bias = _rand(2 * width, dtype=torch.float32, seed=9)
        at = torch.arange(self.l)
        self.pos = torch.stack((at % side, at // side), 1).repeat(boards, 1).int().cuda()
        self.enc_pos = torch.arange(states).repeat(boards)[:, None].expand(-1, 2).int().contiguous().cuda()
        self.freqs = _rand(kv, d // 2, 2, dtype=torch.float32, seed=5, scale=0.3)
        self.lengths = torch.tensor([states, 0, 17], dtype=torch.int32, device="cuda")[:boards]
        e = lambda *s: torch.empty(*s, dtype=dtype, device="cuda")
        self.q, self.kvs, self.a = e(boards * self.l, heads * d), e(boards * states, 2 * kv * d), e(boards * self.l, heads * d)
        self.y, self.up, self.out = torch.empty_like(self.x), e(boards * self.l, 2 * width), torch.empty_like(self.x)
        q, k = self.q.view(boards, self.l, heads, d), self.kvs[:, :kv * d].view(boards, states, kv, d)
        n = max(ops.cross_attention_workspace(q, k, k), ops.linear_workspace(self.x, self.w["up"]), ops.linear_workspace(self.up, self.w["down"]), 16)
        self.ws = torch.empty(n, dtype=torch.uint8, device="cuda")

    def run(self, stream):
        k = self.kvs[:, :self.kv * self.d].unflatten(1, (self.kv, self.d))
        v = self.kvs[:, self.kv * self.d:].unflatten(1, (self.kv, self.d))
        q = self.q.view(-1, self.h, self.d)
        run = dict(workspace=self.ws, stream=stream)
        ops.linear(self.x, self.w["q"], self.q, **run)
        ops.linear(self.enc, self.w["kv"], self.kvs, **run)
        ops.rope_axes(q, self.pos, self.freqs, q, stream=stream)
        ops.rope_axes(k, self.enc_pos, self.freqs, k, stream=stream)
        ops.cross_attention(q.view(self.b, self.l, self.h, self.d), k.unflatten(0, (self.b, self.s)), v.unflatten(0, (self.b, self.s)),
                            self.a.view(self.b, self.l, self.h, self.d), key_lengths=self.lengths, **run)
        ops.linear(self.a, self.w["o"], self.y, residual=self.x, **run)
        ops.linear(self.y, self.w["up"], self.up, bias=self.bias, activation="gelu", **run)
        return ops.linear(self.up, self.w["down"], self.out, residual=self.y, **run)

    def want(self):
        w = {n: t.double().cpu() for n, t in self.w.items()}
        x, enc = self.x.double().cpu(), self.enc.double().cpu()
        q, _ = ref.rope((x @ w["q"].t()).view(-1, self.h, self.d), self.pos, self.freqs)
        k, v = (enc @ w["kv"].t()).view(-1, 2, self.kv, self.d).unbind(1)
        k, _ = ref.rope(k, self.enc_pos, self.freqs)
        a, _ = ref.attention(q.view(self.b, self.l, self.h, self.d), *(t.reshape(self.b, self.s, self.kv, self.d) for t in (k, v)), lengths=self.lengths)
        y = a.view(x.shape[0], -1) @ w["o"].t() + x
        return ref.activate(y @ w["up"].t() + self.bias.double().cpu(), "gelu") @ w["down"].t() + y


# Off by half a step each: the projections, q and k turned, p and the attention,
# the output projection, the two layers: eight roundings, no one of which the
# later steps make more than twice as large against the residual stream.
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_block(dtype):
    block = Block(dtype)
    got, want = block.run(_stream()).double().cpu(), block.want()
    assert (got - want).norm() <= 16 * ref.HALF_STEP[dtype] * want.norm()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=ids)
def test_captured_and_replayed(dtype):
    """A captured block replays to the eager bits, with other work between the
    replays, and follows inputs and lengths that change in place."""
    block = Block(dtype)
    stream = torch.cuda.Stream()
    block.run(_stream())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        block.run(_stream())
    for i in range(4):
        block.x.copy_(_rand(*block.x.shape, dtype=dtype, seed=20 + i))
        block.lengths.copy_(torch.tensor([(5 * i) % 50, 50, i], dtype=torch.int32))
        block.out.fill_(0)
        graph.replay()
        torch.cuda.synchronize()
        replayed = block.out.clone()
        assert torch.equal(block.run(_stream()), replayed), i
        torch.cuda.synchronize()


def test_other_stream_and_null_stream():
    block = Block(torch.float16)
    want = block.run(None).clone()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    block.out.zero_()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = block.run(s.cuda_stream).clone()
    s.synchronize()
    assert torch.equal(got, want)


def test_two_threads_at_once():
    """Calls from two threads on streams and workspaces of their own."""
    blocks = [Block(torch.bfloat16, boards=1 + i) for i in range(2)]
    want = [b.run(None).clone() for b in blocks]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        s = torch.cuda.Stream()
        for _ in range(20):
            blocks[i].out.zero_()
            torch.cuda.current_stream().synchronize()
            blocks[i].run(s.cuda_stream)
            s.synchronize()
            if not torch.equal(blocks[i].out, want[i]):
                bad.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_without_torch_tensors():
    """DeviceTensor views of the library's own buffers."""
    import numpy as np
    rng = np.random.default_rng(0)
    x, w = rng.standard_normal((5, 24)).astype(np.float32), rng.standard_normal((7, 24)).astype(np.float32)
    bx, bw, bo = nn.DeviceBuffer.from_array(x), nn.DeviceBuffer.from_array(w), nn.DeviceBuffer(5 * 7 * 4)
    ops.linear(ops.DeviceTensor(bx.ptr, x.shape, "float32"), ops.DeviceTensor(bw.ptr, w.shape, "float32"),
               ops.DeviceTensor(bo.ptr, (5, 7), "float32"))
    torch.cuda.synchronize()
    ref.check(torch.from_numpy(bo.to_array(np.float32, (5, 7))), ref.linear(torch.from_numpy(x), torch.from_numpy(w)))


def test_refusals_leave_no_error_behind():
    x, w, out = _rand(4, 16), _rand(8, 16), torch.empty(4, 8, dtype=torch.float16, device="cuda")
    with pytest.raises(nn.StringError, match="same device"):
        ops.linear(x, w.cpu(), out)
    with pytest.raises(nn.StringError, match="not on a GPU"):
        ops.linear(x.cpu(), w, out)
    p, _ = ops._linear_params(x, w, out, None, None, None, None)
    assert ops._library().kgh_linear(99, p, None) == 1 and b"no device 99" in nn.hip_library().kgh_last_error()
    assert nn.peek_last_error() == 0
    ref.check(_linear(x, w, out), ref.linear(x, w))


# -- scores, values and masks at the ends of their ranges ---------------------

@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("scale", [1.0, 64.0, 1e22, 1e30], ids=ids)
@pytest.mark.parametrize("lq,lk,d", [(3, 200, 64), (2, 2100, 128), (40, 300, 64), (40, 1100, 32), (512, 130, 64), (512, 70, 128)], ids=ids)
def test_attention_large_scores(dtype, scale, lq, lk, d):
    """Scores of 2^27 to 2^28 in magnitude, times scales of up to the largest one:
    a row's largest has its whole weight whatever its size. The scores are fp32
    numbers (a row's factor of seven bits times 2^21, and multiples of 16 beside
    it), so only exponents have errors: 2^-23 of one, which for 16 (the next score
    below the largest, at scale 1) is less than 2^-18 of a weight of e^-16."""
    g = torch.Generator().manual_seed(lk)
    row = torch.randint(0, 64, (lq,), generator=g).double()
    low = torch.randint(-2, 1, (lk,), generator=g).double() * 16
    for sign in (1.0, -1.0):
        for part in (torch.arange(lk) * 4 // lk, 3 - torch.arange(lk) * 4 // lk):  # quarters of the keys that rise or fall
            q, k = torch.zeros(2, lq, 2, d, dtype=torch.float64), torch.zeros(2, lk, 2, d, dtype=torch.float64)
            q[..., 0], q[..., 1] = ((64 + row) * 2.0 ** 6)[:, None], 1.0
            k[..., 0], k[..., 1] = (sign * 2.0 ** 15 * torch.tensor([0.25, 0.5, 0.75, 1.0], dtype=torch.float64)[part])[:, None], low[:, None]
            q, k = (t.to(dtype).cuda() for t in (q, k))
            v = _rand(2, lk, 2, d, dtype=dtype, seed=3)
            qd, kd, vd = (t.double().cpu().transpose(1, 2) for t in (q, k, v))
            score = qd @ kd.transpose(2, 3).contiguous()
            assert torch.equal(score, score.float().double())
            p = torch.softmax(scale * score, -1)
            want = (p @ vd).transpose(1, 2)
            off = (ref.HALF_STEP[dtype] + 2.0 ** -18 + 2 * (lk + 4) * ref.U32) * (p @ vd.abs()).transpose(1, 2)
            bound = off + ref.HALF_STEP[dtype] * (want.abs() + off) + 2 * ref.SMALLEST[dtype]
            ref.check(_attention(q, k, v, torch.empty_like(q), scale=scale), (want, bound), (sign, part[0]))
            ref.check(ops.cross_attention(q, k, v, torch.empty_like(q), scale=scale, stream=_stream()), (want, bound), (sign, part[0]))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("value", ["inf", "-inf", "nan"])
@pytest.mark.parametrize("lq,lk,d", [(1, 75, 64), (2, 1030, 32), (50, 75, 64), (40, 1100, 128), (600, 70, 64), (768, 40, 128)], ids=ids)
def test_attention_scores_of_minus_infinity_are_zeros_whatever_the_values(dtype, value, lq, lk, d):
    """By every kernel, with a split of the keys and without one."""
    q, k, v = (_rand(3, n, 2, d, dtype=dtype, seed=i) for i, n in enumerate((lq, lk, lk)))
    want = ref.attention(q[::2], k[::2], v[::2])
    q[1].abs_()
    k[1], v[1] = float("-inf"), float(value)
    for run in (_attention, lambda *t: ops.cross_attention(*t, stream=_stream())):
        out = torch.full_like(q, 3.0)
        run(q, k, v, out)
        assert not out[1].any()
        ref.check(out[::2], want)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("lq,lk,h,kv,d", [(1, 75, 2, 2, 64), (3, 33, 8, 1, 31), (2, 1030, 2, 1, 128), (1, 700, 4, 4, 32), (50, 75, 2, 2, 64),
                                          (40, 1100, 2, 2, 128), (600, 70, 2, 2, 64)], ids=ids)
def test_attention_infinite_values_that_take_part(dtype, lq, lk, h, kv, d):
    """An infinite value makes its dim of its head's rows infinite, two of other
    signs or a NaN make it NaN; other dims and heads are what they are."""
    q, k, v = (_rand(2, n, m, d, dtype=dtype, seed=i) for i, (n, m) in enumerate(((lq, h), (lk, kv), (lk, kv))))
    clean = ref.attention(q, k, v)
    v[0, 9, 0, 3], v[0, lk - 2, 0, 7], v[0, 5, 0, 8], v[0, 6, 0, 8], v[0, 30, 0, d - 1] = (float(x) for x in ("inf", "-inf", "inf", "-inf", "nan"))
    g = h // kv
    for run in (_attention, lambda *t: ops.cross_attention(*t, stream=_stream())):
        out = run(q, k, v, torch.empty_like(q))
        assert bool((out[0, :, :g, 3] == float("inf")).all()) and bool((out[0, :, :g, 7] == float("-inf")).all())
        assert bool(out[0, :, :g, [8, d - 1]].isnan().all())
        out, want = out.double().cpu(), clean[0].clone()
        dims = [3, 7, 8, d - 1]
        assert bool(out[0, :, g:].isfinite().all()) and bool(out[1].isfinite().all())
        for t in (out, want):
            t[0, :, :g, dims] = 0.0
        ref.check(out, (want, clean[1]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=ids)
@pytest.mark.parametrize("lq,h,kv,d,workspace", [(1, 2, 2, 64, False), (2, 8, 4, 128, True), (40, 2, 2, 64, False), (512, 4, 2, 128, False), (40, 2, 2, 32, True)],
                         ids=ids)
def test_attention_values_near_the_end_of_the_range(dtype, lq, h, kv, d, workspace):
    """Values of the largest float divided by twice the number of keys, and scores
    that grow by 5.4 (2^7.8 in weight) half way. Exponents are off by less than
    2^-18, p by half a step, its sums by lk * 2^-24."""
    lk = 1024 if workspace else 256
    q, k, v = torch.zeros(1, lq, h, d), torch.zeros(1, lk, kv, d), torch.full((1, lk, kv, d), 2.0 ** 127 / lk)
    q[..., 0] = 1.0
    k[:, lk // 2:, :, 0] = 5.375
    q, k, v = (t.to(dtype).cuda() for t in (q, k, v))
    out = torch.empty_like(q)
    (_attention if workspace else lambda *t, **s: ops.cross_attention(*t, stream=_stream(), **s))(q, k, v, out, scale=1.0)
    off = ref.HALF_STEP[dtype] + 2.0 ** -18 + 2 * (lk + 4) * ref.U32
    want = torch.full(q.shape, 2.0 ** 127 / lk, dtype=torch.float64)
    ref.check(out, (want, want * (off + ref.HALF_STEP[dtype] * (1 + off))))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("act", ops.ACTIVATIONS)
@pytest.mark.parametrize("m,k,pad", [(4, 80, 0), (8, 12296, 0), (90, 80, 0), (70, 4104, 0), (90, 80, 1), (1800, 72, 0), (1800, 72, 1)], ids=ids)
def test_linear_not_finite_through_activations(dtype, act, m, k, pad):
    """A NaN input makes its row NaN whatever the activation, infinite ones what
    the activation of an infinity is; 1800 rows by 1800 columns are large tiles,
    long rows are split over workgroups."""
    n = 1800 if m == 1800 else 40
    x, w = _rand(m, k, dtype=dtype, pad=pad), _rand(n, k, dtype=dtype, seed=1, scale=k ** -0.5, pad=pad)
    x[1, k - 2], x[2, 9], x[3] = float("inf"), float("nan"), float("nan")
    bias = torch.zeros(n, device="cuda")
    bias[5] = float("nan")
    out = torch.empty(m, n, dtype=dtype, device="cuda")
    _linear(x, w, out, bias=bias, activation=act)
    z = x[:4].double().cpu() @ w.double().cpu().t() + bias.double().cpu()
    want = ref.activate(z, act)
    assert bool(out[2:4].isnan().all()) and bool(out[:, 5].isnan().all())
    assert torch.equal(out[:2].double().cpu().isnan(), want[:2].isnan())
    assert torch.equal(out[1].double().cpu().nan_to_num(7.0, 9.0, -9.0), want[1].nan_to_num(7.0, 9.0, -9.0))
    rest = torch.tensor([0] + list(range(4, min(m, 40))))
    keep = torch.arange(n) != 5
    y, bound = ref.linear(x[rest], w, bias, act)
    ref.check(out[rest][:, keep], (y[:, keep], bound[:, keep]), act)


def _every_value(dtype):
    """Every finite number of a type in 16 bits; of fp32 the tails finely, and
    numbers of all sizes."""
    if dtype == torch.float32:
        sizes = torch.logspace(-25, 38, 4000, dtype=torch.float64)
        return torch.cat((torch.linspace(-100, 30, 24000, dtype=torch.float64), sizes, -sizes)).float()
    every = torch.arange(-(1 << 15), 1 << 15, dtype=torch.int32).to(torch.int16).view(dtype)
    return every[every.isfinite()]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("act", ops.ACTIVATIONS)
@pytest.mark.parametrize("kernel", ["few rows", "split", "aligned tiles", "any tiles"])
def test_linear_activations_of_every_value(dtype, act, kernel):
    """Values as they are (products with 1) through the activation, right relative
    to the result down to the type's smallest normal numbers: 2^-15 in 16 bits,
    2^-18 in fp32, and a rounding to the type. Fp32 tiles split a value into pieces
    that are off by 2^-26 of it at most, which a result in a tail follows by |z|
    times as much."""
    z = _every_value(dtype)
    form = 0.0 if act in ("identity", "relu") else 2.0 ** -18 if dtype == torch.float32 else 2.0 ** -15
    if kernel in ("few rows", "split"):
        if kernel == "split":
            z = z[::32]
        w = torch.zeros(len(z), 6144 if kernel == "split" else 8, dtype=dtype)
        w[:, 3] = z
        x = torch.zeros(2, w.shape[1], dtype=dtype)
        x[:, 3] = 1.0
        out = torch.empty(2, len(z), dtype=dtype, device="cuda")
        got = _linear(x.cuda(), w.cuda(), out, activation=act)
        assert ops.linear_workspace(x.cuda(), w.cuda()) == 0 or kernel == "split"
        assert torch.equal(got[0], got[1])
        got = got[0]
    else:
        x = torch.zeros(len(z), 8 if kernel == "aligned tiles" else 1, dtype=dtype)
        x[:, 0] = z
        w = torch.zeros(9, x.shape[1], dtype=dtype)
        w[:, 0] = 1.0
        got = _linear(x.cuda(), w.cuda(), torch.empty(len(z), 9, dtype=dtype, device="cuda"), activation=act)
        assert bool((got == got[:, :1]).all())
        got = got[:, 0]
        if dtype == torch.float32:
            form = form + 2.0 ** -26 * (1 + z.double().abs().clamp_max(110))
    y = ref.activate(z.double(), act)
    smallest = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
    ref.check(got, (y, y.abs() * (form + ref.HALF_STEP[dtype] * (1 + form)) + smallest), act)


@pytest.mark.parametrize("m,n,pad", [(3, 40, 0), (90, 40, 0), (90, 40, 1), (1800, 1900, 0), (1800, 1900, 1)])
@pytest.mark.parametrize("at", [-101, -113, -119, -125])
def test_linear_fp32_small_numbers(m, n, pad, at):
    """Small normal numbers against large ones on the other side, in a whole step
    and in what is left of K, and in one of the two beside ordinary numbers: their
    sums are as right as any."""
    k = 44
    for swap in (False, True):
        for part in (slice(0, k), slice(0, 20), slice(36, k)):
            x, w = _rand(m, k, dtype=torch.float32, pad=pad), _rand(n, k, dtype=torch.float32, seed=1, pad=pad)
            a, b = (w, x) if swap else (x, w)
            a[:, part] = (a[:, part].sign() + a[:, part].clamp(-0.99, 0.99) / 2) * 2.0 ** at
            b[:, part] *= 2.0 ** -at
            a[:, 5], a[:, 40] = 0.0, 0.0
            ref.check(_linear(x, w, torch.empty(m, n, device="cuda")), ref.linear(x, w))


@pytest.mark.parametrize("m,n,pad", [(3, 40, 0), (90, 40, 0), (90, 40, 1), (1800, 1900, 0), (1800, 1900, 1)])
def test_linear_fp32_infinities_times_anything(m, n, pad):
    """An infinity times an infinity or a number of any size is an infinity of the
    product's sign, times 0 NaN."""
    x, w = _rand(m, 70, dtype=torch.float32, pad=pad).abs_(), _rand(n, 70, dtype=torch.float32, seed=1, pad=pad).abs_()
    for row, (at, a, b) in enumerate(((3, "inf", "inf"), (40, "inf", "-inf"), (68, "-inf", "1e-38"))):
        x[row, at] = float(a)
        w[row, at] = float(b)
    w[10, 40] = 0.0
    out = _linear(x, w, torch.empty(m, n, device="cuda")).cpu()
    want = x.double().cpu() @ w.double().cpu().t()
    special = ~want.isfinite()
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out[special].nan_to_num(7.0), want[special].float().nan_to_num(7.0))
    assert bool(out[~special].isfinite().all())


@pytest.mark.parametrize("m,n,pad", [(3, 40, 0), (90, 40, 0), (90, 40, 1), (1800, 1900, 0), (1800, 1900, 1)])
def test_linear_fp32_sums_near_the_largest(m, n, pad):
    """Sums of up to the largest float, whose parts are finite: no infinity before
    that, and one behind it."""
    most = torch.finfo(torch.float32).max
    x, w = torch.zeros(m, 40 + pad, device="cuda")[:, :40], torch.zeros(n, 40 + pad, device="cuda")[:, :40]
    x[:, 3] = most * torch.linspace(0.98, 1.0, m, dtype=torch.float64, device="cuda").float()
    x[:, 38] = 2.0 ** 125
    w[:, 3] = torch.tensor([1.0, -1.0, 0.5, 2.0], device="cuda")[torch.arange(n, device="cuda") % 4]
    w[:, 38] = torch.tensor([0.0, 0.0, 1.0, 0.0], device="cuda")[torch.arange(n, device="cuda") % 4]
    out = _linear(x, w, torch.empty(m, n, device="cuda")).cpu()
    want = x.double().cpu() @ w.double().cpu().t()
    fits = want.abs() <= most
    assert bool(out[:, 3::4].isinf().all()) and bool(fits[:, torch.arange(n) % 4 != 3].all())
    ref.check(out[:, torch.arange(n) % 4 != 3], (want[:, torch.arange(n) % 4 != 3], (want.abs() * 4 * ref.U32)[:, torch.arange(n) % 4 != 3]))


def test_calls_without_a_stream_are_on_torchs():
    """Behind work that is under way on torch's current stream, and in its captures."""
    x, w = _rand(6, 64), _rand(32, 64, seed=1)
    q, k = _rand(1, 3, 2, 32, seed=2), _rand(1, 40, 2, 32, seed=3)
    pos, freqs = torch.arange(6, dtype=torch.int32, device="cuda")[:, None], torch.ones(1, 16, 1, device="cuda")
    calls = [lambda: ops.linear(x, w, torch.empty(6, 32, dtype=x.dtype, device="cuda")),
             lambda: ops.rope_axes(x.view(6, 2, 32), pos, freqs, torch.empty(6, 2, 32, dtype=x.dtype, device="cuda")),
             lambda: ops.cross_attention(q, k, k, torch.empty_like(q))]
    inputs = [x, x, q]
    for call, t in zip(calls, inputs):
        new = torch.randn_like(t)
        old = t.clone()
        t.copy_(new)
        want = call()
        t.copy_(old)
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            torch.cuda._sleep(100_000_000)
            t.copy_(new)
            got = call()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = call()
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


# -- what only large or unusual calls reach -----------------------------------

@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("lq,h,kv,d,lk,kind", [
    (512, 2, 2, 64, 33, "none"), (1000, 1, 1, 80, 200, "none"), (256, 4, 2, 128, 300, "lengths"), (1000, 2, 2, 128, 97, "mask"),
    (1000, 1, 1, 64, 260, "mask"), (500, 2, 1, 40, 64, "lengths"), (999, 1, 1, 127, 129, "none")], ids=ids)
def test_attention_of_eight_waves(dtype, lq, h, kv, d, lk, kind):
    """16 bits, 512 rows a kv head and more of which at most an eighth is empty:
    workgroups of 256 rows."""
    b = 3
    rows = lq * h // kv
    assert rows >= 512 and rows * 8 >= (rows + 255) // 256 * 256 * 7
    q, k, v = (_rand(b, n, m, d, dtype=dtype, seed=i, scale=1.2) for i, (n, m) in enumerate(((lq, h), (lk, kv), (lk, kv))))
    lengths = torch.tensor([lk, 0, lk // 2], dtype=torch.int32, device="cuda") if kind == "lengths" else None
    mask = None
    if kind == "mask":
        mask = torch.rand(b, lk, generator=torch.Generator().manual_seed(lk)).cuda() < 0.5
        mask[1] = False
        mask[2, :lk - 3] = False
    out, untouched = _guarded(b, lq, h, d, dtype=dtype)
    ref.check(_attention(q, k, v, out, key_lengths=lengths, key_mask=mask), ref.attention(q, k, v, lengths=lengths, mask=mask))
    untouched()


@pytest.mark.parametrize("dtype,d,lq,b", [(torch.float16, 64, 40, 1), (torch.bfloat16, 128, 40, 1), (torch.float16, 128, 520, 1), (torch.bfloat16, 72, 1024, 1),
                                          (torch.float32, 32, 40, 1), (torch.float32, 16, 40, 260), (torch.bfloat16, 32, 40, 1)], ids=ids)
@pytest.mark.parametrize("kind", ["none", "all", "empty rounds", "last key", "lengths"])
def test_attention_of_many_keys_in_rounds(dtype, d, lq, b, kind):
    """Many rows, more keys than a round of 256 tiles: three rounds, of which masks
    empty the first, the second, or all but the last key's. The items share keys."""
    lk = 2 * 256 * (32 if (dtype != torch.float32 and d > 64) or b > 256 else 64) + 100
    q = _rand(b, lq, 1, d, dtype=dtype, scale=1.2)
    k, v = _rand(1, lk, 1, d, dtype=dtype, seed=1, scale=1.2), _rand(1, lk, 1, d, dtype=dtype, seed=2)
    mask = lengths = None
    if kind == "lengths":
        lengths = torch.full((b,), lk - 90, dtype=torch.int32, device="cuda")
    elif kind != "none":
        mask = torch.rand(1, lk, generator=torch.Generator().manual_seed(d)) < 0.7
        if kind == "empty rounds":
            mask[0, :lk // 3 - 64] = False
            mask[0, lk * 4 // 9:lk - 70] = False
        if kind == "last key":
            mask[0, :lk - 1] = False
            mask[0, lk - 1] = True
        mask = mask.cuda().expand(b, lk)
    out = torch.empty_like(q)
    ops.cross_attention(q, k.expand(b, lk, 1, d), v.expand(b, lk, 1, d), out, key_lengths=lengths, key_mask=mask, stream=_stream())
    for i in {0, b // 2, b - 1}:
        ref.check(out[i:i + 1], ref.attention(q[i:i + 1], k, v, lengths=lengths, mask=mask), i)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("lq,d", [(40, 64), (40, 50), (600, 128), (3, 64)])
def test_attention_of_tokens_far_apart(dtype, lq, d):
    """Token strides of 2^23 elements, where a tile's offsets pass 32 bits, and keys
    that end 2^31 elements behind the first."""
    lk, stride = 258, 1 << 23
    far = torch.empty((lk - 1) * stride + 4096, dtype=dtype, device="cuda")
    q = _rand(1, lq, 1, d, dtype=dtype)
    k, v = (far.as_strided((1, lk, 1, d), (0, stride, 0, 1), at) for at in (0, 2048))
    k.copy_(_rand(1, lk, 1, d, dtype=dtype, seed=1))
    v.copy_(_rand(1, lk, 1, d, dtype=dtype, seed=2))
    ref.check(_attention(q, k, v, torch.empty_like(q)), ref.attention(q, k, v))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("m,k,n,pad", [(17, 72, 8192, 0), (20, 72, 8200, 0), (32, 264, 8201, 1), (33, 40, 8192, 0), (50, 72, 8195, 0), (64, 200, 8300, 3)], ids=ids)
def test_linear_of_few_rows_and_many_columns(dtype, m, k, n, pad):
    """17 to 64 rows, 8192 columns and more: workgroups of 32 columns."""
    x, w = _rand(m, k, dtype=dtype, pad=pad), _rand(n, k, dtype=dtype, seed=1, scale=k ** -0.5, pad=pad)
    bias, res = _rand(n, dtype=torch.float32, seed=2), _rand(m, n, dtype=dtype, seed=3, pad=pad)
    out, untouched = _guarded(m, n, dtype=dtype)
    ref.check(_linear(x, w, out, bias=bias, activation="silu", residual=res), ref.linear(x, w, bias, "silu", res))
    untouched()


def _split_block(dtype, **kw):
    """A block whose attention and last layer split their keys and their K."""
    block = Block(dtype, states=600, width=1032, **kw)
    q, k = block.q.view(block.b, block.l, block.h, block.d), block.kvs[:, :block.kv * block.d].view(block.b, block.s, block.kv, block.d)
    need = (ops.cross_attention_workspace(q, k, k), ops.linear_workspace(block.up, block.w["down"]))
    assert min(need) > 16 and block.ws.numel() >= max(need)
    return block


# Roundings as in test_block, and four fp32 sums of up to 2064 terms of random signs.
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_split_block(dtype):
    block = _split_block(dtype)
    got, want = block.run(_stream()).double().cpu(), block.want()
    assert (got - want).norm() <= (16 * ref.HALF_STEP[dtype] + 4 * math.sqrt(2064) * ref.U32) * want.norm()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_split_block_captured_and_replayed(dtype):
    """Two graphs with workspaces of their own, replayed at the same time on two
    streams, with the program's own work between; each time the eager bits."""
    blocks = [_split_block(dtype, boards=2 + i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in blocks]
    graphs = [torch.cuda.CUDAGraph() for _ in blocks]
    for block, stream, graph in zip(blocks, streams, graphs):
        block.run(_stream())
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            block.run(stream.cuda_stream)
    for i in range(4):
        for block in blocks:
            block.x.copy_(_rand(*block.x.shape, dtype=dtype, seed=20 + i))
            block.lengths.copy_(torch.tensor([(150 * i) % 600, 600, i], dtype=torch.int32)[:block.b])
            block.out.fill_(0)
            block.ws.fill_(255)
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for block in blocks:
            replayed = block.out.clone()
            assert torch.equal(block.run(_stream()), replayed), i
        torch.cuda.synchronize()


def test_split_blocks_of_two_threads():
    """On streams and workspaces of their own."""
    blocks = [_split_block(torch.bfloat16, boards=2 + i) for i in range(2)]
    want = [b.run(0).clone() for b in blocks]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        s = torch.cuda.Stream()
        for _ in range(20):
            blocks[i].out.zero_()
            torch.cuda.current_stream().synchronize()
            blocks[i].run(s.cuda_stream)
            s.synchronize()
            if not torch.equal(blocks[i].out, want[i]):
                bad.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("lq,lk,h,kv,d,dv", [(3, 90, 4, 2, 64, 64), (40, 90, 2, 2, 64, 64), (520, 130, 2, 1, 64, 64), (40, 200, 2, 2, 128, 128), (300, 70, 4, 2, 128, 128),
                                             (33, 64, 3, 3, 20, 32), (130, 1100, 2, 1, 80, 50), (40, 1200, 2, 2, 32, 32)], ids=ids)
@pytest.mark.parametrize("kind", ["none", "both"])
def test_attention_precise(dtype, lq, lk, h, kv, d, dv, kind):
    """Weights of twice the type's bits: the result is off by its own rounding, and
    by what fp32 scores, exponentials and sums and the weights' second piece leave
    (half a step of it, and half of fp16's smallest number against a weight of at
    least 2^7)."""
    b = 6
    g = torch.Generator().manual_seed(lk)
    q, k, v = _rand(b, lq, h, d, dtype=dtype), _rand(b, lk, kv, d, dtype=dtype, seed=1), _rand(b, lk, kv, dv, dtype=dtype, seed=2)
    lengths, mask = _masks(kind, b, lk, g)
    want, bound = ref.attention(q, k, v, lengths=lengths, mask=mask)
    out, untouched = _guarded(b, lq, h, dv, dtype=dtype)
    need = ops.cross_attention_workspace(q, k, v, precise=True)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
    ops.cross_attention(q, k, v, out, key_lengths=lengths, key_mask=mask, workspace=ws, stream=_stream(), precise=True)
    ref.check(out, (want, bound))
    untouched()
    ref.check(ops.cross_attention(q, k, v, torch.empty_like(out), key_lengths=lengths, key_mask=mask, precise=True), (want, bound))
    size, _ = ref.attention(q, k, v.abs(), lengths=lengths, mask=mask)  # of the weighted values
    terms = d ** -0.5 * torch.einsum("bqhd,bkhd->bhqk", q.double().cpu().abs(), k.double().cpu().abs().repeat_interleave(h // kv, 2)).amax(-1).transpose(1, 2)
    off = (ref.HALF_STEP[dtype] ** 2 + 2 * (d + 4) * ref.U32 * terms[..., None] + 2.0 ** -20 + 2 * (lk + 4) * ref.U32) * size + ref.SMALLEST[dtype] * lk * 2.0 ** -5
    assert (out.double().cpu() - want).norm() <= (want.to(dtype).double() - want).norm() + off.norm() + ref.HALF_STEP[dtype] * off.norm()


@pytest.mark.parametrize("dtype", TYPES[:2], ids=ids)
@pytest.mark.parametrize("lq,lk,d", [(50, 75, 64), (40, 1100, 128), (600, 70, 32)])
def test_attention_precise_infinite_values(dtype, lq, lk, d):
    q, k, v = (_rand(1, n, 2, d, dtype=dtype, seed=i) for i, n in enumerate((lq, lk, lk)))
    clean = ref.attention(q, k, v)
    v[0, 9, 0, 3], v[0, lk - 2, 0, 7], v[0, 30, 0, d - 1] = (float(x) for x in ("inf", "-inf", "nan"))
    out = ops.cross_attention(q, k, v, torch.empty_like(q), precise=True).double().cpu()
    assert bool((out[0, :, 0, 3] == float("inf")).all()) and bool((out[0, :, 0, 7] == float("-inf")).all()) and bool(out[0, :, 0, d - 1].isnan().all())
    dims = [3, 7, d - 1]
    out[0, :, 0, dims] = clean[0][0, :, 0, dims]
    ref.check(out, clean)


@pytest.mark.parametrize("dtype", TYPES[:2], ids=ids)
@pytest.mark.parametrize("lq,d", [(40, 64), (520, 64), (40, 128), (33, 32)])
def test_attention_precise_weights_are_not_rounded(dtype, lq, d):
    """Scores that are exact (multiples of 2^-6 below 8), so that what is left besides
    the result's own rounding is the weights' second piece, exponents of up to 12
    that are off by 2^-23 of themselves, and sums. Weights rounded once are seen."""
    lk, g = 64, torch.Generator().manual_seed(lq)
    q, k = torch.zeros(1, lq, 2, d), torch.zeros(1, lk, 2, d)
    q[..., 0] = torch.randint(1, 5, (1, lq, 2), generator=g) / 4
    k[..., 0] = torch.randint(-32, 33, (1, lk, 2), generator=g) / 16
    q, k, v = q.to(dtype).cuda(), k.to(dtype).cuda(), _rand(1, lk, 2, d, dtype=dtype)
    out = ops.cross_attention(q, k, v, torch.empty_like(q), scale=1.0, precise=True).double().cpu()
    want, _ = ref.attention(q, k, v, scale=1.0)
    size, _ = ref.attention(q, k, v.abs(), scale=1.0)
    off = (ref.HALF_STEP[dtype] ** 2 + 2.0 ** -19 + 2 * (lk + 4) * ref.U32) * size + ref.SMALLEST[dtype] * lk * 2.0 ** -5
    limit = (want.to(dtype).double() - want).norm() + off.norm() * (1 + ref.HALF_STEP[dtype])
    assert (out - want).norm() <= limit
    p = torch.exp((q[..., 0].double().cpu().transpose(1, 2)[..., None] * k[..., 0].double().cpu().transpose(1, 2)[:, :, None]))
    once = (p.to(dtype).double() @ v.double().cpu().transpose(1, 2) / p.sum(-1, keepdim=True)).transpose(1, 2)
    assert (once.to(dtype).double() - want).norm() > 1.02 * limit

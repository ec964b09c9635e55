"""Refusals of the operators on the caller's tensors, by the C ABI and by the
Python calls (no GPU: both look at the arguments before any device is touched),
and the plain forms that the GPU tests compare with."""
import ctypes
import json
import os

import pytest
import torch

import operator_reference as ref
from katago_amd import nn, ops

INVALID = 1
AT = 1 << 20  # an address that nothing reads


class Meta:
    """A tensor that is on a GPU as far as its attributes say."""

    def __init__(self, *shape, dtype="float16", strides=None, device=0, at=AT):
        self._t = ops.DeviceTensor(at, shape, dtype, strides, device)

    def __getattr__(self, name):
        return getattr(self._t, name)


def _refused(call, *words):
    with pytest.raises(nn.StringError) as e:
        call()
    assert e.value.code == INVALID, e.value
    for w in words:
        assert w in str(e.value), e.value


def test_structs_have_the_headers_sizes():
    assert ctypes.sizeof(ops._LinearParams) == 4 * 2 + 8 + 4 * 2 + 8 * 11
    assert ctypes.sizeof(ops._RopeParams) == 4 * 4 + 8 + 4 * 4 + 8 * 9
    assert ctypes.sizeof(ops._AttentionParams) == 4 * 9 + 4 + 8 * 16 + 8 * 5


def _linear(**change):
    a = dict(x=Meta(4, 16), weights=Meta(8, 16), out=Meta(4, 8))
    a.update(change)
    return lambda: ops.linear(a.pop("x"), a.pop("weights"), a.pop("out"), **a)


@pytest.mark.parametrize("change,word", [
    (dict(x=Meta(16)), "axes"), (dict(weights=Meta(8, 15)), "input channels"), (dict(out=Meta(4, 9)), "shape"),
    (dict(out=Meta(3, 8)), "shape"), (dict(weights=Meta(8, 16, dtype="bfloat16")), "type"), (dict(x=Meta(4, 16, dtype="int32")), "type"),
    (dict(x=Meta(4, 16, dtype="float64")), "type"), (dict(bias=Meta(8)), "type"), (dict(bias=Meta(7, dtype="float32")), "shape"),
    (dict(residual=Meta(4, 7)), "shape"), (dict(activation="tanh"), "activation"), (dict(weights=Meta(8, 16, device=1)), "device"),
    (dict(x=Meta(4, 16, strides=(1, 4))), "contiguous"), (dict(out=Meta(4, 8, strides=(7, 1))), "out_stride"),
    (dict(x=Meta(4, 16, at=AT + 1)), "aligned"), (dict(x=Meta(4, 16, at=0)), "null"), (dict(out=Meta(4, 8, at=0)), "null"),
    (dict(x=Meta(4, 16, strides=(-16, 1))), "stride"), (dict(x=Meta(4, 0), weights=Meta(8, 0)), "in_channels"),
    (dict(weights=Meta(0, 16), out=Meta(4, 0)), "out_channels"), (dict(bias=Meta(8, dtype="float32", at=AT + 2)), "aligned"),
    (dict(x=Meta(1 << 31, 16, strides=(0, 1)), out=Meta(1 << 31, 8)), "longer"),
    (dict(x=Meta(1 << 30, 16, strides=(0, 1)), weights=Meta(1 << 20, 16), out=Meta(1 << 30, 1 << 20)), "too large"),
    (dict(weights=Meta((1 << 26) + 1, 16), out=Meta(4, (1 << 26) + 1)), "out_channels"),
    (dict(workspace=Meta(64, dtype="uint8", device=1)), "workspace"), (dict(workspace=Meta(64, dtype="uint8", at=AT + 8)), "aligned"),
])
def test_linear_refuses(change, word):
    _refused(_linear(**change), word)


def _rope(**change):
    a = dict(x=Meta(5, 4, 32), positions=Meta(5, 2, dtype="int32"), freqs=Meta(2, 16, 2, dtype="float32"), out=Meta(5, 4, 32, at=2 * AT))
    a.update(change)
    return lambda: ops.rope_axes(a.pop("x"), a.pop("positions"), a.pop("freqs"), a.pop("out"), **a)


@pytest.mark.parametrize("change,word", [
    (dict(positions=Meta(5, 3, dtype="int32")), "shape"), (dict(positions=Meta(5, 2, dtype="float32")), "type"),
    (dict(freqs=Meta(3, 16, 2, dtype="float32")), "tables"), (dict(freqs=Meta(2, 17, 2, dtype="float32")), "pairs"),
    (dict(freqs=Meta(2, 16, 5, dtype="float32"), positions=Meta(5, 5, dtype="int32")), "axes"),
    (dict(freqs=Meta(2, 16, 2, dtype="float32", strides=(40, 2, 1))), "contiguous"), (dict(layout="thirds"), "layout"),
    (dict(out=Meta(5, 4, 31)), "shape"), (dict(out=Meta(5, 4, 32, strides=(64, 32, 1))), "overlap"),
    (dict(out=Meta(5, 4, 32, strides=(256, 64, 1))), "in place"), (dict(x=Meta(5, 4, 32, dtype="uint8")), "type"),
    (dict(out=Meta(5, 4, 32, dtype="float32")), "type"), (dict(x=Meta(5, 4, 32, at=0)), "null"),
    (dict(positions=Meta(5, 2, dtype="int32", at=AT + 2)), "aligned"), (dict(freqs=Meta(1, 0, 2, dtype="float32")), "positive"),
])
def test_rope_refuses(change, word):
    _refused(_rope(**change), word)


def _attention(**change):
    a = dict(q=Meta(2, 3, 4, 32), k=Meta(2, 9, 2, 32), v=Meta(2, 9, 2, 24), out=Meta(2, 3, 4, 24))
    a.update(change)
    return lambda: ops.cross_attention(a.pop("q"), a.pop("k"), a.pop("v"), a.pop("out"), **a)


@pytest.mark.parametrize("change,word", [
    (dict(k=Meta(2, 9, 2, 31)), "shape"), (dict(k=Meta(1, 9, 2, 32)), "shape"), (dict(v=Meta(2, 8, 2, 24)), "shape"),
    (dict(v=Meta(2, 9, 4, 24)), "shape"), (dict(out=Meta(2, 3, 4, 32)), "shape"), (dict(k=Meta(2, 9, 3, 32), v=Meta(2, 9, 3, 24)), "divide"),
    (dict(q=Meta(2, 3, 4, 129), k=Meta(2, 9, 2, 129)), "head dim"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(key_lengths=Meta(3, dtype="int32")), "shape"),
    (dict(key_lengths=Meta(2, dtype="float32")), "type"), (dict(key_mask=Meta(2, 8, dtype="uint8")), "shape"),
    (dict(key_mask=Meta(2, 9, dtype="int32")), "type"), (dict(out=Meta(2, 3, 4, 24, strides=(288, 96, 23, 1))), "overlap"),
    (dict(out=Meta(2, 3, 4, 24, strides=(0, 96, 24, 1))), "overlap"), (dict(q=Meta(2, 3, 4, 32, at=AT + 1)), "aligned"),
    (dict(v=Meta(2, 9, 2, 24, at=0)), "null"), (dict(key_mask=Meta(2, 9, dtype="bool", device=1)), "device"),
    (dict(q=Meta(2, 1 << 30, 4, 32), out=Meta(2, 1 << 30, 4, 24)), "too many"),
    (dict(q=Meta(70000, 3, 4, 32), k=Meta(70000, 9, 2, 32), v=Meta(70000, 9, 2, 24), out=Meta(70000, 3, 4, 24)), "65535"),
])
def test_attention_refuses(change, word):
    _refused(_attention(**change), word)


def test_c_entries_refuse_null_and_unknown_codes():
    lib = ops._library()
    for name, params in (("kgh_linear", ops._LinearParams), ("kgh_rope_axes", ops._RopeParams), ("kgh_cross_attention", ops._AttentionParams)):
        assert getattr(lib, name)(0, None, None) == INVALID
        p = params()
        p.dtype = 7
        assert getattr(lib, name)(0, p, None) == INVALID
        assert b"dtype 7" in lib.kgh_last_error()
    for name, params in (("kgh_linear_workspace", ops._LinearParams), ("kgh_cross_attention_workspace", ops._AttentionParams)):
        assert getattr(lib, name)(0, None, None) == INVALID
        assert getattr(lib, name)(0, params(), None) == INVALID


def test_outputs_on_inputs_are_refused():
    far = dict(at=2 * AT)
    _refused(_linear(x=Meta(4, 8), weights=Meta(8, 8, **far)), "x itself")
    _refused(_linear(x=Meta(8, 8, **far), weights=Meta(8, 8), out=Meta(8, 8)), "weights itself")
    _refused(_linear(x=Meta(4, 16, **far), weights=Meta(8, 16, **far), residual=Meta(4, 8, strides=(16, 1))), "residual_stride")
    _refused(_attention(k=Meta(2, 9, 2, 32, **far), v=Meta(2, 9, 2, 24, **far)), "q itself")
    _refused(_attention(q=Meta(2, 3, 4, 32, **far), v=Meta(2, 9, 2, 24, **far)), "k itself")
    _refused(_attention(q=Meta(2, 3, 4, 32, **far), k=Meta(2, 9, 2, 32, **far)), "v itself")


def test_largest_sizes_are_refused_in_64_bits():
    """Sizes of the C entries whose counts pass 64 bits."""
    lib = ops._library()
    p = ops._RopeParams(0, 0, 0, 1, 1 << 62, 4, 64, 32, 1, AT, 64, 64, AT, 1, AT, 2 * AT, 256, 64)
    for tokens, heads, dim in ((1 << 62, 4, 64), (1 << 32, (1 << 31) - 1, 1 << 20), (1 << 20, 1 << 20, 64)):
        p.tokens, p.heads, p.head_dim = tokens, heads, dim
        p.out_head_stride, p.out_token_stride = dim, heads * dim
        assert lib.kgh_rope_axes(0, p, None) == INVALID
        assert b"tokens" in lib.kgh_last_error()
    _refused(_attention(scale=1e31), "scale")


def test_kernels_keep_everything_in_registers():
    """No kernel of the operators leaves registers for scratch memory, by the
    compiler's report of the build (see test_host.py's, of the nets' kernels)."""
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "katago_amd", "lib", "kernel_resources.json")
    with open(path) as f:
        usage = json.load(f)
    kernels = ("linearSkinnyKernel", "linearDmaKernel", "linearTileKernel", "linearJoinKernel", "ropeAxesKernel", "attentionFewKernel",
               "attentionManyKernel", "attentionJoinKernel")
    for kernel in kernels:
        found = [u for name, u in usage.items() if kernel in name]
        assert found and all(u["scratch"] == 0 and u["vgpr_spill"] == 0 for u in found), kernel


def test_device_tensor_strides():
    t = ops.DeviceTensor(ctypes.c_void_p(64), (2, 3, 4), "float16")
    assert t.stride() == (12, 4, 1) and t.data_ptr() == 64
    assert ops.DeviceTensor(64, (2, 3, 4), "float16", (100, 8, 1)).stride() == (100, 8, 1)


def test_plain_forms():
    """The oracle against torch's own functions, and its bounds against inputs
    rounded as a kernel would round them."""
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(5, 37, generator=g), torch.randn(11, 37, generator=g)
    y, _ = ref.linear(x, w, torch.ones(11), "gelu")
    torch.testing.assert_close(y, torch.nn.functional.gelu(x.double() @ w.double().t() + 1))
    q, k, v = (torch.randn(2, n, 4, 16, generator=g) for n in (3, 9, 9))
    y, _ = ref.attention(q, k, v)
    t = [z.double().transpose(1, 2) for z in (q, k, v)]
    torch.testing.assert_close(y, torch.nn.functional.scaled_dot_product_attention(*t).transpose(1, 2))
    pos, freqs = torch.randint(0, 50, (5, 3), generator=g), torch.randn(2, 8, 3, generator=g)
    z = torch.randn(5, 4, 16, generator=g)
    for layout in ops.ROPE_LAYOUTS:
        y, _ = ref.rope(z, pos, freqs, layout)
        torch.testing.assert_close(y.norm(dim=-1), z.double().norm(dim=-1))
        back, _ = ref.rope(y, pos, freqs, layout, inverse=True)
        torch.testing.assert_close(back, z.double())
    with pytest.raises(AssertionError):  # a mistake of one step of bf16 is seen
        ref.check(y * (1 + 2.0 ** -7), (y, y.abs() * 2.0 ** -8))


class Trained(Meta):
    requires_grad = True


@pytest.mark.parametrize("call", [
    _linear(x=Trained(4, 16)), _linear(weights=Trained(8, 16)), _linear(bias=Trained(8, dtype="float32")), _linear(residual=Trained(4, 8)),
    _linear(out=Trained(4, 8)), _rope(x=Trained(5, 4, 32)), _rope(freqs=Trained(2, 16, 2, dtype="float32")), _attention(q=Trained(2, 3, 4, 32)),
    _attention(k=Trained(2, 9, 2, 32)), _attention(v=Trained(2, 9, 2, 24))])
def test_tensors_that_require_gradients_are_refused(call):
    """Their results would have no history."""
    _refused(call, "gradients")


def test_tensors_that_require_gradients_are_taken_under_no_grad():
    with torch.no_grad():
        _refused(_linear(x=Trained(4, 16), weights=Trained(8, 16, at=0)), "null")
        _refused(_rope(x=Trained(5, 4, 32), freqs=Trained(2, 16, 2, dtype="float32", at=0)), "null")
        _refused(_attention(q=Trained(2, 3, 4, 32), k=Trained(2, 9, 2, 32, at=0)), "null")
    assert ops.linear_workspace(Trained(4, 16), Trained(8, 16)) == 0  # sizes only
    assert ops.cross_attention_workspace(Trained(2, 3, 4, 32), Trained(2, 9, 2, 32), Trained(2, 9, 2, 24)) == 0


@pytest.mark.parametrize("dtype,size", [("uint8", 1), ("int8", 1), ("bool", 1), ("bfloat16", 2), ("int16", 2), ("float32", 4), ("int32", 4),
                                        ("int64", 8), ("float64", 8)])
def test_workspaces_of_any_type(dtype, size):
    t = torch.empty(5, 3, dtype=getattr(torch, dtype))
    assert size == t.element_size()
    assert ops._workspace("linear", t, -1) == (t.data_ptr(), 15 * size)
    _refused(_linear(workspace=Meta(8, dtype=dtype, at=AT + 8)), "aligned")
    _refused(_attention(workspace=Meta(8, dtype=dtype, device=1)), "workspace")
    _refused(_linear(workspace=Meta(8, 3, dtype=dtype, strides=(4, 1))), "contiguous")


def test_workspaces_of_other_types_are_refused():
    _refused(_linear(workspace=Meta(8, dtype="complex64")), "type")


def test_precise_is_a_truth_value():
    t = Meta(2, 3, 4, 32), Meta(2, 9, 2, 32), Meta(2, 9, 2, 24)
    p, _ = ops._attention_params(*t, None, True)
    assert p.precise == 1
    p.precise = 2
    assert ops._library().kgh_cross_attention(0, p, None) == INVALID
    assert b"precise" in ops._library().kgh_last_error()

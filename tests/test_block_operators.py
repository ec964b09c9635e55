"""Refusals of the 8-bit and normalising operators, by the C ABI and by the Python
calls (no GPU: both look at the arguments before any device is touched), and the
formulas that the GPU tests compare with."""
import ctypes
import json
import os

import pytest
import torch

import block_reference as ref
import operator_reference
from katago_amd import nn, ops

INVALID = 1
AT = 1 << 20  # an address that nothing reads


class Meta:
    """A tensor that is on a GPU as far as its attributes say."""

    def __init__(self, *shape, dtype="float16", strides=None, device=0, at=AT):
        self._t = ops.DeviceTensor(at, shape, dtype, strides, device)

    def __getattr__(self, name):
        return getattr(self._t, name)


class Trained(Meta):
    requires_grad = True


def _refused(call, *words):
    with pytest.raises(nn.StringError) as e:
        call()
    assert e.value.code == INVALID, e.value
    for w in words:
        assert w in str(e.value), e.value


def test_structs_have_the_headers_sizes():
    assert ctypes.sizeof(ops._QuantizeParams) == 4 * 2 + 8 * 6
    assert ctypes.sizeof(ops._LinearInt8Params) == 4 * 2 + 8 + 4 * 2 + 8 * 13
    assert ctypes.sizeof(ops._GroupNormParams) == 4 * 7 + 4 + 8 * 15
    assert ctypes.sizeof(ops._GroupNormBackwardParams) == 4 * 6 + 8 * 19


F32, I8 = {"dtype": "float32"}, {"dtype": "int8"}


def _quantize(**change):
    a = dict(x=Meta(4, 16), out=Meta(4, 16, at=2 * AT, **I8), scales=Meta(4, at=3 * AT, **F32))
    a.update(change)
    return lambda: ops.quantize_rows(**a)


@pytest.mark.parametrize("change,word", [
    (dict(x=Meta(4, 4, 4)), "axes"), (dict(x=Meta(4, 16, dtype="int8")), "type"), (dict(x=Meta(4, 16, dtype="float64")), "type"),
    (dict(out=Meta(4, 16)), "type"), (dict(out=Meta(4, 16, dtype="uint8")), "type"), (dict(out=Meta(4, 15, **I8)), "shape"),
    (dict(scales=Meta(5, **F32)), "shape"), (dict(scales=Meta(4)), "type"), (dict(scales=Meta(4, 1, **F32)), "axes"),
    (dict(scales=Meta(4, strides=(2,), **F32)), "contiguous"), (dict(x=Meta(4, 16, strides=(1, 4))), "contiguous"),
    (dict(out=Meta(4, 16, at=2 * AT, strides=(15, 1), **I8)), "out_stride"), (dict(x=Meta(4, 16, strides=(-16, 1))), "stride"),
    (dict(x=Meta(4, 16, at=AT + 1)), "aligned"), (dict(x=Meta(4, 16, at=0)), "null"), (dict(out=Meta(4, 16, at=0, **I8)), "null"),
    (dict(scales=Meta(4, at=0, **F32)), "null"), (dict(scales=Meta(4, at=AT + 2, **F32)), "aligned"), (dict(out=Meta(4, 16, device=1, **I8)), "device"),
    (dict(x=Meta(4, 0), out=Meta(4, 0, **I8)), "channels"), (dict(out=Meta(4, 16, **I8)), "x itself"), (dict(scales=Meta(4, **F32)), "x itself"),
    (dict(scales=Meta(4, at=2 * AT, **F32)), "scales itself"), (dict(x=Trained(4, 16)), "gradients"),
    (dict(x=Meta(1 << 31, 1, strides=(0, 1)), out=Meta(1 << 31, 1, **I8), scales=Meta(1 << 31, **F32)), "longer"),
])
def test_quantize_refuses(change, word):
    _refused(_quantize(**change), word)


def _linear(**change):
    a = dict(x=Meta(4, 16, **I8), x_scales=Meta(4, **F32), weights=Meta(8, 16, **I8), weight_scales=Meta(8, **F32), out=Meta(4, 8, at=2 * AT))
    a.update(change)
    return lambda: ops.linear_int8(**a)


@pytest.mark.parametrize("change,word", [
    (dict(x=Meta(16, **I8)), "axes"), (dict(x=Meta(4, 16)), "type"), (dict(x=Meta(4, 16, dtype="uint8")), "type"), (dict(weights=Meta(8, 16)), "type"),
    (dict(weights=Meta(8, 15, **I8)), "input channels"), (dict(out=Meta(4, 9)), "shape"), (dict(out=Meta(4, 8, dtype="int32")), "type"),
    (dict(x_scales=Meta(3, **F32)), "shape"), (dict(x_scales=Meta(4)), "type"), (dict(weight_scales=Meta(4, **F32)), "shape"),
    (dict(weight_scales=Meta(8, strides=(2,), **F32)), "contiguous"), (dict(bias=Meta(8)), "type"), (dict(bias=Meta(7, **F32)), "shape"),
    (dict(residual=Meta(4, 7)), "shape"), (dict(residual=Meta(4, 8, dtype="bfloat16")), "type"), (dict(activation="tanh"), "activation"),
    (dict(weights=Meta(8, 16, device=1, **I8)), "device"), (dict(x=Meta(4, 16, strides=(1, 4), **I8)), "contiguous"),
    (dict(out=Meta(4, 8, at=2 * AT, strides=(7, 1))), "out_stride"), (dict(out=Meta(4, 8, at=2 * AT + 1)), "aligned"), (dict(x=Meta(4, 16, at=0, **I8)), "null"),
    (dict(x_scales=Meta(4, at=0, **F32)), "x_scales is null"), (dict(weight_scales=Meta(8, at=0, **F32)), "weight_scales is null"),
    (dict(x=Meta(4, 16, strides=(-16, 1), **I8)), "stride"), (dict(x=Meta(4, 0, **I8), weights=Meta(8, 0, **I8)), "in_channels"),
    (dict(x=Meta(4, 131072, **I8), weights=Meta(8, 131072, **I8)), "32 bits"), (dict(weights=Meta(0, 16, **I8), weight_scales=Meta(0, **F32), out=Meta(4, 0)), "out_channels"),
    (dict(bias=Meta(8, at=AT + 2, **F32)), "aligned"), (dict(workspace=Meta(64, dtype="uint8", at=AT + 8)), "aligned"),
    (dict(workspace=Meta(64, dtype="uint8", device=1)), "workspace"), (dict(out=Meta(4, 8)), "x itself"),
    (dict(out=Meta(4, 8), x=Meta(4, 16, at=3 * AT, **I8), x_scales=Meta(4, at=3 * AT, **F32)), "weights itself"),
    (dict(residual=Meta(4, 8, at=2 * AT, strides=(16, 1))), "residual_stride"), (dict(x_scales=Trained(4, **F32)), "gradients"),
    (dict(weight_scales=Trained(8, **F32)), "gradients"), (dict(bias=Trained(8, **F32)), "gradients"), (dict(residual=Trained(4, 8)), "gradients"),
    (dict(x=Meta(1 << 30, 16, strides=(0, 1), **I8), x_scales=Meta(1 << 30, **F32), weights=Meta(1 << 20, 16, **I8), weight_scales=Meta(1 << 20, **F32),
          out=Meta(1 << 30, 1 << 20, at=2 * AT)), "too large"),
])
def test_linear_int8_refuses(change, word):
    _refused(_linear(**change), word)


WORK = dict(workspace=Meta(1 << 20, dtype="uint8", at=9 * AT))


def _norm(**change):
    a = dict(x=Meta(2, 9, 24), out=Meta(2, 9, 24, at=2 * AT), groups=4, **WORK)
    a.update(change)
    return lambda: ops.group_norm(**a)


NORM_INPUTS = [
    (dict(groups=5), "divide"), (dict(groups=0), "divide"), (dict(groups=-4), "divide"), (dict(weight=Meta(24)), "type"), (dict(weight=Meta(23, **F32)), "shape"),
    (dict(bias=Meta(25, **F32)), "shape"), (dict(bias=Meta(24, strides=(2,), **F32)), "contiguous"), (dict(lengths=Meta(3, dtype="int32")), "shape"),
    (dict(lengths=Meta(2, **F32)), "type"), (dict(lengths=Meta(2, dtype="int32", at=AT + 2)), "aligned"), (dict(mask=Meta(2, 8, dtype="bool")), "shape"),
    (dict(mask=Meta(2, 9, dtype="int32")), "type"), (dict(mask=Meta(2, 9, dtype="bool", device=1)), "device"), (dict(activation="tanh"), "activation"),
    (dict(weight=Meta(24, at=AT + 1, **F32)), "aligned"), (dict(workspace=Meta(64, dtype="uint8", device=1)), "workspace"), (dict(workspace=Meta(64, dtype="uint8", at=AT + 8)), "aligned"),
    (dict(x=Meta(2, 9, 24, strides=(-216, 24, 1))), "negative"), (dict(x=Meta(2, 9, 24, strides=(216, 1, 9))), "contiguous"), (dict(x=Meta(18, 24)), "axes"),
    (dict(x=Meta(2, 9, 24, at=AT + 1)), "aligned"), (dict(x=Meta(2, 9, 24, at=0)), "null"), (dict(x=Meta(2, 9, 24, dtype="int32")), "type"),
    (dict(mask=Meta(2, 9, dtype="bool", strides=(-9, 1))), "negative"), (dict(weight=Trained(24, **F32)), "gradients"), (dict(x=Trained(2, 9, 24)), "gradients"),
]


@pytest.mark.parametrize("change,word", NORM_INPUTS + [
    (dict(out=Meta(2, 9, 23)), "shape"), (dict(out=Meta(2, 9, 24, dtype="float32")), "type"), (dict(out=Meta(2, 9, 24, **I8)), "type"),
    (dict(out=Meta(2, 9, 24, at=2 * AT, strides=(216, 23, 1))), "overlap"), (dict(out=Meta(2, 9, 24, at=2 * AT, strides=(100, 24, 1))), "overlap"),
    (dict(out=Meta(2, 9, 24, strides=(240, 24, 1))), "in place"), (dict(out=Meta(2, 9, 24, **I8), out_scales=Meta(2, 9, **F32)), "x itself"),
    (dict(out_scales=Meta(2, 9, **F32)), "type"), (dict(out=Meta(2, 9, 24, at=2 * AT, **I8), out_scales=Meta(2, 8, **F32)), "shape"),
    (dict(out=Meta(2, 9, 24, at=2 * AT, **I8), out_scales=Meta(2, 9, strides=(10, 1), **F32)), "contiguous"), (dict(stats=Meta(2, 4, 3, **F32)), "shape"),
    (dict(stats=Meta(2, 4, 2)), "type"), (dict(stats=Meta(2, 4, 2, strides=(16, 2, 1), **F32)), "contiguous"), (dict(eps=0.0), "eps"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(eps=1e-39), "eps"), (dict(out=Meta(2, 9, 24, at=0)), "null"),
])
def test_group_norm_refuses(change, word):
    _refused(_norm(**change), word)


def test_group_norm_of_no_positions_refuses_statistics():
    """They are written where nothing else is."""
    none = dict(x=Meta(2, 0, 24), out=Meta(2, 0, 24, at=2 * AT))
    _refused(_norm(stats=Meta(2, 4, 2, at=AT + 2, **F32), **none), "statistics", "aligned")
    _refused(_norm(stats=Meta(2, 3, 2, **F32), **none), "shape")


def _backward(**change):
    a = dict(x=Meta(2, 9, 24), grad_out=Meta(2, 9, 24, at=2 * AT), stats=Meta(2, 4, 2, at=3 * AT, **F32), grad_x=Meta(2, 9, 24, at=4 * AT), groups=4, **WORK)
    a.update(change)
    return lambda: ops.group_norm_backward(**a)


@pytest.mark.parametrize("change,word", NORM_INPUTS + [
    (dict(grad_out=Meta(2, 9, 23)), "shape"), (dict(grad_out=Meta(2, 9, 24, **F32)), "type"), (dict(grad_x=Meta(2, 8, 24)), "shape"),
    (dict(grad_x=Meta(2, 9, 24, dtype="bfloat16")), "type"), (dict(grad_x=Meta(2, 9, 24, at=4 * AT, strides=(216, 20, 1))), "overlap"),
    (dict(grad_x=Meta(2, 9, 24)), "x itself"), (dict(grad_x=Meta(2, 9, 24, at=2 * AT)), "grad_out itself"), (dict(stats=Meta(2, 5, 2, **F32)), "shape"),
    (dict(stats=Meta(2, 4, 2, at=0, **F32)), "null"), (dict(stats=Meta(2, 4, 2, at=AT + 1, **F32)), "aligned"), (dict(grad_weight=Meta(23, **F32)), "shape"),
    (dict(grad_bias=Meta(24)), "type"), (dict(grad_weight=Meta(24, **F32), grad_bias=Meta(24, **F32)), "grad_bias itself"),
    (dict(grad_out=Meta(2, 9, 24, at=0)), "null"), (dict(grad_x=Meta(2, 9, 24, at=0)), "null"), (dict(grad_out=Trained(2, 9, 24)), "gradients"),
])
def test_group_norm_backward_refuses(change, word):
    _refused(_backward(**change), word)


def _apart(**change):
    return dict(dict(x=Meta(2, 9, 24), weight=Meta(24, at=10 * AT, **F32), bias=Meta(24, at=11 * AT, **F32), lengths=Meta(2, dtype="int32", at=12 * AT),
                     mask=Meta(2, 9, dtype="bool", at=13 * AT)), **change)


@pytest.mark.parametrize("name,at", [("weight", 10), ("bias", 11), ("lengths", 12), ("mask", 13)])
def test_outputs_that_are_inputs_are_refused(name, at):
    q = dict(out=Meta(2, 9, 24, at=2 * AT, **I8))
    scales, stats = (lambda at: Meta(2, 9, at=at * AT, **F32)), (lambda at: Meta(2, 4, 2, at=at * AT, **F32))
    _refused(_norm(**_apart(out=Meta(2, 9, 24, at=at * AT))), "out is " + name + " itself")
    _refused(_norm(**_apart(out_scales=scales(at), **q)), "out_scales is " + name + " itself")
    _refused(_norm(**_apart(stats=stats(at))), "statistics is " + name + " itself")
    _refused(_backward(**_apart(grad_x=Meta(2, 9, 24, at=at * AT))), "grad_x is " + name + " itself")
    for grad in ("grad_weight", "grad_bias"):
        _refused(_backward(**_apart(**{grad: Meta(24, at=at * AT, **F32)})), grad + " is " + name + " itself")


def test_outputs_that_are_each_other_are_refused():
    f32 = lambda *shape, at: Meta(*shape, at=at * AT, **F32)
    q = dict(out=Meta(2, 9, 24, at=2 * AT, **I8))
    _refused(_norm(**_apart(out_scales=f32(2, 9, at=2), **q)), "out is out_scales itself")
    _refused(_norm(**_apart(stats=f32(2, 4, 2, at=2))), "out is statistics itself")
    _refused(_norm(**_apart(out_scales=f32(2, 9, at=5), stats=f32(2, 4, 2, at=5), **q)), "out_scales is statistics itself")
    _refused(_norm(**_apart(out_scales=f32(2, 9, at=1), **q)), "out_scales is x itself")
    _refused(_norm(**_apart(stats=f32(2, 4, 2, at=1))), "statistics is x itself")
    _refused(_backward(**_apart(grad_x=Meta(2, 9, 24, at=3 * AT))), "grad_x is statistics itself")
    for grad in ("grad_weight", "grad_bias"):
        for name, at in (("x", 1), ("grad_out", 2), ("statistics", 3), ("grad_x", 4)):
            _refused(_backward(**_apart(**{grad: f32(24, at=at)})), grad + " is " + name + " itself")


def test_workspaces_that_are_needed():
    """A call that needs a workspace names the bytes."""
    x, q = Meta(3, 16384, 512), Meta(3, 16384, 512, at=2 * AT, **I8)
    need = ops.group_norm_workspace(x, q, 32)
    assert need > 0
    small = Meta(need - 1, dtype="uint8", at=9 * AT)
    scales = Meta(3, 16384, at=3 * AT, **F32)
    for space in (None, small):
        _refused(_norm(x=x, out=q, groups=32, out_scales=scales, workspace=space), "workspace of %d bytes" % need)
    need = ops.group_norm_backward_workspace(x, 32)
    assert need > 0
    for space in (None, Meta(need - 1, dtype="uint8", at=9 * AT)):
        _refused(_backward(x=x, grad_out=Meta(3, 16384, 512, at=2 * AT), grad_x=Meta(3, 16384, 512, at=4 * AT), stats=Meta(3, 32, 2, **F32), groups=32,
                           workspace=space), "workspace of %d bytes" % need)


def test_c_entries_refuse_null_and_unknown_codes():
    lib = ops._library()
    for name in ("kgh_quantize_rows", "kgh_linear_int8", "kgh_group_norm", "kgh_group_norm_backward"):
        p = ops._CALLS[name]()
        assert getattr(lib, name)(0, None, None) == INVALID
        p.dtype = 7
        assert getattr(lib, name)(0, p, None) == INVALID
        assert b"dtype 7" in lib.kgh_last_error()
        if name != "kgh_quantize_rows":
            p.dtype, p.activation = 1, 9
            assert getattr(lib, name)(0, p, None) == INVALID
            assert b"activation 9" in lib.kgh_last_error()
            assert getattr(lib, name + "_workspace")(0, None, None) == INVALID
            assert getattr(lib, name + "_workspace")(0, ops._CALLS[name](), None) == INVALID


def test_largest_sizes_are_refused_in_64_bits():
    lib = ops._library()
    for name, batch, positions in (("kgh_group_norm", 1 << 30, 1 << 30), ("kgh_group_norm_backward", (1 << 31) - 1, (1 << 31) - 1)):
        p = ops._CALLS[name](1, 0, batch, positions, 64, 8)
        assert getattr(lib, name)(0, p, None) == INVALID
        assert b"product" in lib.kgh_last_error()
    p = ops._QuantizeParams(1, 64, 1 << 62, AT, 64, 2 * AT, 64, 3 * AT)
    assert lib.kgh_quantize_rows(0, p, None) == INVALID
    assert b"rows" in lib.kgh_last_error()


def test_kernels_keep_everything_in_registers():
    """No kernel of these operators leaves registers for scratch memory, by the
    compiler's report of the build."""
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "katago_amd", "lib", "kernel_resources.json")
    with open(path) as f:
        usage = json.load(f)
    for kernel in ("quantizeRows", "linear8", "norm"):
        found = {name: u for name, u in usage.items() if any(c + kernel in name for c in "0123456789")}
        assert found and not {n: u for n, u in found.items() if u["scratch"] != 0 or u["vgpr_spill"] != 0}, kernel


def test_formulas():
    """The oracle against torch's own functions, and that its checks see mistakes."""
    g = torch.Generator().manual_seed(1)
    x, w, b = torch.randn(3, 7, 24, generator=g), torch.randn(24, generator=g), torch.randn(24, generator=g)
    y, _ = ref.group_norm(x, 4, weight=w, bias=b, act="silu")
    want = torch.nn.functional.silu(torch.nn.functional.group_norm(x.double().transpose(1, 2), 4, w.double(), b.double())).transpose(1, 2)
    torch.testing.assert_close(y, want)
    for act in ops.ACTIVATIONS:
        t = [v.double().requires_grad_(True) for v in (x, w, b)]
        f = {"identity": lambda v: v, "relu": torch.relu, "mish": torch.nn.functional.mish, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[act]
        dy = torch.randn(3, 7, 24, generator=g)
        out = f(torch.nn.functional.group_norm(t[0].transpose(1, 2), 4, t[1], t[2]).transpose(1, 2))
        grads = torch.autograd.grad(out, t, dy.double())
        mean, rstd, _, _ = ref.statistics(x, 4)
        for got, want in zip(ref.group_norm_backward(x, dy, torch.stack((mean, rstd), -1), 4, w, b, act), grads):
            torch.testing.assert_close(got[0], want)
    q, s = ref.quantize(x[0])
    assert int(q.abs().max()) == 127 and float((q * s[:, None] - x[0]).abs().max()) <= float(s.max()) * 0.5001
    ref.check_rows(q, s, (x[0].double(), torch.zeros(7, 24, dtype=torch.float64)))
    with pytest.raises(AssertionError):
        ref.check_rows(q + (q == 0), s, (x[0].double(), torch.zeros(7, 24, dtype=torch.float64)))
    rows = torch.tensor([[0.0, 0.0], [float("nan"), 1.0], [2.0, float("-inf")], [2.0 ** -121, 0.0], [2.0 ** -120, -1e-40]])
    q, s = ref.quantize(rows)
    assert q.tolist() == [[0, 0], [0, 0], [0, 0], [0, 0], [127, 0]]
    assert s.isnan().tolist() == [False, True, True, False, False] and s[0] == 0 and s[3] == 0 and s[4] > 0
    y, bound = ref.linear_int8(q, s[4:].expand(5), torch.ones(3, 2, dtype=torch.int8), torch.ones(3), torch.float32)
    operator_reference.check(y, (y, bound))
    x1, _ = ref.group_norm(x, 4, lengths=torch.tensor([0, 7, 3]))
    assert not x1[0].any() and not x1[2, 3:].any()
    torch.testing.assert_close(x1[2, :3], ref.group_norm(x[2:, :3], 4)[0][0])


def test_gradients_are_taken_under_no_grad():
    with torch.no_grad():
        _refused(_norm(x=Trained(2, 9, 24), out=Meta(2, 9, 24, at=0)), "null")
        _refused(_backward(x=Trained(2, 9, 24), grad_out=Meta(2, 9, 24, at=0)), "null")
        _refused(_quantize(x=Trained(4, 16), out=Meta(4, 16, at=0, **I8)), "null")


def test_tangents_are_refused():
    """A dual tensor's result would silently have no tangent; in a Function's forward it
    has what the Function's jvp gives it."""
    x = torch.randn(2, 3)
    seen = []

    class Function(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            ops._no_gradients("group_norm", x, None)
            seen.append(True)
            return x * 2

        @staticmethod
        def backward(ctx, grad):
            return grad * 2

        @staticmethod
        def jvp(ctx, tangent):
            return tangent * 2

    ops._no_gradients("group_norm", x, None)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        ops._no_gradients("group_norm", x, None, Meta(4, 16))
        for tensors in ((dual,), (x, None, dual)):
            _refused(lambda: ops._no_gradients("group_norm", *tensors), "group_norm", "tangent")
            with torch.no_grad():
                _refused(lambda: ops._no_gradients("group_norm", *tensors), "tangent")
        assert bool((torch.autograd.forward_ad.unpack_dual(Function.apply(dual)).tangent == 2).all()) and seen
    ops._no_gradients("group_norm", x, None)

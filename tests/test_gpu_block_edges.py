"""Edges of the 8-bit and normalising operators: numbers of the types' far ends, bits
that may not depend on the kernel, sums of very many terms."""
import pytest
import torch

import block_reference as ref
from katago_amd import ops
from operator_reference import U32, check
from test_gpu_block_operators import TYPES, _backward, _bytes, _forward_statistics, _laid, _linear, _norm, _rand, ids

pytestmark = pytest.mark.gpu

CURVED = [a for a in ops.ACTIVATIONS if a not in ("identity", "relu")]
LARGEST = torch.finfo(torch.float32).max


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

"""The workloads of the 8-bit and normalising operators of this backend.

A case is what a program does that builds pre-activation blocks (norm, activation,
1x1 convolution, residual) on tensors that are already on the GPU
(``katago_amd.ops``): the matrix product of 8-bit integers with scales for each row
and output channel, after quantising the rows or on rows that came quantised; group
norm with an activation, channels last; its gradient; and the norm with 8-bit rows
and the product that reads them. With ``own`` false the same outputs come from
elementary torch operations in 32 bits.

A case:
  op          "linear", "norm", "backward" or "block"
  dtype       "fp32", "fp16" or "bf16": the tensors that are not 8-bit
  act         "identity", "relu", "mish", "silu" or "gelu"
  linear      rows, in_c, out_c; quantize: whether the rows come in `dtype` and are
              quantised in the pass; bias, residual (truth values); pad: channels
              between rows
  norm        batch, positions, channels, groups; mask: "none", "lengths" (padded
              items, some empty where `least` is 0) or "boards" (square boards of
              several sides in one grid); least: the smallest length as a share of
              positions; pad: channels between positions
  backward    the same
  block       the same, and out_c, residual (the norm's input, where out_c is channels)
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ACTS = ("identity", "relu", "mish", "silu", "gelu")
EPS = 1e-5


def _linear(name, dtype, rows, in_c, out_c, act="identity", quantize=False, bias=True, residual=False, pad=0):
    return {"name": name, "op": "linear", "dtype": dtype, "rows": rows, "in_c": in_c, "out_c": out_c, "act": act, "quantize": quantize,
            "bias": bias, "residual": residual, "pad": pad}


def _norm(name, dtype, batch, positions, channels, groups, act, mask="none", least=1.0, pad=0, op="norm"):
    return {"name": name, "op": op, "dtype": dtype, "batch": batch, "positions": positions, "channels": channels, "groups": groups,
            "act": act, "mask": mask, "least": least, "pad": pad}


def _block(name, dtype, batch, positions, channels, groups, act, out_c, residual, mask="none", least=1.0, pad=0):
    return {**_norm(name, dtype, batch, positions, channels, groups, act, mask, least, pad, "block"), "out_c": out_c, "residual": residual}


def listed():
    return [
        # One token through a feed-forward layer of the 384-channel transformer, quantised on its way in: latency.
        _linear("linear fp16 1x384x1024 silu", "fp16", 1, 384, 1024, "silu", True),
        # A serving step of eight streams on rows that came in 8 bits: the weights are read once.
        _linear("linear bf16 8x4096x8192 gelu", "bf16", 8, 4096, 8192, "gelu"),
        # The second feed-forward layer over 128 boards of 19x19, added to the trunk.
        _linear("linear fp16 46208x1024x384 res", "fp16", 128 * 361, 1024, 384, residual=True),
        # A prompt through a wide layer: quantised, multiplied, everything in the epilogue.
        _linear("linear bf16 8192x4096x8192", "bf16", 8192, 4096, 8192, "gelu", True, True, True),
        # One token's layer norm (one group) in front of a layer.
        _norm("norm fp16 1 token", "fp16", 1, 1, 384, 1, "identity"),
        # The trunk of 256 boards of several sizes in a 19x19 grid.
        _norm("norm fp16 256 boards mish", "fp16", 256, 361, 384, 32, "mish", "boards"),
        # Pictures of 128 x 128 positions: a group does not fit a workgroup.
        _norm("norm bf16 4 pictures silu", "bf16", 4, 16384, 512, 32, "silu"),
        # Padded sequences of odd lengths in fp32, rows of a wider tensor.
        _norm("norm fp32 ragged gelu", "fp32", 24, 1531, 190, 19, "gelu", "lengths", 0.2, 7),
        # The gradient over 128 boards, as a program has it that fits a block's norm.
        _norm("backward bf16 128 boards mish", "bf16", 128, 361, 384, 32, "mish", "boards", op="backward"),
        # The gradient over pictures of 64 x 64 positions in fp32.
        _norm("backward fp32 8 pictures silu", "fp32", 8, 4096, 320, 32, "silu", op="backward"),
        # A residual block's 1x1 layer over 8 boards: norm and activation in 8-bit rows, product, residual.
        _block("block fp16 8 boards", "fp16", 8, 361, 384, 32, "mish", 384, True, "boards"),
        # The fused projection of 128 boards behind its norm.
        _block("block bf16 128 boards 1152", "bf16", 128, 361, 384, 32, "silu", 1152, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges: sizes over their logarithm, odd and
    even, every type, activation, mask and direction."""
    op = rng.choice(("linear", "linear", "linear", "norm", "norm", "backward", "block"))
    dtype = rng.choice(("fp16", "bf16", "bf16", "fp32")) if op != "block" else rng.choice(("fp16", "bf16"))
    # (not the gradient's step of relu: which side a value next to it falls on is its rounding's)
    act = rng.choice(ACTS if op != "backward" else [a for a in ACTS if a != "relu"])
    whole = rng.random() < 0.7  # widths in sixteens, as most nets have them
    pad = rng.choice((0, 0, 64, 7))
    if op == "linear":
        rows, in_c = _log(rng, 1, 46208), _log(rng, 24, 8192)
        out_c = max(1, min(_log(rng, 24, 8192), (1 << 25) // in_c))
        if whole:
            in_c, out_c = max(16, in_c // 16 * 16), max(16, out_c // 16 * 16)
        rows = max(1, min(rows, int(1.3e11 / (in_c * out_c)), (1 << 26) // max(in_c, out_c)))
        return _linear("", dtype, rows, in_c, out_c, act, rng.random() < 0.5, rng.random() < 0.7, rng.random() < 0.4, pad)
    per = rng.choice((4, 8, 12, 16, 16, 32, 64)) if whole else rng.randint(1, 80)
    groups = rng.choice((1, 8, 16, 32, 32)) if whole else _log(rng, 1, 40)
    channels = per * groups
    mask = rng.choice(("none", "lengths", "boards"))
    least = rng.choice((0.0, 0.3, 0.9)) if mask == "lengths" else 1.0
    positions = rng.choice((7, 9, 13, 19, 25)) ** 2 if mask == "boards" else _log(rng, 1, 16384)
    room = (1 << 24) // (2 if dtype == "fp32" else 1)  # values
    batch = max(1, min(_log(rng, 1, 4096 if positions < 64 else 256), room // (positions * channels)))
    positions = max(1, min(positions, room // (batch * channels))) if mask != "boards" else positions
    if op == "block":
        residual = rng.random() < 0.5
        return _block("", dtype, batch, positions, channels, groups, act, channels if residual else _log(rng, 24, 1200), residual, mask, least, pad)
    return _norm("", dtype, batch, positions, channels, groups, act, mask, least, pad, op)


# -- inputs -------------------------------------------------------------------

def _lengths(case):
    """Positions of each item that take part, from the smallest share to all."""
    n, most = case["batch"], case["positions"]
    low, step = case["least"] * most, 7 if n % 7 else 11
    return [int(low + (most - low) * ((step * i + 3) % n) / (n - 1)) for i in range(n)] if n > 1 else [most]


def _sides(case):
    """Boards of three sides in a square grid, cycled over the items."""
    grid = math.isqrt(case["positions"])
    return [max(1, (grid, grid * 2 // 3, grid // 2)[i % 3]) for i in range(case["batch"])]


def _rows(g, shape, pad, dtype, scale=1.0):
    """Normal values; rows of the last axis lie `pad` channels apart."""
    row = torch.randn(*shape[:-1], shape[-1] + pad, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)
    return row[..., :shape[-1]]


def _bytes(g, rows, channels, pad):
    """8-bit rows as a quantiser leaves them (normal values, the largest of a row
    about 4 standard deviations), and their scales."""
    q = torch.randn(rows, channels + pad, generator=g, device="cuda").mul_(127 / 4).round_().clamp_(-127, 127).to(torch.int8)
    return q[:, :channels], torch.rand(rows, generator=g, device="cuda").mul_(0.5).add_(0.75).mul_(4 / 127)


def _weights(g, s, out_c, in_c, pad):
    """Weights of a trained net's size, in 8 bits with a scale for each channel."""
    s["w"], s["w_scales"] = _bytes(g, out_c, in_c, pad)
    s["w_scales"] = s["w_scales"] * in_c ** -0.5
    s["b"] = torch.randn(out_c, generator=g, device="cuda") * 0.3


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t, pad = DTYPES[case["dtype"]], case["pad"]
    s = {"case": case}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["in_c"], case["out_c"]
        if case["quantize"]:
            s["x"] = _rows(g, (m, k), pad, t)
        else:
            s["x"], s["x_scales"] = _bytes(g, m, k, pad)
        _weights(g, s, n, k, pad)
        if not case["bias"]:
            s["b"] = None
        s["residual"] = _rows(g, (m, n), pad, t) if case["residual"] else None
        s["out"] = torch.empty(m, n + pad, device="cuda", dtype=t)[:, :n]
        return s
    b, p, c = case["batch"], case["positions"], case["channels"]
    # Channels of a trunk: each with a mean and a spread of its own.
    spread = torch.rand(c, generator=g, device="cuda") + 0.5
    mean = torch.randn(c, generator=g, device="cuda")
    x = torch.randn(b, p, c + pad, generator=g, device="cuda")
    x[..., :c].mul_(spread).add_(mean)
    s["x"] = x.to(t)[..., :c]
    s["gamma"] = torch.randn(c, generator=g, device="cuda") * 0.2 + 1
    s["beta"] = torch.randn(c, generator=g, device="cuda") * 0.2
    s["lengths"] = s["mask"] = None
    if case["mask"] == "lengths":
        s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    elif case["mask"] == "boards":
        grid = math.isqrt(p)
        side = torch.tensor(_sides(case), device="cuda")[:, None]
        at = torch.arange(p, device="cuda")
        s["mask"] = (at // grid < side) & (at % grid < side)
    if case["op"] == "backward":
        s["grad"] = _rows(g, (b, p, c), pad, t)
        s["stats"] = _statistics(s)
        s["grad_x"] = torch.empty(b, p, c, device="cuda", dtype=t)
        return s
    if case["op"] == "norm":
        if s["lengths"] is not None:  # what lies behind an item's positions was never written
            s["x"].masked_fill_((torch.arange(p, device="cuda") >= s["lengths"][:, None])[..., None], math.nan)
        s["out"] = torch.empty(b, p, c, device="cuda", dtype=t)
        return s
    _weights(g, s, case["out_c"], c, 0)
    s["out"] = torch.empty(b * p, case["out_c"], device="cuda", dtype=t)
    return s


def _statistics(s):
    """Mean and reciprocal standard deviation of each item's groups, as a forward
    pass keeps them for its gradient."""
    c = s["case"]
    x = s["x"].double().unflatten(2, (c["groups"], -1))
    on = _valid(s)
    n = (torch.full((c["batch"],), c["positions"], device="cuda") if on is None else on.sum(1)) * x.shape[-1]
    n = n.clamp_min(1)[:, None]
    if on is not None:
        x = x * on[:, :, None, None]
    mean = x.sum((1, 3)) / n
    d = x - mean[:, None, :, None]
    if on is not None:
        d = d * on[:, :, None, None]
    var = (d * d).sum((1, 3)) / n
    return torch.stack((mean, (var + EPS).rsqrt()), -1).float()


# -- plain forms --------------------------------------------------------------

def _activate(v, act):
    if act == "relu":
        return v.clamp_min(0)
    if act == "mish":
        return v * torch.tanh(torch.log1p(torch.exp(v.clamp_max(20))) + v.clamp_min(20) - 20)
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return v * 0.5 * (1 + torch.erf(v * math.sqrt(0.5)))
    return v


def _slope(v, act):
    """The activation's derivative."""
    if act == "relu":
        return (v > 0).float()
    if act == "mish":
        t = torch.tanh(torch.log1p(torch.exp(v.clamp_max(20))) + v.clamp_min(20) - 20)
        return t + v * (1 - t * t) / (1 + torch.exp(-v))
    if act == "silu":
        e = 1 / (1 + torch.exp(-v))
        return e * (1 + v * (1 - e))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(v * math.sqrt(0.5))) + v * torch.exp(-0.5 * v * v) * (1 / math.sqrt(2 * math.pi))
    return torch.ones_like(v)


def _valid(s):
    """Which positions of an item take part, or None for all."""
    if s["mask"] is not None:
        return s["mask"]
    if s["lengths"] is not None:
        return torch.arange(s["x"].shape[1], device="cuda") < s["lengths"][:, None]
    return None


def _quantized(x):
    """Rows in 8 bits, as the whole numbers they hold, and their scales."""
    top = x.abs().amax(-1, keepdim=True)
    # (a number over a tensor would be its reciprocal's product)
    factor = torch.where(top > 0, torch.full_like(top, 127.0) / top, 0.0)
    return torch.round(x * factor), top / 127.0


def _product(s, q, q_scales):
    v = (q @ s["w"].float().t()) * q_scales * s["w_scales"]
    if s["b"] is not None:
        v = v + s["b"]
    return v


def _plain_linear(s):
    q, scales = _quantized(s["x"].float()) if s["case"]["quantize"] else (s["x"].float(), s["x_scales"][:, None])
    v = _activate(_product(s, q, scales), s["case"]["act"])
    if s["residual"] is not None:
        v = v + s["residual"].float()
    return v.to(s["out"].dtype)


def _plain_values(s):
    """The norm with its activation, before it is rounded."""
    c = s["case"]
    on = _valid(s)
    x = s["x"].float().unflatten(2, (c["groups"], -1))
    if on is not None:
        x = x.masked_fill(~on[:, :, None, None], 0)
        n = (on.sum(1) * x.shape[-1]).clamp_min(1)[:, None, None, None]
    else:
        n = c["positions"] * x.shape[-1]
    # Many values are summed: in 64 bits.
    mean = x.sum((1, 3), keepdim=True, dtype=torch.float64) / n
    d = x - mean.float()
    if on is not None:
        d = d * on[:, :, None, None]
    var = (d * d).sum((1, 3), keepdim=True, dtype=torch.float64) / n
    y = (d * torch.rsqrt(var + EPS).float()).flatten(2) * s["gamma"] + s["beta"]
    y = _activate(y, c["act"])
    return y if on is None else y * on[:, :, None]


def _plain_norm(s):
    return _plain_values(s).to(s["x"].dtype)


def _plain_backward(s):
    c = s["case"]
    on = _valid(s)
    x, grad = s["x"].float().unflatten(2, (c["groups"], -1)), s["grad"].float()
    mean, rstd = s["stats"][:, None, :, None, 0], s["stats"][:, None, :, None, 1]
    h = (x - mean) * rstd
    grad = grad * _slope(h.flatten(2) * s["gamma"] + s["beta"], c["act"])
    n = c["positions"] * x.shape[-1]
    if on is not None:
        grad = grad * on[:, :, None]
        n = (on.sum(1) * x.shape[-1]).clamp_min(1)[:, None, None, None]
    flat = h.flatten(2)
    grad_gamma = (grad * flat).sum((0, 1), dtype=torch.float64).float()
    grad_beta = grad.sum((0, 1), dtype=torch.float64).float()
    inner = (grad * s["gamma"]).unflatten(2, (c["groups"], -1))
    a1 = (inner.sum((1, 3), keepdim=True, dtype=torch.float64) / n).float()
    a2 = ((inner * h).sum((1, 3), keepdim=True, dtype=torch.float64) / n).float()
    out = (rstd * (inner - a1 - h * a2)).flatten(2)
    if on is not None:
        out = out * on[:, :, None]
    return out.to(s["x"].dtype), grad_gamma, grad_beta


def _plain_block(s):
    q, scales = _quantized(_plain_values(s).flatten(0, 1))
    v = _product(s, q, scales)
    if s["case"]["residual"]:
        v = v + s["x"].float().flatten(0, 1)
    return v.to(s["out"].dtype)


# -- the framework's operators ------------------------------------------------

def _space(s, name, need):
    """A workspace that is kept with the layer."""
    if name not in s:
        s[name] = torch.empty(need(), dtype=torch.uint8, device="cuda")
    return s[name]


def _own(s):
    from katago_amd import ops

    c = s["case"]
    if c["op"] == "linear":
        x, scales = s["x"], s.get("x_scales")
        if c["quantize"]:
            if "q" not in s:
                s["q"] = torch.empty(c["rows"], c["in_c"], dtype=torch.int8, device="cuda")
                s["q_scales"] = torch.empty(c["rows"], device="cuda")
            x, scales = s["q"], s["q_scales"]
            ops.quantize_rows(s["x"], x, scales)
        space = _space(s, "workspace", lambda: ops.linear_int8_workspace(x, s["w"]))
        return ops.linear_int8(x, scales, s["w"], s["w_scales"], s["out"], bias=s["b"], activation=c["act"], residual=s["residual"], workspace=space)
    kw = {"weight": s["gamma"], "bias": s["beta"], "eps": EPS, "activation": c["act"], "lengths": s["lengths"], "mask": s["mask"]}
    if c["op"] == "norm":
        space = _space(s, "workspace", lambda: ops.group_norm_workspace(s["x"], s["out"], c["groups"]))
        return ops.group_norm(s["x"], s["out"], c["groups"], workspace=space, **kw)
    if c["op"] == "backward":
        if "grad_gamma" not in s:
            s["grad_gamma"], s["grad_beta"] = torch.empty_like(s["gamma"]), torch.empty_like(s["beta"])
        space = _space(s, "workspace", lambda: ops.group_norm_backward_workspace(s["x"], c["groups"]))
        del kw["eps"]
        ops.group_norm_backward(s["x"], s["grad"], s["stats"], s["grad_x"], c["groups"], grad_weight=s["grad_gamma"], grad_bias=s["grad_beta"],
                                workspace=space, **kw)
        return s["grad_x"], s["grad_gamma"], s["grad_beta"]
    if "q" not in s:
        s["q"] = torch.empty(s["x"].shape, dtype=torch.int8, device="cuda")
        s["q_scales"] = torch.empty(s["x"].shape[:2], device="cuda")
    space = _space(s, "workspace", lambda: ops.group_norm_workspace(s["x"], s["q"], c["groups"]))
    ops.group_norm(s["x"], s["q"], c["groups"], out_scales=s["q_scales"], workspace=space, **kw)
    q = s["q"].flatten(0, 1)
    space = _space(s, "product", lambda: ops.linear_int8_workspace(q, s["w"]))
    residual = s["x"].flatten(0, 1) if c["residual"] else None
    return ops.linear_int8(q, s["q_scales"].flatten(), s["w"], s["w_scales"], s["out"], bias=s["b"], residual=residual, workspace=space)


def run(state):
    if own:
        return _own(state)
    return {"linear": _plain_linear, "norm": _plain_norm, "backward": _plain_backward, "block": _plain_block}[state["case"]["op"]](state)


# -- what a pass cannot do without --------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "linear":
        m, k, n = case["rows"], case["in_c"], case["out_c"]
        rows = m * k * size if case["quantize"] else m * (k + 4)
        return {"bytes": rows + n * (k + 4) + size * m * n * (2 if case["residual"] else 1) + (4 * n if case["bias"] else 0), "flops": 2 * m * k * n}
    places = case["batch"] * case["positions"]
    on = {"none": lambda: places, "lengths": lambda: sum(_lengths(case)), "boards": lambda: sum(v * v for v in _sides(case))}[case["mask"]]()
    c = case["channels"]
    if case["op"] == "norm":
        return {"bytes": size * (on + places) * c + 8 * c, "flops": 8 * on * c}
    if case["op"] == "backward":
        return {"bytes": size * (2 * on + places) * c + 8 * case["batch"] * case["groups"] + 16 * c, "flops": 20 * on * c}
    n = case["out_c"]
    return {"bytes": size * (places if case["residual"] else on) * c + 8 * c + n * (c + 8) + size * places * n, "flops": 2 * places * c * n}


# -- the definitions in 64 bits -----------------------------------------------

def _exact_activation(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "mish":
        return z * torch.tanh(torch.logaddexp(z, torch.zeros_like(z)))
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * torch.erfc(-z / math.sqrt(2.0))
    return z


def _exact_derivative(z, act):
    if act == "relu":
        return torch.where(z > 0, 1.0, 0.0).double()
    if act == "mish":
        w = torch.tanh(torch.logaddexp(z, torch.zeros_like(z)))
        return w + z * torch.sigmoid(z) * (1 - w.square())
    if act == "silu":
        return torch.sigmoid(z) + z * torch.sigmoid(z) * torch.sigmoid(-z)
    if act == "gelu":
        return 0.5 * torch.erfc(-z / math.sqrt(2.0)) + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def _exact_rows(y):
    """(whole numbers, scales) of rows: the factor and its products are fp32
    numbers by definition."""
    most = y.abs().max(1).values
    factor = (127.0 / most).float().double()
    factor[most == 0] = 0.0
    return torch.round((y * factor[:, None]).float().double()), most / 127.0


def _exact_product(s, q, scales):
    z = torch.mm(q.double(), s["w"].double().t().contiguous())
    z = z * torch.outer(scales.double(), s["w_scales"].double())
    return z if s["b"] is None else z + s["b"].double()


def _exact_normal(s, item):
    """An item's positions that take part, its values there in groups, and these
    normalised."""
    c = s["case"]
    if s["mask"] is not None:
        keep = s["mask"][item].nonzero()[:, 0]
    else:
        keep = torch.arange(c["positions"] if s["lengths"] is None else int(s["lengths"][item]), device="cuda")
    x = s["x"][item, keep].double().reshape(len(keep), c["groups"], c["channels"] // c["groups"])
    if not len(keep):
        return keep, x, None
    dev = torch.sqrt(x.var((0, 2), correction=0) + EPS)
    return keep, (x - x.mean((0, 2))[None, :, None]) / dev[None, :, None], dev


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        out = torch.empty(case["rows"], case["out_c"], dtype=torch.float64, device="cuda")
        for i in range(0, case["rows"], 4096):
            rows = s["x"][i:i + 4096]
            q, scales = _exact_rows(rows.double()) if case["quantize"] else (rows, s["x_scales"][i:i + 4096])
            z = _exact_activation(_exact_product(s, q, scales), case["act"])
            out[i:i + 4096] = z + s["residual"][i:i + 4096].double() if case["residual"] else z
        return out
    b, p, c = case["batch"], case["positions"], case["channels"]
    gamma, beta = s["gamma"].double(), s["beta"].double()
    out = torch.zeros(b, p, c, dtype=torch.float64, device="cuda")
    if case["op"] == "backward":
        d_gamma, d_beta = torch.zeros_like(gamma), torch.zeros_like(beta)
        for i in range(b):
            keep, h, dev = _exact_normal(s, i)
            if not len(keep):
                continue
            flat = h.flatten(1)
            grad = s["grad"][i, keep].double() * _exact_derivative(flat * gamma + beta, case["act"])
            d_gamma += (grad * flat).sum(0)
            d_beta += grad.sum(0)
            u = (grad * gamma).view_as(h)
            u = u - u.mean((0, 2))[None, :, None] - h * (u * h).mean((0, 2))[None, :, None]
            out[i, keep] = (u / dev[None, :, None]).flatten(1)
        return out, d_gamma, d_beta
    for i in range(b):
        keep, h, _ = _exact_normal(s, i)
        if len(keep):
            out[i, keep] = _exact_activation(h.flatten(1) * gamma + beta, case["act"])
    if case["op"] == "norm":
        return out
    q, scales = _exact_rows(out.flatten(0, 1))
    z = _exact_product(s, q, scales)
    return z + s["x"].double().flatten(0, 1) if case["residual"] else z

"""The workloads that the device-level operators of this backend are measured on.

A case is one call of one operator on tensors that are already on the GPU, as a
program makes it that builds transformer blocks around the nets it evaluates
(``katago_amd.ops``): a matrix product with its epilogue, rotary positions with
several axes, and attention to an encoder's states. With ``own`` false the same
outputs come from elementary torch operations in 32 bits.

A case:
  op          "linear", "rope" or "attention"
  dtype       "fp32", "fp16" or "bf16": inputs and outputs
  linear      rows, in_c, out_c; act ("identity", "relu", "mish", "silu", "gelu");
              bias, residual (truth values); pad: channels between rows
  rope        tokens, heads, dim, pairs, axes; tables: frequency tables (heads of
              a group share one); layout: "interleaved" or "halves"; far: largest
              position; pad: channels between tokens (rows of a larger tensor)
  attention   batch, lq, lk, heads, kv_heads, dq, dv; mask: "none", "lengths"
              (padded encoder states, some empty where `least` is 0) or "boards"
              (square boards of several sides in one grid); least: the smallest
              length as a share of lk; pad: channels between tokens
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ACTS = ("identity", "relu", "mish", "silu", "gelu")


def _linear(name, dtype, rows, in_c, out_c, act="identity", bias=True, residual=False, pad=0):
    return {"name": name, "op": "linear", "dtype": dtype, "rows": rows, "in_c": in_c, "out_c": out_c, "act": act, "bias": bias,
            "residual": residual, "pad": pad}


def _rope(name, dtype, tokens, heads, dim, pairs, axes, tables=1, layout="interleaved", far=19, pad=0):
    return {"name": name, "op": "rope", "dtype": dtype, "tokens": tokens, "heads": heads, "dim": dim, "pairs": pairs, "axes": axes,
            "tables": tables, "layout": layout, "far": far, "pad": pad}


def _attention(name, dtype, batch, lq, lk, heads, kv_heads, dq, dv, mask="none", least=1.0, pad=0):
    return {"name": name, "op": "attention", "dtype": dtype, "batch": batch, "lq": lq, "lk": lk, "heads": heads,
            "kv_heads": kv_heads, "dq": dq, "dv": dv, "mask": mask, "least": least, "pad": pad}


def listed():
    return [
        # One token through a feed-forward layer of the 384-channel transformer: latency.
        _linear("linear fp16 1x384x1024 silu", "fp16", 1, 384, 1024, "silu"),
        # A serving step of eight streams: the weights are read once.
        _linear("linear bf16 8x4096x8192 gelu", "bf16", 8, 4096, 8192, "gelu"),
        # The second feed-forward layer over eight boards of 19x19 in fp32, added to the trunk.
        _linear("linear fp32 2888x1024x384 res", "fp32", 2888, 1024, 384, "identity", True, True),
        # A prompt through a wide layer, everything in the epilogue.
        _linear("linear bf16 8192x4096x8192", "bf16", 8192, 4096, 8192, "gelu", True, True),
        # The query of one token.
        _rope("rope fp16 1 token", "fp16", 1, 6, 64, 32, 2, 6),
        # Queries and keys of 128 boards, in place of the fused projection's rows, learned frequencies.
        _rope("rope fp16 128 boards", "fp16", 128 * 361, 12, 64, 32, 2, 6, pad=384),
        # A video's patches: time, height and width, halves of a head rotated against each other.
        _rope("rope bf16 video", "bf16", 20011, 32, 128, 64, 3, 1, "halves", 4096),
        # One query to the states of a board.
        _attention("attention fp16 1 query", "fp16", 1, 1, 361, 6, 6, 64, 64),
        # A decoding step of 32 streams, each with its own length of encoder states.
        _attention("attention bf16 32 streams", "bf16", 32, 1, 4096, 32, 8, 128, 128, "lengths", 0.25),
        # 64 boards' positions to the states of boards of several sizes.
        _attention("attention fp16 64 boards", "fp16", 64, 361, 361, 6, 6, 64, 64, "boards", pad=384),
        # A long text to a long encoding, grouped heads.
        _attention("attention bf16 4096x5000", "bf16", 2, 4096, 5000, 32, 8, 128, 128),
        # Eight boards in fp32 to shorter states.
        _attention("attention fp32 8 boards", "fp32", 8, 361, 169, 6, 6, 64, 64, "lengths", 0.5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges: sizes over their logarithm, odd and
    even, every type, activation, layout and mask."""
    op = rng.choice(("linear", "linear", "rope", "attention", "attention"))
    dtype = rng.choice(("fp16", "bf16", "bf16", "fp32")) if op != "rope" else rng.choice(tuple(DTYPES))
    whole = rng.random() < 0.7  # widths in eights, as most nets have them
    if op == "linear":
        rows = _log(rng, 1, 8192)
        most = 1 << (23 if dtype == "fp32" else 25)  # weights
        in_c = _log(rng, 24, 8192)
        out_c = max(1, min(_log(rng, 24, 8192), most // in_c))
        if whole:
            in_c, out_c = max(8, in_c // 8 * 8), max(8, out_c // 8 * 8)
        return _linear("", dtype, rows, in_c, out_c, rng.choice(ACTS), rng.random() < 0.7, rng.random() < 0.4, rng.choice((0, 0, 64, 7)))
    if op == "rope":
        tokens, heads = _log(rng, 1, 46208), _log(rng, 1, 40)
        pairs = rng.randint(8, 64)
        pairs = pairs // 4 * 4 if whole else pairs
        dim = 2 * pairs + rng.choice((0, 0, 0, 8, 1 if not whole else 16))
        tokens = max(1, min(tokens, 150_000_000 // (heads * dim * (2 if dtype != "fp32" else 4))))
        tables = rng.choice([t for t in (1, 2, heads) if heads % t == 0])
        return _rope("", dtype, tokens, heads, dim, pairs, rng.randint(1, 4), tables, rng.choice(("interleaved", "halves")),
                     _log(rng, 2, 1 << 20), rng.choice((0, 0, 64, 3)))
    kv_heads = rng.choice((1, 2, 4, 6, 8))
    heads = kv_heads * rng.choice((1, 1, 2, 4))
    dq = rng.choice((32, 64, 64, 80, 128, 128)) if whole else rng.randint(9, 128)
    dv = dq if rng.random() < 0.8 else rng.choice((16, 32, 64, 128))
    lq = 1 if rng.random() < 0.4 else _log(rng, 1, 4096)
    mask = rng.choice(("none", "lengths", "lengths", "boards"))
    lk = rng.randint(7, 25) ** 2 if mask == "boards" else _log(rng, 1, 16384)
    batch = _log(rng, 1, 64)
    room = min(1.3e9, (4e10 if dtype == "fp32" else 2e11) / (dq + dv))  # scores
    size = 4 if dtype == "fp32" else 2
    batch = max(1, min(batch, int(room / (heads * lq * lk)), int(3.5e8 / ((lk * kv_heads + lq * heads) * (dq + dv) * size))))
    lq = max(1, min(lq, int(room / (batch * heads * lk))))
    return _attention("", dtype, batch, lq, lk, heads, kv_heads, dq, dv, mask, rng.choice((0.0, 0.3, 0.9)) if mask == "lengths" else 1.0,
                      rng.choice((0, 0, 64, 5)))


# -- inputs -------------------------------------------------------------------

def _lengths(case):
    """Valid encoder states of each item, from the smallest share to all."""
    n, most = case["batch"], case["lk"]
    low, step = case["least"] * most, 7 if n % 7 else 11
    return [int(low + (most - low) * ((step * i + 3) % n) / (n - 1)) for i in range(n)] if n > 1 else [most]


def _sides(case):
    """Boards of three sides in a square grid, cycled over the items."""
    grid = math.isqrt(case["lk"])
    return [max(1, (grid, grid * 2 // 3, grid // 2)[i % 3]) for i in range(case["batch"])]


def _rows(g, shape, pad, dtype, scale=1.0):
    """Normal values; rows of the last two axes lie `pad` channels apart."""
    outer, (heads, dim) = shape[:-2], shape[-2:]
    row = torch.randn(*outer, heads * dim + pad, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)
    return row[..., :heads * dim].unflatten(-1, (heads, dim))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = DTYPES[case["dtype"]]
    if case["op"] == "linear":
        m, k, n, pad = case["rows"], case["in_c"], case["out_c"], case["pad"]
        # Weights of a trained net's size: products of unit rows are of unit size.
        s = {"case": case, "x": _rows(g, (m, 1, k), pad, t)[:, 0], "w": _rows(g, (n, 1, k), pad, t, k ** -0.5)[:, 0],
             "bias": torch.randn(n, generator=g, device="cuda") * 0.3 if case["bias"] else None,
             "residual": _rows(g, (m, 1, n), pad, t)[:, 0] if case["residual"] else None,
             "out": torch.empty(m, n + pad, device="cuda", dtype=t)[:, :n]}
        return s
    if case["op"] == "rope":
        n, a, far = case["tokens"], case["axes"], case["far"]
        # Axes of a grid: the first one runs slowest and goes farthest.
        at = torch.randint(0, far, (n, a), generator=g, device="cuda", dtype=torch.int32)
        p = torch.arange(case["pairs"], device="cuda", dtype=torch.float32)
        if case["tables"] > 1:  # learned: every pair turns with every axis
            freqs = torch.randn(case["tables"], case["pairs"], a, generator=g, device="cuda") * 0.5
        else:  # each axis has a run of the pairs, from fast to slow
            theta = 10000.0 ** (-p / max(1, case["pairs"]))
            runs = torch.arange(case["pairs"], device="cuda") * a // case["pairs"]
            freqs = torch.zeros(1, case["pairs"], a, device="cuda").scatter_(2, runs.view(1, -1, 1), theta.view(1, -1, 1))
        x = _rows(g, (n, case["heads"], case["dim"]), case["pad"], t)
        return {"case": case, "x": x, "positions": at, "freqs": freqs, "out": torch.empty(n, case["heads"], case["dim"], device="cuda", dtype=t)}
    b, lq, lk, pad = case["batch"], case["lq"], case["lk"], case["pad"]
    s = {"case": case, "q": _rows(g, (b, lq, case["heads"], case["dq"]), pad, t, 1.5),
         "k": _rows(g, (b, lk, case["kv_heads"], case["dq"]), pad, t, 1.5),
         "v": _rows(g, (b, lk, case["kv_heads"], case["dv"]), pad, t),
         "lengths": None, "mask": None,
         "out": torch.empty(b, lq, case["heads"], case["dv"], device="cuda", dtype=t)}
    if case["mask"] == "lengths":
        s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
        # What lies behind an item's states was never written.
        behind = torch.arange(lk, device="cuda") >= s["lengths"][:, None]
        s["k"].masked_fill_(behind[:, :, None, None], math.nan)
        s["v"].masked_fill_(behind[:, :, None, None], math.nan)
    elif case["mask"] == "boards":
        grid = math.isqrt(lk)
        side = torch.tensor(_sides(case), device="cuda")[:, None]
        at = torch.arange(lk, device="cuda")
        s["mask"] = (at // grid < side) & (at % grid < side)
    return s


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


def _plain_linear(s):
    v = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        v = v + s["bias"]
    v = _activate(v, s["case"]["act"])
    if s["residual"] is not None:
        v = v + s["residual"].float()
    return v.to(s["x"].dtype)


def _plain_rope(s):
    c = s["case"]
    x, p = s["x"].float(), c["pairs"]
    # Far positions turn many times: angles in 64 bits.
    angle = (s["positions"].double()[:, None, None, :] * s["freqs"].double()).sum(-1)
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    group = c["heads"] // c["tables"]
    cos, sin = cos.repeat_interleave(group, 1), sin.repeat_interleave(group, 1)
    if c["layout"] == "interleaved":
        x0, x1 = x[..., 0:2 * p:2], x[..., 1:2 * p:2]
    else:
        x0, x1 = x[..., :p], x[..., p:2 * p]
    y0, y1 = x0 * cos - x1 * sin, x0 * sin + x1 * cos
    turned = torch.stack((y0, y1), -1).flatten(-2) if c["layout"] == "interleaved" else torch.cat((y0, y1), -1)
    return torch.cat((turned, x[..., 2 * p:]), -1).to(s["x"].dtype)


def _valid(s):
    """Which keys an item attends to, or None for all."""
    if s["mask"] is not None:
        return s["mask"]
    if s["lengths"] is not None:
        return torch.arange(s["k"].shape[1], device="cuda") < s["lengths"][:, None]
    return None


def _plain_attention(s):
    c = s["case"]
    group = c["heads"] // c["kv_heads"]
    on = _valid(s)
    k, v = s["k"].float(), s["v"].float()
    if on is not None:
        k, v = k.masked_fill(~on[:, :, None, None], 0), v.masked_fill(~on[:, :, None, None], 0)
    # Heads of a group share their keys: (batch, kv head, group and query, ...).
    q = s["q"].float().unflatten(2, (c["kv_heads"], group)).permute(0, 2, 3, 1, 4).flatten(2, 3).contiguous()
    score = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * (c["dq"] ** -0.5)
    if on is not None:
        score = score.masked_fill(~on[:, None, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - top.masked_fill(top == -math.inf, 0))
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e, v.permute(0, 2, 1, 3).contiguous()) / total.masked_fill(total == 0, 1)
    return out.unflatten(2, (group, c["lq"])).permute(0, 3, 1, 2, 4).flatten(2, 3).to(s["q"].dtype)


# -- the framework's operators ------------------------------------------------

def _own(s):
    from katago_amd import ops

    c = s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "linear":
        if "workspace" not in s:  # kept with the layer
            need = ops.linear_workspace(s["x"], s["w"])
            s["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
        return ops.linear(s["x"], s["w"], s["out"], bias=s["bias"], activation=c["act"], residual=s["residual"],
                          workspace=s["workspace"], stream=stream)
    if c["op"] == "rope":
        return ops.rope_axes(s["x"], s["positions"], s["freqs"], s["out"], layout=c["layout"], stream=stream)
    if "workspace" not in s:  # kept with the layer
        need = ops.cross_attention_workspace(s["q"], s["k"], s["v"])
        s["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
    return ops.cross_attention(s["q"], s["k"], s["v"], s["out"], key_lengths=s["lengths"], key_mask=s["mask"],
                               workspace=s["workspace"], stream=stream)


def run(state):
    if own:
        return _own(state)
    return {"linear": _plain_linear, "rope": _plain_rope, "attention": _plain_attention}[state["case"]["op"]](state)


# -- what a pass cannot do without --------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "linear":
        m, k, n = case["rows"], case["in_c"], case["out_c"]
        return {"bytes": size * (m * k + k * n + m * n * (2 if case["residual"] else 1)) + (4 * n if case["bias"] else 0), "flops": 2 * m * k * n}
    if case["op"] == "rope":
        values = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * size * values + 4 * case["axes"] * (case["tokens"] + case["tables"] * case["pairs"]),
                "flops": 6 * case["tokens"] * case["heads"] * case["pairs"]}
    keys = {"none": lambda: case["batch"] * case["lk"], "lengths": lambda: sum(_lengths(case)),
            "boards": lambda: sum(v * v for v in _sides(case))}[case["mask"]]()
    dims = case["dq"] + case["dv"]
    return {"bytes": size * (case["batch"] * case["lq"] * case["heads"] + keys * case["kv_heads"]) * dims,
            "flops": 2 * case["heads"] * case["lq"] * keys * dims}


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


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        wt = s["w"].double().t().contiguous()
        out = torch.empty(case["rows"], case["out_c"], dtype=torch.float64, device="cuda")
        for i in range(0, case["rows"], 1024):
            z = torch.mm(s["x"][i:i + 1024].double(), wt)
            if case["bias"]:
                z += s["bias"].double()
            z = _exact_activation(z, case["act"])
            out[i:i + 1024] = z + s["residual"][i:i + 1024].double() if case["residual"] else z
        return out
    if case["op"] == "rope":
        p, group = case["pairs"], case["heads"] // case["tables"]
        out = s["x"].double()
        for i in range(0, case["tokens"], 4096):
            at = s["positions"][i:i + 4096].double()
            for h in range(case["heads"]):
                angle = at @ s["freqs"][h // group].double().t().contiguous()
                turn = torch.polar(torch.ones_like(angle), angle)
                x = out[i:i + 4096, h]
                if case["layout"] == "interleaved":
                    z = torch.complex(x[:, 0:2 * p:2].contiguous(), x[:, 1:2 * p:2].contiguous()) * turn
                    x[:, 0:2 * p:2], x[:, 1:2 * p:2] = z.real, z.imag
                else:
                    z = torch.complex(x[:, :p].contiguous(), x[:, p:2 * p].contiguous()) * turn
                    x[:, :p], x[:, p:2 * p] = z.real, z.imag
        return out
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(case["batch"], case["lq"], case["heads"], case["dv"], dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        if s["mask"] is not None:
            keep = s["mask"][b].nonzero()[:, 0]
        else:
            keep = torch.arange(case["lk"] if s["lengths"] is None else int(s["lengths"][b]), device="cuda")
        if not len(keep):
            continue
        for h in range(case["heads"]):
            k, v = s["k"][b, keep, h // group].double(), s["v"][b, keep, h // group].double()
            z = torch.mm(s["q"][b, :, h].double(), k.t().contiguous()) / math.sqrt(case["dq"])
            out[b, :, h] = torch.mm(torch.softmax(z, -1), v)
    return out

"""Operators of an image / video transformer's training and serving step: what they compute, in plain torch operations,
the sizes they are measured at, and the calls a user makes of this framework's kernels for them.

  layer norm     h = (s - mean(s)) / sqrt(var(s) + eps) * w + b with s = x (+ delta), the residual sum a transformer block
                 forms on the way; the gradients of x, delta, w and b
  rotary axes    rotary positions whose angles come from several position axes (time, height, width): each pair of a head
                 turns by position[axis of the pair] * frequency of the pair; q and k in one call, apart or as parts of a
                 fused q / k / v projection, and the inverse turn of their gradients
  fp8 linear     y = x W^T + b with both operands in e4m3 and a power-of-two scale for each block of 128: 1 x 128 blocks
                 of the activation and of the gradient along the contraction, 128 x 128 blocks of the weight; dx, dW, db;
                 the serving form takes a weight that was packed once

`own = False` runs the plain forms (32-bit arithmetic on the inputs as they are), `own = True` the framework's kernels.
"""
import math
import os
import sys

import torch

own = False
DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _framework():
    folder = os.path.join(os.getcwd(), "sm120-nvfp4-training_b200")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import nvfp4_training
    return nvfp4_training


# ---- the cases ------------------------------------------------------------------------------------------------------
def _norm(name, rows, cols, x, delta, out, train):
    return dict(name=name, op="norm", rows=rows, cols=cols, x=x, delta=delta, out=out, train=train)


def _rotary(name, batch, seq, heads, kv_heads, dim, sections, layout, frequencies, dtype, fused, train, far=0):
    return dict(name=name, op="rotary", batch=batch, seq=seq, heads=heads, kv_heads=kv_heads, dim=dim, sections=sections, layout=layout,
                frequencies=frequencies, dtype=dtype, fused=fused, train=train, far=far)


def _linear(name, tokens, inputs, outputs, dtype, bias, train):
    return dict(name=name, op="linear", tokens=tokens, inputs=inputs, outputs=outputs, dtype=dtype, bias=bias, train=train)


def listed():
    return [
        # the block entry of a few tokens being generated: residual sum and norm, latency only
        _norm("norm_4_tokens", 4, 4096, "bf16", "bf16", "bf16", False),
        # GPT-2-small width at 16 sequences of 1024: an FP32 residual stream, BF16 branch and BF16 result, as under autocast
        _norm("norm_autocast_train", 16384, 768, "fp32", "bf16", "bf16", True),
        # a ragged batch of a model whose width suits no vector load
        _norm("norm_odd_train", 2051, 1027, "fp16", "", "fp16", True),
        # a wide model's training step, everything in BF16
        _norm("norm_wide_train", 16384, 5120, "bf16", "bf16", "bf16", True),
        # one generated token at a far time position of a vision language model, grouped key heads
        _rotary("rotary_1_token", 1, 1, 32, 8, 128, "16,24,24", "half", "shared", "bf16", False, False, far=1000000),
        # image training: fused projection in, one gradient of it out; 24 heads of 128 as in the decoder
        _rotary("rotary_image_train", 4, 4352, 24, 24, 128, "8,28,28", "interleaved", "axis", "bf16", True, True),
        # a small FP32 encoder whose heads turn only in part, ragged length
        _rotary("rotary_partial_fp32", 3, 1021, 16, 16, 72, "16,16", "half", "axis", "fp32", False, True),
        # a video of 21 x 45 x 80 latent positions, forward only
        _rotary("rotary_video", 1, 75600, 40, 40, 128, "22,21,21", "interleaved", "axis", "bf16", False, False),
        # one token against a weight that was packed when the model was loaded
        _linear("linear_1_token", 1, 4096, 4096, "bf16", False, False),
        # a ragged batch through odd widths, with its bias, forward and backward
        _linear("linear_odd_train", 1000, 1152, 4304, "bf16", True, True),
        # the layer of the framework's GEMM benchmark: 8192 tokens, 4096 x 4096, the whole training step's three products
        _linear("linear_square_train", 8192, 4096, 4096, "bf16", False, True),
        # a feed-forward layer's training step
        _linear("linear_ffn_train", 16384, 4096, 14336, "bf16", False, True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "rotary", "linear"])
    if op == "norm":
        cols = _log(rng, 64, 8192)
        if rng.random() < 0.75:
            cols = (cols + 7) // 8 * 8
        rows = max(1, min(_log(rng, 1, 32768), 16384 * 5120 // cols))
        x, delta, out = rng.choice([("bf16", "", "bf16"), ("bf16", "bf16", "bf16"), ("fp16", "fp16", "fp16"), ("fp32", "fp32", "fp32"),
                                    ("fp32", "", "bf16"), ("fp32", "bf16", "bf16"), ("fp32", "bf16", "fp32")])
        case = _norm("", rows, cols, x, delta, out, rng.random() < 0.6)
        if x == "fp32" or (cols % 8 and rows * cols > 2 ** 23):   # wider types and odd widths within the largest case's cost
            case["rows"] = max(1, min(rows, 2 ** 25 // cols))
    elif op == "rotary":
        dim = rng.choice([32, 64, 72, 80, 96, 128, 256])
        axes = rng.choice([1, 2, 3, 3, 4])
        pairs = dim // 2 if rng.random() < 0.7 else max(axes, dim // 4)
        cuts = sorted(rng.sample(range(1, pairs), axes - 1))
        sections = [b - a for a, b in zip([0] + cuts, cuts + [pairs])]
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 3, 4, 5])
        batch = rng.choice([1, 1, 2, 3, 4])
        seq = _log(rng, 1, 32768)
        seq = max(1, min(seq, 75600 * 80 * 128 // 4 // (batch * (heads + 2 * kv) * dim)))
        case = _rotary("", batch, seq, heads, kv, dim, ",".join(map(str, sections)), rng.choice(["half", "interleaved"]),
                       rng.choice(["shared", "axis"]), rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.random() < 0.5, rng.random() < 0.5,
                       far=rng.choice([0, 0, 100000, 1000000]))
    else:
        train = rng.random() < 0.6
        inputs, outputs = _log(rng, 128, 8192), _log(rng, 128, 8192)
        if rng.random() < 0.7:
            inputs, outputs = (inputs + 15) // 16 * 16, (outputs + 15) // 16 * 16
        tokens = max(1, min(_log(rng, 1, 16384), 2 ** 38 // (inputs * outputs)))
        case = _linear("", tokens, inputs, outputs, rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"]), rng.random() < 0.4, train)
    del case["name"]
    return case


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4, "": 0}
    if case["op"] == "norm":
        n = case["rows"] * case["cols"]
        sx, sd, so = size[case["x"]], size[case["delta"]], size[case["out"]]
        total = sx if case["delta"] else 0
        moved = n * (sx + sd + total + so)                       # x, delta in; sum, h out
        flops = 9 * n
        if case["train"]:                                      # dh, d sum in, dx, d delta out; the sum is read again
            apart = sd if (case["delta"] and case["delta"] != case["x"]) else 0   # d delta is dx itself where the types agree
            moved += n * (so + sx + (sx if case["delta"] else 0) + sx + apart)
            flops += 16 * n
        return dict(bytes=moved + 8 * case["cols"], flops=flops)
    if case["op"] == "rotary":
        tokens = case["batch"] * case["seq"]
        s = size[case["dtype"]]
        turned = tokens * (case["heads"] + case["kv_heads"]) * case["dim"]
        moved = 2 * turned * s + tokens * 8 * len(case["sections"].split(","))
        flops = 3 * turned
        if case["train"]:
            moved += 2 * turned * s + (2 * tokens * case["kv_heads"] * case["dim"] * s if case["fused"] else 0)
            flops += 3 * turned
        return dict(bytes=moved, flops=flops)
    m, k, n = case["tokens"], case["inputs"], case["outputs"]
    s = size[case["dtype"]]
    if not case["train"]:
        return dict(bytes=n * k + (m * k + m * n) * s, flops=2 * m * n * k)
    return dict(bytes=(2 * m * k + 2 * m * n + 2 * n * k) * s, flops=6 * m * n * k)   # x, w, dy in; y, dx, dw out


# ---- the inputs -----------------------------------------------------------------------------------------------------
def _grid_positions(batch, seq, axes, far, g):
    """Positions of a flattened grid with `axes` axes, row major, behind an offset on the first axis (the text or the
    frames that came before)."""
    side = max(1, round(seq ** (1.0 / axes)))
    t = torch.arange(seq, device=DEVICE)
    cols = []
    for a in range(axes - 1, 0, -1):
        extent = side + a
        cols.append(t % extent)
        t = t // extent
    cols.append(t)
    grid = torch.stack(cols[::-1], dim=-1)
    start = torch.randint(0, 50, (batch, 1, 1), device=DEVICE, generator=g)
    pos = grid[None].expand(batch, seq, axes).clone()
    pos[..., :1] += start + far
    return pos


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    rand = lambda *shape: torch.randn(*shape, device=DEVICE, generator=g)
    state = dict(case=dict(case))
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        x = rand(rows, cols) * (0.5 + rand(cols).abs()) + 0.3 * rand(cols)      # channels of different size and offset
        state["x"] = x.to(DTYPES[case["x"]])
        state["delta"] = (0.5 * rand(rows, cols)).to(DTYPES[case["delta"]]) if case["delta"] else None
        state["w"], state["b"] = 1 + 0.1 * rand(cols), 0.1 * rand(cols)
        if case["train"]:
            state["dh"] = (rand(rows, cols) * torch.exp(rand(rows, 1))).to(DTYPES[case["out"]])
            state["dsum"] = rand(rows, cols).to(DTYPES[case["x"]]) if case["delta"] else None
    elif case["op"] == "rotary":
        b, s, h, hk, d = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["dim"]
        dt = DTYPES[case["dtype"]]
        state["sections"] = tuple(int(v) for v in case["sections"].split(","))
        state["positions"] = _grid_positions(b, s, len(state["sections"]), case["far"], g)
        if case["fused"]:
            state["qkv"] = rand(b, s, (h + 2 * hk) * d).to(dt)
        else:
            state["q"], state["k"] = rand(b, s, h, d).to(dt), rand(b, s, hk, d).to(dt)
        if case["train"]:
            # gradients arrive as an attention kernel leaves them: [batch, heads, seq, dim] seen as [batch, seq, heads, dim]
            state["dq"], state["dk"], state["dv"] = (rand(b, n, s, d).to(dt).transpose(1, 2) for n in (h, hk, hk))
    else:
        m, k, n = case["tokens"], case["inputs"], case["outputs"]
        dt = DTYPES[case["dtype"]]
        x = rand(m, k)
        x *= torch.exp(0.5 * rand(k))                                            # channels of different size
        state["x"] = x.to(dt)
        del x
        state["w"] = (rand(n, k) / math.sqrt(k)).to(dt)
        state["b"] = (0.1 * rand(n)).to(dt) if case["bias"] else None
        if case["train"]:
            state["dy"] = (1e-3 * rand(m, n) * torch.exp(rand(m, 1))).to(dt)    # tokens of different loss
        elif own:
            state["packed"] = _framework().fp8_pack(state["w"])
        else:
            state["packed"] = _fp8_values(state["w"], 128, 128)
    if own:
        _framework()
        for name in ("x", "delta", "w", "b", "qkv", "q", "k"):
            if case["train"] and state.get(name) is not None:
                state[name].requires_grad_(True)
    return state


# ---- plain forms ----------------------------------------------------------------------------------------------------
EPS = 1e-5


def _norm_plain(st):
    x, delta, w, b = st["x"], st["delta"], st["w"], st["b"]
    out_dtype = DTYPES[st["case"]["out"]]
    total = x if delta is None else (x.float() + delta.float()).to(x.dtype)
    s = total.float()
    centred = s - s.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    xhat = centred * rstd
    out = dict(h=(xhat * w + b).to(out_dtype))
    if delta is not None:
        out["sum"] = total
    if st["case"]["train"]:
        dh = st["dh"].float()
        u = dh * w
        dx = rstd * (u - u.mean(-1, keepdim=True) - xhat * (u * xhat).mean(-1, keepdim=True))
        if delta is not None:
            dx = dx + st["dsum"].float()
            out["ddelta"] = dx.to(delta.dtype)
        out["dx"] = dx.to(x.dtype)
        out["dw"], out["db"] = (dh * xhat).sum(0), dh.sum(0)
    return out


def _frequencies(sections, kind, theta=10000.0):
    if kind == "axis":
        exponents = torch.cat([torch.arange(n, dtype=torch.float64) / n for n in sections])
    else:
        exponents = torch.arange(sum(sections), dtype=torch.float64) / sum(sections)
    return torch.exp(-math.log(theta) * exponents).to(DEVICE)


def _angles(st):
    """[batch, seq, pairs] in 64 bits: far positions need more than 24 bits of angle."""
    sections = st["sections"]
    axis = torch.repeat_interleave(torch.arange(len(sections), device=DEVICE), torch.tensor(sections, device=DEVICE))
    return st["positions"].double()[..., axis] * _frequencies(sections, st["case"]["frequencies"])


def _turn(x, cos, sin, layout, dtype):
    """x [batch, seq, heads, dim]; cos, sin [batch, seq, 1, pairs]; features behind the turned ones pass unchanged."""
    pairs = cos.shape[-1]
    y = x.to(dtype).clone()
    if layout == "half":
        a, b = x[..., :pairs].to(dtype), x[..., pairs:2 * pairs].to(dtype)
        y[..., :pairs] = a * cos - b * sin
        y[..., pairs:2 * pairs] = b * cos + a * sin
    else:
        a, b = x[..., 0:2 * pairs:2].to(dtype), x[..., 1:2 * pairs:2].to(dtype)
        y[..., 0:2 * pairs:2] = a * cos - b * sin
        y[..., 1:2 * pairs:2] = b * cos + a * sin
    return y


def _parts(st):
    c = st["case"]
    if not c["fused"]:
        return st["q"], st["k"], None
    b, s, h, hk, d = c["batch"], c["seq"], c["heads"], c["kv_heads"], c["dim"]
    q, k, v = st["qkv"].split([h * d, hk * d, hk * d], dim=-1)
    return q.view(b, s, h, d), k.view(b, s, hk, d), v.view(b, s, hk, d)


def _rotary_math(st, dtype):
    c = st["case"]
    angles = _angles(st)[:, :, None]
    cos, sin = torch.cos(angles).to(dtype), torch.sin(angles).to(dtype)
    del angles
    q, k, v = _parts(st)
    turn = lambda t, sn: _turn(t, cos, sn, c["layout"], dtype).to(t.dtype if dtype == torch.float32 else dtype)
    out = dict(q=turn(q, sin), k=turn(k, sin))
    if v is not None:
        out["v"] = v if dtype == torch.float32 else v.to(dtype)
    if c["train"]:
        back = [turn(st["dq"], -sin), turn(st["dk"], -sin)]
        if v is not None:
            dv = st["dv"] if dtype == torch.float32 else st["dv"].to(dtype)
            out["dqkv"] = torch.cat([t.flatten(2) for t in (*back, dv)], dim=-1)
        else:
            out["dq"], out["dk"] = back
    return out


def _block_scale(amax):
    """Smallest power of two 2^e with amax / 2^e <= 448, the largest e4m3 number; e = 0 for an empty block."""
    mantissa, exponent = torch.frexp(amax)                       # amax = mantissa * 2^exponent, mantissa in [0.5, 1)
    e = exponent - 9 + (mantissa > 0.875).to(exponent.dtype)
    return torch.where(amax > 0, e.clamp(min=-127), torch.zeros_like(e))


def _blocks(x, block_rows, block_cols):
    rows, cols = x.shape
    x = torch.nn.functional.pad(x, (0, -cols % block_cols, 0, -rows % block_rows))
    return x.view(x.shape[0] // block_rows, block_rows, x.shape[1] // block_cols, block_cols)


def _fp8_values(x, block_rows, block_cols):
    """The numbers that the e4m3 codes of x stand for, in 32 bits."""
    rows, cols = x.shape
    t = _blocks(x.float(), block_rows, block_cols)
    e = _block_scale(t.abs().amax((1, 3), keepdim=True)).int()
    scale = torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22)).view(torch.float32)     # 2^e from its bits
    q = (t / scale).to(torch.float8_e4m3fn).float() * scale
    return q.reshape(t.shape[0] * t.shape[1], -1)[:rows, :cols]


def _linear_plain(st):
    x, b, dt = st["x"], st["b"], st["x"].dtype
    w = st["packed"] if not st["case"]["train"] else _fp8_values(st["w"], 128, 128)
    y = _fp8_values(x, 1, 128) @ w.t()
    if b is not None:
        y = y + b.float()
    out = dict(y=y.to(dt))
    if st["case"]["train"]:
        dy = st["dy"]
        out["dx"] = (_fp8_values(dy, 1, 128) @ w).to(dt)
        out["dw"] = (_fp8_values(dy, 128, 1).t() @ _fp8_values(x, 128, 1)).to(dt)
        if b is not None:
            out["db"] = dy.float().sum(0).to(b.dtype)
    return out


# ---- the framework's calls ------------------------------------------------------------------------------------------
def _norm_own(st):
    nv, c = _framework(), st["case"]
    x, delta, w, b = st["x"], st["delta"], st["w"], st["b"]
    out_dtype = DTYPES[c["out"]]
    if not c["train"]:
        with torch.no_grad():
            if delta is None:
                return dict(h=nv.layer_norm(x, w, b, eps=EPS, out_dtype=out_dtype))
            total, h = nv.add_layer_norm(x, delta, w, b, eps=EPS, out_dtype=out_dtype)
            return dict(h=h, sum=total)
    if delta is None:
        h = nv.layer_norm(x, w, b, eps=EPS, out_dtype=out_dtype)
        dx, dw, db = torch.autograd.grad(h, (x, w, b), st["dh"])
        return dict(h=h.detach(), dx=dx, dw=dw, db=db)
    total, h = nv.add_layer_norm(x, delta, w, b, eps=EPS, out_dtype=out_dtype)
    dx, dd, dw, db = torch.autograd.grad((h, total), (x, delta, w, b), (st["dh"], st["dsum"]))
    return dict(h=h.detach(), sum=total.detach(), ddelta=dd, dx=dx, dw=dw, db=db)


def _rotary_own(st):
    nv, c = _framework(), st["case"]
    how = dict(layout=c["layout"], frequencies=c["frequencies"])
    with torch.set_grad_enabled(c["train"]):
        if c["fused"]:
            q, k, v = nv.rotary_axes_qkv(st["qkv"], st["positions"], st["sections"], c["heads"], c["kv_heads"], **how)
        else:
            (q, k), v = nv.rotary_axes(st["q"], st["k"], st["positions"], st["sections"], **how), None
    out = dict(q=q.detach(), k=k.detach())
    if v is not None:
        out["v"] = v.detach()
    if c["train"]:
        if v is not None:
            out["dqkv"], = torch.autograd.grad((q, k, v), st["qkv"], (st["dq"], st["dk"], st["dv"]))
        else:
            out["dq"], out["dk"] = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["dq"], st["dk"]))
    return out


def _linear_own(st):
    nv = _framework()
    if not st["case"]["train"]:
        with torch.no_grad():
            return dict(y=nv.fp8_linear(st["x"], st["packed"], st["b"]))
    leaves = [st["x"], st["w"]] + ([st["b"]] if st["b"] is not None else [])
    y = nv.fp8_linear(st["x"], st["w"], st["b"])
    return dict(zip(["y", "dx", "dw", "db"], [y.detach(), *torch.autograd.grad(y, leaves, st["dy"])]))


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _norm_own, "rotary": _rotary_own, "linear": _linear_own}[op](state)
    with torch.no_grad():
        if op == "norm":
            return _norm_plain(state)
        return _rotary_math(state, torch.float32) if op == "rotary" else _linear_plain(state)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------
def _norm_exact(st):
    x, delta, w, b = st["x"].double(), st["delta"], st["w"].double(), st["b"].double()
    n = x.shape[1]
    out = {}
    s = x
    if delta is not None:
        total = (st["x"].float() + delta.float()).to(st["x"].dtype)     # the residual stream is held in x's type
        out["sum"] = x + delta.double()
        s = total.double()
    mu = s.sum(-1, keepdim=True) / n
    var = ((s - mu) ** 2).sum(-1, keepdim=True) / n
    z = (s - mu) / (var + EPS) ** 0.5
    out["h"] = z * w + b
    if st["case"]["train"]:
        dh = st["dh"].double()
        dz = dh * w
        # d/ds of (s - mu) / sigma, written out as the projection off the constant and off z
        ds = (dz - dz.sum(-1, keepdim=True) / n - z * ((dz * z).sum(-1, keepdim=True) / n)) / (var + EPS) ** 0.5
        if delta is not None:
            ds = ds + st["dsum"].double()
            out["ddelta"] = ds
        out["dx"], out["dw"], out["db"] = ds, torch.einsum("ij,ij->j", dh, z), torch.einsum("ij->j", dh)
    return out


def _rotary_exact(st):
    """The turn as a product of complex numbers."""
    c, sections = st["case"], st["sections"]
    pairs = sum(sections)
    angle = torch.empty(*st["positions"].shape[:2], 1, pairs, dtype=torch.float64, device=DEVICE)
    first = 0
    for a, n in enumerate(sections):
        for i in range(n):
            j = first + i
            power = i / n if c["frequencies"] == "axis" else j / pairs
            angle[..., 0, j] = st["positions"][..., a].double() * 10000.0 ** -power
        first += n
    unit = torch.polar(torch.ones_like(angle), angle)

    def turned(t, by):
        t = t.double()
        head, rest = t[..., :2 * pairs], t[..., 2 * pairs:]
        halves = head.unflatten(-1, (2, pairs)).movedim(-2, -1) if c["layout"] == "half" else head.unflatten(-1, (pairs, 2))
        z = torch.view_as_real(torch.view_as_complex(halves.contiguous()) * by)
        z = z.movedim(-1, -2).flatten(-2) if c["layout"] == "half" else z.flatten(-2)
        return torch.cat([z, rest], dim=-1)

    q, k, v = _parts(st)
    out = dict(q=turned(q, unit), k=turned(k, unit))
    if v is not None:
        out["v"] = v.double()
    if c["train"]:
        dq, dk = turned(st["dq"], unit.conj()), turned(st["dk"], unit.conj())
        if v is not None:
            out["dqkv"] = torch.cat([dq.flatten(2), dk.flatten(2), st["dv"].double().flatten(2)], dim=-1)
        else:
            out["dq"], out["dk"] = dq, dk
    return out


def _two_to(n):
    """2^n as a float64 made from its bits (pow may be one unit off, which turns ties)."""
    return ((n.long() + 1023) << 52).view(torch.float64)


def _fp8_exact(x, along_rows, block):
    """x rounded to e4m3 under a power-of-two scale per block, in 64 bits: the grid of spacing 2^(e - 3), e at least -6."""
    t = x.double()
    rows, cols = t.shape
    br, bc = (block, block) if along_rows is None else ((1, block) if along_rows else (block, 1))
    pad = torch.zeros(-(-rows // br) * br, -(-cols // bc) * bc, dtype=torch.float64, device=DEVICE)
    pad[:rows, :cols] = t
    tiles = pad.view(pad.shape[0] // br, br, pad.shape[1] // bc, bc)
    top = tiles.abs().amax(3, keepdim=True).amax(1, keepdim=True)
    power = torch.ceil(torch.log2(torch.where(top > 0, top, torch.full_like(top, 448.0)) / 448.0))
    scale = _two_to(power)
    scale = torch.where(top > 448.0 * scale, scale * 2, torch.where(top <= 224.0 * scale, scale / 2, scale))   # log2 rounds next to a border
    v = tiles / torch.where(top > 0, scale, torch.ones_like(scale))
    _, e = torch.frexp(v)
    step = _two_to((e - 1).clamp(min=-6) - 3)
    q = torch.round(v / step) * step * torch.where(top > 0, scale, torch.ones_like(scale))
    return q.view_as(pad)[:rows, :cols]


def _linear_exact(st):
    x, w = st["x"], st["w"]
    wq = _fp8_exact(w, None, 128)
    y = _fp8_exact(x, True, 128) @ wq.t()
    if st["b"] is not None:
        y = y + st["b"].double()
    out = dict(y=y)
    if st["case"]["train"]:
        dy = st["dy"]
        out["dx"] = _fp8_exact(dy, True, 128) @ wq
        out["dw"] = _fp8_exact(dy, False, 128).t() @ _fp8_exact(x, False, 128)
        if st["b"] is not None:
            out["db"] = dy.double().sum(0)
    return out


def exact(case, seed):
    if case["op"] == "rotary" and case["batch"] * case["seq"] * (case["heads"] + case["kv_heads"]) * case["dim"] > 10 ** 9:
        return None      # 64-bit complex copies of the largest calls would not leave room for anything else
    global own
    asked, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = asked
    with torch.no_grad():
        if case["op"] == "norm":
            return _norm_exact(st)
        return _rotary_exact(st) if case["op"] == "rotary" else _linear_exact(st)

"""The operators of a context layer over all the tokens of a study, and of its training.

The encoder's last map has 256 positions an image at 512 px and 81 at 288 px, so a 24-slice study is 6144
tokens and one of 88 windows 22528.  A transformer layer over them normalises rows, turns queries and keys
by each token's slice, row and column, attends within a window of neighbours plus a few first summary
tokens, and is trained with AdamW.  `run` computes each operator in its plain form, from elementary torch
operations in 32 bits, or with the framework's kernels where `own` is set.
"""
from __future__ import annotations

import importlib
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5                                             # layer norm's
BASE = 10000.0                                         # rotary positions'
LR, BETA1, BETA2, ADAM_EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
BLOCK = 256                                            # elements of a tensor that share one scale
SLOTS = 8                                              # runs of tokens a study's key mask switches


# --- the cases ----------------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # one study's 88 windows at the head's context width: the smallest call, inference
        dict(name="norm_study", op="norm", rows=88, width=256, dtype="f32", train=False),
        # the features of 8 studies of 88 windows in a training step of a head on the encoder's output
        dict(name="norm_features", op="norm", rows=704, width=1664, dtype="f32", train=True),
        # the tokens of 16 24-slice studies in a training step, an odd row short
        dict(name="norm_tokens", op="norm", rows=98303, width=1024, dtype="bf16", train=True),
        # queries and keys of one 88-window study at 288 px (81 positions an image), as the layer calls it
        dict(name="rotary_study", op="rotary", batch=1, slices=88, rows=9, cols=9, heads=8, dim=64,
             dtype="bf16", inverse=False),
        # the gradient of queries and keys of 8 24-slice studies at 512 px
        dict(name="rotary_batch", op="rotary", batch=8, slices=24, rows=16, cols=16, heads=20, dim=128,
             dtype="f16", inverse=True),
        # forward over every token of one 88-window study at 512 px: two slices to either side, 12 summary
        # tokens, two of the eight slots absent
        dict(name="attention_study", op="attention", batch=1, tokens=22528, heads=4, key_heads=4, dim=64,
             dtype="bf16", left=512, right=512, sinks=12, absent=2, train=False),
        # a training step over two short studies of an odd number of tokens, shared key heads, causal
        dict(name="attention_step_small", op="attention", batch=2, tokens=2499, heads=8, key_heads=2, dim=64,
             dtype="bf16", left=511, right=0, sinks=4, absent=1, train=True),
        # a training step at the largest width: long rows, wide window, eight shared heads' gradients
        dict(name="attention_step_large", op="attention", batch=2, tokens=8199, heads=16, key_heads=4, dim=128,
             dtype="f16", left=1023, right=0, sinks=4, absent=0, train=True),
        # one new image token against one study's cache: a single request's latency
        dict(name="token_one", op="token", batch=1, cache=6144, heads=4, key_heads=4, dim=64, dtype="bf16",
             left=2047, sinks=12, shortest=6144),
        # one new token of each of 64 requests with caches of every length
        dict(name="token_many", op="token", batch=64, cache=8192, heads=32, key_heads=8, dim=128, dtype="f16",
             left=4095, sinks=4, shortest=1),
        # the head's 22 parameter tensors, full-width states
        dict(name="adamw_head", op="adamw", layers=0, width=256, dtype="f32", grad="f32", bits=32),
        # five context layers of width 1280, 60 tensors, 8-bit states, gradients as autocast leaves them
        dict(name="adamw_layers", op="adamw", layers=5, width=1280, dtype="f32", grad="bf16", bits=8),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng) -> dict:
    op = rng.choice(["norm", "rotary", "attention", "attention", "token", "adamw"])
    if op == "norm":
        width = _log(rng, 16, 8192)
        return dict(op=op, rows=_log(rng, 1, min(100000, 100_000_000 // width)), width=width,
                    dtype=rng.choice(list(TYPES)), train=rng.random() < 0.7)
    if op == "rotary":
        img = rng.randint(5, 20)
        return dict(op=op, batch=rng.randint(1, 8), slices=_log(rng, 1, 96), rows=img, cols=rng.randint(5, 20),
                    heads=rng.randint(1, 16), dim=rng.choice([32, 64, 96, 128]), dtype=rng.choice(list(TYPES)),
                    inverse=rng.random() < 0.5)
    if op == "attention":
        key_heads = rng.choice([1, 2, 4])
        heads = key_heads * rng.choice([1, 2, 4])
        tokens = _log(rng, 1, 8000)
        batch = rng.randint(1, 2 if tokens > 2000 else 4)
        left = _log(rng, 1, 2048)
        return dict(op=op, batch=batch, tokens=tokens, heads=heads, key_heads=key_heads, dim=rng.choice([64, 128]),
                    dtype=rng.choice(["bf16", "f16"]), left=left, right=rng.choice([0, 0, left]),
                    sinks=rng.choice([0, 1, 4, 12, 70]), absent=rng.choice([0, 1, 3]), train=rng.random() < 0.6)
    if op == "token":
        key_heads = rng.choice([1, 2, 4, 8])
        cache = _log(rng, 16, 16384)
        return dict(op=op, batch=_log(rng, 1, 32), cache=cache, heads=key_heads * rng.choice([1, 2, 4, 8]),
                    key_heads=key_heads, dim=rng.choice([64, 128]), dtype=rng.choice(["bf16", "f16"]),
                    left=_log(rng, 8, 8192), sinks=rng.choice([0, 1, 4, 12]), shortest=rng.randint(1, cache))
    layers = rng.randint(0, 5)
    dtype = rng.choice(["f32", "f32", "bf16"])
    return dict(op=op, layers=layers, width=256 if layers == 0 else _log(rng, 33, 1000), dtype=dtype,
                grad=rng.choice(["f32", "bf16"]), bits=rng.choice([8, 32]))


def _sections(dim: int) -> tuple[int, int, int]:
    """Pairs per axis: a quarter of the channels for the slice, three eighths each for row and column."""
    half = dim // 2
    rest = 3 * half // 8
    return half - 2 * rest, rest, rest


def _shapes(case: dict) -> list[tuple[int, ...]]:
    """The parameter tensors: the head's (no layers), or those of some context layers."""
    w = case["width"]
    layer = [(3 * w, w), (3 * w,), (w, w), (w,), (w,), (w,), (w,), (w,), (4 * w, w), (4 * w,), (w, 4 * w), (w,)]
    if case["layers"]:
        return layer * case["layers"]
    head = [(8, 1664), (w, 1664), (w,), (11, w)]
    block = [(3 * w, w), (3 * w,), (w, w), (w,), (w,), (w,), (w,), (w,), (2 * w, w), (2 * w,), (w, 2 * w), (w,)]
    return head + block + [(1664, w), (1664,), (12, 1664), (12,), (12, 1664), (12,)]


def _lengths(case: dict) -> list[int]:
    n = case["batch"]
    return [case["shortest"] + (case["cache"] - case["shortest"]) * i // max(1, n - 1) for i in range(n)]


# --- the inputs ---------------------------------------------------------------------------------
def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": case}

    def normal(*shape, dtype="f32", scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=g, device=DEV) * scale + shift).to(TYPES[dtype])

    if case["op"] == "norm":
        rows, width, t = case["rows"], case["width"], case["dtype"]
        s |= dict(x=normal(rows, width, dtype=t, scale=1.5, shift=0.3), weight=normal(width, scale=0.1, shift=1.0),
                  bias=normal(width, scale=0.1))
        if case["train"]:
            s["dy"] = normal(rows, width, dtype=t)
    elif case["op"] == "rotary":
        b, z, y, x = case["batch"], case["slices"], case["rows"], case["cols"]
        grid = torch.stack(torch.meshgrid(torch.arange(z), torch.arange(y), torch.arange(x), indexing="ij"), -1)
        pos = grid.reshape(-1, 3).to(DEV, torch.int32)
        # studies begin at slices of their own, so each has its own positions
        first = torch.randint(0, 32, (b, 1, 1), generator=g, device=DEV, dtype=torch.int32)
        s["pos"] = (pos[None] + torch.cat([first, torch.zeros_like(first), torch.zeros_like(first)], -1)).contiguous()
        s["x"] = normal(b, z * y * x, case["heads"], case["dim"], dtype=case["dtype"])
    elif case["op"] == "attention":
        b, n, h, hk, d, t = (case[k] for k in ("batch", "tokens", "heads", "key_heads", "dim", "dtype"))
        s |= dict(q=normal(b, n, h, d, dtype=t, scale=1.5), k=normal(b, n, hk, d, dtype=t), v=normal(b, n, hk, d, dtype=t))
        if case["train"]:
            s["dout"] = normal(b, n, h, d, dtype=t)
        if case["absent"]:
            off = torch.rand((b, SLOTS), generator=g, device=DEV).argsort(1) < case["absent"]
            at = torch.arange(n, device=DEV) * SLOTS // n
            s["mask"] = ~off[:, at] | (torch.arange(n, device=DEV) < case["sinks"])
        else:
            s["mask"] = None
    elif case["op"] == "token":
        b, n, h, hk, d, t = (case[k] for k in ("batch", "cache", "heads", "key_heads", "dim", "dtype"))
        s |= dict(q=normal(b, h, d, dtype=t, scale=1.5), k=normal(b, n, hk, d, dtype=t), v=normal(b, n, hk, d, dtype=t))
        order = torch.randperm(b, generator=torch.Generator().manual_seed(seed))
        s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32)[order].to(DEV)
    else:
        shapes = _shapes(case)
        s["params"] = [normal(*sh, dtype=case["dtype"], scale=0.05) for sh in shapes]
        s["grads"] = [normal(*sh, dtype=case["grad"], scale=0.01) for sh in shapes]
        s["sizes"] = [math.prod(sh) for sh in shapes]
        s["padded"] = [-(-n // BLOCK) * BLOCK for n in s["sizes"]]
        # states as they are after some steps; the blocks' padding holds zeros
        inside = torch.cat([torch.arange(p, device=DEV) < n for n, p in zip(s["sizes"], s["padded"])])
        total = inside.numel()
        s["t"] = 100
        if case["bits"] == 8:
            s["m_code"] = torch.randint(-127, 128, (total,), generator=g, device=DEV, dtype=torch.int8) * inside
            s["v_code"] = torch.randint(1, 256, (total,), generator=g, device=DEV, dtype=torch.int32).to(torch.uint8) * inside
            s["m_scale"] = torch.rand(total // BLOCK, generator=g, device=DEV) * 0.01 + 0.005
            s["v_scale"] = torch.rand(total // BLOCK, generator=g, device=DEV) * 0.01 + 0.005
        else:
            s["m"] = torch.randn(total, generator=g, device=DEV) * 0.003 * inside
            s["v"] = torch.rand(total, generator=g, device=DEV) * 1e-4 * inside
        if own:
            s["handle"] = _optimizer(s)
    return s


def _optimizer(s: dict):
    """The optimizer that a training program keeps, at the state's step."""
    opt = _own("optim").AdamW(s["params"], lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=DECAY,
                              state_bits=s["case"]["bits"])
    names = ("m_code", "v_code", "m_scale", "v_scale") if s["case"]["bits"] == 8 else ("m", "v")
    opt.load_state_dict({"step": s["t"], **{n: s[n] for n in names}})
    return opt


def _own(module: str):
    import __graft_entry__
    __graft_entry__.load_package()
    return importlib.import_module("rsna_knee_efficiency_amd." + module)


# --- one pass -----------------------------------------------------------------------------------
def run(s: dict):
    return (_run_own if own else _run_plain)(s)


def _run_own(s: dict):
    case = s["case"]
    if case["op"] == "adamw":
        s["handle"].step(s["grads"])
        return (s["params"], *s["handle"].moments())
    ops = _own("context")
    if case["op"] == "norm":
        y, mean, rstd = ops.layer_norm_forward(s["x"], s["weight"], s["bias"], EPS)
        if not case["train"]:
            return y
        return (y, *ops.layer_norm_backward(s["dy"], s["x"], s["weight"], mean, rstd))
    if case["op"] == "rotary":
        return ops.rotary(s["x"], s["pos"], _sections(case["dim"]), BASE, inverse=case["inverse"])
    if case["op"] == "attention":
        how = dict(left=case["left"], right=case["right"], sinks=case["sinks"], key_mask=s["mask"])
        out, lse = ops.window_attention_forward(s["q"], s["k"], s["v"], **how)
        if not case["train"]:
            return out
        return (out, *ops.window_attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, **how))
    return ops.window_attention_token(s["q"], s["k"], s["v"], s["lengths"], left=case["left"], sinks=case["sinks"])


def _run_plain(s: dict):
    return {"norm": _norm, "rotary": _rotary, "attention": _attention, "token": _token, "adamw": _adamw}[s["case"]["op"]](s)


def _norm(s: dict):
    x = s["x"].float()
    centred = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt(centred.square().mean(1, keepdim=True) + EPS)
    unit = centred * rstd
    y = (unit * s["weight"] + s["bias"]).to(s["x"].dtype)
    if "dy" not in s:
        return y
    dy = s["dy"].float()
    g = dy * s["weight"]
    dx = rstd * (g - g.mean(1, keepdim=True) - unit * (g * unit).mean(1, keepdim=True))
    return y, dx.to(s["x"].dtype), (dy * unit).sum(0), dy.sum(0)


def _rotary(s: dict):
    x, sections = s["x"].float(), _sections(s["case"]["dim"])
    freq = torch.cat([BASE ** (-torch.arange(n, device=x.device, dtype=torch.float32) / n) for n in sections])
    axis = torch.cat([torch.full((n,), a, device=x.device) for a, n in enumerate(sections)])
    angle = (s["pos"].float()[..., axis] * freq)[:, :, None]
    cos, sin = angle.cos(), angle.sin()
    sin = -sin if s["case"]["inverse"] else sin
    half = x.shape[-1] // 2
    u, v = x[..., :half], x[..., half:]
    return torch.cat([u * cos - v * sin, u * sin + v * cos], -1).to(s["x"].dtype)


def _attention(s: dict):
    case, t = s["case"], s["q"].dtype
    b, n, h, d = s["q"].shape
    hk = case["key_heads"]
    scale = 1.0 / math.sqrt(d)
    # heads first, the query heads of one key head beside each other: (b, hk, h / hk, n, d)
    q = s["q"].float().permute(0, 2, 1, 3).reshape(b, hk, h // hk, n, d)
    k, v = (s[name].float().permute(0, 2, 1, 3)[:, :, None] for name in ("k", "v"))
    i, j = torch.arange(n, device=q.device)[:, None], torch.arange(n, device=q.device)[None]
    seen = (j <= i + case["right"]) & ((j >= i - case["left"]) | (j < case["sinks"]))
    hidden = ~seen if s["mask"] is None else ~(seen & s["mask"][:, None, None, None, :])
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).masked_fill_(hidden, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top.isfinite(), top, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, 1.0))

    def laid(x):                                       # (b, hk, g, n, d) -> (b, n, heads, d), rounded
        return x.reshape(b, -1, n, d).permute(0, 2, 1, 3).contiguous().to(t)

    out = laid(torch.matmul(p, v))
    if "dout" not in s:
        return out
    do = s["dout"].float().permute(0, 2, 1, 3).reshape(b, hk, h // hk, n, d)
    o = out.float().permute(0, 2, 1, 3).reshape(b, hk, h // hk, n, d)
    dv = torch.matmul(p.transpose(-1, -2), do).sum(2)
    ds = torch.matmul(do, v.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    dq = torch.matmul(ds, k) * scale
    dk = (torch.matmul(ds.transpose(-1, -2), q) * scale).sum(2)
    return out, laid(dq), laid(dk), laid(dv)


def _token(s: dict):
    case = s["case"]
    b, h, d = s["q"].shape
    hk = case["key_heads"]
    q = s["q"].float().reshape(b, hk, h // hk, d)
    k, v = (s[name].float().permute(0, 2, 1, 3) for name in ("k", "v"))
    j, last = torch.arange(case["cache"], device=q.device)[None], (s["lengths"] - 1)[:, None]
    seen = (j <= last) & ((j >= last - case["left"]) | (j < case["sinks"]))
    p = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(d)
    p = p.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True))
    out = torch.matmul(p / p.sum(-1, keepdim=True), v)
    return out.reshape(b, h, d).to(s["q"].dtype)


def _flat(tensors: list, padded: list) -> torch.Tensor:
    """The tensors one after the other in 32 bits, each padded with zeros to whole blocks."""
    pads = [t.new_zeros(p - t.numel(), dtype=torch.float32) for t, p in zip(tensors, padded)]
    return torch.cat([part for t, z in zip(tensors, pads) for part in (t.reshape(-1).float(), z)])


def _adamw(s: dict):
    case = s["case"]
    p, g = _flat(s["params"], s["padded"]), _flat(s["grads"], s["padded"])
    if case["bits"] == 8:
        c = s["m_code"].float().view(-1, BLOCK)
        m = (c * c.abs() * (s["m_scale"] * (1 / 127 ** 2))[:, None]).view(-1)
        c = s["v_code"].float().view(-1, BLOCK)
        v = (c * c * (s["v_scale"] * (1 / 255 ** 2))[:, None]).view(-1).square()
    else:
        m, v = s["m"], s["v"]
    s["t"] += 1
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + g * g * (1 - BETA2)
    root = v.sqrt()
    p = p * (1 - LR * DECAY) - m / (root * (1 / math.sqrt(1 - BETA2 ** s["t"])) + ADAM_EPS) * (LR / (1 - BETA1 ** s["t"]))
    pieces = torch.split(p, [n for a, b in zip(s["sizes"], s["padded"]) for n in (a, b - a)])[::2]
    torch._foreach_copy_(s["params"], [x.view_as(t) for x, t in zip(pieces, s["params"])])
    if case["bits"] == 8:
        # the square of a signed code is the first moment, the square of an unsigned one the second's root
        # (at least one step above zero, so that no moment that is not zero divides as zero)
        size, root = m.abs().view(-1, BLOCK), root.view(-1, BLOCK)
        s["m_scale"], s["v_scale"] = _scale(size), _scale(root)
        c = torch.clamp(((size * _inverse(s["m_scale"])).sqrt() * 127).round(), max=127)
        c = c * m.view(-1, BLOCK).sign()
        s["m_code"] = c.view(-1).to(torch.int8)
        m = (c * c.abs() * (s["m_scale"] * (1 / 127 ** 2))[:, None]).view(-1)
        low = ((root > 0) & (s["v_scale"][:, None] > 0)).float()
        c = torch.maximum(torch.clamp(((root * _inverse(s["v_scale"])).sqrt() * 255).round(), max=255), low)
        s["v_code"] = c.view(-1).to(torch.uint8)
        v = (c * c * (s["v_scale"] * (1 / 255 ** 2))[:, None]).view(-1).square()
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    return s["params"], m, v


def _scale(size: torch.Tensor) -> torch.Tensor:
    """A block's scale: its largest value, or none where that is too small to divide by."""
    top = size.amax(1)
    return torch.where(top >= 2.0 ** -100, top, 0.0)


def _inverse(scale: torch.Tensor) -> torch.Tensor:
    return torch.where(scale > 0, 1 / scale, 0.0)[:, None]


# --- what a pass cannot do without ----------------------------------------------------------------
def _pairs(n: int, left: int, right: int, sinks: int) -> int:
    """Visible (query, key) pairs of n tokens."""
    i = np.arange(n, dtype=np.int64)
    last, first = np.minimum(n - 1, i + right), np.maximum(0, i - left)
    return int((last - first + 1 + np.minimum(first, min(sinks, n))).sum())


def work(case: dict) -> dict:
    op = case["op"]
    if op == "norm":
        n = case["rows"] * case["width"]
        return {"bytes": n * SIZE[case["dtype"]] * (4 if case["train"] else 2) + 16 * case["width"],
                "flops": n * (22 if case["train"] else 8)}
    if op == "rotary":
        tokens = case["batch"] * case["slices"] * case["rows"] * case["cols"]
        n = tokens * case["heads"] * case["dim"]
        return {"bytes": 2 * n * SIZE[case["dtype"]] + 12 * tokens, "flops": 3 * n}
    if op == "attention":
        rows = case["batch"] * case["tokens"] * case["dim"] * SIZE[case["dtype"]]
        each = 2 * case["heads"] + 2 * case["key_heads"]
        pairs = _pairs(case["tokens"], case["left"], case["right"], case["sinks"]) * (SLOTS - case["absent"]) / SLOTS
        return {"bytes": rows * each * (2 if case["train"] else 1),
                "flops": case["batch"] * case["heads"] * pairs * case["dim"] * (14 if case["train"] else 4)}
    if op == "token":
        seen = sum(min(n, case["left"] + 1) + min(case["sinks"], max(0, n - 1 - case["left"])) for n in _lengths(case))
        return {"bytes": SIZE[case["dtype"]] * case["dim"] * 2 * (seen * case["key_heads"] + case["batch"] * case["heads"]),
                "flops": 4 * seen * case["heads"] * case["dim"]}
    n = sum(math.prod(sh) for sh in _shapes(case))
    state = 16 if case["bits"] == 32 else 4 + 8        # both moments read and written; the values of 8-bit ones given
    return {"bytes": n * (2 * SIZE[case["dtype"]] + SIZE[case["grad"]] + state), "flops": 14 * n}


# --- the definitions in 64 bits -------------------------------------------------------------------
def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return {"norm": _norm64, "rotary": _rotary64, "attention": _attention64, "token": _token64,
            "adamw": _adamw64}[case["op"]](s)


def _norm64(s: dict):
    x, w = s["x"].double(), s["weight"].double()
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    sd = torch.sqrt(var + EPS)
    unit = (x - mean) / sd
    y = torch.addcmul(s["bias"].double(), unit, w)
    if "dy" not in s:
        return y
    dy = s["dy"].double()
    # dx is the gradient through the row: (I - 1 1^T / n - unit unit^T / n) (dy w) / sd
    z, n = dy * w, x.shape[1]
    dx = (z - z.sum(1, keepdim=True) / n - unit * ((z * unit).sum(1, keepdim=True) / n)) / sd
    return y, dx, torch.einsum("rc,rc->c", dy, unit), dy.sum(0)


def _rotary64(s: dict):
    x, case = s["x"].double(), s["case"]
    half = case["dim"] // 2
    z = torch.complex(x[..., :half], x[..., half:])
    turn, at = [], 0
    for axis, n in enumerate(_sections(case["dim"])):
        for t in range(n):
            turn.append(s["pos"][..., axis].double() * math.pow(BASE, -t / n))
    angle = torch.stack(turn, -1)[:, :, None]
    z = z * torch.polar(torch.ones_like(angle), -angle if case["inverse"] else angle)
    return torch.cat([z.real, z.imag], -1)


def _attention64(s: dict):
    """Head by head, a run of queries at a time against the keys any of them can see."""
    case = s["case"]
    b, n, h, d = s["q"].shape
    per = h // case["key_heads"]
    out = torch.zeros((b, n, h, d), dtype=torch.float64, device=DEV)
    train = "dout" in s
    dq, dk, dv = out.clone(), *(torch.zeros(s["k"].shape, dtype=torch.float64, device=DEV) for _ in range(2))
    step = max(256, 1 << 22 >> max(0, (case["left"] + case["right"]).bit_length()))
    for i0 in range(0, n, step):
        i1 = min(n, i0 + step)
        lo, hi = max(0, i0 - case["left"]), min(n, i1 + case["right"])
        keys = torch.cat([torch.arange(min(case["sinks"], lo), device=DEV), torch.arange(lo, hi, device=DEV)])
        i = torch.arange(i0, i1, device=DEV)[:, None]
        inside = (keys <= i + case["right"]) & ((keys >= i - case["left"]) | (keys < case["sinks"]))
        for row in range(b):
            see = inside if s["mask"] is None else inside & s["mask"][row, keys]
            for head in range(h):
                kh = head // per
                q, k, v = s["q"][row, i0:i1, head].double(), s["k"][row, keys, kh].double(), s["v"][row, keys, kh].double()
                w = torch.where(see, q @ k.T / math.sqrt(d), -math.inf)
                p = torch.softmax(w, -1).nan_to_num(0.0)          # a row that sees nothing is zero
                out[row, i0:i1, head] = p @ v
                if train:
                    do = s["dout"][row, i0:i1, head].double()
                    dp = do @ v.T
                    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(d)
                    dq[row, i0:i1, head] = ds @ k
                    dk[row, :, kh].index_add_(0, keys, ds.T @ q)
                    dv[row, :, kh].index_add_(0, keys, p.T @ do)
    return (out, dq, dk, dv) if train else out


def _token64(s: dict):
    case = s["case"]
    b, h, d = s["q"].shape
    per = h // case["key_heads"]
    out = torch.zeros((b, h, d), dtype=torch.float64, device=DEV)
    for row, n in enumerate(s["lengths"].tolist()):
        lo = max(0, n - 1 - case["left"])
        keys = torch.cat([torch.arange(min(case["sinks"], lo), device=DEV), torch.arange(lo, n, device=DEV)])
        k, v = (s[name][row, keys].double().repeat_interleave(per, 1) for name in ("k", "v"))
        p = torch.softmax(torch.einsum("hd,jhd->hj", s["q"][row].double(), k) / math.sqrt(d), -1)
        out[row] = torch.einsum("hj,jhd->hd", p, v)
    return out


def _adamw64(s: dict):
    case, t = s["case"], s["t"] + 1
    new, ms, vs, at = [], [], [], 0
    for p, g, n, padded in zip(s["params"], s["grads"], s["sizes"], s["padded"]):
        where, blocks = slice(at, at + n), slice(at // BLOCK, (at + padded) // BLOCK)
        if case["bits"] == 8:
            sm, sv = (s[k][blocks].double().repeat_interleave(BLOCK)[:n] for k in ("m_scale", "v_scale"))
            cm, cv = s["m_code"][where].double(), s["v_code"][where].double()
            m, v = sm * cm.sign() * (cm / 127) ** 2, (sv * (cv / 255) ** 2) ** 2
        else:
            m, v = s["m"][where].double(), s["v"][where].double()
        g, q = g.reshape(-1).double(), p.reshape(-1).double()
        m = BETA1 * m + (1 - BETA1) * g
        v = BETA2 * v + (1 - BETA2) * g ** 2
        q = q - LR * DECAY * q
        q = q - LR * (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + ADAM_EPS)
        new.append(q.view(p.shape))
        both = torch.zeros((2, padded), dtype=torch.float64, device=DEV)
        both[0, :n], both[1, :n] = m, v
        if case["bits"] == 8:
            m, r = both[0].view(-1, BLOCK), both[1].sqrt().view(-1, BLOCK)
            sm, sr = m.abs().amax(1, keepdim=True).clamp(min=1e-300), r.amax(1, keepdim=True).clamp(min=1e-300)
            cm = torch.round(127 * torch.sqrt(m.abs() / sm))
            cr = torch.where(r > 0, torch.round(255 * torch.sqrt(r / sr)).clamp(min=1), 0.0)
            both = torch.stack([(sm * m.sign() * (cm / 127) ** 2).view(-1), ((sr * (cr / 255) ** 2) ** 2).view(-1)])
        ms.append(both[0])
        vs.append(both[1])
        at += padded
    return new, torch.cat(ms), torch.cat(vs)

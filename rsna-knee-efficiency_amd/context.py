"""The operators of a context layer over all the tokens of a study, on the GPU (`d8s_layer_norm`, `d8s_rotary`,
`d8s_attention` and their gradients, include/d8s_hip.h).

The reference's head attends over one feature vector a window, at most 128 of them (src/knee/models/baseline.py:
954-977).  A layer over every position of the encoder's last map has thousands of tokens a study, placed by slice,
row and column; its attention is kept to a window of neighbours and a few first summary tokens.  Each operator has a
differentiable form (`layer_norm`, `rotary`, `window_attention`), the forward and backward calls it is made of, and
for tokens that arrive one at a time `window_attention_token`.  Calls run on the current stream and may be recorded
into HIP graphs.  There is no CPU path: without the library the calls raise.  Tensors with a forward-mode tangent are
refused.
"""
from __future__ import annotations

import functools
import math

import torch
from torch.autograd import forward_ad

from . import hip

def _fail(message: str):
    raise ValueError(message)


def _on_gpu(first: torch.Tensor, *others: torch.Tensor) -> None:
    index = first.get_device()                 # (an int, -1 on the CPU: a call has up to six tensors to look at)
    if index < 0:
        _fail("the tensors must be on one GPU")
    for t in others:
        if t.get_device() != index:
            _fail("the tensors must be on one GPU")


def _no_tangents(*tensors: torch.Tensor | None) -> None:
    """Every call begins with this: a kernel would leave out a forward-mode tangent without a word (a tensor that has one
    need not require a gradient)."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError("forward-mode derivatives are not implemented: a tensor has a tangent")


def _like(x: torch.Tensor) -> torch.Tensor:
    """A new contiguous tensor of x's shape and type"""
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


# --- layer norm -----------------------------------------------------------------------------------
NORM_MAX = 16384


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x as rows of its last dimension, evenly apart; copied only where its strides allow no such view"""
    x = x.reshape(-1, x.shape[-1]) if x.dim() != 2 else x
    apart, step = x.stride()
    return x if step == 1 and (apart >= x.shape[1] or x.shape[0] == 1) else x.contiguous()


def _norm_types(x: torch.Tensor, weight: torch.Tensor) -> tuple[int, int, int]:
    """(width, type of x, type of weight)"""
    shape = x.shape
    if not shape or not 1 <= shape[-1] <= NORM_MAX:
        _fail(f"x must have a last dimension of 1 .. {NORM_MAX}")
    if x.dtype not in hip.ELEMENTS:
        _fail("x must be float32, bfloat16 or float16")
    if weight.shape != shape[-1:] or weight.dtype not in (torch.float32, x.dtype):
        _fail("weight must have x's last dimension, in float32 or x's type")
    return shape[-1], hip.ELEMENTS[x.dtype], hip.ELEMENTS[weight.dtype]


def layer_norm_forward(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, eps: float = 1e-5,
                       statistics: bool = True) -> tuple:
    """x (..., width) in float32, bfloat16 or float16; weight and bias (width,) in float32 or x's type ->
    (y like x, mean, rstd), the last two float32, one a row, for `layer_norm_backward` (None without
    `statistics`)."""
    _no_tangents(x, weight, bias)
    width, dtype, wdtype = _norm_types(x, weight)
    if bias is not None and (bias.shape != weight.shape or bias.dtype != weight.dtype):
        _fail("bias must be like weight")
    device = x.device
    _on_gpu(x, weight, weight if bias is None else bias)
    y = _like(x)
    n = x.numel() // width
    mean = rstd = None
    if statistics:
        mean = x.new_empty(n, dtype=torch.float32)
        rstd = torch.empty_like(mean)
    if n:
        rows, weight = _rows(x), weight.contiguous()
        bias = None if bias is None else bias.contiguous()
        a = hip.NormArgs(rows.data_ptr(), weight.data_ptr(), 0 if bias is None else bias.data_ptr(), y.data_ptr(),
                         mean.data_ptr() if statistics else 0, rstd.data_ptr() if statistics else 0, 0, 0, 0, 0, 0, 0,
                         n, rows.stride(0), 0, width, dtype, wdtype, eps)
        hip.launch("d8s_layer_norm", device, a)
    return y, mean, rstd


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, mean: torch.Tensor,
                        rstd: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The gradients (dx like x, dweight, dbias like weight) of `layer_norm_forward` at dy like x."""
    _no_tangents(dy, x, weight, mean, rstd)
    width, dtype, wdtype = _norm_types(x, weight)
    n = x.numel() // width
    if dy.shape != x.shape or dy.dtype != x.dtype:
        _fail("dy must be like x")
    if mean.shape != (n,) or rstd.shape != (n,) or mean.dtype != torch.float32 or rstd.dtype != torch.float32:
        _fail("mean and rstd must be float32, one a row")
    device = x.device
    _on_gpu(x, dy, weight, mean, rstd)
    dx = _like(x)
    if not n:
        return dx, torch.zeros_like(weight), torch.zeros_like(weight)
    rows, grad, weight, mean, rstd = _rows(x), _rows(dy), weight.contiguous(), mean.contiguous(), rstd.contiguous()
    dw, db = torch.empty_like(weight), torch.empty_like(weight)
    a = hip.NormArgs(rows.data_ptr(), weight.data_ptr(), 0, 0, mean.data_ptr(), rstd.data_ptr(), grad.data_ptr(),
                     dx.data_ptr(), dw.data_ptr(), db.data_ptr(), 0, 0, n, rows.stride(0), grad.stride(0), width, dtype,
                     wdtype, 0.0)
    work = hip.work_buffer("d8s_layer_norm_workspace", device, a)
    a.partial, a.partial_bytes = work.data_ptr(), work.numel()
    hip.launch("d8s_layer_norm_backward", device, a)
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.has_bias = bias is not None
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        dx, dw, db = layer_norm_backward(dy, *ctx.saved_tensors)
        return dx, dw, db if ctx.has_bias else None, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over x's last dimension, differentiable in x, weight and bias (types as in
    `layer_norm_forward`)."""
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        _no_tangents(x, weight, bias)
        return _LayerNorm.apply(x, weight, bias, eps)
    return layer_norm_forward(x, weight, bias, eps, statistics=False)[0]


# --- rotary positions -------------------------------------------------------------------------------
_POSITIONS = {torch.int32: 0, torch.int64: 1, torch.float32: 2}


@functools.lru_cache(maxsize=64)
def _rotary_plan(sections: tuple, base: float) -> bytes:
    """The arguments that depend on the layer alone: each pair's axis and its turns per position."""
    if not sections or any(not isinstance(n, int) or n < 0 for n in sections) or not 1 <= sum(sections) <= hip.ROTARY_PAIRS:
        _fail(f"sections must be pairs per axis, 1 .. {hip.ROTARY_PAIRS} in all")
    if len(sections) > 255 or not base > 0 or not math.isfinite(base):
        _fail("at most 255 axes, and a positive base")
    a = hip.RotaryArgs()
    at = 0
    for axis, n in enumerate(sections):
        for t in range(n):
            a.freq[at], a.axis[at] = base ** (-t / n) / (2 * math.pi), axis
            at += 1
    a.pairs, a.axes = at, len(sections)
    return bytes(a)


def _may_meet(x: torch.Tensor, y: torch.Tensor) -> bool:
    """Whether two tensors of one shape and type may have an element in common.  Exact where their strides are the same
    and nested: then the distance between them must not be a sum of strides times differences of indices."""
    def span(sizes, strides):
        return sum((n - 1) * s for n, s in zip(sizes, strides))
    size, apart = x.element_size(), y.data_ptr() - x.data_ptr()
    if not -size * span(y.shape, y.stride()) <= apart <= size * span(x.shape, x.stride()):
        return False
    if apart % size or x.stride() != y.stride():
        return True
    dims = sorted(zip(x.stride(), x.shape), reverse=True)

    def reached(distance: int, at: int) -> bool:
        if at == len(dims):
            return distance == 0
        stride, n = dims[at]
        rest = span([m for _, m in dims[at + 1:]], [t for t, _ in dims[at + 1:]])
        if stride == 0:
            return reached(distance, at + 1)
        low, high = max(1 - n, -((rest - distance) // stride)), min(n - 1, (distance + rest) // stride)
        return high - low > 4 or any(reached(distance - i * stride, at + 1) for i in range(low, high + 1))
    return reached(apart // size, 0)


def _rotate(x, positions, sections, base, adjacent, inverse, out):
    _no_tangents(x, positions, out)
    a = hip.RotaryArgs.from_buffer_copy(_rotary_plan(tuple(sections), float(base)))
    if x.dim() != 4 or x.dtype not in hip.ELEMENTS or x.shape[3] < 2 * a.pairs:
        _fail(f"x must be (batch, tokens, heads, channels) of at least {2 * a.pairs} channels in float32, bfloat16 or "
              "float16")
    if positions.dtype not in _POSITIONS or positions.shape not in ((*x.shape[:2], a.axes), (x.shape[1], a.axes)):
        _fail(f"positions must be (batch, tokens, {a.axes}) or (tokens, {a.axes}) in int32, int64 or float32")
    _on_gpu(x, positions)
    x = x if x.stride(3) == 1 else x.contiguous()
    positions = positions if positions.stride(-1) == 1 else positions.contiguous()
    if out is None:
        out = _like(x)
    elif out.shape != x.shape or out.dtype != x.dtype or out.device != x.device or out.stride(3) != 1:
        _fail("out must be like x, its channels contiguous")
    elif any(s == 0 and n > 1 for n, s in zip(out.shape, out.stride())):
        _fail("out must not have several elements in one place")
    elif out.data_ptr() == x.data_ptr():
        if out.stride() != x.stride():
            _fail("out must be x itself, or memory of its own")
    elif x.numel() and _may_meet(x, out):      # (a token's values could be read after another's were written there)
        x = x.clone(memory_format=torch.contiguous_format)
    if not x.numel():
        return out
    a.x, a.y, a.pos = x.data_ptr(), out.data_ptr(), positions.data_ptr()
    a.x_sb, a.x_ss, a.x_sh = x.stride()[:3]
    a.y_sb, a.y_ss, a.y_sh = out.stride()[:3]
    a.pos_ss = positions.stride(-2)
    a.pos_sb = positions.stride(0) if positions.dim() == 3 else 0
    a.B, a.S, a.H, a.D = x.shape
    a.dtype, a.pos_type, a.adjacent, a.inverse = hip.ELEMENTS[x.dtype], _POSITIONS[positions.dtype], adjacent, inverse
    hip.launch("d8s_rotary", x.device, a)
    return out


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, sections, base, adjacent, inverse):
        ctx.save_for_backward(positions)
        ctx.how = (sections, base, adjacent, not inverse)
        return _rotate(x, positions, sections, base, adjacent, inverse, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        return _rotate(dy, ctx.saved_tensors[0], *ctx.how, None), None, None, None, None, None


def rotary(x: torch.Tensor, positions: torch.Tensor, sections, base: float = 10000.0, *, adjacent: bool = False,
           inverse: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """Turns x (batch, tokens, heads, channels) by its tokens' positions on several axes (slice, row, column ...).

    sections[a] pairs of channels turn with axis a, pair t of them by positions[..., a] * base^(-t / sections[a]);
    pairs are channels (i, i + pairs), or (2 i, 2 i + 1) when `adjacent`; channels past the pairs are copied.
    positions: (batch, tokens, axes) or, for all of a batch, (tokens, axes).  `inverse` turns back (the gradient; the
    call is differentiable in x).  `out` may be x itself, where no gradient is asked for, and elements of other places in x's
    memory (x is then copied first); it must not be expanded.  Queries and keys that lie
    beside each other in one tensor are turned in one call, as x of all their heads."""
    if torch.is_grad_enabled() and x.requires_grad:
        _no_tangents(x, positions, out)
        if out is not None:
            _fail("out is not taken where x requires a gradient")
        return _Rotary.apply(x, positions, tuple(sections), base, adjacent, inverse)
    given = out
    out = _rotate(x, positions, sections, base, adjacent, inverse, out)
    if given is not None:
        hip.written(out)
    return out


# --- attention within a window ------------------------------------------------------------------------
_FAR = 1 << 30


def _last(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 else t.contiguous()


def _extent(n: int | None, name: str) -> int:
    if n is None:
        return _FAR
    if n < 0:
        _fail(f"{name} must not be negative (None: no limit)")
    return min(int(n), _FAR)


def _attn_args(q, k, v, left, right, sinks, key_mask, scale):
    """The call's arguments, and the tensors they point into (copies where the channels were not contiguous), which the
    caller holds until the call has been made"""
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        _fail("q must be (batch, tokens, heads, channels), k and v (batch, tokens, key heads, channels)")
    B, S, H, D = q.shape
    HK = k.shape[2]
    if k.shape != (B, S, HK, D) or HK < 1 or H % HK:
        _fail("k and v must have q's batch, tokens and channels, and heads that divide q's")
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        _fail("q, k and v must be bfloat16, or float16")
    if D not in (64, 128):
        _fail("64 or 128 channels a head")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 2.0 ** -100 <= scale <= 2.0 ** 100:
        _fail("scale must be positive: 2^-100 .. 2^100")
    q, k, v = _last(q), _last(k), _last(v)
    _on_gpu(q, k, v)
    mask_at, mask_sb = 0, 0
    if key_mask is not None:
        if key_mask.shape != (B, S) or key_mask.dtype not in (torch.bool, torch.uint8):
            _fail("key_mask must be (batch, tokens) of bool or uint8")
        _on_gpu(q, key_mask)
        key_mask = _last(key_mask)
        mask_at, mask_sb = key_mask.data_ptr(), key_mask.stride(0)
    a = hip.AttnArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), mask_at, 0, 0, 0, 0, 0, 0, 0, 0, *q.stride()[:3],
                     *k.stride()[:3], *v.stride()[:3], 0, 0, 0, mask_sb, B, S, H, HK, D, hip.ELEMENTS[q.dtype],
                     _extent(left, "left"), _extent(right, "right"), _extent(sinks, "sinks"), scale)
    return a, (q, k, v, key_mask)


def window_attention_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, left: int | None = None,
                             right: int | None = 0, sinks: int = 0, key_mask: torch.Tensor | None = None,
                             scale: float | None = None, statistics: bool = True) -> tuple:
    """Attention of q (batch, tokens, heads, channels) over k, v (batch, tokens, key heads, channels), bfloat16 or
    float16, 64 or 128 channels; query head h uses key head h // (heads / key heads).

    Token i sees token j iff j <= i + right, and j >= i - left or j < sinks, and key_mask[batch, j] (bool, or uint8
    with 0 for absent).  None: no limit on that side.  A token that sees nothing has zeros.  Strides are free (the
    channels are copied where they are not contiguous).  scale: 1 / sqrt(channels) unless given
    (2^-100 .. 2^100).

    -> (out like q, lse (batch, heads, tokens) float32: the logarithm of the sum of exponentials, -inf where nothing
    is seen; None without `statistics`)"""
    _no_tangents(q, k, v)
    a, _kept = _attn_args(q, k, v, left, right, sinks, key_mask, scale)
    out = _like(q)
    lse = q.new_empty((a.B, a.H, a.S), dtype=torch.float32) if statistics else None
    if q.numel():
        a.out, a.lse = out.data_ptr(), lse.data_ptr() if statistics else 0
        hip.launch("d8s_attention", q.device, a)
    return out, lse


def window_attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                              lse: torch.Tensor, left: int | None = None, right: int | None = 0, sinks: int = 0,
                              key_mask: torch.Tensor | None = None, scale: float | None = None) -> tuple:
    """The gradients (dq, dk, dv) of `window_attention_forward` at dout like out."""
    _no_tangents(dout, q, k, v, out, lse)
    a, _kept = _attn_args(q, k, v, left, right, sinks, key_mask, scale)
    if dout.shape != q.shape or dout.dtype != q.dtype or out.shape != q.shape or out.dtype != q.dtype:
        _fail("dout and out must be like q")
    if lse.shape != (a.B, a.H, a.S) or lse.dtype != torch.float32:
        _fail("lse must be (batch, heads, tokens) float32")
    _on_gpu(q, dout, out, lse)
    dq, dk, dv = _like(q), _like(k), _like(v)
    if not q.numel():
        return dq, dk.zero_(), dv.zero_()
    dout, out, lse = _last(dout), out.contiguous(), lse.contiguous()
    a.dout, a.out, a.lse = dout.data_ptr(), out.data_ptr(), lse.data_ptr()
    a.do_sb, a.do_ss, a.do_sh = dout.stride()[:3]
    a.dq, a.dk, a.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    work = hip.work_buffer("d8s_attention_workspace", q.device, a)
    a.workspace, a.ws_bytes = work.data_ptr(), work.numel()
    hip.launch("d8s_attention_backward", q.device, a)
    return dq, dk, dv


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, left, right, sinks, key_mask, scale):
        out, lse = window_attention_forward(q, k, v, left, right, sinks, key_mask, scale)
        ctx.save_for_backward(q, k, v, out, lse, key_mask)
        ctx.how = (left, right, sinks)
        ctx.scale = scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        *saved, key_mask = ctx.saved_tensors
        return (*window_attention_backward(dout, *saved, *ctx.how, key_mask, ctx.scale), None, None, None, None, None)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, left: int | None = None, right: int | None = 0,
                     sinks: int = 0, key_mask: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """`window_attention_forward`'s out, differentiable in q, k and v."""
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        _no_tangents(q, k, v)
        return _WindowAttention.apply(q, k, v, left, right, sinks, key_mask, scale)
    return window_attention_forward(q, k, v, left, right, sinks, key_mask, scale, statistics=False)[0]


def window_attention_token(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: torch.Tensor,
                           left: int | None = None, sinks: int = 0, scale: float | None = None) -> torch.Tensor:
    """One new token a row against its cache: q (batch, heads, channels), k_cache and v_cache (batch, capacity, key
    heads, channels), types as in `window_attention_forward`.  Row b's token is the last of the lengths[b] (int32, on
    the GPU) tokens in its cache, whose keys and values are already there; it sees the last left + 1 of them and the
    first `sinks`.  Lengths are not checked (that would synchronise): they are taken as 0 .. capacity, and length 0
    (or scores that are all -infinity) gives zeros.  What the cache holds from a row's length on is not read."""
    _no_tangents(q, k_cache, v_cache)
    if q.dim() != 3 or k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        _fail("q must be (batch, heads, channels), k_cache and v_cache (batch, capacity, key heads, channels)")
    B, H, D = q.shape
    HK = k_cache.shape[2]
    if k_cache.shape[0] != B or k_cache.shape[3] != D or HK < 1 or H % HK:
        _fail("the caches must have q's batch and channels, and heads that divide q's")
    if q.dtype not in (torch.bfloat16, torch.float16) or k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        _fail("q, k_cache and v_cache must be bfloat16, or float16")
    if D not in (64, 128):
        _fail("64 or 128 channels a head")
    if lengths.shape != (B,) or lengths.dtype != torch.int32:
        _fail("lengths must be (batch,) int32")
    _on_gpu(q, k_cache, v_cache, lengths)
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 2.0 ** -100 <= scale <= 2.0 ** 100:
        _fail("scale must be positive: 2^-100 .. 2^100")
    out = _like(q)
    if not out.numel() or not k_cache.shape[1]:
        return out.zero_()
    if k_cache.stride(3) != 1 or v_cache.stride(3) != 1:
        _fail("the caches' channels must be contiguous")
    q, lengths = _last(q), lengths.contiguous()
    a = hip.TokenArgs(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), lengths.data_ptr(), out.data_ptr(), 0, 0,
                      *q.stride()[:2], *k_cache.stride()[:3], *v_cache.stride()[:3], B, k_cache.shape[1], H, HK, D,
                      hip.ELEMENTS[q.dtype], _extent(left, "left"), _extent(sinks, "sinks"), scale, 0)
    work = hip.work_buffer("d8s_attention_token_workspace", q.device, a)
    a.workspace, a.ws_bytes = work.data_ptr(), work.numel()
    hip.launch("d8s_attention_token", q.device, a)
    return out

"""A context layer's cache of keys and values in 8 bits, and attention of new tokens over it, on the GPU
(`d8s_cache_append`, `d8s_cache_read`, `d8s_cache_attention`, include/d8s_hip.h).

    cache = QuantizedCache(batch, capacity, key_heads, channels)
    cache.append(k, v)                                   # the keys and values of an image's tokens, or of one token
    out = cached_attention(q, cache, left=512, sinks=12)  # their queries over all that the cache holds

Half the bytes of a 16-bit cache, and half the time of the attention of many requests' tokens, which is bound by reading it (64 requests of 8192
tokens, 32 heads on 8 of 128 channels: 190 us, over a 16-bit cache 387; a single request's is a matter of latency, 13 and 14).  Calls run on
the current stream of the cache's device and may be recorded into HIP graphs: lengths are kept on the GPU, so a replay
appends its tokens behind those of the one before.  There is no CPU path: without the library the calls raise.  None
of this has gradients (`context.window_attention` has): tensors that require one are refused outside `torch.no_grad()`.
"""
from __future__ import annotations

import functools
import math

import torch

from . import hip
from .context import _extent, _fail, _last, _like, _no_tangents, _on_gpu

_BLOCK = hip.CACHE_BLOCK


def _no_gradients(*tensors: torch.Tensor) -> None:
    _no_tangents(*tensors)
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        _fail("the cache has no gradients: call under torch.no_grad()")


def _counts(counts: torch.Tensor | None, batch: int, like: torch.Tensor) -> torch.Tensor | None:
    if counts is None:
        return None
    if counts.shape != (batch,) or counts.dtype != torch.int32:
        _fail("counts must be (batch,) int32")
    _on_gpu(like, counts)
    return counts.contiguous()


class QuantizedCache:
    """Keys and values of up to `capacity` tokens of `batch` rows, `key_heads` heads of 64 or 128 channels.

    64 tokens in a row of a key head are a block.  Once a block is full it is held as 8-bit codes with one float32 scale, its largest
    |x| over the largest code: int8 codes (127 steps to either side), or float8_e4m3fn ones (3 bits behind the leading one, for blocks
    whose values span decades).  The last block stays in `dtype` until it is full.  So a token is rounded once, and any split
    of the tokens over calls gives the same cache.  A block with a key (value) that is not finite reads as not a number.

    lengths (batch,) int32: tokens of every row, on the GPU.  A row may be set back to 0 (a new request in its place; `clear`
    does it), to a multiple of 64 below its length, or, while its last block is not full, to fewer tokens of that (tokens that were
    only tried); nothing else of the cache need be touched then.  To any other length the tokens are no longer there in 16 bits.
    dropped (batch,) int32: tokens that found no room.  Appending past the capacity loses them and counts them there (the host does
    not know the lengths, and finding out would synchronise); what their queries get means nothing."""

    def __init__(self, batch: int, capacity: int, key_heads: int, channels: int, codes: torch.dtype = torch.int8,
                 dtype: torch.dtype = torch.bfloat16, device="cuda:0") -> None:
        if batch < 1 or capacity < 1 or key_heads < 1:
            _fail("batch, capacity and key_heads must be positive")
        if capacity > 1 << 29:
            _fail("at most 2^29 tokens")
        if batch * key_heads >= 1 << 22:
            _fail("too many heads: batch times key_heads must be below 2^22")
        if channels not in (64, 128):
            _fail("64 or 128 channels a head")
        if codes not in hip.CODES:
            _fail("codes must be int8 or float8_e4m3fn")
        if dtype not in (torch.bfloat16, torch.float16):
            _fail("dtype must be bfloat16 or float16")
        device = torch.device(device)
        if device.type != "cuda":
            _fail("the cache must be on a GPU")
        self.batch, self.capacity, self.key_heads, self.channels, self.codes, self.dtype = (
            batch, capacity, key_heads, channels, codes, dtype)
        block, blocks = _BLOCK, max(1, capacity // _BLOCK)

        def empty(*shape, of):
            return torch.empty((batch, key_heads, *shape), dtype=of, device=device)
        self._held = (empty(blocks, block, channels, of=torch.uint8), empty(blocks, channels, block, of=torch.uint8),
                      empty(blocks, of=torch.float32), empty(blocks, of=torch.float32),
                      empty(block, channels, of=dtype), empty(channels, block, of=dtype))
        self._lengths, self._dropped, self._arrived = (torch.zeros(n, dtype=torch.int32, device=device)
                                                       for n in (batch, batch, batch * hip.CACHE_ARRIVED))
        self.device = self._lengths.device
        self._sizes = (batch, capacity, key_heads, channels, hip.ELEMENTS[dtype], hip.CODES[codes])
        self._made: hip.Cache | None = None

    # (the tensors themselves are never replaced: their addresses are formed once)
    lengths = property(lambda self: self._lengths)
    dropped = property(lambda self: self._dropped)

    def _args(self) -> hip.Cache:
        if self._made is None:
            self._made = hip.Cache(*(t.data_ptr() for t in self._held), self._lengths.data_ptr(), *self._sizes)
        return self._made

    def __getstate__(self) -> dict:            # a copy has tensors, and addresses, of its own
        return {**self.__dict__, "_made": None}

    def append(self, k: torch.Tensor, v: torch.Tensor, counts: torch.Tensor | None = None) -> None:
        """Appends k and v (batch, tokens, key heads, channels) in the cache's dtype, any strides (the channels are copied
        where they are not contiguous).  counts (batch,) int32 on the GPU: only the first counts[b] (taken as 0 .. tokens)
        are there.  One launch; calls on one cache must follow each other.  (At most 2^29 tokens, and 2^24 blocks of all heads.)"""
        _no_gradients(k, v)
        shape = (self.batch, k.shape[1] if k.dim() == 4 else 0, self.key_heads, self.channels)
        if k.shape != shape or v.shape != shape:
            _fail(f"k and v must be ({self.batch}, tokens, {self.key_heads}, {self.channels})")
        if k.dtype != self.dtype or v.dtype != self.dtype:
            _fail("k and v must have the cache's dtype")
        if shape[1] > 1 << 29 or self.batch * self.key_heads * ((shape[1] + 2 * _BLOCK - 2) // _BLOCK) >= 1 << 24:
            _fail("too many heads and tokens for one call")
        _on_gpu(self._lengths, k, v)
        counts = _counts(counts, self.batch, self._lengths)
        if not shape[1]:
            return
        k, v = _last(k), _last(v)
        a = hip.CacheAppendArgs(self._args(), k.data_ptr(), v.data_ptr(), 0 if counts is None else counts.data_ptr(),
                                self._arrived.data_ptr(), self._dropped.data_ptr(), *k.stride()[:3], *v.stride()[:3], shape[1], 0)
        hip.launch("d8s_cache_append", self.device, a)
        torch.autograd.graph.increment_version([*self._held, self._lengths, self._dropped])

    def read(self, tokens: int | None = None, dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """(k, v) (batch, tokens, key heads, channels): the values that the first `tokens` (default: all the capacity) stand
        for, zeros from a row's length on, in the cache's dtype (each rounded once more) or, exactly, in float32."""
        tokens = self.capacity if tokens is None else tokens
        dtype = self.dtype if dtype is None else dtype
        if not 0 <= tokens <= self.capacity:
            _fail("tokens must be 0 .. capacity")
        if dtype not in (torch.float32, self.dtype):
            _fail("dtype must be float32 or the cache's")
        k, v = (torch.empty((self.batch, tokens, self.key_heads, self.channels), dtype=dtype, device=self.device) for _ in range(2))
        if tokens:
            hip.launch("d8s_cache_read", self.device,
                       hip.CacheReadArgs(self._args(), k.data_ptr(), v.data_ptr(), tokens, hip.ELEMENTS[dtype]))
        return k, v

    def clear(self, rows=None) -> None:
        """Empties all rows, or those of an index (a number, a list, a tensor)."""
        if rows is None:
            self._lengths.zero_()
        else:
            self._lengths[rows] = 0


@functools.lru_cache(maxsize=4096)
def _workspace(device: torch.device, sizes: tuple, T: int, H: int, left: int, right: int, sinks: int) -> int:
    """Bytes of workspace that a call of these sizes needs on a device"""
    at = 1 << 20                               # (a pointer that is not followed)
    a = hip.CacheAttnArgs(hip.Cache(at, at, at, at, at, at, at, *sizes), T=T, H=H, left=left, right=right, sinks=sinks, scale=1.0)
    need = hip.u64()
    with torch.cuda.device(device):
        hip.call("d8s_cache_attention_workspace", a, need)
    return need.value


def checked(q: torch.Tensor, cache: QuantizedCache, left: int | None, right: int | None, sinks: int,
            counts: torch.Tensor | None, scale: float | None = None) -> tuple:
    """`cached_attention`'s checks of its arguments -> the others of `attend`.  (Apart, for a caller that appends between them: a call that
    is refused should leave the cache as it was.)"""
    _no_gradients(q)
    shape = q.shape
    if len(shape) != 4 or shape[0] != cache.batch or shape[3] != cache.channels or shape[2] < 1 or shape[2] % cache.key_heads:
        _fail(f"q must be ({cache.batch}, tokens, heads, {cache.channels}), heads a multiple of {cache.key_heads}")
    if q.dtype != cache.dtype:
        _fail("q must have the cache's dtype")
    if shape[0] * shape[1] * shape[2] >= 1 << 27:
        _fail("too many heads and tokens for one call: batch times tokens times heads must be below 2^27")
    _on_gpu(cache._lengths, q)
    counts = _counts(counts, cache.batch, cache._lengths)
    scale = 1.0 / math.sqrt(cache.channels) if scale is None else float(scale)
    if not 2.0 ** -100 <= scale <= 2.0 ** 100:
        _fail("scale must be positive: 2^-100 .. 2^100")
    return _extent(left, "left"), _extent(right, "right"), _extent(sinks, "sinks"), counts, scale


def attend(q: torch.Tensor, cache: QuantizedCache, left: int, right: int, sinks: int, counts: torch.Tensor | None, scale: float) -> torch.Tensor:
    """`cached_attention` of arguments that `checked` has returned"""
    out = _like(q)
    if not q.numel():
        return out
    q = _last(q)
    _, T, H, _ = q.shape
    made = cache._args()
    need = _workspace(cache.device, cache._sizes, T, H, left, right, sinks)
    work = torch.empty(need, dtype=torch.uint8, device=cache.device) if need else None
    hip.launch("d8s_cache_attention", cache.device, hip.CacheAttnArgs(
        made, q.data_ptr(), 0 if counts is None else counts.data_ptr(), out.data_ptr(), 0 if work is None else work.data_ptr(),
        need, *q.stride()[:3], T, H, left, right, sinks, scale))
    return out


def cached_attention(q: torch.Tensor, cache: QuantizedCache, left: int | None = None, right: int | None = 0, sinks: int = 0,
                     counts: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """Attention of new tokens over a cache that holds them already: q (batch, tokens, heads, channels) in the cache's dtype are
    the queries of every row's last tokens, or, with counts (batch,) int32 on the GPU (taken as 0 .. tokens), the first
    counts[b] of them are.  Query head h uses key head h // (heads / key heads).

    The token at position i of its row sees token j iff j <= i + right, and j >= i - left or j < sinks (None: no limit on that
    side): as in `context.window_attention` over all of the row.  -> out like q: zeros for a query that sees nothing or is past
    its row's count.  scale: 1 / sqrt(channels) unless given (2^-100 .. 2^100).  (A value of the last, 16-bit block that is not
    finite can spoil the queries beside those that see it.  A query that sees bfloat16 values above 2^64, or some token of a full
    block that has one, loses digits of what others below 2^-70 add to its result.)"""
    return attend(q, cache, *checked(q, cache, left, right, sinks, counts, scale))

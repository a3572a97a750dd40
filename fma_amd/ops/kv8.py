"""A KV cache held in 8 bits, its store, and causal attention over it.

Keys and values are held in blocks of 32 tokens, each with one fp32 scale for
each kv head, K and V apart:

- ``fp8`` (e4m3): scale = the smallest power of two that brings the block's
  largest finite magnitude to 448 or less, code = e4m3(x / scale);
- ``int8``: scale = amax / 127, code = rint(x * (127 / amax)).

The largest magnitude counts as at least 2^-100. A block is coded once, when
its last token arrives; until then its tokens are held as they came, in 16
bits. Codes are made from 16-bit values, so what the cache holds does not
depend on how tokens were spread over calls. In a coded block NaN is 0 and an
infinity the block's largest value; attention takes a V that is still raw
alike, an infinity as the type's largest value.

The raw values of the last two blocks stay, so a caller may go back a few
tokens (a rejected draft) and append again: to any position not before the
block that precedes the incomplete one, or to the first token of any block.

On a GPU the calls run kernels of the native extension, one launch each
(attention: two where a long axis is split). On the CPU the same layout is
filled and read with torch operations.
"""

from __future__ import annotations

from functools import lru_cache
from typing import List, Optional, Tuple, Union

import torch

from fma_amd.ops import actuation

#: tokens that share a scale
BLOCK = 32
#: head widths that the kernels are built for; head_dim is padded to the next
WIDTHS = (32, 64, 96, 128, 192, 256)
FORMATS = ("fp8", "int8")

Position = Union[int, torch.Tensor]


class KV8Cache:
    """8-bit cache of ``batch`` sequences for ``num_layers`` layers.

    Where positions are given as numbers the cache follows each layer's
    length and refuses calls that would leave a hole or build on values it no
    longer holds; where they live on the GPU the caller answers for that,
    tokens behind max_seq are dropped, and so are all of a sequence whose
    position is negative. The same holds for a layer that a captured graph
    appends to, whose replays the host does not see.
    """

    def __init__(self, num_layers: int, batch: int, max_seq: int,
                 kv_heads: int, head_dim: int, fmt: str = "fp8",
                 dtype: torch.dtype = torch.bfloat16, device="cpu"):
        if fmt not in FORMATS:
            raise ValueError(f"unknown cache format {fmt!r}: one of {FORMATS}")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"keys and values must have 16 bits, got {dtype}")
        if not 1 <= head_dim <= WIDTHS[-1]:
            raise ValueError(f"head_dim must be 1..{WIDTHS[-1]}, "
                             f"got {head_dim}")
        if min(num_layers, batch, max_seq, kv_heads) < 1 \
                or max_seq >= 1 << 30:
            raise ValueError("cache sizes must be positive, max_seq < 2^30")
        self.num_layers, self.batch = num_layers, batch
        self.max_seq, self.kv_heads = max_seq, kv_heads
        self.head_dim, self.fmt, self.dtype = head_dim, fmt, dtype
        self.width = next(w for w in WIDTHS if w >= head_dim)
        blocks = (max_seq + BLOCK - 1) // BLOCK
        lead = (num_layers, 2, batch, kv_heads)
        self.codes = torch.zeros((*lead, blocks, BLOCK * self.width),
                                 dtype=torch.uint8, device=device)
        self.scales = torch.zeros((*lead, blocks), dtype=torch.float32,
                                  device=device)
        self.tail = torch.zeros((*lead, 2, BLOCK * self.width), dtype=dtype,
                                device=device)
        self.device = self.codes.device
        # layers without a store that a graph repeats
        self._followed = [True] * num_layers
        self._native = None
        if self.device.type == "cuda":
            self._native = actuation.require_native().Kv8Buffers(
                self.codes, self.scales, self.tail, max_seq, head_dim,
                fmt == "fp8")
        self.reset()

    def _check_scale(self, scale: float) -> None:
        if not abs(scale) < 3.4e38:
            raise ValueError(f"scale must be finite in fp32, got {scale}")

    def reset(self) -> None:
        """Forget all tokens (nothing is cleared)."""
        # None: appended at positions that only the GPU knows
        self._length: List[Optional[int]] = [
            0 if followed else None for followed in self._followed]
        self._raw_from = [0] * self.num_layers

    @property
    def nbytes(self) -> int:
        return self.codes.nbytes + self.scales.nbytes + self.tail.nbytes

    def free(self) -> None:
        self._native = None
        self.codes = self.scales = self.tail = None  # type: ignore

    # -- bookkeeping of positions that the host knows -----------------------

    def _check_layer(self, layer: int) -> None:
        if self.codes is None:
            raise ValueError("the cache was freed")
        if not 0 <= layer < self.num_layers:
            raise ValueError(f"no layer {layer}: the cache has "
                             f"{self.num_layers}")

    def _check_rows(self, x: torch.Tensor, name: str, heads: int) -> None:
        if x.dim() != 4 or x.shape[0] != self.batch \
                or x.shape[3] != self.head_dim \
                or (x.shape[2] != heads if heads else
                    x.shape[2] < 1 or x.shape[2] % self.kv_heads):
            raise ValueError(
                f"{name} must be [{self.batch}, T, "
                f"{heads or f'a multiple of {self.kv_heads}'}, "
                f"{self.head_dim}], got {list(x.shape)}")
        if x.dtype != self.dtype or x.device != self.device:
            raise ValueError(f"{name} must be {self.dtype} on {self.device}, "
                             f"got {x.dtype} on {x.device}")
        if x.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} requires a gradient; the 8-bit cache "
                             "has no backward pass")

    def _check_span(self, *given: Optional[Position]) -> None:
        for t in given:
            if isinstance(t, torch.Tensor):
                self._check_ints(t, "start, counts or length")

    def _check_ints(self, t: torch.Tensor, name: str) -> None:
        if t.dtype != torch.int32 or t.shape != (self.batch,) \
                or t.device != self.device or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous int32 "
                             f"[{self.batch}] on {self.device}")

    def _may(self, layer: int, start: int, T: int, store: bool,
             counts: Optional[torch.Tensor]) -> None:
        """Refuse what does not fit the tokens held, as far as the host knows
        them."""
        end = start + T
        if start < 0 or end > self.max_seq:
            raise ValueError(f"tokens [{start}, {end}) lie outside the "
                             f"cache's {self.max_seq}")
        known = self._length[layer]
        if known is None or not T:
            return
        if not store:
            if counts is None and end > known:
                raise ValueError(f"attention over {end} tokens, but the "
                                 f"cache holds {known}")
        elif start > known:
            raise ValueError(f"appending at {start} would leave a hole "
                             f"behind the {known} tokens held")
        elif start % BLOCK and start < self._raw_from[layer]:
            raise ValueError(
                f"cannot append at {start}: raw values are held from "
                f"{self._raw_from[layer]} on (or start at a multiple of "
                f"{BLOCK})")

    def _stored(self, layer: int, start: Position, T: int,
                counts: Optional[torch.Tensor]) -> None:
        if not T:
            return
        if self._native is not None and self._native.capturing():
            self._followed[layer] = False
        if counts is not None or isinstance(start, torch.Tensor) \
                or not self._followed[layer]:
            self._length[layer] = None
            return
        known, end = self._length[layer], start + T
        if known is None:
            if start:
                return
            self._raw_from[layer] = 0
        self._length[layer] = end
        self._raw_from[layer] = max(
            min(self._raw_from[layer], start // BLOCK * BLOCK),
            (end // BLOCK - 1) * BLOCK)


def _check_pair(q: torch.Tensor, k: torch.Tensor) -> None:
    if q.shape[1] != k.shape[1]:
        raise ValueError(f"q has {q.shape[1]} tokens and k {k.shape[1]}")


def kv8_append(cache: KV8Cache, layer: int, k: torch.Tensor, v: torch.Tensor,
               start: Position, counts: Optional[torch.Tensor] = None
               ) -> None:
    """Store keys and values [B, T, kvH, hd] at positions start..start+T-1.

    start: a number, or int32 [B] on the cache's device; counts (int32 [B]):
    how many of the T tokens are each sequence's own, the rest is padding.
    Any strides but a contiguous last dimension."""
    cache._check_layer(layer)
    given = isinstance(start, torch.Tensor)
    T = k.shape[1] if k.dim() == 4 else 0
    if not given:
        cache._may(layer, start, T, True, counts)
    if cache._native is not None:
        cache._native.append(layer, k, v, start if given else None,
                             0 if given else start, counts)
    else:
        cache._check_rows(k, "k", cache.kv_heads)
        cache._check_rows(v, "v", cache.kv_heads)
        _check_pair(v, k)
        cache._check_span(start, counts)
        _store(cache, layer, k, v, start, counts)
    cache._stored(layer, start, T, counts)


def qk_norm_rope_kv8(cache: KV8Cache, layer: int, q: torch.Tensor,
                     k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor,
                     sin: torch.Tensor, start: Position,
                     q_norm: Optional[torch.Tensor] = None,
                     k_norm: Optional[torch.Tensor] = None,
                     counts: Optional[torch.Tensor] = None,
                     eps: float = 1e-6, interleaved: bool = True
                     ) -> torch.Tensor:
    """:func:`~fma_amd.ops.decode_ops.fast_qk_norm_rope` of q and k at
    positions start.. and :func:`kv8_append` of the result and v, in one
    launch; the same bits as the two calls. Returns the queries, zeros behind
    each sequence's count. The tables must cover the cache's max_seq."""
    cache._check_layer(layer)
    given = isinstance(start, torch.Tensor)
    T = k.shape[1] if k.dim() == 4 else 0
    if not given:
        cache._may(layer, start, T, True, counts)
    if cache._native is not None:
        out = cache._native.norm_rope_append(
            layer, q, k, v, cos, sin, start if given else None,
            0 if given else start, q_norm, k_norm, counts, eps, interleaved)
        cache._stored(layer, start, T, counts)
        return out
    from fma_amd.ops.decode_ops import _check_rope, rope_rows
    cache._check_rows(q, "q", 0)
    cache._check_rows(k, "k", cache.kv_heads)
    cache._check_rows(v, "v", cache.kv_heads)
    _check_pair(q, k)
    _check_pair(v, k)
    _check_rope(q, k, cos, sin, q_norm, k_norm)
    cache._check_span(start, counts)
    if cos.shape[0] < cache.max_seq:
        raise ValueError(f"the cos/sin tables hold {cos.shape[0]} positions, "
                         f"the cache {cache.max_seq}")
    starts, ns = _host_span(cache, start, T, counts)
    pos = starts[:, None] + torch.arange(T)
    pos = pos.clamp(0, cache.max_seq - 1)
    live = (torch.arange(T) < ns[:, None])[:, :, None, None]
    qo = rope_rows(q, q_norm, cos, sin, pos, eps, interleaved)
    ko = rope_rows(k, k_norm, cos, sin, pos, eps, interleaved)
    _store(cache, layer, ko, v, start, counts)
    cache._stored(layer, start, T, counts)
    return torch.where(live, qo, torch.zeros((), dtype=qo.dtype))


def kv8_attention(q: torch.Tensor, cache: KV8Cache, layer: int,
                  start: Position, counts: Optional[torch.Tensor] = None,
                  scale: Optional[float] = None) -> torch.Tensor:
    """Causal attention of q [B, T, qH, hd], whose tokens lie at positions
    start.. and are in the cache already, over everything up to themselves:
    softmax(scale * q K^T) V, scale = head_dim ** -0.5 by default, qH a
    multiple of kvH. start and counts as in :func:`kv8_append`; rows behind a
    sequence's count come out as zeros, and outputs saturate at the type's
    largest value, as which an infinity in V counts. Where the cache knows its length the
    queries may lie anywhere in it; else, and in a captured graph, each
    sequence's last query has to be the last token stored, which says what of
    it is coded already."""
    cache._check_layer(layer)
    given = isinstance(start, torch.Tensor)
    if not given:
        cache._may(layer, start, q.shape[1] if q.dim() == 4 else 0, False,
                   counts)
    if scale is None:
        scale = cache.head_dim ** -0.5
    cache._check_scale(scale)
    if cache._native is not None:
        held = cache._length[layer]
        if held is not None and cache._native.capturing():
            # the length at a replay is not today's
            if not given and counts is None and start + q.shape[1] != held:
                raise ValueError(
                    f"a captured call's queries must end at the last of the "
                    f"{held} tokens held")
            held = None
        return cache._native.attention(q, layer, start if given else None,
                                       0 if given else start, counts, scale,
                                       held or 0)
    cache._check_rows(q, "q", 0)
    cache._check_span(start, counts)
    return _attend(q, cache, layer, start, counts, scale)


def kv8_read(cache: KV8Cache, layer: int, start: Position, n: int,
             length: Position) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values [B, n, kvH, hd] that the cache stands for at
    positions start..start+n-1 of sequences of ``length`` tokens (all that
    were stored: that says which are coded), in its 16-bit type, where they
    saturate; zeros behind the length."""
    cache._check_layer(layer)
    known = cache._length[layer]
    if known is not None and not isinstance(length, torch.Tensor) \
            and length != known:
        raise ValueError(f"length {length}, but the cache holds {known}")
    if not 0 <= n < 1 << 29:
        raise ValueError(f"cannot read {n} tokens")
    args = []
    for value, name in ((start, "start"), (length, "length")):
        if isinstance(value, torch.Tensor):
            args += [value, 0]
        else:
            if not 0 <= value <= cache.max_seq:
                raise ValueError(f"{name} {value} lies outside the cache's "
                                 f"{cache.max_seq}")
            args += [None, value]
    if cache._native is not None:
        return cache._native.read(layer, args[0], args[1], n, args[2],
                                  args[3])
    cache._check_span(args[0], args[2])
    out = torch.zeros((2, cache.batch, n, cache.kv_heads, cache.head_dim),
                      dtype=cache.dtype)
    for b in range(cache.batch):
        s = max(int(start[b]) if args[0] is not None else int(start), 0)
        end = min(int(length[b]) if args[2] is not None else int(length),
                  cache.max_seq)
        m = min(n, end - s)
        if m > 0:
            for w, x in enumerate(_held(cache, layer, b, end)):
                top = torch.finfo(cache.dtype).max
                coded = max(min(end // BLOCK * BLOCK - s, m), 0)
                x = x[s:s + m]
                out[w, b, :coded] = x[:coded].clamp(-top, top).to(cache.dtype)
                out[w, b, coded:m] = x[coded:].to(cache.dtype)
    return out[0], out[1]


# -- the same on the CPU -------------------------------------------------------

@lru_cache(maxsize=None)
def _places(width: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Where value (token, d) of a block lies, for K and for V: the order in
    which the matrix unit's lanes take them (kidx / vidx in csrc/kv8.hip)."""
    tok = torch.arange(BLOCK)[:, None]
    d = torch.arange(width)[None]
    k = ((((d >> 5) * 64 + ((d >> 3) & 3) * 16 + (tok & 15)) * 2
          + (tok >> 4)) * 8 + (d & 7))
    v = ((((d >> 5) * 64 + ((tok >> 2) & 3) * 16 + (d & 15)) * 2
          + ((d >> 4) & 1)) * 8 + (tok >> 4) * 4 + (tok & 3))
    return k, v


def _host_span(cache: KV8Cache, start: Position, T: int,
               counts: Optional[torch.Tensor]
               ) -> Tuple[torch.Tensor, torch.Tensor]:
    s = start.long() if isinstance(start, torch.Tensor) \
        else torch.full((cache.batch,), start, dtype=torch.long)
    n = counts.long().clamp(max=T) if counts is not None \
        else torch.full((cache.batch,), T, dtype=torch.long)
    n = torch.where((s < 0) | (s > cache.max_seq), torch.zeros_like(n),
                    torch.minimum(n, cache.max_seq - s)).clamp(min=0)
    return s, n


def encode(x: torch.Tensor, fmt: str) -> Tuple[torch.Tensor, torch.Tensor]:
    """Codes (as uint8) and scale of one block [32, hd] of 16-bit values."""
    x = x.float()
    fine = torch.isfinite(x)
    a = torch.where(fine, x.abs(), torch.zeros(())).amax()
    x = torch.where(torch.isnan(x), torch.zeros(()), x.clamp(-a, a))
    a = a.clamp(min=2.0 ** -100)
    if fmt == "fp8":
        m, e = torch.frexp(a)
        scale = torch.ldexp(torch.ones(()), torch.where(m <= 0.875, e - 9,
                                                        e - 8))
        return (x / scale).to(torch.float8_e4m3fn).view(torch.uint8), scale
    # both quotients correctly rounded (torch divides by a number by way of
    # its reciprocal, which is not)
    mul, scale = (127 / a.double()).float(), (a.double() / 127).float()
    code = (x * mul).round().clamp(-127, 127)
    return (code + 128).to(torch.uint8), scale


def _store(cache: KV8Cache, layer: int, k: torch.Tensor, v: torch.Tensor,
           start: Position, counts: Optional[torch.Tensor]) -> None:
    starts, ns = _host_span(cache, start, k.shape[1], counts)
    hd = cache.head_dim
    for b in range(cache.batch):
        s, n = int(starts[b]), int(ns[b])
        end = s + n
        for blk in range(s // BLOCK, (end + BLOCK - 1) // BLOCK if n else 0):
            lo, hi = max(s, blk * BLOCK), min(end, (blk + 1) * BLOCK)
            rows = slice(lo - blk * BLOCK, hi - blk * BLOCK)
            for h in range(cache.kv_heads):
                for w, (src, place) in enumerate(zip((k, v),
                                                     _places(cache.width))):
                    raw = cache.tail[layer, w, b, h, blk & 1]
                    x = raw[place[:, :hd]].clone()
                    x[rows] = src[b, lo - s:hi - s, h]
                    if hi == (blk + 1) * BLOCK:
                        flat, scale = encode(x, cache.fmt)
                        codes = cache.codes[layer, w, b, h, blk]
                        codes.fill_(0 if cache.fmt == "fp8" else 128)
                        codes[place[:, :hd]] = flat
                        cache.scales[layer, w, b, h, blk] = scale
                    if blk >= end // BLOCK - 1:
                        raw[place[rows, :hd]] = x[rows]


def _held(cache: KV8Cache, layer: int, b: int, length: int
          ) -> Tuple[torch.Tensor, torch.Tensor]:
    """What the cache holds of one sequence: two [length, kvH, hd], fp32."""
    full, left = divmod(length, BLOCK)
    hd = cache.head_dim
    out = []
    for w, place in enumerate(_places(cache.width)):
        at = place[:, :hd]
        codes = cache.codes[layer, w, b, :, :full][..., at]
        if cache.fmt == "fp8":
            x = codes.view(torch.float8_e4m3fn).float()
        else:
            x = codes.float() - 128
        x = (x * cache.scales[layer, w, b, :, :full, None, None]) \
            .flatten(1, 2)
        raw = cache.tail[layer, w, b, :, full & 1][..., at][:, :left].float()
        out.append(torch.cat((x, raw), 1).transpose(0, 1))
    return out[0], out[1]


def _attend(q: torch.Tensor, cache: KV8Cache, layer: int, start: Position,
            counts: Optional[torch.Tensor], scale: float) -> torch.Tensor:
    T, group = q.shape[1], q.shape[2] // cache.kv_heads
    starts, ns = _host_span(cache, start, T, counts)
    out = torch.zeros(q.shape, dtype=torch.float32)
    top = torch.finfo(cache.dtype).max
    for b in range(cache.batch):
        s, n = int(starts[b]), int(ns[b])
        if not n:
            continue
        k, v = (x[:s + n].repeat_interleave(group, 1).transpose(0, 1)
                for x in _held(cache, layer, b,
                               max(cache._length[layer] or 0, s + n)))
        v = torch.nan_to_num(v, posinf=top, neginf=-top)
        score = q[b, :n].float().transpose(0, 1) @ k.transpose(1, 2) * scale
        late = torch.arange(s + n) > s + torch.arange(n)[:, None]
        p = torch.softmax(score.masked_fill(late, float("-inf")), -1)
        out[b, :n] = (p @ v).transpose(0, 1)
    return out.clamp(-top, top).to(q.dtype)

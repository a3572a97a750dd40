"""Fused decode elementwise ops with eager fallbacks.

One launch each for rmsnorm / silu*up / RoPE on the single-token decode
path (profiling showed the fragmented eager versions cost more GPU time
than the GEMVs). Fallbacks implement identical math for CPU and for
non-decode shapes; numerics are compared in tests/gpu.
"""

from __future__ import annotations

import os

import torch
import torch.nn.functional as F

from fma_amd.ops import actuation

_ENABLED = None


def available() -> bool:
    global _ENABLED
    if _ENABLED is None:
        _ENABLED = (torch.cuda.is_available()
                    and actuation.native_available()
                    and os.environ.get("FMA_DISABLE_FUSED_OPS") != "1")
    return _ENABLED


def _fusable(x: torch.Tensor) -> bool:
    return (available() and x.is_cuda and x.dtype == torch.bfloat16
            and x.is_contiguous() and (x.numel() & 7) == 0)


def fast_rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    """Single-token rmsnorm; x may be [..., H] with numel == H."""
    H = x.shape[-1]
    if _fusable(x) and x.numel() == H and w.is_contiguous():
        return actuation._C.rmsnorm1_bf16(x.reshape(-1), w, eps).view(x.shape)
    xf = x.float()
    xf = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    return (xf * w.float()).to(x.dtype)


def fast_silu_mul(g: torch.Tensor, u: torch.Tensor) -> torch.Tensor:
    if _fusable(g) and u.is_contiguous():
        return actuation._C.silu_mul_bf16(
            g.reshape(-1), u.reshape(-1)).view(g.shape)
    return F.silu(g) * u


def fast_rope1(x: torch.Tensor, cos_row: torch.Tensor, sin_row: torch.Tensor
               ) -> torch.Tensor:
    """RoPE for one position: x [B=1, 1, heads, hd]; cos/sin_row [hd/2] fp32.
    In-place on the fused path (x is a fresh projection output)."""
    B, T, heads, hd = x.shape
    if _fusable(x) and B == 1 and T == 1:
        actuation._C.rope1_bf16_(x.reshape(-1), cos_row.reshape(-1),
                                 sin_row.reshape(-1), heads, hd)
        return x
    c = cos_row.view(1, 1, 1, hd // 2)
    s = sin_row.view(1, 1, 1, hd // 2)
    xf = x.float().view(B, T, heads, hd // 2, 2)
    x0, x1 = xf[..., 0], xf[..., 1]
    out = torch.stack((x0 * c - x1 * s, x0 * s + x1 * c), dim=-1)
    return out.view(B, T, heads, hd).to(x.dtype)


def _check_rope(q, k, cos, sin, q_norm, k_norm) -> None:
    hd = q.shape[-1]
    if cos.dim() != 2 or cos.shape != sin.shape \
            or cos.dtype != torch.float32 or sin.dtype != torch.float32 \
            or not (cos.is_contiguous() and sin.is_contiguous()) \
            or cos.device != q.device or sin.device != q.device:
        raise ValueError("cos/sin must be contiguous fp32 [S, rot/2] on "
                         f"{q.device}")
    if not 1 <= cos.shape[1] <= hd // 2 or cos.shape[0] < 1:
        raise ValueError(f"tables of {list(cos.shape)} cannot rotate heads "
                         f"of {hd}")
    for w in (q_norm, k_norm):
        if w is not None and (w.shape != (hd,) or w.dtype != q.dtype
                              or w.device != q.device
                              or not w.is_contiguous()):
            raise ValueError(f"norm weights must be contiguous {q.dtype} "
                             f"[{hd}] on {q.device}")
        if w is not None and w.requires_grad and torch.is_grad_enabled():
            raise ValueError("a norm weight requires a gradient; this has no "
                             "backward pass")


def rope_rows(x, w, cos, sin, pos, eps: float, interleaved: bool):
    """The plain form of :func:`fast_qk_norm_rope` for one of its tensors;
    pos [B, T] within the tables."""
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + eps) * w.float()
    c, s = cos[pos].unsqueeze(2), sin[pos].unsqueeze(2)
    n = cos.shape[1]
    if interleaved:
        a, b = y[..., 0:2 * n:2], y[..., 1:2 * n:2]
        r = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    else:
        a, b = y[..., :n], y[..., n:2 * n]
        r = torch.cat((a * c - b * s, a * s + b * c), -1)
    return torch.cat((r, y[..., 2 * n:]), -1).to(x.dtype)


def fast_qk_norm_rope(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor,
                      sin: torch.Tensor, pos, q_norm=None, k_norm=None,
                      eps: float = 1e-6, interleaved: bool = True):
    """RMSNorm of each query and key head over its head_dim, then the position
    rotation, in one pass: fp32 inside, rounded once. Returns new (q, k).

    q [B, T, qH, hd], k [B, T, kvH, hd] in bf16, fp16 or fp32, any strides
    but a contiguous last dimension (views of a fused projection need no
    copy). q_norm / k_norm [hd]: gains, None leaves that norm out. cos / sin
    fp32 [S, rot/2]: the first rot of hd values turn, the rest passes; a
    factor for long contexts belongs into the tables. Pairs are (2i, 2i+1),
    or with interleaved=False (i, i + rot/2). pos: the first token's position
    as a number, or int32 / int64 [B] of first positions, or [B, T] of every
    token's. A position outside the tables is refused where the host knows
    it; one that only the GPU knows gives NaN.

    One launch on the GPU for any T; torch operations on the CPU."""
    if q.is_cuda:
        given = isinstance(pos, torch.Tensor)
        return actuation.require_native().qk_norm_rope(
            q, k, cos, sin, pos if given else None, 0 if given else pos,
            q_norm, k_norm, eps, interleaved)
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] \
            or q.shape[3] != k.shape[3] or q.shape[2] < 1 or k.shape[2] < 1:
        raise ValueError(f"q {list(q.shape)} and k {list(k.shape)} must be "
                         "[B, T, heads, head_dim] alike but for the heads")
    if q.dtype != k.dtype or q.device != k.device or q.dtype not in (
            torch.bfloat16, torch.float16, torch.float32):
        raise ValueError("q and k must both be bf16, fp16 or fp32 on one "
                         "device")
    B, T, _, hd = q.shape
    if not 2 <= hd <= 256:
        raise ValueError(f"head_dim must be 2..256, got {hd}")
    if (q.requires_grad or k.requires_grad) and torch.is_grad_enabled():
        raise ValueError("q or k requires a gradient; this has no backward "
                         "pass")
    _check_rope(q, k, cos, sin, q_norm, k_norm)
    given = isinstance(pos, torch.Tensor)
    if given:
        if pos.dtype not in (torch.int32, torch.int64) \
                or pos.device != q.device \
                or pos.shape not in ((B,), (B, T)):
            raise ValueError(f"pos must be int32 or int64 [{B}] or "
                             f"[{B}, {T}] on {q.device}")
    elif pos < 0 or pos + T > cos.shape[0]:
        raise ValueError(f"positions [{pos}, {pos + T}) lie outside the "
                         f"tables' {cos.shape[0]}")
    if not given:
        pos = torch.full((B,), pos, dtype=torch.long)
    if pos.dim() == 1:
        pos = pos.long()[:, None] + torch.arange(T)
    pos = pos.long()
    out = (pos < 0) | (pos >= cos.shape[0])
    pos = pos.clamp(0, cos.shape[0] - 1)
    nan = torch.full((), float("nan"), dtype=q.dtype)
    return tuple(torch.where(out[:, :, None, None], nan, rope_rows(
        x, w, cos, sin, pos, eps, interleaved))
        for x, w in ((q, q_norm), (k, k_norm)))


def fast_rope_qkv_store(q, k, v, kcache, vcache, cos_tab, sin_tab,
                        pos=None, pos_dev=None) -> bool:
    """RoPE(q in place) + RoPE(k)->cache + v->cache in ONE launch
    (replaces 2 rope + 2 cache-write kernels on the decode path).
    q [1,1,qH,hd]; k/v [1,1,kvH,hd]; k/vcache [S,kvH,hd]. Returns False
    when the fused kernel does not apply (caller uses the unfused ops)."""
    if not available():
        return False
    if not (q.is_cuda and q.dtype == torch.bfloat16 and q.is_contiguous()
            and k.is_contiguous() and v.is_contiguous()
            and kcache.is_contiguous() and vcache.is_contiguous()):
        return False
    qh, hd = q.shape[-2], q.shape[-1]
    kvh = k.shape[-2]
    actuation._C.rope_qkv_store_bf16_(
        q.reshape(qh, hd), k.reshape(kvh, hd), v.reshape(kvh, hd),
        kcache, vcache, cos_tab, sin_tab, pos_dev,
        0 if pos is None else int(pos))
    return True


def fast_attn_prefill(q: torch.Tensor, k_cache: torch.Tensor,
                      v_cache: torch.Tensor, pos0: int):
    """Causal GQA prefill on MFMA matrix cores. q [1,T,qH,hd]; k/v_cache
    [S,kvH,hd] holding keys [0, pos0+T). Returns [1,T,qH*hd] or None when
    the kernel does not apply (caller falls back to SDPA).

    Dispatch is measured, not aspirational (tools/prefill_bench.py on
    MI355X): the hand-written kernel beats torch SDPA up to T~128 and
    trails it beyond (0.56x at 4K ctx), so by default it serves short
    prefills only. FMA_MFMA_PREFILL=1 forces it always, =0 never."""
    mode = os.environ.get("FMA_MFMA_PREFILL", "auto")
    if not available() or mode == "0":
        return None
    b, t, qh, hd = q.shape
    # FMA_PREFILL_16=1 opts into the 16-row fragment kernel (occupancy 4,
    # doubled tile grid — built for exactly the mid-T range the 32-row
    # kernel loses; numerics hardware-validated, perf unmeasured), so the
    # short-prefill cutoff does not apply to it
    p16 = os.environ.get("FMA_PREFILL_16") == "1"
    if mode != "1" and not p16 and t > 128:
        return None
    if (b != 1 or hd not in (64, 128) or not q.is_cuda
            or q.dtype != torch.bfloat16
            or qh % k_cache.shape[1] != 0
            or pos0 + t > k_cache.shape[0]):
        return None
    out = actuation._C.attn_prefill_bf16(
        q.reshape(t, qh, hd).contiguous(), k_cache, v_cache, pos0)
    return out.view(1, t, qh * hd)


def fast_attn_decode(q: torch.Tensor, k_cache: torch.Tensor,
                     v_cache: torch.Tensor, t: int):
    """q [1,1,qH,hd]; k/v_cache [S,kvH,hd] (one layer, batch 1). Returns
    [1,1,qH*hd] or None when the fused kernel does not apply."""
    if not available():
        return None
    _, _, qh, hd = q.shape
    if (hd % 64 != 0 or hd > 256 or t > (1 << 17) or not q.is_cuda
            or q.dtype != torch.bfloat16
            or qh % k_cache.shape[1] != 0):
        return None
    out = actuation._C.attn_decode_bf16(
        q.reshape(qh, hd).contiguous(), k_cache, v_cache, t)
    return out.view(1, 1, qh * hd)

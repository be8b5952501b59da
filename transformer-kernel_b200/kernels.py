"""Attention forward on the B200 kernel.

Same contract as the reference's ``src/kernels.py`` ``flash_attention``
(:250-294) and ``attention_supported`` (:96-103): ``q``/``k``/``v`` are
logically ``[B, H, S, hd]`` fp16 with arbitrary strides and a contiguous
last dimension (e.g. views straight out of the fused ``[B, S, 3, H, hd]``
QKV projection); the result is the context written directly as
``[B, S, H*hd]``. Scores are scaled after ``q.k`` (the baseline's order),
softmax statistics are fp32. Backed by ``tk_attn_fwd`` of libtk_b200; no
SDPA fallback.
"""

from __future__ import annotations

from typing import Optional

import torch

import _tklib as tk

__all__ = ["kernels_available", "attention_supported", "flash_attention", "window_attention"]


def kernels_available() -> bool:
    try:
        tk.lib()
        return True
    except tk.TKError:
        return False


def attention_supported(head_dim: int, dtype: torch.dtype, device: torch.device) -> bool:
    return (
        device.type == "cuda"
        and dtype == torch.float16
        and bool(tk.lib().tk_attn_supported(int(head_dim)))
    )


def flash_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    scale: float,
    causal: bool,
    kv_len: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Exact attention; returns the context in ``[B, S, H*hd]`` fp16.

    ``kv_len`` (int32 ``[B]``, optional) masks keys ``>= kv_len[b]`` -- the
    harness's prefix key-padding mask."""
    if not (q.shape == k.shape == v.shape) or q.dim() != 4:
        raise ValueError(f"q/k/v must share a [B, H, S, hd] shape, got {q.shape}, {k.shape}, {v.shape}")
    if not (q.dtype == k.dtype == v.dtype == torch.float16):
        raise tk.TKError("flash_attention", -2, "q/k/v must be float16")
    if not (q.stride() == k.stride() == v.stride()) or q.stride(-1) != 1:
        raise tk.TKError("flash_attention", -1, "q/k/v need identical strides and a contiguous last dimension")
    dev = tk.require_cuda(q, k, v, kv_len, out)
    B, H, S, hd = q.shape
    if out is None:
        out = torch.empty((B, S, H * hd), dtype=torch.float16, device=dev)
    elif out.shape != (B, S, H * hd) or out.stride(-1) != 1 or out.stride(0) != S * out.stride(1):
        raise ValueError("out must be [B, S, H*hd] with unit last stride and rows S*ld apart per batch")
    if kv_len is not None:
        kv_len = kv_len.to(dtype=torch.int32).contiguous()
    with torch.cuda.device(dev):
        tk.call(
            "tk_attn_fwd",
            q.data_ptr(), k.data_ptr(), v.data_ptr(),
            q.stride(0), q.stride(1), q.stride(2),
            out.data_ptr(), out.stride(1),
            B, S, H, hd, float(scale), int(bool(causal)),
            tk.ptr(kv_len), tk.stream_handle(dev),
        )
    return out


def window_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    scale: float,
    window: int,
    sinks: int = 0,
    kv_len: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Causal attention in which query i sees key j when ``i - j < window`` or
    ``j < sinks``; returns the context in ``[B, S, H*hd]`` fp16.

    ``q`` is ``[B, H, S, hd]``, ``k`` and ``v`` ``[B, Hkv, S, hd]`` with H a
    multiple of Hkv (query head h reads head ``h // (H // Hkv)``), any strides
    with a contiguous last dimension, shared by k and v (in dimensions of more
    than one entry). ``kv_len`` (int32
    ``[B]``, optional) masks keys ``>= kv_len[b]``; what they hold is never
    used. Rows that see no key are zero. The other values of k and v must be
    finite: inside a tile a masked weight is 0 times the value. Backed by
    ``tk_attn_window``; a window of S or more is plain causal attention."""
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError(f"q must be [B, H, S, hd] and k, v [B, Hkv, S, hd], got {q.shape}, {k.shape}, {v.shape}")
    B, H, S, hd = q.shape
    Bk, Hkv, Sk, hdk = k.shape
    if (B, S, hd) != (Bk, Sk, hdk):
        raise ValueError(f"q must be [B, H, S, hd] and k, v [B, Hkv, S, hd], got {q.shape}, {k.shape}, {v.shape}")
    if B * H * S * hd * Hkv == 0 or H % Hkv != 0:
        raise ValueError(f"sizes must be positive and {H} query heads a multiple of {Hkv} key-value heads")
    if not (q.dtype == k.dtype == v.dtype == torch.float16):
        raise tk.TKError("window_attention", -2, "q/k/v must be float16")
    q_b, q_h, q_s, q_1 = q.stride()
    k_b, k_h, k_s, k_1 = strides = k.stride()
    # the stride of a dimension of one entry means nothing
    if q_1 != 1 or k_1 != 1 or (strides != v.stride() and any(
            n > 1 and a != b for n, a, b in zip(k.shape, strides, v.stride()))):
        raise tk.TKError("window_attention", -1, "k and v need identical strides, and all a contiguous last dimension")
    dev = q.device
    if dev.type != "cuda" or k.device != dev or v.device != dev:
        tk.require_cuda(q, k, v)
    ld = H * hd
    if out is None:
        out = q.new_empty((B, S, ld))
    else:
        tk.require_cuda(q, out)
        if S > 1 or out.stride(1) > ld:
            ld = out.stride(1)
        if (out.shape != (B, S, H * hd) or out.dtype != torch.float16 or out.stride(2) != 1
                or (B > 1 and out.stride(0) != S * ld)):
            raise ValueError("out must be fp16 [B, S, H*hd] with unit last stride and rows S*ld apart per batch")
    kv_ptr = None
    if kv_len is not None:
        tk.require_cuda(q, kv_len)
        if kv_len.shape != (B,):
            raise ValueError(f"kv_len must have shape ({B},), got {tuple(kv_len.shape)}")
        kv_len = kv_len.to(dtype=torch.int32).contiguous()
        kv_ptr = kv_len.data_ptr()
    tk.call_on(dev, "tk_attn_window", q.data_ptr(), q_b, q_h, q_s, k.data_ptr(), v.data_ptr(), k_b, k_h, k_s,
               out.data_ptr(), ld, B, S, H, Hkv, hd, scale, window, sinks, kv_ptr)
    return out

"""Fused per-layer attention preparation on the GPU.

``qk_norm_rope_write`` does, in one kernel, what Qwen3Attention.__call__ of the
reference does between the QKV projection and the attention call
(src/nano_vllm_metal/models/qwen3.py:100-116): RMSNorm of every q and k head row
(q_norm / k_norm), RoPE of q and k at each token's position, and the paged write of
the rotated K and the raw V (int8-quantised for int8 pools), returning q in the layout
``paged_attention`` takes.
"""

from __future__ import annotations

import torch

from .. import _native as nv
from .rotary_embedding import RoPE


def _token_rows(x: torch.Tensor) -> tuple[torch.Tensor, int]:
    """[B, L, H, D] -> (tensor whose rows are read in place, elements between tokens).
    Views of a fused QKV projection ([B, L, (Hq + 2 Hkv) * D] split along the last
    axis) keep their token stride and are read without a copy."""
    B, L, H, D = x.shape
    sb, st, sh, sd = x.stride()
    if L == 1:  # the stride of one token says nothing (a view of a decode step's projection gives H * D)
        st = sb if B > 1 else H * D
    if sd == 1 and sh == D and (B == 1 or sb == L * st) and st >= H * D:
        return x, st
    return x.contiguous(), H * D


def _on_vectors(x: torch.Tensor, stride: int, elements: int) -> tuple[torch.Tensor, int]:
    """Rows as ``_token_rows`` gives them, copied where they do not start on the vectors that the kernels move."""
    if stride % elements == 0 and x.data_ptr() % (2 * elements) == 0:
        return x, stride
    return x.clone(memory_format=torch.contiguous_format), x.shape[2] * x.shape[3]


def qk_norm_rope_write(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_norm_weight: torch.Tensor | None,
                       k_norm_weight: torch.Tensor | None, rope: RoPE, positions: torch.Tensor, key_pages: torch.Tensor,
                       value_pages: torch.Tensor, slot_mapping: torch.Tensor, *, eps: float = 1e-5,
                       key_scales: torch.Tensor | None = None, value_scales: torch.Tensor | None = None,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """q [B, L, Hq, D], k/v [B, L, Hkv, D] (the projections, f16/bf16); positions [B, L]
    (request offset + index); slot_mapping [B * L] int64 (page_id * page_size + offset,
    negative = skip).  Returns q normalised and rotated, [B, Hq, L, D]; K (normalised,
    rotated) and V are written into key_pages / value_pages [P, Hkv, page_size, D], of q's
    dtype, int8 or packed 4-bit codes (uint8 [P, Hkv, page_size, D / 2] with scales of q's
    dtype, see ``cache.paged.write_slots``).  Without norm weights (both None: models that
    have no q/k norm) the rows are rotated as they are."""
    dev = nv.require_cuda("qk_norm_rope_write", q, k, v, q_norm_weight, k_norm_weight, positions, key_pages, value_pages,
                          slot_mapping, key_scales, value_scales, out)
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape:
        raise RuntimeError("qk_norm_rope_write: q must be [B, L, Hq, D], k and v [B, L, Hkv, D]")
    B, L, Hq, D = q.shape
    Hkv = k.shape[2]
    if k.shape[0] != B or k.shape[1] != L or k.shape[3] != D:
        raise RuntimeError("qk_norm_rope_write: q, k, v disagree on batch, length or head dim")
    if q.dtype != k.dtype or q.dtype != v.dtype or q.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("qk_norm_rope_write: q, k, v must share one dtype, float16 or bfloat16")
    if rope.dims != D:
        raise RuntimeError("qk_norm_rope_write: the RoPE tables are for a different head dim")
    T = B * L
    vec = 4 if key_pages.dtype is torch.uint8 else max(D // 32, 1)  # elements a lane moves at a time
    qc, q_st = _on_vectors(*_token_rows(q), vec)
    kc, k_st = _on_vectors(*_token_rows(k), vec)
    vc, v_st = _on_vectors(*_token_rows(v), vec)
    if k_st != v_st:
        kc, vc = (x if st == Hkv * D else x.contiguous() for x, st in ((kc, k_st), (vc, v_st)))
        k_st = v_st = Hkv * D
    if (q_norm_weight is None) != (k_norm_weight is None):
        raise RuntimeError("qk_norm_rope_write: q and k are normalised both or not at all")
    wq = wk = None
    if q_norm_weight is not None:
        wq, wk = nv.packed(q_norm_weight, q.dtype), nv.packed(k_norm_weight, q.dtype)
    if positions.numel() != T or slot_mapping.numel() != T:
        raise RuntimeError("qk_norm_rope_write: positions and slot_mapping need one entry per token")
    pos, slots = nv.packed(positions, torch.int32), nv.packed(slot_mapping, torch.int64)
    cos, sin = rope.cos_freqs, rope.sin_freqs
    if cos.device != dev or sin.device != dev:
        cos, sin = cos.to(dev), sin.to(dev)
    cos, sin = cos.contiguous(), sin.contiguous()
    kp, vp = key_pages, value_pages
    P, Hkv_p, ps, D_p = kp.shape
    int8, u4 = kp.dtype == torch.int8, kp.dtype == torch.uint8
    if Hkv_p != Hkv or (D_p != D and not u4) or vp.shape != kp.shape:
        raise RuntimeError("qk_norm_rope_write: page pools must be [P, Hkv, page_size, D] matching k")
    if not (kp.is_contiguous() and vp.is_contiguous()):
        raise RuntimeError("qk_norm_rope_write: page pools must be contiguous (written in place)")
    if u4:
        nv.require_u4("qk_norm_rope_write", D, kp, vp, key_scales, value_scales)
        if key_scales.dtype != q.dtype:
            raise RuntimeError("qk_norm_rope_write: scales of 4-bit pages must be of q's dtype")
    if int8:
        if key_scales is None or value_scales is None:
            raise RuntimeError("qk_norm_rope_write: int8 pages need key_scales and value_scales")
        for sc in (key_scales, value_scales):
            if tuple(sc.shape) != (P, Hkv, ps, 1) or not sc.is_contiguous() or not sc.is_floating_point():
                raise RuntimeError("qk_norm_rope_write: scales must be contiguous float [P, Hkv, page_size, 1]")
        if key_scales.dtype != value_scales.dtype:
            raise RuntimeError("qk_norm_rope_write: key and value scales must share one dtype")
    if out is None:
        out = q.new_empty((B, Hq, L, D))
    elif tuple(out.shape) != (B, Hq, L, D) or out.dtype != q.dtype or not out.is_contiguous():
        raise RuntimeError("qk_norm_rope_write: out must be a contiguous [B, Hq, L, D] tensor of q's dtype")
    ks = key_scales if int8 or u4 else None
    vs = value_scales if int8 or u4 else None
    with nv.on_device(dev):
        nv.check(nv.lib().nvm_qk_norm_rope_write(
            qc.data_ptr(), kc.data_ptr(), vc.data_ptr(), nv.dtype_code(q.dtype), q_st, k_st, nv.ptr(wq), nv.ptr(wk),
            float(eps), cos.data_ptr(), sin.data_ptr(), cos.shape[0], 1 if rope.traditional else 0, pos.data_ptr(), out.data_ptr(), L,
            kp.data_ptr(), vp.data_ptr(), nv.dtype_code(kp.dtype), nv.ptr(ks), nv.ptr(vs),
            nv.dtype_code(ks.dtype) if ks is not None else nv.NVM_F16, slots.data_ptr(), T, Hq, Hkv, D, P, ps,
            nv.stream_ptr(dev)))
    return out

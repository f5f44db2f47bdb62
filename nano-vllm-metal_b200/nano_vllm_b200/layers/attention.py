"""Attention operators with the reference's signatures, running on libnvm_attn.

Mirrors ``src/nano_vllm_metal/layers/attention.py`` of nano-vllm-metal:

* ``paged_attention`` (reference ``attention.py:154-230``): same arguments, same
  mask rules (None or "causal"; an array mask raises NotImplementedError), same
  default scale ``1/sqrt(D)``, same fp32 ``[B, Hq, L, D]`` result.  int8 pages with
  ``key_scales`` / ``value_scales`` are dequantised inside the kernel for every L
  (the reference dequantises the whole pool for L > 1, ``attention.py:204-215``).
* ``flash_attention`` (reference ``attention.py:103-151``): dense attention with
  GQA and an optional additive mask; "causal" never materialises a mask tensor.
* ``causal_mask`` / ``scaled_dot_product_attention_grouped`` (``attention.py:59-100``):
  plain-torch dense references, used by tests and callers that want them.

Extensions (keyword-only, defaults keep the reference behaviour): ``out_dtype``
lets the model receive bf16/fp16 directly instead of casting the fp32 result;
``window`` / ``sinks`` limit every query token to the last ``window`` positions (its own
included) and the first ``sinks``; ``key_mass`` accumulates the attention weight that
every cached key receives, by which ``cache.evict`` trims a cache.
Query tensors are read in their own dtype (fp32, fp16 or bf16); the reference's
``query.astype(float32)`` is exact for 16-bit queries, so it is skipped.
"""

from __future__ import annotations

import torch

from .. import _native as nv

__all__ = [
    "causal_mask",
    "scaled_dot_product_attention_grouped",
    "flash_attention",
    "paged_attention",
]


def _check_window(op: str, window: int | None, sinks: int) -> None:
    if window is not None and not 1 <= window < 2 ** 31:
        raise RuntimeError(f"{op}: window must be at least 1 and below 2^31 (None for no window), got {window}")
    if not 0 <= sinks < 2 ** 31:
        raise RuntimeError(f"{op}: sinks must not be negative, nor 2^31 or more, got {sinks}")


def _row_strides(what: str, x: torch.Tensor) -> tuple[int, int]:
    """The first two strides of x [B, H, S], whose rows must be contiguous along S and must not
    overlap one another."""
    B, H, S = x.shape
    if x.is_contiguous():
        return H * S, S
    sb, sh, ss = x.stride()
    ok = S <= 1 or ss == 1
    if H > 1:
        ok = ok and sh >= S
    if B > 1:
        ok = ok and (sb >= (H - 1) * sh + S or (H > 1 and sh >= (B - 1) * sb + S and sb >= S))
    if not ok:
        raise RuntimeError(f"{what} must be contiguous along its last axis, its rows apart from one another")
    return sb, sh


def causal_mask(L: int, S: int, dtype: torch.dtype = torch.float32, device=None) -> torch.Tensor:
    """0 where key s <= l + (S - L), -inf elsewhere (reference attention.py:59-61)."""
    allowed = torch.ones((L, S), dtype=torch.bool, device=device).tril(diagonal=S - L)
    zero = torch.zeros((), dtype=dtype, device=device)
    ninf = torch.full((), float("-inf"), dtype=dtype, device=device)
    return torch.where(allowed, zero, ninf)


def scaled_dot_product_attention_grouped(query, key, value, scale=None, mask=None):
    """Dense grouped-query SDPA with plain torch ops (reference attention.py:64-100)."""
    expected_shape = query.shape
    Hq, L, D = query.shape[-3:]
    Hkv, S, _ = key.shape[-3:]
    batch = query.shape[:-3]
    assert Hq % Hkv == 0
    rep = Hq // Hkv
    q = query.reshape(*batch, 1, Hkv, rep, L, D)
    k = key.reshape(*batch, 1, Hkv, 1, S, D)
    v = value.reshape(*batch, 1, Hkv, 1, S, D)
    factor = scale if scale is not None else 1.0 / (D ** 0.5)
    scores = torch.matmul(q, k.transpose(-2, -1)) * factor
    if isinstance(mask, str):
        assert mask == "causal"
        scores = scores + causal_mask(L, S, scores.dtype, scores.device)
    elif mask is not None:
        m = torch.broadcast_to(mask, (*batch, Hq, L, S)).reshape(*batch, 1, Hkv, rep, L, S)
        scores = scores + m
    out = torch.matmul(torch.softmax(scores, dim=-1), v)
    return out.reshape(expected_shape)


def flash_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, scale: float | None = None,
                    mask: torch.Tensor | str | None = None, *, out_dtype: torch.dtype | None = None,
                    window: int | None = None, sinks: int = 0) -> torch.Tensor:
    """Dense flash attention (reference attention.py:103-151).

    query ``[..., Hq, L, E]``, key/value ``[B, Hkv, S, E]`` (fp32, fp16 or bf16, all
    the same dtype).  ``mask`` is None, "causal", or a float tensor broadcastable to
    ``[..., Hq, L, S]`` that is added to the scaled scores.  Returns ``[..., Hq, L, E]``
    in ``out_dtype`` (default: the query dtype, i.e. fp32 for the reference's fp32
    inputs).

    ``window``: the token at position ``pos = l + S - L`` sees key ``s`` only if ``s < sinks``
    or ``s > pos - window``; not together with a mask tensor.  A row that sees no key is zero.
    """
    _check_window("flash_attention", window, sinks)
    factor = scale if scale is not None else 1.0 / (query.shape[-1] ** 0.5)
    *batch_shape, Hq, L, D = query.shape
    _, Hkv, S, _ = key.shape
    assert Hq % Hkv == 0
    dev = nv.require_cuda("flash_attention", query, key, value)
    if not (query.dtype == key.dtype == value.dtype):
        raise RuntimeError("flash_attention: query, key and value must have the same dtype")
    N = query.numel() // (L * D) if query.numel() else 0
    B = N // Hq
    q = query.contiguous()
    k = key.contiguous()
    v = value.contiguous()
    is_causal = isinstance(mask, str) and mask == "causal"
    if isinstance(mask, str) and mask != "causal":
        raise NotImplementedError(f"flash_attention: unknown mask {mask!r}")
    if window is not None:
        if isinstance(mask, torch.Tensor):
            raise NotImplementedError("flash_attention: window goes with mask=None or causal only")
        if q.dim() < 3 or tuple(k.shape) != (B, Hkv, S, D) or v.shape != k.shape:
            raise RuntimeError("flash_attention: key and value must be [B, Hkv, S, E] with the query's B and E")
        out = torch.empty((*batch_shape, Hq, L, D), dtype=out_dtype or query.dtype, device=dev)
        with nv.on_device(dev):
            nv.check(nv.lib().nvm_flash_attention_window(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), nv.dtype_code(q.dtype), out.data_ptr(),
                nv.dtype_code(out.dtype), B, Hq, Hkv, L, S, D, float(factor), int(is_causal), window, sinks,
                nv.stream_ptr(dev)))
        return out
    m = None
    ms = (0, 0, 0)
    if isinstance(mask, torch.Tensor):
        mb = torch.broadcast_to(mask.to(device=dev, dtype=torch.float32), (*batch_shape, Hq, L, S))
        m = mb.reshape(N, L, S)
        ms = m.stride()
    od = out_dtype or query.dtype
    out = torch.empty((*batch_shape, Hq, L, D), dtype=od, device=dev)
    L_ = nv.lib()
    with torch.cuda.device(dev):
        nv.check(L_.nvm_flash_attention(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), nv.dtype_code(q.dtype), nv.ptr(m), ms[0], ms[1], ms[2],
            out.data_ptr(), nv.dtype_code(od), B, Hq, Hkv, L, S, D, float(factor), int(is_causal),
            nv.stream_ptr(dev)))
    return out


def _int32_rows(x: torch.Tensor) -> torch.Tensor:
    return x if x.dtype is torch.int32 and x.is_contiguous() else x.to(torch.int32).contiguous()


def _paged_attention_window(query, key_pages, value_pages, block_table, context_lens, page_size, key_scales, value_scales,
                            scale, mask, out_dtype, out, window, sinks, key_mass):
    """paged_attention with a window or key scores."""
    op = "paged_attention"
    _check_window(op, window, sinks)
    if isinstance(mask, torch.Tensor):
        raise NotImplementedError("Paged attention only supports mask=None or causal")
    if mask is not None and mask != "causal":
        raise NotImplementedError
    B, Hq, L, D = query.shape
    P, Hkv, ps, pd = key_pages.shape
    assert Hq % Hkv == 0
    dev = nv.require_cuda(op, query, key_pages, value_pages, block_table, context_lens, key_scales, value_scales, key_mass,
                          out)
    if key_pages.dtype != value_pages.dtype:
        raise RuntimeError(f"{op}: key_pages and value_pages must have the same dtype")
    if key_pages.shape != value_pages.shape:
        raise RuntimeError(f"{op}: key_pages and value_pages must have the same shape")
    if pd != D:
        raise RuntimeError(f"{op}: q and page tensors must have the same head dimension")
    if ps != page_size:
        raise RuntimeError(f"{op}: pages must be [P, Hkv, page_size, D]")
    if block_table.dim() != 2 or context_lens.dim() != 1:
        raise RuntimeError(f"{op}: block_table must be 2D and context_lens must be 1D")
    MP = block_table.shape[1]
    if block_table.shape[0] != B or context_lens.shape[0] != B:
        raise RuntimeError(f"{op}: q batch size must match block_table batch size")
    q, kp, vp = query.contiguous(), key_pages.contiguous(), value_pages.contiguous()
    bt, cl = _int32_rows(block_table), _int32_rows(context_lens)
    ks = vs = None
    sdt = nv.NVM_F16
    if kp.dtype is torch.int8:
        assert key_scales is not None
        assert value_scales is not None
        ks, vs = key_scales.contiguous(), value_scales.contiguous()
        if tuple(ks.shape) != (P, Hkv, ps, 1) or vs.shape != ks.shape:
            raise RuntimeError(f"{op}: scales must be [P, Hkv, page_size, 1]")
        if ks.dtype != vs.dtype:
            vs = vs.to(ks.dtype)
        sdt = nv.dtype_code(ks.dtype)
    mp, msb, msh, ml = None, 0, 0, 0
    if key_mass is not None:
        if key_mass.dim() != 3 or key_mass.shape[0] != B or key_mass.shape[1] != Hkv or key_mass.dtype is not torch.float32:
            raise RuntimeError(f"{op}: key_mass must be float32 [B, Hkv, S]")
        msb, msh = _row_strides(f"{op}: key_mass", key_mass)
        mp, ml = key_mass.data_ptr(), key_mass.shape[2]
    if out is None:
        out = torch.empty_like(q) if out_dtype is q.dtype else q.new_empty((B, Hq, L, D), dtype=out_dtype)
    elif tuple(out.shape) != (B, Hq, L, D) or not out.is_contiguous():
        raise RuntimeError(f"{op}: out must be a contiguous [B, Hq, L, D] tensor")
    factor = scale if scale is not None else 1.0 / (D ** 0.5)
    lib = nv.lib()
    kvc = nv.dtype_code(kp.dtype)
    with nv.on_device(dev):
        nv.call_with_workspace(
            dev,
            lambda: lib.nvm_paged_attention_window_workspace_size(B, Hq, Hkv, L, D, ps, MP, kvc, window or 0, sinks,
                                                                  int(mp is not None)),
            lambda ws, ws_bytes, stream: lib.nvm_paged_attention_window(
                q.data_ptr(), nv.dtype_code(q.dtype), kp.data_ptr(), vp.data_ptr(), kvc, nv.ptr(ks), nv.ptr(vs), sdt,
                bt.data_ptr(), cl.data_ptr(), out.data_ptr(), nv.dtype_code(out.dtype), B, Hq, Hkv, L, D, P, ps, MP,
                factor, mask == "causal", window or 0, sinks, mp, msb, msh, ml, ws, ws_bytes, stream))
    return out


def paged_attention(query: torch.Tensor, key_pages: torch.Tensor, value_pages: torch.Tensor,
                    block_table: torch.Tensor, context_lens: torch.Tensor, page_size: int,
                    key_scales: torch.Tensor | None = None, value_scales: torch.Tensor | None = None,
                    scale: float | None = None, mask: torch.Tensor | str | None = None, *,
                    out_dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None,
                    window: int | None = None, sinks: int = 0,
                    key_mass: torch.Tensor | None = None) -> torch.Tensor:
    """Paged attention over block-paged K/V pools (reference attention.py:154-230).

    query ``[B, Hq, L, D]``; key_pages/value_pages ``[P, Hkv, page_size, D]`` (fp32,
    fp16, bf16, or int8 with ``key_scales``/``value_scales`` ``[P, Hkv, page_size, 1]``);
    block_table ``[B, max_pages]`` (-1 padded); context_lens ``[B]`` (tokens of each
    sequence, the new L included).  Returns ``[B, Hq, L, D]`` (fp32 by default).

    ``window``: the query token at position ``pos = l + context_len - L`` sees key ``s`` only if
    ``s < sinks`` or ``s > pos - window``; pages wholly between are not read.  ``key_mass``
    (float32 ``[B, Hkv, S]``, last axis contiguous) is updated in place: every key gains the
    softmax weights it gets from the rows of its kv head, and the newest L keys start at zero,
    so the buffer needs no clearing between requests whose tokens scored calls append (zero the
    entries of others, as ``DevicePageTable.attach`` does for an attached prefix); keys at or past
    S gain nothing.  A row that sees no key is zero, and a key that no row sees has no influence
    whatever it holds.
    """
    if window is not None or key_mass is not None or sinks != 0:
        return _paged_attention_window(query, key_pages, value_pages, block_table, context_lens, page_size, key_scales,
                                       value_scales, scale, mask, out_dtype, out, window, sinks, key_mass)
    if isinstance(mask, torch.Tensor):
        raise NotImplementedError("Paged attention only supports mask=None or causal")
    if mask is not None and mask != "causal":
        raise NotImplementedError
    factor = scale if scale is not None else 1.0 / (query.shape[-1] ** 0.5)
    B, Hq, L, D = query.shape
    P, Hkv, ps, _ = key_pages.shape
    assert Hq % Hkv == 0
    dev = nv.require_cuda("paged_attention", query, key_pages, value_pages, block_table, context_lens,
                          key_scales, value_scales)
    if key_pages.dtype != value_pages.dtype:
        raise RuntimeError("paged_attention: key_pages and value_pages must have the same dtype")
    if key_pages.shape != value_pages.shape:
        raise RuntimeError("paged_attention: key_pages and value_pages must have the same shape")
    if key_pages.shape[3] != D:
        raise RuntimeError("paged_attention: q and page tensors must have the same head dimension")
    q = query.contiguous()
    kp = key_pages.contiguous()
    vp = value_pages.contiguous()
    bt = block_table.to(torch.int32).contiguous()
    cl = context_lens.to(torch.int32).contiguous()
    if bt.dim() != 2 or cl.dim() != 1:
        raise RuntimeError("paged_attention: block_table must be 2D and context_lens must be 1D")
    if bt.shape[0] != cl.shape[0] or bt.shape[0] != B:
        raise RuntimeError("paged_attention: q batch size must match block_table batch size")
    ks = vs = None
    sdt = nv.NVM_F16
    if kp.dtype == torch.int8:
        assert key_scales is not None
        assert value_scales is not None
        ks = key_scales.contiguous()
        vs = value_scales.contiguous()
        if ks.dtype != vs.dtype:
            vs = vs.to(ks.dtype)
        sdt = nv.dtype_code(ks.dtype)
    if out is None:
        out = torch.empty((B, Hq, L, D), dtype=out_dtype, device=dev)
    L_ = nv.lib()
    kvc = nv.dtype_code(kp.dtype)
    with nv.on_device(dev):
        nv.call_with_workspace(
            dev, lambda: L_.nvm_paged_attention_workspace_size(B, Hq, Hkv, L, D, ps, bt.shape[1], kvc),
            lambda ws, ws_bytes, stream: L_.nvm_paged_attention(
                q.data_ptr(), nv.dtype_code(q.dtype), kp.data_ptr(), vp.data_ptr(), kvc, nv.ptr(ks), nv.ptr(vs), sdt,
                bt.data_ptr(), cl.data_ptr(), out.data_ptr(), nv.dtype_code(out.dtype), B, Hq, Hkv, L, D, P, ps,
                bt.shape[1], float(factor), int(mask == "causal"), ws, ws_bytes, stream))
    return out

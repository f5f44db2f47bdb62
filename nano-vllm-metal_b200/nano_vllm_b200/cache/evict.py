"""Eviction of cached tokens by accumulated attention weight.

``paged_attention(..., key_mass=mass)`` adds to ``mass[b, h, s]`` the softmax weight that key
``s`` gets in every step.  ``evict_tokens`` trims each request that has grown past a budget to
the tokens that matter: its first ``sinks``, its last ``recent`` and, of the rest, the heaviest,
chosen separately for every kv head.  Their K/V rows move in order to the front of the request's
own pages, so attention, append and rewind go on as if the request had always been that short
(keys carry their rotary positions already; ``positions`` of new tokens stay the caller's).  The
reference has no counterpart.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _native as nv
from ..layers.attention import _int32_rows, _row_strides

__all__ = ["EvictResult", "evict_tokens"]

_PAGE_DTYPES = (torch.float32, torch.float16, torch.bfloat16, torch.int8)


class EvictResult(NamedTuple):
    keep_index: torch.Tensor  # [B, Hkv, budget] int32: old position of each kept token, -1 behind them
    kept: torch.Tensor        # [B] int32 tokens kept
    dropped: torch.Tensor     # [B] int32 tokens given up: what to rewind the request by
    refused: torch.Tensor     # [B] int32, not zero for a request that could not be trimmed


def evict_tokens(key_pages: torch.Tensor, value_pages: torch.Tensor, block_table: torch.Tensor,
                 context_lens: torch.Tensor, key_mass: torch.Tensor, budget: int, *, sinks: int = 0, recent: int = 0,
                 key_scales: torch.Tensor | None = None, value_scales: torch.Tensor | None = None,
                 page_refcount: torch.Tensor | None = None, mass_out: torch.Tensor | None = None,
                 status: torch.Tensor | None = None) -> EvictResult:
    """Trim every request of more than ``budget`` tokens to ``budget``, in place.

    key_pages/value_pages ``[P, Hkv, page_size, D]`` (fp32, fp16, bf16, or int8 with
    ``key_scales``/``value_scales`` ``[P, Hkv, page_size, 1]``), contiguous; block_table
    ``[B, max_pages]`` and context_lens ``[B]`` int32; key_mass float32 ``[B, Hkv, S]``, last
    axis contiguous.  Ties go to the lowest position, NaN ranks below every number.  The kept
    tokens' weights move along (into ``mass_out`` when given, which must not overlap key_mass,
    else in place) and are zero from there to the old length.

    ``context_lens`` is left alone: rewind each request by ``dropped``
    (``DevicePageTable.evict`` does both).  The pages from position ``sinks`` on must belong to
    the request alone; ``page_refcount`` ([P] int32 or longer) makes the kernel check it.  A
    request with a shared or unmapped page there, or longer than S or its row, is left as it
    is, with ``dropped`` 0 and ``refused`` not zero; ``status`` (one int32, optional) is then set
    too and is never cleared.
    """
    return plan_evict(key_pages, value_pages, block_table, context_lens, key_mass, budget, sinks, recent, key_scales,
                      value_scales, page_refcount, mass_out, status).launch()


class EvictPlan:
    """One checked call of ``evict_tokens``: nothing can refuse it any more.  ``args`` are those of
    nvm_paged_evict up to the stream, ``written`` the page pools and scales that it rewrites, ``mass``
    the weights that it selects by; ``held`` keeps converted inputs alive until the launch."""

    __slots__ = ("device", "args", "result", "written", "mass", "held")

    def __init__(self, device, args, result, written, mass, held):
        self.device, self.args, self.result, self.written, self.mass, self.held = device, args, result, written, mass, held

    def launch(self) -> EvictResult:
        with nv.on_device(self.device):
            nv.check(nv.lib().nvm_paged_evict(*self.args, nv.stream_ptr(self.device)))
        return self.result


def overlap(tensors) -> bool:
    """Do any two of these contiguous tensors share memory."""
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in tensors if t.numel())
    return any(a[1] > b[0] for a, b in zip(spans, spans[1:]))


def plan_evict(key_pages, value_pages, block_table, context_lens, key_mass, budget, sinks=0, recent=0, key_scales=None,
               value_scales=None, page_refcount=None, mass_out=None, status=None) -> EvictPlan:
    """Every check and allocation of ``evict_tokens``, and no launch."""
    op = "evict"
    out = key_mass if mass_out is None else mass_out
    dev = nv.require_cuda(op, key_pages, value_pages, block_table, context_lens, key_mass, key_scales, value_scales,
                          page_refcount, mass_out, status)
    dtype = key_pages.dtype
    if key_pages.dim() != 4 or key_pages.shape != value_pages.shape or dtype is not value_pages.dtype:
        raise RuntimeError(f"{op}: key_pages and value_pages must be [P, Hkv, page_size, D] of one dtype")
    if not (key_pages.is_contiguous() and value_pages.is_contiguous()):
        raise RuntimeError(f"{op}: page pools must be contiguous (written in place)")
    P, Hkv, ps, D = key_pages.shape
    if block_table.dim() != 2 or context_lens.dim() != 1 or block_table.shape[0] != context_lens.shape[0]:
        raise RuntimeError(f"{op}: block_table must be [B, max_pages] and context_lens [B]")
    B, MP = block_table.shape
    if budget < 1 or sinks < 0 or recent < 0 or sinks + recent > budget:
        raise RuntimeError(f"{op}: need budget >= 1, sinks >= 0, recent >= 0 and sinks + recent <= budget")
    if key_mass.dim() != 3 or key_mass.shape[0] != B or key_mass.shape[1] != Hkv or key_mass.dtype is not torch.float32:
        raise RuntimeError(f"{op}: key_mass must be float32 [B, Hkv, S]")
    msb, msh = _row_strides(f"{op}: key_mass", key_mass)
    osb, osh = msb, msh
    if mass_out is not None:
        if mass_out.shape != key_mass.shape or mass_out.dtype is not torch.float32:
            raise RuntimeError(f"{op}: mass_out must be float32 with the shape of key_mass")
        osb, osh = _row_strides(f"{op}: mass_out", mass_out)
        S = key_mass.shape[2]
        if 0 < abs(mass_out.data_ptr() - key_mass.data_ptr()) < 4 * B * Hkv * S and msb == osb == Hkv * S and msh == osh == S:
            raise RuntimeError(f"{op}: mass_out must be key_mass itself or share no memory with it")
    sdt = nv.NVM_F16
    if dtype not in _PAGE_DTYPES:
        raise RuntimeError(f"{op}: pages must be float32, float16, bfloat16 or int8")
    if D > 256:
        raise RuntimeError(f"{op}: head dimension must be <= 256 (got {D})")
    if dtype is torch.int8:
        if key_scales is None or value_scales is None:
            raise RuntimeError(f"{op}: int8 pages need key_scales and value_scales")
        for s in (key_scales, value_scales):
            if tuple(s.shape) != (P, Hkv, ps, 1) or not s.is_contiguous() or s.dtype != key_scales.dtype:
                raise RuntimeError(f"{op}: scales must be contiguous [P, Hkv, page_size, 1] of one dtype")
        if key_scales.dtype not in _PAGE_DTYPES[:3]:
            raise RuntimeError(f"{op}: int8 pages need floating-point key and value scales")
        sdt = nv.dtype_code(key_scales.dtype)
    else:
        key_scales = value_scales = None
    if page_refcount is not None and (page_refcount.dtype != torch.int32 or page_refcount.numel() < P or
                                      not page_refcount.is_contiguous()):
        raise RuntimeError(f"{op}: page_refcount must be contiguous int32 with an entry per page")
    if status is not None and (status.dtype != torch.int32 or status.numel() != 1):
        raise RuntimeError(f"{op}: status must be one int32")
    bt, cl = _int32_rows(block_table), _int32_rows(context_lens)
    keep = bt.new_empty((B, Hkv, budget))
    kept, dropped, refused = bt.new_empty((3, B)).unbind(0)
    kp, vp = key_pages.data_ptr(), value_pages.data_ptr()
    written = (key_pages, value_pages) if key_scales is None else (key_pages, value_pages, key_scales, value_scales)
    if abs(kp - vp) < P * Hkv * ps * D * dtype.itemsize or (key_scales is not None and overlap(written)):
        raise RuntimeError(f"{op}: page pools and scales must not share memory with one another")
    args = (kp, vp, nv.dtype_code(dtype), nv.ptr(key_scales), nv.ptr(value_scales), sdt, bt.data_ptr(),
            cl.data_ptr(), nv.ptr(page_refcount), key_mass.data_ptr(), msb, msh, key_mass.shape[2], out.data_ptr(), osb, osh,
            B, Hkv, D, P, ps, MP, budget, sinks, recent, keep.data_ptr(), kept.data_ptr(), dropped.data_ptr(),
            refused.data_ptr(), nv.ptr(status))
    return EvictPlan(dev, args, EvictResult(keep, kept, dropped, refused), written, key_mass, (bt, cl))

"""Passes of more than one token over cached sequences (csrc/seq_attn.cu,
csrc/seq_cache.cu): whole prompts of different lengths packed into one pass,
and trees of drafted tokens. They stand beside the single-token kernels of
tp_ops and are what TPDecoder.forward_packed, forward_tree and
generate_speculative_tree run between their projections.

A cache is [B, nkv, max_len, hd], one sequence per batch entry. Packed rows
are described by `cu`, int64 [B + 1]: sequence b has the rows cu[b] ..
cu[b + 1] - 1. All tensors are BF16 CUDA tensors on one device except
lengths, positions and indices (int64, on the device so that a captured pass
reads the current values), `inv_freq` (fp32) and masks (bool). Values on the
device that point outside a tensor are cut off or skipped, never followed.
Work runs on the current stream of the tensors' device; nothing synchronises.
"""
from __future__ import annotations

import contextlib
import ctypes

import torch

from .. import _lib
from . import _device

_BF16 = torch.bfloat16
_I64 = torch.int64
MAX_HEAD_SIZE = 256
MAX_KEEP = 256


def _on(dev: torch.device):
    """The C entry points launch on the current device."""
    return contextlib.nullcontext() if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _need(ok: bool, text: str) -> None:
    if not ok:
        raise ValueError(text)


def _check_device(who: str, first: torch.Tensor, *others) -> None:
    for t in (first, *others):
        if t is not None and t.device != first.device:
            raise ValueError(f"{who}: tensors on {first.device} and {t.device}")


def _check_cuda(who: str, dev: torch.device) -> None:
    if dev.type != "cuda":
        raise ValueError(f"{who} runs on CUDA tensors (got {dev}); there is no CPU fallback")


def _check_bf16(who: str, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and (t.dtype != _BF16 or (t.numel() and t.stride(-1) != 1 and t.shape[-1] > 1)):
            raise ValueError(f"{who}: {name} must be bf16 with unit stride along the head size")


def _check_index(who: str, shape: tuple, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and (t.dtype != _I64 or tuple(t.shape) != shape or not t.is_contiguous()):
            raise ValueError(f"{who}: {name} must be a contiguous int64 tensor of shape {shape}")


def _no_grad(who: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{who} has no backward pass: run it under torch.no_grad()")


def _check_out(who: str, out: torch.Tensor, q: torch.Tensor) -> None:
    _need(out.shape == q.shape, f"{who}: out must have q's shape")
    for size, stride in zip(out.shape, out.stride()):
        _need(size < 2 or stride != 0, f"{who}: out must not be an expanded tensor")


def _attend(entry: str, who: str, d: _lib.AttnDesc, dev: torch.device) -> None:
    _check_cuda(who, dev)
    L = _lib.load()
    with _on(dev):
        need = L.aib_attention_workspace_floats(d)
        if need:
            ws = torch.empty(need, dtype=torch.float32, device=dev)
            d.workspace, d.workspace_floats = ws.data_ptr(), need
        _lib.check(getattr(L, entry)(d, _device.status_word(dev).data_ptr(), _device.stream_ptr(dev)), who)


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, scale: float, *,
                     cu_k: torch.Tensor | None = None, len_k: torch.Tensor | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of packed prompts: q [N, nh, hd], cu_q [B + 1].

    Keys are packed too (k, v [Nk, nkv, hd], cu_k [B + 1], default cu_q), or
    lie in caches (k, v [B, nkv, max_len, hd], len_k [B] keys each, the
    prompt's own among them). A sequence's queries are the last of its keys:
    row i of m sees the keys j <= L - m + i. Rows that see nothing are zero;
    rows of q in no sequence are not computed and their rows of `out` not
    written. Returns out [N, nh, hd] (new unless given)."""
    who = "prompt_attention"
    _check_device(who, q, k, v, cu_q, cu_k, len_k, out)
    _check_bf16(who, q=q, k=k, v=v, out=out)
    _no_grad(who, q, k, v)
    _need(q.dim() == 3, f"{who}: q must be [tokens, heads, head size]")
    n, nh, hd = q.shape
    _need(cu_q.dim() == 1 and cu_q.shape[0] >= 1, f"{who}: cu_q must be int64 [sequences + 1]")
    b = cu_q.shape[0] - 1
    _check_index(who, (b + 1,), cu_q=cu_q, cu_k=cu_k)
    _check_index(who, (b,), len_k=len_k)
    _need(v.shape == k.shape and k.shape[-1] == hd, f"{who}: k and v must have one shape and q's head size")
    d = _lib.AttnDesc()
    if k.dim() == 4:
        _need(len_k is not None and cu_k is None, f"{who}: caches [B, nkv, max_len, hd] need len_k, and no cu_k")
        _need(k.shape[0] == b, f"{who}: {k.shape[0]} caches for {b} sequences")
        nkv, rows = k.shape[1], k.shape[2]
        d.k_batch_stride, d.k_head_stride, d.k_token_stride = k.stride()[:3]
        d.v_batch_stride, d.v_head_stride, d.v_token_stride = v.stride()[:3]
        d.len_k = len_k.data_ptr()
    else:
        _need(k.dim() == 3 and len_k is None, f"{who}: packed k and v are [tokens, kv heads, head size], without len_k")
        _need(cu_k is not None or k.shape[0] == n, f"{who}: k and v need cu_k unless they have q's rows")
        rows, nkv = k.shape[0], k.shape[1]
        d.k_token_stride, d.k_head_stride = k.stride()[:2]
        d.v_token_stride, d.v_head_stride = v.stride()[:2]
        d.cu_k = (cu_q if cu_k is None else cu_k).data_ptr()
    _need(nkv > 0 and nh > 0 and nh % nkv == 0, f"{who}: {nh} heads do not divide into {nkv} kv heads")
    _need(1 <= hd <= MAX_HEAD_SIZE, f"{who}: head size {hd} outside 1..{MAX_HEAD_SIZE}")
    if out is None:
        out = torch.empty(n, nh, hd, dtype=_BF16, device=q.device)
    _check_out(who, out, q)
    d.q, d.k, d.v, d.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    d.q_token_stride, d.q_head_stride = q.stride()[:2]
    d.out_token_stride, d.out_head_stride = out.stride()[:2]
    d.tokens, d.batch, d.key_rows = n, b, rows
    d.nh, d.nkv, d.hd, d.scale = nh, nkv, hd, scale
    d.cu_q = cu_q.data_ptr()
    _attend("aib_prompt_attention_bf16", who, d, q.device)
    return out


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, pos: torch.Tensor,
                   mask: torch.Tensor, scale: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of T drafted tokens per sequence over its cache: q
    [B, T, nh, hd], caches [B, nkv, max_len, hd], pos int64 [B].

    Every query of sequence b sees the slots before pos[b]; the C drafted
    tokens are at the slots pos[b] .. pos[b] + C - 1, and query i sees those
    with mask[i, j] (mask bool [T, C] for all sequences or [B, T, C]; see
    tree_mask). T = C = 1 is the single-token step of a batch. A query that
    sees nothing gives zeros. Returns [B, T, nh, hd] (new unless given)."""
    who = "tree_attention"
    _check_device(who, q, k_cache, v_cache, pos, mask, out)
    _check_bf16(who, q=q, k_cache=k_cache, v_cache=v_cache, out=out)
    _no_grad(who, q, k_cache, v_cache)
    _need(q.dim() == 4, f"{who}: q must be [sequences, tokens, heads, head size]")
    b, t, nh, hd = q.shape
    _need(k_cache.dim() == 4 and v_cache.shape == k_cache.shape and k_cache.shape[0] == b and k_cache.shape[3] == hd,
          f"{who}: caches must be [{b}, kv heads, max_len, {hd}]")
    nkv, rows = k_cache.shape[1], k_cache.shape[2]
    _need(nkv > 0 and nh > 0 and nh % nkv == 0, f"{who}: {nh} heads do not divide into {nkv} kv heads")
    _need(1 <= hd <= MAX_HEAD_SIZE, f"{who}: head size {hd} outside 1..{MAX_HEAD_SIZE}")
    _check_index(who, (b,), pos=pos)
    _need(mask.dtype == torch.bool and mask.dim() in (2, 3) and mask.shape[-2] == t
          and (mask.dim() == 2 or mask.shape[0] == b), f"{who}: mask must be bool [{t}, C] or [{b}, {t}, C]")
    cols = mask.shape[-1]
    _need(cols <= rows, f"{who}: {cols} drafted tokens for caches of {rows} rows")
    if out is None:
        out = torch.empty(b, t, nh, hd, dtype=_BF16, device=q.device)
    _check_out(who, out, q)
    d = _lib.AttnDesc()
    d.q, d.k, d.v, d.out = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr()
    d.q_batch_stride, d.q_token_stride, d.q_head_stride = q.stride()[:3]
    d.k_batch_stride, d.k_head_stride, d.k_token_stride = k_cache.stride()[:3]
    d.v_batch_stride, d.v_head_stride, d.v_token_stride = v_cache.stride()[:3]
    d.out_batch_stride, d.out_token_stride, d.out_head_stride = out.stride()[:3]
    d.tokens, d.batch, d.key_rows = t, b, rows
    d.nh, d.nkv, d.hd, d.scale = nh, nkv, hd, scale
    # a mask without columns still says "tree" to the C entry: any address serves, none is read
    d.pos, d.mask = pos.data_ptr(), mask.data_ptr() or pos.data_ptr()
    d.mask_batch_stride = mask.stride(0) if mask.dim() == 3 else 0
    d.mask_row_stride, d.mask_col_stride = mask.stride()[-2:]
    d.mask_cols = cols
    _attend("aib_tree_attention_bf16", who, d, q.device)
    return out


def rope_cache_packed(qkv: torch.Tensor, nh: int, nkv: int, hd: int, cu: torch.Tensor, start: torch.Tensor,
                      inv_freq: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, *,
                      depth: torch.Tensor | None = None, q_norm: torch.Tensor | None = None,
                      k_norm: torch.Tensor | None = None, eps: float = 1e-6,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """qkv [N, (nh + 2 nkv) * hd] -> q [N, nh, hd] (returned; new unless
    given), k and v written into the caches [B, nkv, max_len, hd].

    Row cu[b] + i is token i of sequence b; its keys and values go to row
    start[b] + i of the sequence's caches, and its rotary place is
    start[b] + depth[row] (int64 [N]: a drafted node's depth) or, without
    depth, start[b] + i. q and k take RMSNorm over the head first where both
    norm weights are given. Rows outside [0, max_len) are not written, nor
    the q rows of rows in no sequence. fp32 inside, one rounding at the end
    (tp_ops.qk_rope_cache rounds where transformers does)."""
    who = "rope_cache_packed"
    _check_device(who, qkv, cu, start, inv_freq, k_cache, v_cache, depth, q_norm, k_norm, out)
    _check_bf16(who, qkv=qkv, k_cache=k_cache, v_cache=v_cache, q_norm=q_norm, k_norm=k_norm, out=out)
    _no_grad(who, qkv, q_norm, k_norm)
    _need(nh > 0 and nkv > 0 and hd >= 2 and hd % 2 == 0 and hd <= 1024, f"{who}: bad heads or head size")
    _need(qkv.dim() == 2 and qkv.shape[1] == (nh + 2 * nkv) * hd, f"{who}: qkv must be [N, {(nh + 2 * nkv) * hd}]")
    n = qkv.shape[0]
    _need(cu.dim() == 1 and cu.shape[0] >= 1, f"{who}: cu must be int64 [sequences + 1]")
    b = cu.shape[0] - 1
    _check_index(who, (b + 1,), cu=cu)
    _check_index(who, (b,), start=start)
    _check_index(who, (n,), depth=depth)
    _need(k_cache.dim() == 4 and v_cache.shape == k_cache.shape and tuple(k_cache.shape[:2]) == (b, nkv)
          and k_cache.shape[3] == hd and k_cache.shape[2] > 0, f"{who}: caches must be [{b}, {nkv}, max_len, {hd}]")
    _need(inv_freq.dtype == torch.float32 and tuple(inv_freq.shape) == (hd // 2,) and inv_freq.is_contiguous(),
          f"{who}: inv_freq must be fp32 [{hd // 2}]")
    _need(k_cache.data_ptr() != v_cache.data_ptr() or k_cache.numel() == 0, f"{who}: k_cache and v_cache are the same")
    _need((q_norm is None) == (k_norm is None), f"{who}: give both q and k norm weights or neither")
    _need(q_norm is None or (tuple(q_norm.shape) == (hd,) and tuple(k_norm.shape) == (hd,)),
          f"{who}: norm weights must be [{hd}]")
    for c in (k_cache, v_cache):
        _need(all(size < 2 or stride != 0 for size, stride in zip(c.shape, c.stride())),
              f"{who}: caches must not be expanded tensors")
    if out is None:
        out = torch.empty(n, nh, hd, dtype=_BF16, device=qkv.device)
    _need(tuple(out.shape) == (n, nh, hd) and out.is_contiguous(), f"{who}: out must be contiguous [N, {nh}, {hd}]")
    _check_cuda(who, qkv.device)
    L = _lib.load()
    with _on(qkv.device):
        _lib.check(L.aib_rope_cache_packed_bf16(
            qkv.data_ptr(), qkv.stride(0), n, b, nh, nkv, hd, cu.data_ptr(), start.data_ptr(),
            None if depth is None else depth.data_ptr(), None if q_norm is None else q_norm.data_ptr(),
            None if k_norm is None else k_norm.data_ptr(), eps, inv_freq.data_ptr(), out.data_ptr(),
            k_cache.data_ptr(), v_cache.data_ptr(), (ctypes.c_int64 * 3)(*k_cache.stride()[:3]),
            (ctypes.c_int64 * 3)(*v_cache.stride()[:3]), k_cache.shape[2], _device.stream_ptr(qkv.device)), who)
    return out


def keep_cache_rows(caches: list, pos: torch.Tensor, keep: torch.Tensor) -> None:
    """The rows that stay after a draft was accepted, moved together, in
    every cache of `caches` (tensors [B, nkv, max_len, hd] of one shape and
    one set of strides: the keys and the values of all layers) at once: row
    pos[b] + i <- row pos[b] + keep[b, i] as it was before the call, for the
    n <= 256 columns of keep (int64 [B, n]). keep < 0, and rows outside the
    cache, leave the row as it is."""
    who = "keep_cache_rows"
    if not caches:
        return
    first = caches[0]
    _check_device(who, first, pos, keep)
    _need(first.dim() == 4, f"{who}: caches must be [B, kv heads, max_len, head size]")
    b, nkv, max_len, hd = first.shape
    shape, strides, dev = first.shape, first.stride(), first.device
    for t in caches:
        _need(t.dtype == _BF16 and t.shape == shape and t.stride() == strides and t.device == dev,
              f"{who}: caches must be bf16 tensors of one shape, one set of strides and one device")
    _need(strides[3] == 1 or hd == 1, f"{who}: caches need unit stride along the head size")
    _need(all(size < 2 or stride != 0 for size, stride in zip(shape, strides)),
          f"{who}: caches must not be expanded tensors")
    ptrs = [t.data_ptr() for t in caches]
    _need(len(set(ptrs)) == len(ptrs), f"{who}: a cache is given twice")
    _need(keep.dim() == 2, f"{who}: keep must be int64 [B, n]")
    n = keep.shape[1]
    _need(n <= MAX_KEEP, f"{who}: {n} rows, at most {MAX_KEEP}")
    _check_index(who, (b,), pos=pos)
    _check_index(who, (b, n), keep=keep)
    _check_cuda(who, dev)
    if first.numel() == 0:
        return
    L = _lib.load()
    with _on(dev):
        _lib.check(L.aib_keep_cache_rows_bf16((ctypes.c_void_p * len(ptrs))(*ptrs), len(ptrs), b, nkv, max_len, hd,
                                              (ctypes.c_int64 * 3)(*strides[:3]), pos.data_ptr(), keep.data_ptr(), n,
                                              _device.stream_ptr(dev)), who)


def tree_mask(parents, device=None) -> tuple[torch.Tensor, torch.Tensor]:
    """(mask, depth) of a drafted tree: parents[i] < i is node i's parent, or
    -1 for a node that continues the committed tokens. mask bool [T, T]: a
    node sees itself and its ancestors; depth int64 [T]: its distance from
    the committed tokens, 0 for parent -1."""
    parents = [int(x) for x in parents]
    n = len(parents)
    mask = torch.zeros(n, n, dtype=torch.bool)
    depth = torch.zeros(n, dtype=_I64)
    for i, p in enumerate(parents):
        if not -1 <= p < i:
            raise ValueError(f"tree_mask: node {i} has parent {p}; parents come before their children")
        if p >= 0:
            mask[i] = mask[p]
            depth[i] = depth[p] + 1
        mask[i, i] = True
    return mask.to(device), depth.to(device)


__all__ = ["prompt_attention", "tree_attention", "rope_cache_packed", "keep_cache_rows", "tree_mask"]

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

import array
import ctypes
import struct

import torch

from .. import _lib
from . import _device

_BF16 = torch.bfloat16
_I64 = torch.int64
_F32 = torch.float32
MAX_HEAD_SIZE = 256
MAX_KEEP = 256

# aib_attn_desc, packed in one go: a step makes two calls a layer, and setting 37 ctypes fields one by one takes
# longer than the kernel of a short tree
_DESC = struct.Struct("@4P15q3if5P5q")
assert _DESC.size == ctypes.sizeof(_lib.AttnDesc)

# (absent from a torch without CUDA, which has no tensors that get as far)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _need(ok: bool, text: str) -> None:
    if not ok:
        raise ValueError(text)


def _check_device(who: str, first: torch.Tensor, *others) -> None:
    for t in (first, *others):
        if t is not None and t.device != first.device:
            raise ValueError(f"{who}: tensors on {first.device} and {t.device}")


def _check_cuda(who: str, first: torch.Tensor) -> None:
    if not first.is_cuda:
        raise ValueError(f"{who} runs on CUDA tensors (got {first.device}); there is no CPU fallback")


def _check_bf16(who: str, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and (t.dtype != _BF16 or (t.numel() and t.stride(-1) != 1 and t.shape[-1] > 1)):
            raise ValueError(f"{who}: {name} must be bf16 with unit stride along the head size")


def _check_index(who: str, shape: tuple, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and (t.dtype != _I64 or tuple(t.shape) != shape or not t.is_contiguous()):
            raise ValueError(f"{who}: {name} must be a contiguous int64 tensor of shape {shape}")


def _check_no_grad(who: str, *tensors) -> None:
    if any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{who} has no backward pass: run it under torch.no_grad()")


def _check_out(who: str, out: torch.Tensor, q: torch.Tensor) -> None:
    _need(out.shape == q.shape, f"{who}: out must have q's shape")
    _check_not_expanded(who, "out", out)


def _check_not_expanded(who: str, name: str, t: torch.Tensor) -> None:
    for size, stride in zip(t.shape, t.stride()):
        _need(size < 2 or stride != 0, f"{who}: {name} must not be an expanded tensor")


def _check_heads(who: str, nh: int, nkv: int, hd: int) -> None:
    _need(nkv > 0 and nh > 0 and nh % nkv == 0, f"{who}: {nh} heads do not divide into {nkv} kv heads")
    _need(1 <= hd <= MAX_HEAD_SIZE, f"{who}: head size {hd} outside 1..{MAX_HEAD_SIZE}")


def _call(entry: str, who: str, q: torch.Tensor, desc: bytes) -> None:
    """The C entry points launch on the current device."""
    dev = q.get_device()
    if torch._C._cuda_getDevice() != dev:
        with torch.cuda.device(dev):
            return _call(entry, who, q, desc)
    L = _lib.load()
    floats = L.aib_attention_workspace_floats(desc)
    ws = torch.empty(floats, dtype=_F32, device=q.device) if floats else None
    rc = getattr(L, entry)(desc, ws.data_ptr() if floats else None, floats,
                           _device.status_word(q.device).data_ptr(), _raw_stream(dev))
    if rc:
        _lib.check(rc, who)


# Each operator looks its arguments over in one expression (`usual`) that only the common, valid calls pass; the
# others go through its _check function, which says what is wrong, or nothing where a call is unusual and valid.


def _no_grad(*tensors) -> bool:
    return not torch.is_grad_enabled() or not any(t is not None and t.requires_grad for t in tensors)


def _check_prompt(q, k, v, cu_q, cu_k, len_k, out) -> None:
    who = "prompt_attention"
    _check_device(who, q, k, v, cu_q, cu_k, len_k, out)
    _check_bf16(who, q=q, k=k, v=v, out=out)
    if torch.is_grad_enabled():
        _check_no_grad(who, q, k, v, out)
    _need(q.dim() == 3, f"{who}: q must be [tokens, heads, head size]")
    n, nh, hd = q.shape
    _need(cu_q.dim() == 1 and cu_q.shape[0] >= 1, f"{who}: cu_q must be int64 [sequences + 1]")
    b = cu_q.shape[0] - 1
    _check_index(who, (b + 1,), cu_q=cu_q, cu_k=cu_k)
    _check_index(who, (b,), len_k=len_k)
    _need(v.shape == k.shape and k.shape[-1] == hd, f"{who}: k and v must have one shape and q's head size")
    if k.dim() == 4:
        _need(len_k is not None and cu_k is None, f"{who}: caches [B, nkv, max_len, hd] need len_k, and no cu_k")
        _need(k.shape[0] == b, f"{who}: {k.shape[0]} caches for {b} sequences")
    else:
        _need(k.dim() == 3 and len_k is None, f"{who}: packed k and v are [tokens, kv heads, head size], without len_k")
        _need(cu_k is not None or k.shape[0] == n, f"{who}: k and v need cu_k unless they have q's rows")
    _check_heads(who, nh, k.shape[1], hd)
    if out is not None:
        _check_out(who, out, q)


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, scale: float, *,
                     cu_k: torch.Tensor | None = None, len_k: torch.Tensor | None = None,
                     out: torch.Tensor | None = None, sms: int = 0) -> torch.Tensor:
    """Causal attention of packed prompts: q [N, nh, hd], cu_q [B + 1].

    Keys are packed too (k, v [Nk, nkv, hd], cu_k [B + 1], default cu_q), or
    lie in caches (k, v [B, nkv, max_len, hd], len_k [B] keys each, the
    prompt's own among them). A sequence's queries are the last of its keys:
    row i of m sees the keys j <= L - m + i. Rows that see nothing are zero;
    rows of q in no sequence are not computed and their rows of `out` not
    written. Returns out [N, nh, hd] (new unless given; it may be q). `sms`:
    how many SMs the work is cut for while kernels of other streams hold
    some, without clusters, which wait for several free SMs at once (0: all
    of them, with clusters where they pay)."""
    shape, kshape = q.shape, k.shape
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    dev = q.get_device()
    lens = cu_q if len_k is None else len_k
    usual = (out is None and cu_k is None and len(shape) == 3 and q.dtype is _BF16 and k.dtype is _BF16
             and v.dtype is _BF16 and cu_q.dtype is _I64 and lens.dtype is _I64 and cu_q.dim() == 1
             and (len(kshape) == 3 and kshape[0] == shape[0] if len_k is None else
                  len(kshape) == 4 and kshape[0] == cu_q.shape[0] - 1 and len_k.shape == kshape[:1])
             and v.shape == kshape and kshape[-1] == shape[2] and qs[2] == 1 and ks[-1] == 1 and vs[-1] == 1
             and cu_q.is_contiguous() and lens.is_contiguous() and shape[1] and kshape[1] and cu_q.shape[0]
             and shape[1] % kshape[1] == 0 and 0 < shape[2] <= MAX_HEAD_SIZE and dev >= 0 and k.get_device() == dev
             and v.get_device() == dev and cu_q.get_device() == dev and lens.get_device() == dev
             and _no_grad(q, k, v))
    if not usual:
        _check_prompt(q, k, v, cu_q, cu_k, len_k, out)
        _check_cuda("prompt_attention", q)
    n, nh, hd = shape
    if out is None:
        out = torch.empty(n, nh, hd, dtype=_BF16, device=q.device)
    if len_k is not None:
        nkv, rows = kshape[1], kshape[2]
        strides = ks[0], ks[1], ks[2], vs[0], vs[1], vs[2]
        starts, lens = 0, lens.data_ptr()
    else:
        rows, nkv = kshape[0], kshape[1]
        strides = 0, ks[1], ks[0], 0, vs[1], vs[0]
        starts, lens = (cu_q if cu_k is None else cu_k).data_ptr(), 0
    os = out.stride()
    _call("aib_prompt_attention_bf16", "prompt_attention", q, _DESC.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 0, qs[0], qs[1], *strides, 0, os[0], os[1],
        n, cu_q.shape[0] - 1, rows, nh, nkv, hd, scale, cu_q.data_ptr(), starts, lens, 0, 0, 0, 0, 0, 0, sms))
    return out


def _check_tree(q, k_cache, v_cache, pos, mask, out) -> None:
    who = "tree_attention"
    _check_device(who, q, k_cache, v_cache, pos, mask, out)
    _check_bf16(who, q=q, k_cache=k_cache, v_cache=v_cache, out=out)
    if torch.is_grad_enabled():
        _check_no_grad(who, q, k_cache, v_cache, out)
    _need(q.dim() == 4, f"{who}: q must be [sequences, tokens, heads, head size]")
    b, t, nh, hd = q.shape
    _need(k_cache.dim() == 4 and v_cache.shape == k_cache.shape and k_cache.shape[0] == b and k_cache.shape[3] == hd,
          f"{who}: caches must be [{b}, kv heads, max_len, {hd}]")
    _check_heads(who, nh, k_cache.shape[1], hd)
    _check_index(who, (b,), pos=pos)
    _need(mask.dtype == torch.bool and mask.dim() in (2, 3) and mask.shape[-2] == t
          and (mask.dim() == 2 or mask.shape[0] == b), f"{who}: mask must be bool [{t}, C] or [{b}, {t}, C]")
    _need(mask.shape[-1] <= k_cache.shape[2],
          f"{who}: {mask.shape[-1]} drafted tokens for caches of {k_cache.shape[2]} rows")
    if out is not None:
        _check_out(who, out, q)


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, pos: torch.Tensor,
                   mask: torch.Tensor, scale: float, out: torch.Tensor | None = None, sms: int = 0) -> torch.Tensor:
    """Attention of T drafted tokens per sequence over its cache: q
    [B, T, nh, hd], caches [B, nkv, max_len, hd], pos int64 [B].

    Every query of sequence b sees the slots before pos[b]; the C drafted
    tokens are at the slots pos[b] .. pos[b] + C - 1, and query i sees those
    with mask[i, j] (mask bool [T, C] for all sequences or [B, T, C]; see
    tree_mask). T = C = 1 is the single-token step of a batch. A query that
    sees nothing gives zeros. Returns [B, T, nh, hd] (new unless given; it
    may be q). `sms`: as for prompt_attention."""
    shape, kshape, mshape = q.shape, k_cache.shape, mask.shape
    qs, ks, vs, ms = q.stride(), k_cache.stride(), v_cache.stride(), mask.stride()
    dev = q.get_device()
    usual = (out is None and len(shape) == 4 and len(kshape) == 4 and q.dtype is _BF16 and k_cache.dtype is _BF16
             and v_cache.dtype is _BF16 and pos.dtype is _I64 and mask.dtype is torch.bool
             and v_cache.shape == kshape and kshape[0] == shape[0] and kshape[3] == shape[3] and qs[3] == 1
             and ks[3] == 1 and vs[3] == 1 and pos.shape == shape[:1] and pos.is_contiguous() and len(mshape) == 2
             and mshape[0] == shape[1] and mshape[1] <= kshape[2] and shape[2] and kshape[1]
             and shape[2] % kshape[1] == 0 and 0 < shape[3] <= MAX_HEAD_SIZE and dev >= 0
             and k_cache.get_device() == dev and v_cache.get_device() == dev and pos.get_device() == dev
             and mask.get_device() == dev and _no_grad(q, k_cache, v_cache))
    if not usual:
        _check_tree(q, k_cache, v_cache, pos, mask, out)
        _check_cuda("tree_attention", q)
    b, t, nh, hd = shape
    if out is None:
        out = torch.empty(b, t, nh, hd, dtype=_BF16, device=q.device)
    at = pos.data_ptr()
    # a mask without columns still says "tree" to the C entry: any address serves, none is read
    _call("aib_tree_attention_bf16", "tree_attention", q, _DESC.pack(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), *qs[:3], *ks[:3], *vs[:3],
        *out.stride()[:3], t, b, kshape[2], nh, kshape[1], hd, scale, 0, 0, 0, at, mask.data_ptr() or at,
        ms[0] if len(ms) == 3 else 0, ms[-2], ms[-1], mshape[-1], sms))
    return out


def _check_rope(qkv, nh, nkv, hd, cu, start, inv_freq, k_cache, v_cache, depth, q_norm, k_norm, out) -> None:
    who = "rope_cache_packed"
    _check_device(who, qkv, cu, start, inv_freq, k_cache, v_cache, depth, q_norm, k_norm, out)
    _check_bf16(who, qkv=qkv, k_cache=k_cache, v_cache=v_cache, q_norm=q_norm, k_norm=k_norm, out=out)
    if torch.is_grad_enabled():
        _check_no_grad(who, qkv, inv_freq, k_cache, v_cache, q_norm, k_norm, out)
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
    _need(inv_freq.dtype == _F32 and tuple(inv_freq.shape) == (hd // 2,) and inv_freq.is_contiguous(),
          f"{who}: inv_freq must be fp32 [{hd // 2}]")
    _need(k_cache.data_ptr() != v_cache.data_ptr() or k_cache.numel() == 0, f"{who}: k_cache and v_cache are the same")
    _need((q_norm is None) == (k_norm is None), f"{who}: give both q and k norm weights or neither")
    _need(q_norm is None or (tuple(q_norm.shape) == (hd,) and tuple(k_norm.shape) == (hd,)),
          f"{who}: norm weights must be [{hd}]")
    _check_not_expanded(who, "k_cache", k_cache)
    _check_not_expanded(who, "v_cache", v_cache)
    _need(out is None or (tuple(out.shape) == (n, nh, hd) and out.is_contiguous()),
          f"{who}: out must be contiguous [N, {nh}, {hd}]")


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
    shape, kshape = qkv.shape, k_cache.shape
    xs, ks, vs = qkv.stride(), k_cache.stride(), v_cache.stride()
    dev = qkv.get_device()
    usual = (out is None and len(shape) == 2 and len(kshape) == 4 and qkv.dtype is _BF16 and k_cache.dtype is _BF16
             and v_cache.dtype is _BF16 and cu.dtype is _I64 and start.dtype is _I64 and inv_freq.dtype is _F32
             and nh > 0 and nkv > 0 and hd % 2 == 0 and 0 < hd <= 1024 and shape[1] == (nh + 2 * nkv) * hd and xs[1] == 1
             and ks[3] == 1 and vs[3] == 1 and min(ks) > 0 and min(vs) > 0 and v_cache.shape == kshape
             and kshape[1] == nkv and kshape[3] == hd and start.shape == kshape[:1] and kshape[2] > 0 and cu.dim() == 1
             and cu.shape[0] == kshape[0] + 1 and inv_freq.dim() == 1 and inv_freq.shape[0] == hd // 2
             and cu.is_contiguous() and start.is_contiguous() and inv_freq.is_contiguous() and dev >= 0
             and cu.get_device() == dev and start.get_device() == dev and inv_freq.get_device() == dev
             and k_cache.get_device() == dev and v_cache.get_device() == dev
             and k_cache.data_ptr() != v_cache.data_ptr()
             and (depth is None or (depth.dtype is _I64 and depth.dim() == 1 and depth.shape[0] == shape[0]
                                    and depth.is_contiguous() and depth.get_device() == dev))
             and (q_norm is None and k_norm is None
                  or q_norm is not None and k_norm is not None and q_norm.dtype is _BF16 and k_norm.dtype is _BF16
                  and q_norm.dim() == 1 and k_norm.dim() == 1 and q_norm.shape[0] == hd and k_norm.shape[0] == hd
                  and q_norm.stride(0) == 1 and k_norm.stride(0) == 1 and q_norm.get_device() == dev
                  and k_norm.get_device() == dev)
             and _no_grad(qkv, inv_freq, k_cache, v_cache, q_norm, k_norm))
    if not usual:
        _check_rope(qkv, nh, nkv, hd, cu, start, inv_freq, k_cache, v_cache, depth, q_norm, k_norm, out)
        _check_cuda("rope_cache_packed", qkv)
    n = shape[0]
    if out is None:
        out = torch.empty(n, nh, hd, dtype=_BF16, device=qkv.device)

    def call():
        return _lib.load().aib_rope_cache_packed_bf16(
            qkv.data_ptr(), xs[0], n, cu.shape[0] - 1, nh, nkv, hd, cu.data_ptr(), start.data_ptr(),
            None if depth is None else depth.data_ptr(), None if q_norm is None else q_norm.data_ptr(),
            None if k_norm is None else k_norm.data_ptr(), eps, inv_freq.data_ptr(), out.data_ptr(),
            k_cache.data_ptr(), v_cache.data_ptr(), struct.pack("3q", *ks[:3]), struct.pack("3q", *vs[:3]), kshape[2],
            _raw_stream(dev))

    if torch._C._cuda_getDevice() == dev:
        rc = call()
    else:
        with torch.cuda.device(dev):
            rc = call()
    if rc:
        _lib.check(rc, "rope_cache_packed")
    return out


_shape_of, _dtype_of = torch.Tensor.shape.__get__, torch.Tensor.dtype.__get__


def _all_are(values, value, n: int) -> bool:
    return list(values).count(value) == n


def _check_keep(caches, pos, keep, ptrs) -> None:
    who = "keep_cache_rows"
    first = caches[0]
    _check_device(who, first, pos, keep)
    if torch.is_grad_enabled():
        _check_no_grad(who, *caches)
    _need(first.dim() == 4, f"{who}: caches must be [B, kv heads, max_len, head size]")
    for t in caches:
        _need(t.dtype == _BF16 and t.shape == first.shape and t.stride() == first.stride() and t.device == first.device,
              f"{who}: caches must be bf16 tensors of one shape, one set of strides and one device")
    _need(first.stride(3) == 1 or first.shape[3] == 1, f"{who}: caches need unit stride along the head size")
    _check_not_expanded(who, "a cache", first)
    _need(first.numel() == 0 or len(set(ptrs)) == len(ptrs), f"{who}: a cache is given twice")
    _need(keep.dim() == 2, f"{who}: keep must be int64 [B, n]")
    _need(keep.shape[1] <= MAX_KEEP, f"{who}: {keep.shape[1]} rows, at most {MAX_KEEP}")
    _check_index(who, (first.shape[0],), pos=pos)
    _check_index(who, (first.shape[0], keep.shape[1]), keep=keep)


def keep_cache_rows(caches: list, pos: torch.Tensor, keep: torch.Tensor) -> None:
    """The rows that stay after a draft was accepted, moved together, in
    every cache of `caches` (tensors [B, nkv, max_len, hd] of one shape and
    one set of strides: the keys and the values of all layers) at once: row
    pos[b] + i <- row pos[b] + keep[b, i] as it was before the call, for the
    n <= 256 columns of keep (int64 [B, n]). keep < 0, and rows outside the
    cache, leave the row as it is. The caches must not overlap."""
    if not caches:
        return
    first = caches[0]
    shape, strides, dev = first.shape, first.stride(), first.get_device()
    n = len(caches)
    ptrs = list(map(torch.Tensor.data_ptr, caches))
    # (map over the type's own accessors: 80 tensors of a 40-layer model are looked at in each call)
    usual = (len(shape) == 4 and _all_are(map(_dtype_of, caches), _BF16, n)
             and _all_are(map(_shape_of, caches), shape, n)
             and (_all_are(map(torch.Tensor.is_contiguous, caches), True, n)
                  or _all_are(map(torch.Tensor.stride, caches), strides, n))
             and _all_are(map(torch.Tensor.get_device, caches), dev, n) and len(set(ptrs)) == n and dev >= 0
             and strides[3] == 1 and min(strides) > 0 and pos.dtype is _I64 and keep.dtype is _I64
             and pos.get_device() == dev and keep.get_device() == dev and pos.shape == shape[:1] and keep.dim() == 2
             and keep.shape[0] == shape[0] and keep.shape[1] <= MAX_KEEP and pos.is_contiguous()
             and keep.is_contiguous() and not (torch.is_grad_enabled() and torch._C._any_requires_grad(*caches)))
    if not usual:
        _check_keep(caches, pos, keep, ptrs)
        _check_cuda("keep_cache_rows", first)
    if first.numel() == 0:
        return

    def call():
        table = array.array("Q", ptrs)
        return _lib.load().aib_keep_cache_rows_bf16(table.buffer_info()[0], n, *shape,
                                                    struct.pack("3q", *strides[:3]), pos.data_ptr(), keep.data_ptr(),
                                                    keep.shape[1], _raw_stream(dev))

    if torch._C._cuda_getDevice() == dev:
        rc = call()
    else:
        with torch.cuda.device(dev):
            rc = call()
    if rc:
        _lib.check(rc, "keep_cache_rows")


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

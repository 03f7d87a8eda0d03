"""A paged cache of keys and values: new tokens enter it normed and rotated, and attention reads it.

- ``paged_kv_append``: keys and values of new tokens into their pages, with RMSNorm and the rotary embedding on the way, and
  the queries beside them;
- ``paged_attention``: the new tokens' attention over the cache: single tokens, pieces of a prompt, trees of drafted tokens,
  with a sliding window and first tokens that stay visible (``window_attention``'s form for serving).

The cache is a pair of tensors ``[pages, HKV, page_size, D]`` that the caller owns; any strides with a contiguous last axis do
(``[pages, page_size, HKV, D]`` transposed is one). ``page_table [N, width]`` (int32) names each sequence's pages in order,
``lengths [N]`` its tokens in the cache with the new ones counted, in both calls. Tables and lengths are not read on the host, and
``cu_seqlens`` only where ``cu_seqlens_cpu`` is missing: with it both calls can be captured, and replayed with new tables, lengths
and bounds. Replayed and compiled calls take ``cu_seqlens`` unchecked, in ascending order; a sequence may then be without new
tokens. The reference has no cache and no decoding (``sore/model/lm.py:206-208``).
"""
from __future__ import annotations

import torch
from torch import Tensor

from sorernn_amd import _lib
from sorernn_amd.linear import _launch, _strided, _weight
from sorernn_amd.ops import _check_cuda, _cu_info, _no_grad_check
from sorernn_amd.window import _CODES, _whole

__all__ = ["paged_kv_append", "paged_attention"]


def _cache_strides(name: str, c: Tensor):
    """Strides between pages, heads and tokens; of a dimension of one, which may have any, 0."""
    st = c.stride()
    if c.shape[0] == 1 or c.shape[1] == 1:
        st = tuple(0 if n == 1 else s for n, s in zip(c.shape, st))
    if st[3] != 1 or c.data_ptr() & 15 or (st[0] | st[1] | st[2]) & 7 or st[2] > 1 << 23:
        raise ValueError(f"{name}: rows of the caches must be contiguous and 16-byte aligned, strides {c.stride()}")
    return st[:3]


def _cache_args(name: str, x: Tensor, k_cache: Tensor, v_cache: Tensor, page_table: Tensor, lengths: Tensor,
                cu_seqlens: Tensor | None, cu_seqlens_cpu: Tensor | None):
    """Checks of what both calls take, ``x [B,T,heads,D]`` among it. Returns the caches' strides, the table with contiguous rows,
    the lengths, the number of sequences and the flags."""
    b, t, _, d = x.shape
    if d not in (64, 128):
        raise NotImplementedError(f"{name}: head dim {d} unsupported (64 or 128)")
    if x.dtype not in _CODES:
        raise NotImplementedError(f"{name}: bf16 or fp16 only, got {x.dtype}")
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.shape[3] != d:
        raise ValueError(f"{name}: caches must be [pages,HKV,page_size,{d}], got {tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
    if k_cache.dtype != x.dtype or v_cache.dtype != x.dtype:
        raise ValueError(f"{name}: new tokens and caches must share a dtype ({x.dtype}, {k_cache.dtype}, {v_cache.dtype})")
    pages, hkv, size, _ = k_cache.shape
    if not b or not pages or not hkv or not x.shape[2]:
        raise ValueError(f"{name}: no batch, no heads or no pages in {tuple(x.shape)}, {tuple(k_cache.shape)}")
    if size < 16 or size > 65536 or size & (size - 1):
        raise NotImplementedError(f"{name}: page size {size} unsupported (a power of two from 16 to 65536)")
    kst, vst = _cache_strides(name, k_cache), _cache_strides(name, v_cache)
    n, flags = _cu_info(name, cu_seqlens, cu_seqlens_cpu, b, t)
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != n or not page_table.shape[1]:
        raise ValueError(f"{name}: page_table must be int32 [{n}, width], got {page_table.dtype} {tuple(page_table.shape)}")
    if lengths.dtype not in (torch.int32, torch.int64) or lengths.shape != (n,):
        raise ValueError(f"{name}: lengths must be int32 or int64 [{n}], got {lengths.dtype} {tuple(lengths.shape)}")
    if page_table.stride(1) != 1:
        page_table = page_table.contiguous()
    return kst, vst, page_table, lengths.contiguous(), n, flags


def paged_kv_append(k: Tensor, v: Tensor, k_cache: Tensor, v_cache: Tensor, page_table: Tensor, lengths: Tensor,
                    q: Tensor | None = None, q_weight: Tensor | None = None, k_weight: Tensor | None = None,
                    positions: Tensor | None = None, rot_dim: int | None = None, theta: float = 1e7, eps: float = 1e-6,
                    cu_seqlens: Tensor | None = None, cu_seqlens_cpu: Tensor | None = None) -> Tensor | None:
    """Puts new tokens' keys and values into a paged cache, keys normed and rotated on the way; returns the queries likewise.

    ``k, v [N,T,HKV,D]`` and ``q [N,T,HQ,D]`` or ``None`` (bf16 or fp16, D 64 or 128; views of a projection's output are read
    in place), or ``[1,total,heads,D]`` with ``cu_seqlens [N+1]`` for uneven numbers of new tokens. New token t of sequence n
    goes to place ``lengths[n] - T_n + t``: row ``place % page_size`` of page ``page_table[n, place // page_size]``. With
    ``q_weight`` / ``k_weight`` (``[D]``) the heads of q / k take an RMSNorm first; their first ``rot_dim`` entries (default D,
    a multiple of 16, 0 for none) turn as in ``qk_norm_rope``, by the token's place or by ``positions`` (int32 or int64,
    ``[B,T]`` or ``[T]``: a drafted token's depth in its tree). fp32 inside, one rounding. Returns q contiguous, or ``None``
    without it. Forward only.

    Tokens at a place below 0 (a batch padded in front) or on a page that the cache does not have, and all of a sequence whose
    length its row of the table cannot hold, are not written; the rest of the cache is left as it is. No two new tokens may
    have one place.
    """
    name = "paged_kv_append"
    _check_cuda(name, k, v, k_cache, v_cache, page_table, lengths, q, q_weight, k_weight, positions, cu_seqlens)
    _no_grad_check(name, k, v, q, q_weight, k_weight, k_cache, v_cache)
    if k.dim() != 4 or k.shape != v.shape or (q is not None and (q.dim() != 4 or q.shape[:2] != k.shape[:2] or
                                                                 q.shape[3] != k.shape[3] or not q.shape[2])):
        raise ValueError(f"{name}: expected k,v [B,T,HKV,D] and q [B,T,HQ,D], got {tuple(k.shape)}, {tuple(v.shape)}, "
                         f"{None if q is None else tuple(q.shape)}")
    if v.dtype != k.dtype or (q is not None and q.dtype != k.dtype):
        raise ValueError(f"{name}: q, k, v must share a dtype")
    kcs, vcs, table, lens, n, flags = _cache_args(name, k, k_cache, v_cache, page_table, lengths, cu_seqlens, cu_seqlens_cpu)
    b, t, hkv, d = k.shape
    pages, _, size, _ = k_cache.shape
    if k_cache.shape[1] != hkv:
        raise ValueError(f"{name}: caches have {k_cache.shape[1]} heads, k and v {hkv}")
    for w in (q_weight, k_weight):
        if w is not None and w.shape != (d,):
            raise ValueError(f"{name}: weights must be [{d}], got {tuple(w.shape)}")
    if q_weight is not None and q is None:
        raise ValueError(f"{name}: q_weight without q")
    rot_dim = d if rot_dim is None else int(rot_dim)
    if rot_dim < 0 or rot_dim > d or rot_dim % 16:
        raise NotImplementedError(f"{name}: rot_dim={rot_dim} unsupported (a multiple of 16 up to D={d})")
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64) or positions.shape not in ((b, t), (t,)):
            raise ValueError(f"{name}: positions must be int32 or int64 {(b, t)} or {(t,)}, got {positions.dtype} "
                             f"{tuple(positions.shape)}")
        if positions.dim() == 1:
            positions = positions.expand(b, t)
    (ks, kst), (vs, vst) = _strided(k), _strided(v)
    qw, kw = _weight(q_weight), _weight(k_weight)
    cu = None if cu_seqlens is None else cu_seqlens.contiguous()
    out, hq, qa = None, 0, (None, 0, 0, 0)
    if q is not None:
        qs, qst = _strided(q)
        out, hq, qa = torch.empty(q.shape, device=q.device, dtype=q.dtype), q.shape[2], (qs.data_ptr(), *qst[:3])
    ps = (None, 0, 0, 0) if positions is None else (positions.data_ptr(), *positions.stride(), positions.dtype == torch.int32)
    _launch("gdn_paged_append", k, *qa, ks.data_ptr(), *kst[:3], vs.data_ptr(), *vst[:3], None if qw is None else qw.data_ptr(),
            None if kw is None else kw.data_ptr(), None if out is None else out.data_ptr(), k_cache.data_ptr(),
            *kcs, v_cache.data_ptr(), *vcs, table.data_ptr(), table.stride(0), lens.data_ptr(),
            lens.dtype == torch.int32, *ps, None if cu is None else cu.data_ptr(), b, t, hq, hkv, d, n, pages, size,
            table.shape[1], _CODES[k.dtype], rot_dim, float(theta), float(eps), flags)
    torch.autograd.graph.increment_version((k_cache, v_cache))  # a graph that saved them must not use what they hold now
    return out


def paged_attention(q: Tensor, k_cache: Tensor, v_cache: Tensor, page_table: Tensor, lengths: Tensor,
                    window: int | None = None, sinks: int = 0, tree: Tensor | None = None, scale: float | None = None,
                    cu_seqlens: Tensor | None = None, cu_seqlens_cpu: Tensor | None = None) -> Tensor:
    """Attention of new tokens over a paged cache that holds their keys and values too (``paged_kv_append`` put them there).

    ``q [N,T,HQ,D]`` (bf16 or fp16, D 64 or 128; query head i reads head ``i // (HQ/HKV)``), or ``[1,total,HQ,D]`` with
    ``cu_seqlens [N+1]`` for uneven numbers of new tokens; single tokens and long pieces of a prompt are both meant. The new
    tokens are the last ``T_n`` of ``lengths[n]``. A token at place i sees place ``j <= i`` if ``i - j < window`` (``None``:
    all) or ``j < sinks``. ``scale`` (positive) defaults to ``D**-0.5``. Returns ``o [B,T,HQ,D]``. Forward only.

    ``tree`` (int64, ``[B,T]``, at most 64 new tokens a sequence): the new tokens are a drafted tree; bit t of a token's word
    says that it sees its sequence's new token t (itself and its ancestors). The tokens before them are seen through the window
    from the place behind as many as the token's ancestors, ``lengths[n] - T_n + (bits set) - 1``.

    Rows that see nothing are zero: tokens at a place below 0, of no sequence, without a length. A length above what its row of
    the table can hold counts as that. Keys on pages that the cache does not have are not seen. An infinity or NaN in the cache
    reaches the tokens that see it, not the others; where all scores that a token sees are -inf, its row is NaN.
    """
    name = "paged_attention"
    _check_cuda(name, q, k_cache, v_cache, page_table, lengths, tree, cu_seqlens)
    _no_grad_check(name, q, k_cache, v_cache)
    if q.dim() != 4:
        raise ValueError(f"{name}: expected q [B,T,HQ,D], got {tuple(q.shape)}")
    b, t, hq, d = q.shape
    if tree is not None:
        if tree.dtype != torch.int64 or tree.shape != (b, t):
            raise ValueError(f"{name}: tree must be int64 {(b, t)}, got {tree.dtype} {tuple(tree.shape)}")
        if cu_seqlens is not None and cu_seqlens_cpu is None and not torch.compiler.is_compiling():
            cu_seqlens_cpu = cu_seqlens.detach().cpu()
    kcs, vcs, table, lens, n, flags = _cache_args(name, q, k_cache, v_cache, page_table, lengths, cu_seqlens, cu_seqlens_cpu)
    if tree is not None:
        longest = t if cu_seqlens is None else 0 if cu_seqlens_cpu is None else int(cu_seqlens_cpu.diff().max())
        if longest > 64:
            raise NotImplementedError(f"{name}: trees of up to 64 drafted tokens, got {longest}")
    pages, hkv, size, _ = k_cache.shape
    if hq % hkv:
        raise ValueError(f"{name}: query heads ({hq}) must be a multiple of the caches' ({hkv})")
    window = 0 if window is None else _whole(name, "window", window, 1)
    sinks = _whole(name, "sinks", sinks, 0)
    qs, qst = _strided(q)
    cu = None if cu_seqlens is None else cu_seqlens.contiguous()
    o = torch.empty(b, t, hq, d, device=q.device, dtype=q.dtype)
    width = table.shape[1]
    nbytes = int(_lib.load().gdn_paged_attn_workspace_size(b, t, hq, hkv, d, n, size, width, window, sinks, int(cu is not None)))
    ws = torch.empty(nbytes, device=q.device, dtype=torch.uint8) if nbytes else None
    words = (None, 0, 0) if tree is None else (tree.data_ptr(), *tree.stride())
    _launch("gdn_paged_attn_fwd", q, qs.data_ptr(), *qst[:3], k_cache.data_ptr(), *kcs, v_cache.data_ptr(),
            *vcs, table.data_ptr(), table.stride(0), lens.data_ptr(), lens.dtype == torch.int32, *words,
            o.data_ptr(), None if cu is None else cu.data_ptr(), b, t, hq, hkv, d, n, pages, size, width, _CODES[q.dtype],
            window, sinks, float(d**-0.5 if scale is None else scale), flags, None if ws is None else ws.data_ptr(), nbytes)
    return o

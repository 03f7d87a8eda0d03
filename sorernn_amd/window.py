"""Attention with a sliding window and a few first tokens that stay visible (sinks), with its backward.

``window_attention`` is the attention of whole sequences, prompts and training: causal, grouped query heads, batches or
packed documents, on the kernels of ``gdn_window.hip``. ``paged_attention`` (``sorernn_amd/paged.py``) is its form over a
cache.

It has no counterpart in the reference, whose attention is causal over whole documents (``sore/model/attention.py:124-135``)
and whose native engine has a forward and backward of local attention for its own layer
(``legacy/cpp/src/cuda/ops.cu:1227-1320``). The operator is a pair of ``torch.library`` ops
(``sorernn::window_attention_fwd`` / ``_bwd``) with fake implementations and a registered autograd formula; plain eager
calls run their implementations directly.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from sorernn_amd import _lib
from sorernn_amd import library as _library
from sorernn_amd.linear import _launch, _rows, _strided
from sorernn_amd.ops import _check_cuda, _cu_info

__all__ = ["window_attention"]

_CODES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_MOST_BETWEEN = 1 << 23  # elements between two tokens that the kernels' 32-bit offsets inside a block take


def _heads(x: Tensor):
    """``x [B,T,H,D]`` and its strides if the kernels can read it where it is, else a copy's."""
    x, st = _strided(x)
    if st[1] > _MOST_BETWEEN:
        x = x.clone(memory_format=torch.contiguous_format)
        _, t, h, d = x.shape
        st = (t * h * d, h * d, d, 1)
    return x, st


def _kept_size(q: Tensor):
    """Floats that a forward keeps for its backward: what o's rounding left, in 16 bits, and a logarithm a row."""
    b, t, hq, d = q.shape
    return b * t * hq * (d // 2 + 1)


def fwd_impl(q: Tensor, k: Tensor, v: Tensor, cu_seqlens: Optional[Tensor], window: int, sinks: int, scale: float,
             flags: int, num_seqs: int, save: bool) -> tuple[Tensor, Tensor]:
    b, t, hq, d = q.shape
    (qs, qst), (ks, kst), (vs, vst) = _heads(q), _heads(k), _heads(v)
    cu = None if cu_seqlens is None else cu_seqlens.contiguous()
    o = torch.empty(b, t, hq, d, device=q.device, dtype=q.dtype)
    kept = torch.empty(_kept_size(q) if save else 0, device=q.device, dtype=torch.float32)
    ptr = _lib.ptr
    _launch("gdn_window_attn_fwd", q, ptr(qs), *qst[:3], ptr(ks), *kst[:3], ptr(vs), *vst[:3], ptr(o),
            ptr(kept if save else None), ptr(cu), b, t, hq, k.shape[2], d, num_seqs, _CODES[q.dtype], window, sinks, scale,
            flags)
    return o, kept


fwd = torch.library.custom_op("sorernn::window_attention_fwd", mutates_args=())(fwd_impl)


@fwd.register_fake
def _fwd_fake(q, k, v, cu_seqlens, window, sinks, scale, flags, num_seqs, save):
    b, t, hq, d = q.shape
    return q.new_empty(b, t, hq, d), q.new_empty((_kept_size(q) if save else 0,), dtype=torch.float32)


def bwd_impl(q: Tensor, k: Tensor, v: Tensor, o: Tensor, kept: Tensor, d_o: Tensor, cu_seqlens: Optional[Tensor], window: int,
             sinks: int, scale: float, flags: int, num_seqs: int) -> tuple[Tensor, Tensor, Tensor]:
    b, t, hq, d = q.shape
    hkv = k.shape[2]
    (qs, qst), (ks, kst), (vs, vst), oc, do = _heads(q), _heads(k), _heads(v), _rows(o), _rows(d_o.to(q.dtype))
    cu = None if cu_seqlens is None else cu_seqlens.contiguous()
    dq, dk, dv = (torch.empty(x.shape, device=q.device, dtype=x.dtype) for x in (q, k, v))
    nbytes = int(_lib.load().gdn_window_attn_bwd_workspace_size(b, t, hq, hkv, d, num_seqs, window, sinks, int(cu is not None)))
    ws = torch.empty(nbytes, device=q.device, dtype=torch.uint8)
    ptr = _lib.ptr
    _launch("gdn_window_attn_bwd", q, ptr(qs), *qst[:3], ptr(ks), *kst[:3], ptr(vs), *vst[:3], ptr(oc), ptr(kept), ptr(do),
            ptr(cu), b, t, hq, hkv, d, num_seqs, window, sinks, scale, flags, ptr(dq), ptr(dk), ptr(dv), ptr(ws), nbytes)
    return dq, dk, dv


bwd = torch.library.custom_op("sorernn::window_attention_bwd", mutates_args=())(bwd_impl)


@bwd.register_fake
def _bwd_fake(q, k, v, o, kept, d_o, cu_seqlens, window, sinks, scale, flags, num_seqs):
    return q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)


def _setup(ctx, inputs, output):
    q, k, v, cu_seqlens, *meta, save = inputs
    if not save:
        raise RuntimeError("sorernn::window_attention_fwd: a backward needs save=True")
    ctx.save_for_backward(q, k, v, *output, cu_seqlens)
    ctx.meta = tuple(meta)
    ctx.set_materialize_grads(False)


def _backward(ctx, d_o, _d_kept):
    q, k, v, o, kept, cu_seqlens = ctx.saved_tensors
    if d_o is None:
        d_o = torch.zeros_like(o)
    return *_library._run_bwd(bwd, bwd_impl, q, k, v, o, kept, d_o, cu_seqlens, *ctx.meta), *(None,) * 7


fwd.register_autograd(_backward, setup_context=_setup)
_fwd_eager = _library._eager_function(fwd_impl, _setup, _backward)


def _whole(name: str, what: str, x, least: int) -> int:
    """``x`` as a whole number of at least ``least`` that fits the kernels' 64-bit arguments."""
    if isinstance(x, bool) or not isinstance(x, int) or x < least:
        raise ValueError(f"{name}: {what} must be a whole number from {least} on, got {x!r}")
    return min(x, 1 << 40)


def window_attention(q: Tensor, k: Tensor, v: Tensor, window: int | None = None, sinks: int = 0, scale: float | None = None,
                     cu_seqlens: Tensor | None = None, cu_seqlens_cpu: Tensor | None = None) -> Tensor:
    """Causal attention in which token i sees token j if ``i - j < window`` or ``j < sinks``, with its backward.

    ``q [B,T,HQ,D]``, ``k, v [B,T,HKV,D]`` (bf16 or fp16, D 64 or 128; query head i reads head ``i // (HQ/HKV)``; views of a
    projection's output are read in place). ``window=None``: every earlier token is seen. Places count from 0 in every batch
    row, or in every document of ``cu_seqlens`` (``[N+1]``, needs ``B == 1``); ``cu_seqlens_cpu`` lets the bounds be checked
    without a device sync. ``scale`` (positive) defaults to ``D**-0.5``; scaled scores have to fit fp32. Returns
    ``o [B,T,HQ,D]``; differentiable in q, k and v in bf16. An infinity or NaN in a token reaches the tokens that see it, not
    the others; where all scores that a token sees are -inf, its row is NaN.

    Replayed and compiled calls take ``cu_seqlens`` unchecked, in ascending order: a document may be empty, and tokens before
    the first or behind the last have zeros in ``o`` and in the gradients.
    """
    name = "window_attention"
    _check_cuda(name, q, k, v, cu_seqlens)
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3]:
        raise ValueError(f"{name}: expected q [B,T,HQ,D] and k,v [B,T,HKV,D], got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    b, t, hq, d = q.shape
    hkv = k.shape[2]
    if not b or not hkv or not hq or hq % hkv:
        raise ValueError(f"{name}: query heads ({hq}) must be a multiple of key heads ({hkv}), with a batch (B = {b})")
    if d not in (64, 128):
        raise NotImplementedError(f"{name}: head dim {d} unsupported (64 or 128)")
    if q.dtype != k.dtype or q.dtype != v.dtype:
        raise ValueError(f"{name}: q, k, v must share a dtype ({q.dtype}, {k.dtype}, {v.dtype})")
    if q.dtype not in _CODES:
        raise NotImplementedError(f"{name}: bf16 or fp16 only, got {q.dtype}")
    train = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    if train and q.dtype != torch.bfloat16:
        raise NotImplementedError(f"{name}: the backward exists for bf16 only, got {q.dtype} (inputs require grad); run under "
                                  "torch.no_grad() or detach the inputs")
    window = 0 if window is None else _whole(name, "window", window, 1)
    sinks = _whole(name, "sinks", sinks, 0)
    n, flags = _cu_info(name, cu_seqlens, cu_seqlens_cpu, b, t)
    return _library._eager(fwd, fwd_impl, _fwd_eager, q, k, v, cu_seqlens, window, sinks,
                           float(d**-0.5 if scale is None else scale), flags, n, train)[0]

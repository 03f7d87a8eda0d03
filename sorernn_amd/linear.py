"""Linear attention with a decay for each head, and the q/k norm with rotation that goes before it.

The gated delta rule without its correction term: ``S_t = exp(g_t) S_{t-1} + k_t v_t^T``,
``o_t = scale S_t^T q_t``, with the layouts and arguments of ``chunk_gated_delta_rule``.

- ``chunk_decay_linear_attention``: prompts and training (bf16, chunks of 64 tokens, forward and backward);
- ``fused_recurrent_decay_linear_attention``: single tokens, or any number of them one after the other, in fp32;
- ``qk_norm_rope``: RMSNorm of every query and key head and the rotary embedding in one pass, with its backward.

None has a counterpart in the reference, whose attention layer norms and rotates forward and backward in torch ops
(``sore/model/attention.py:105-116``). The chunked operator and the norm are ``torch.library`` ops
(``sorernn::chunk_decay_linear_attention_fwd`` / ``_bwd``, ``sorernn::qk_norm_rope_fwd`` / ``_bwd``) with fake
implementations and registered autograd formulas; plain eager calls run their implementations directly.
"""
from __future__ import annotations

import warnings
from typing import Optional

import torch
from torch import Tensor

from sorernn_amd import _lib
from sorernn_amd import library as _library
from sorernn_amd.ops import _check_cuda, _cu_info, _no_grad_check

__all__ = ["chunk_decay_linear_attention", "fused_recurrent_decay_linear_attention", "qk_norm_rope"]


def _launch(name: str, x: Tensor, *args) -> None:
    """``_lib.call`` on ``x``'s device and its current stream (a launch goes to the current device)."""
    if x.is_cuda:
        index = x.get_device()
        if index != torch.cuda.current_device():
            with torch.cuda.device(index):
                _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(index))
            return
        _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(index))
    else:
        _lib.call(name, *args, _lib.stream_of(x))


def _rows(x: Tensor) -> Tensor:
    """``x`` contiguous and 16-byte aligned, as the kernels read it."""
    x = x.contiguous()
    return x.clone() if x.data_ptr() & 15 else x


def _state(x: Optional[Tensor]) -> Optional[Tensor]:
    return None if x is None else _rows(x if x.dtype == torch.float32 else x.float())


_CODES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}


# ---------------------------------------------------------------------------------------------------
# sorernn::chunk_decay_linear_attention_fwd / _bwd
# ---------------------------------------------------------------------------------------------------
def _align256(x):
    return (x + 255) // 256 * 256


def states_bytes(b, t, hv, kd, vd, varlen: bool):
    """``gdn_decay_attn_states_size`` in Python: the fp32 states entering the segments of the flat token axis, and the
    segments' decays; 0 where no segment's border cuts a sequence."""
    tokens, most = b * t, 256 // hv if hv <= 128 else 3 if hv <= 170 else 1
    seg = max(128, ((tokens + most - 1) // most + 63) // 64 * 64)
    if (not varlen and t <= max(seg, 384)) or tokens <= 384:
        return 0
    segs = (tokens + seg - 1) // seg
    return 0 if segs == 1 else _align256(segs * hv * kd * vd * 4) + _align256(segs * hv * 4)


def _gate_args(g: Optional[Tensor]):
    """dtype code and element strides of ``g`` ``[B, T, HV]`` (0 where it was expanded)."""
    return (_lib.DTYPE_F32, 0, 0, 0) if g is None else (_CODES[g.dtype], *g.stride())


def attention_fwd_impl(q: Tensor, k: Tensor, v: Tensor, g: Optional[Tensor], initial_state: Optional[Tensor],
                       cu_seqlens: Optional[Tensor], scale: float, flags: int, num_seqs: int,
                       output_final_state: bool) -> tuple[Tensor, Tensor, Tensor]:
    b, t, h, kd = q.shape
    hv, vd = v.shape[2], v.shape[3]
    qc, kc, vc = _rows(q), _rows(k), _rows(v)
    h0 = _state(initial_state)
    cu = None if cu_seqlens is None else cu_seqlens.contiguous()
    o = torch.empty_like(vc)
    final = torch.empty((num_seqs, hv, kd, vd) if output_final_state else (0,), device=q.device, dtype=torch.float32)
    states = torch.empty(states_bytes(b, t, hv, kd, vd, cu is not None), device=q.device, dtype=torch.uint8)
    if t > 0:
        _launch("gdn_decay_attn_fwd", qc, _lib.ptr(qc), _lib.ptr(kc), _lib.ptr(vc), _lib.ptr(g), _lib.ptr(h0), _lib.ptr(o),
                _lib.ptr(final if output_final_state else None), _lib.ptr(cu), b, t, h, hv, kd, vd, num_seqs,
                *_gate_args(g), scale, flags, _lib.ptr(states), states.numel())
    elif output_final_state:
        final.copy_(h0 if h0 is not None else torch.zeros_like(final))
    return o, final, states


attention_fwd = torch.library.custom_op("sorernn::chunk_decay_linear_attention_fwd", mutates_args=())(attention_fwd_impl)


@attention_fwd.register_fake
def _attention_fwd_fake(q, k, v, g, initial_state, cu_seqlens, scale, flags, num_seqs, output_final_state):
    b, t, _, kd = q.shape
    hv, vd = v.shape[2], v.shape[3]
    return (q.new_empty(b, t, hv, vd), q.new_empty((num_seqs, hv, kd, vd) if output_final_state else (0,),
                                                   dtype=torch.float32),
            q.new_empty(states_bytes(b, t, hv, kd, vd, cu_seqlens is not None), dtype=torch.uint8))


def attention_bwd_impl(q: Tensor, k: Tensor, v: Tensor, g: Optional[Tensor], initial_state: Optional[Tensor],
                       final_state: Optional[Tensor], d_o: Tensor, d_final_state: Optional[Tensor], states: Tensor,
                       cu_seqlens: Optional[Tensor], scale: float, flags: int, num_seqs: int, gate_grad: bool,
                       initial_state_grad: bool) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    b, t, h, kd = q.shape
    hv, vd = v.shape[2], v.shape[3]
    qc, kc, vc, do = _rows(q), _rows(k), _rows(v), _rows(d_o.to(q.dtype))
    h0, dht = _state(initial_state), _state(d_final_state)
    cu = None if cu_seqlens is None else cu_seqlens.contiguous()
    dev = q.device
    dq, dk, dv = (torch.empty(x.shape, device=dev, dtype=x.dtype) for x in (q, k, v))
    dg = torch.empty((b, t, hv) if gate_grad else (0,), device=dev, dtype=g.dtype if gate_grad else torch.float32)
    dh0 = torch.empty((num_seqs, hv, kd, vd) if initial_state_grad else (0,), device=dev, dtype=torch.float32)
    if t > 0:
        nbytes = int(_lib.load().gdn_decay_attn_bwd_workspace_size(b, t, h, hv, kd, vd, num_seqs, int(cu is not None)))
        ws = torch.empty(nbytes, device=dev, dtype=torch.uint8)
        _launch("gdn_decay_attn_bwd", qc, _lib.ptr(qc), _lib.ptr(kc), _lib.ptr(vc), _lib.ptr(g), _lib.ptr(h0),
                _lib.ptr(final_state), _lib.ptr(do), _lib.ptr(dht), _lib.ptr(states), _lib.ptr(cu), b, t, h, hv, kd, vd,
                num_seqs, *_gate_args(g), scale, flags, _lib.ptr(dq), _lib.ptr(dk), _lib.ptr(dv),
                _lib.ptr(dg if gate_grad else None), _lib.ptr(dh0 if initial_state_grad else None), _lib.ptr(ws), nbytes)
    elif initial_state_grad:
        dh0.copy_(dht if dht is not None else torch.zeros_like(dh0))
    return dq, dk, dv, dg, dh0


attention_bwd = torch.library.custom_op("sorernn::chunk_decay_linear_attention_bwd", mutates_args=())(attention_bwd_impl)


@attention_bwd.register_fake
def _attention_bwd_fake(q, k, v, g, initial_state, final_state, d_o, d_final_state, states, cu_seqlens, scale, flags,
                        num_seqs, gate_grad, initial_state_grad):
    b, t, _, kd = q.shape
    hv, vd = v.shape[2], v.shape[3]
    return (q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape),
            q.new_empty((b, t, hv) if gate_grad else (0,), dtype=g.dtype if gate_grad else torch.float32),
            q.new_empty((num_seqs, hv, kd, vd) if initial_state_grad else (0,), dtype=torch.float32))


def _attention_setup(ctx, inputs, output):
    q, k, v, g, initial_state, cu_seqlens, scale, flags, num_seqs, output_final_state = inputs
    _, final, states = output
    ctx.save_for_backward(q, k, v, g, initial_state, final if output_final_state else None, cu_seqlens, states)
    ctx.meta = (scale, flags, num_seqs)
    ctx.set_materialize_grads(False)


def _attention_backward(ctx, d_o, d_final, _d_states):
    q, k, v, g, initial_state, final, cu_seqlens, states = ctx.saved_tensors
    scale, flags, num_seqs = ctx.meta
    if d_o is None:
        d_o = torch.zeros(q.shape[0], q.shape[1], v.shape[2], v.shape[3], device=q.device, dtype=q.dtype)
    if d_final is not None and d_final.numel() == 0:
        d_final = None
    want_g = g is not None and ctx.needs_input_grad[3]
    want_h0 = initial_state is not None and ctx.needs_input_grad[4]
    dq, dk, dv, dg, dh0 = _library._run_bwd(attention_bwd, attention_bwd_impl, q, k, v, g, initial_state,
                                            final if want_g and d_final is not None else None, d_o, d_final, states,
                                            cu_seqlens, scale, flags, num_seqs, want_g, want_h0)
    return (dq, dk, dv, dg if want_g else None, dh0.to(initial_state.dtype) if want_h0 else None, None, None, None, None,
            None)


attention_fwd.register_autograd(_attention_backward, setup_context=_attention_setup)
_attention_fwd_eager = _library._eager_function(attention_fwd_impl, _attention_setup, _attention_backward)


def attention_fwd_call(*args):
    """``attention_fwd`` as the entry point calls it: directly when nothing traces or records."""
    return _library._eager(attention_fwd, attention_fwd_impl, _attention_fwd_eager, *args)


def _attention_args(name, q, k, v, g, scale, initial_state, cu_seqlens, cu_seqlens_cpu):
    _check_cuda(name, q, k, v, g, initial_state, cu_seqlens)
    if q.dim() != 4 or k.shape != q.shape or v.dim() != 4 or v.shape[:2] != q.shape[:2]:
        raise ValueError(f"{name}: expected q,k [B,T,H,K] and v [B,T,HV,V], got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    b, t, h, kd = q.shape
    hv, vd = v.shape[2], v.shape[3]
    if not b or not h or not hv or hv % h:
        raise ValueError(f"{name}: value heads ({hv}) must be a multiple of q/k heads ({h}), with a batch (B = {b})")
    if kd not in (64, 128) or vd not in (64, 128):
        raise NotImplementedError(f"{name}: head dims K={kd}, V={vd} unsupported (each must be 64 or 128)")
    if q.dtype != k.dtype or q.dtype != v.dtype:
        raise ValueError(f"{name}: q, k, v must share a dtype ({q.dtype}, {k.dtype}, {v.dtype})")
    _lib.dtype_code(q.dtype)
    if g is not None:
        _lib.dtype_code(g.dtype)
        if g.dim() == 1 and g.shape[0] == hv:
            if g.dtype != torch.float32 and g.requires_grad and torch.is_grad_enabled():
                g = g.float()  # its gradient is a sum over the tokens: summed in fp32, rounded once
            g = g.expand(b, t, hv)
        if tuple(g.shape) != (b, t, hv):
            raise ValueError(f"{name}: g must be [B,T,HV] = {(b, t, hv)} or [HV], got {tuple(g.shape)}")
    n, flags = _cu_info(name, cu_seqlens, cu_seqlens_cpu, b, t)
    if cu_seqlens is not None:  # a replayed or compiled call may leave tokens out
        flags |= _lib.FLAG_ZERO_REST
    if initial_state is not None and tuple(initial_state.shape) != (n, hv, kd, vd):
        raise ValueError(f"{name}: initial_state must be [N,HV,K,V] = {(n, hv, kd, vd)}, got {tuple(initial_state.shape)}")
    return g, n, flags, float(kd**-0.5 if scale is None else scale)


_noted: set = set()


def chunk_decay_linear_attention(q: Tensor, k: Tensor, v: Tensor, g: Tensor | None = None, scale: float | None = None,
                                 initial_state: Tensor | None = None, output_final_state: bool = False,
                                 cu_seqlens: Tensor | None = None, cu_seqlens_cpu: Tensor | None = None):
    """Linear attention with a decay for each head over whole sequences (prompts, training), on matrix cores.

    ``q,k [B,T,H,K]``, ``v [B,T,HV,V]`` bf16 (K, V each 64 or 128; value head i reads q/k head ``i // (HV/H)``);
    ``g`` holds log decays, ``[B,T,HV]`` or one a head ``[HV]`` (fp32, bf16 or fp16; ``None``: no decay; -inf resets the
    state). Returns ``(o [B,T,HV,V], final_state [N,HV,K,V] fp32 or None)``. ``scale`` defaults to ``K**-0.5``. With
    ``cu_seqlens`` (``[N+1]``, needs ``B == 1``) the state restarts at every document; ``cu_seqlens_cpu`` lets the bounds
    be checked without a device sync. Differentiable in q, k, v, g and initial_state. Decays may exceed 1; weights past
    fp32's range (``exp`` of the sum of g over a sequence) are infinite. An infinity or NaN in a token reaches that token
    and those after it (in the backward, the gradients of those before it), not the others. The gradient of g is a sum
    over the tokens from there on, rounded as such: next to 0, where a decay leaves nothing of the state, it is noise of
    about 1e-6 of the terms.

    Replayed and compiled calls take ``cu_seqlens`` unchecked, in ascending order: a document may be empty (its state goes
    through), and tokens before the first or behind the last have zeros in ``o`` and in the gradients.

    fp32 and fp16 q/k/v run on the recurrent kernel, forward only (a ``RuntimeWarning`` says so once per dtype).
    """
    name = "chunk_decay_linear_attention"
    if q.dtype != torch.bfloat16:
        if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, v, g, initial_state)):
            raise NotImplementedError(f"{name}: the backward exists for bf16 q/k/v only, got {q.dtype} (inputs require "
                                      "grad); run under torch.no_grad() or detach the inputs")
        if q.dtype not in _noted and q.is_floating_point():
            _noted.add(q.dtype)
            warnings.warn(f"{name}: {q.dtype} q/k/v run on the fp32 recurrent kernel, not on matrix cores (bf16 q/k/v "
                          "only); reported once per dtype", RuntimeWarning, stacklevel=2)
        return _recurrent(name, q, k, v, g, scale, initial_state, output_final_state, False, cu_seqlens, cu_seqlens_cpu)
    g, n, flags, scale = _attention_args(name, q, k, v, g, scale, initial_state, cu_seqlens, cu_seqlens_cpu)
    o, final, _ = attention_fwd_call(q, k, v, g, initial_state, cu_seqlens, scale, flags, n, bool(output_final_state))
    return o, (final if output_final_state else None)


def _recurrent(name, q, k, v, g, scale, initial_state, output_final_state, inplace, cu_seqlens, cu_seqlens_cpu):
    _no_grad_check(name, q, k, v, g, initial_state)
    g, n, flags, scale = _attention_args(name, q, k, v, g, scale, initial_state, cu_seqlens, cu_seqlens_cpu)
    b, t, h, kd = q.shape
    hv, vd = v.shape[2], v.shape[3]
    q, k, v, h0 = q.contiguous(), k.contiguous(), v.contiguous(), initial_state
    if h0 is not None and not (h0.dtype == torch.float32 and h0.is_contiguous() and h0.data_ptr() % 16 == 0):
        if inplace:
            raise ValueError(f"{name}: inplace_final_state needs a contiguous, 16-byte aligned fp32 initial_state")
        h0 = _state(h0)
    if inplace and h0 is None:
        raise ValueError(f"{name}: inplace_final_state needs an initial_state")
    final = h0 if inplace else None
    if output_final_state and not inplace:
        final = torch.empty(n, hv, kd, vd, device=q.device, dtype=torch.float32)
    o = torch.empty_like(v)
    if t > 0 or (final is not None and not inplace):
        cu = None if cu_seqlens is None else cu_seqlens.contiguous()
        ptr = _lib.ptr
        _launch("gdn_decay_attn_recurrent_fwd", q, ptr(q), ptr(k), ptr(v), ptr(g), ptr(h0), ptr(o), ptr(final), ptr(cu), b, t,
                h, hv, kd, vd, n, _CODES[q.dtype], *_gate_args(g), scale, flags)
        if inplace:  # a graph that saved the state must not use what it holds now
            torch.autograd.graph.increment_version(h0)
    return o, final


def fused_recurrent_decay_linear_attention(q: Tensor, k: Tensor, v: Tensor, g: Tensor | None = None,
                                           scale: float | None = None, initial_state: Tensor | None = None,
                                           output_final_state: bool = False, inplace_final_state: bool = False,
                                           cu_seqlens: Tensor | None = None, cu_seqlens_cpu: Tensor | None = None):
    """The recurrence of ``chunk_decay_linear_attention`` token by token in fp32 (the decode step at ``T == 1``).

    The same arguments, with q/k/v in bf16, fp16 or fp32. With ``inplace_final_state`` the final state overwrites
    ``initial_state`` (contiguous fp32) and is returned. Forward only.
    """
    return _recurrent("fused_recurrent_decay_linear_attention", q, k, v, g, scale, initial_state, output_final_state,
                      inplace_final_state, cu_seqlens, cu_seqlens_cpu)


# ---------------------------------------------------------------------------------------------------
# sorernn::qk_norm_rope_fwd / _bwd
# ---------------------------------------------------------------------------------------------------
def _strided(x: Tensor):
    """``x`` and its strides if its rows can be read where they are (contiguous, each on a 16-byte address), else a copy's."""
    st = x.stride()
    if st[3] != 1 or x.data_ptr() & 15 or (st[0] | st[1] | st[2]) & (16 // x.element_size() - 1):
        x = _rows(x)
        _, t, h, d = x.shape
        st = (t * h * d, h * d, d, 1)  # where a size is 1, a contiguous tensor may have any stride
    return x, st


def _weight(w: Optional[Tensor]) -> Optional[Tensor]:
    return w if w is None or (w.dtype == torch.float32 and w.is_contiguous()) else w.float().contiguous()


def rope_fwd_impl(q: Tensor, k: Tensor, q_weight: Optional[Tensor], k_weight: Optional[Tensor], positions: Optional[Tensor],
                  cu_seqlens: Optional[Tensor], rot_dim: int, theta: float, eps: float, flags: int,
                  num_seqs: int) -> tuple[Tensor, Tensor]:
    b, t, hq, d = q.shape
    (qs, qst), (ks, kst) = _strided(q), _strided(k)
    qw, kw = _weight(q_weight), _weight(k_weight)
    cu = None if cu_seqlens is None else cu_seqlens.contiguous()
    qo = torch.empty_like(q, memory_format=torch.contiguous_format)
    ko = torch.empty_like(k, memory_format=torch.contiguous_format)
    ptr = _lib.ptr
    ps = (None, 0, 0, 0) if positions is None else (ptr(positions), *positions.stride(), positions.dtype == torch.int32)
    _launch("gdn_qk_norm_rope_fwd", qs, ptr(qs), qst[0], qst[1], qst[2], ptr(ks), kst[0], kst[1], kst[2], ptr(qw), ptr(kw),
            *ps, ptr(qo), ptr(ko), ptr(cu), b, t, hq, k.shape[2], d, num_seqs, _CODES[q.dtype], rot_dim, theta, eps, flags)
    return qo, ko


rope_fwd = torch.library.custom_op("sorernn::qk_norm_rope_fwd", mutates_args=())(rope_fwd_impl)


@rope_fwd.register_fake
def _rope_fwd_fake(q, k, q_weight, k_weight, positions, cu_seqlens, rot_dim, theta, eps, flags, num_seqs):
    return q.new_empty(q.shape), k.new_empty(k.shape)


def rope_bwd_impl(q: Tensor, k: Tensor, q_weight: Optional[Tensor], k_weight: Optional[Tensor], positions: Optional[Tensor],
                  cu_seqlens: Optional[Tensor], dq_out: Tensor, dk_out: Tensor, rot_dim: int, theta: float, eps: float,
                  flags: int, num_seqs: int, weight_grads: bool) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    b, t, hq, d = q.shape
    (qs, qst), (ks, kst), dqo, dko = _strided(q), _strided(k), _rows(dq_out.to(q.dtype)), _rows(dk_out.to(q.dtype))
    qw, kw = _weight(q_weight), _weight(k_weight)
    cu = None if cu_seqlens is None else cu_seqlens.contiguous()
    dq = torch.empty_like(q, memory_format=torch.contiguous_format)
    dk = torch.empty_like(k, memory_format=torch.contiguous_format)
    dw = [torch.empty(d if weight_grads and x is not None else 0, device=q.device, dtype=torch.float32)
          for x in (q_weight, k_weight)]
    nbytes = int(_lib.load().gdn_qk_norm_rope_bwd_workspace_size(b, t, d)) if weight_grads else 0
    ws = torch.empty(nbytes, device=q.device, dtype=torch.uint8)
    ptr = _lib.ptr
    ps = (None, 0, 0, 0) if positions is None else (ptr(positions), *positions.stride(), positions.dtype == torch.int32)
    _launch("gdn_qk_norm_rope_bwd", qs, ptr(qs), qst[0], qst[1], qst[2], ptr(ks), kst[0], kst[1], kst[2], ptr(qw), ptr(kw),
            *ps, ptr(dqo), ptr(dko), ptr(dq), ptr(dk), *(ptr(x) if x.numel() else None for x in dw), ptr(cu), b, t, hq,
            k.shape[2], d, num_seqs, _CODES[q.dtype], rot_dim, theta, eps, flags, ptr(ws), nbytes)
    return dq, dk, dw[0], dw[1]


rope_bwd = torch.library.custom_op("sorernn::qk_norm_rope_bwd", mutates_args=())(rope_bwd_impl)


@rope_bwd.register_fake
def _rope_bwd_fake(q, k, q_weight, k_weight, positions, cu_seqlens, dq_out, dk_out, rot_dim, theta, eps, flags, num_seqs,
                   weight_grads):
    d = q.shape[3]
    dw = [q.new_empty(d if weight_grads and x is not None else 0, dtype=torch.float32) for x in (q_weight, k_weight)]
    return q.new_empty(q.shape), k.new_empty(k.shape), dw[0], dw[1]


def _rope_setup(ctx, inputs, output):
    q, k, q_weight, k_weight, positions, cu_seqlens, *meta = inputs
    ctx.save_for_backward(q, k, q_weight, k_weight, positions, cu_seqlens)
    ctx.meta = tuple(meta)


def _rope_backward(ctx, dq_out, dk_out):
    q, k, q_weight, k_weight, positions, cu_seqlens = ctx.saved_tensors
    want = [w is not None and ctx.needs_input_grad[i] for i, w in ((2, q_weight), (3, k_weight))]
    dq, dk, dqw, dkw = _library._run_bwd(rope_bwd, rope_bwd_impl, q, k, q_weight, k_weight, positions, cu_seqlens, dq_out,
                                         dk_out, *ctx.meta, any(want))
    return (dq, dk, dqw.to(q_weight.dtype) if want[0] else None, dkw.to(k_weight.dtype) if want[1] else None,
            None, None, None, None, None, None, None)


rope_fwd.register_autograd(_rope_backward, setup_context=_rope_setup)
_rope_fwd_eager = _library._eager_function(rope_fwd_impl, _rope_setup, _rope_backward)


def rope_fwd_call(*args):
    """``rope_fwd`` as the entry point calls it: directly when nothing traces or records."""
    return _library._eager(rope_fwd, rope_fwd_impl, _rope_fwd_eager, *args)


def qk_norm_rope(q: Tensor, k: Tensor, q_weight: Tensor | None = None, k_weight: Tensor | None = None,
                 positions: Tensor | None = None, rot_dim: int | None = None, theta: float = 1e7, eps: float = 1e-6,
                 cu_seqlens: Tensor | None = None, cu_seqlens_cpu: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """RMSNorm of every query and key head, then the rotary embedding of its first ``rot_dim`` entries, in one pass.

    ``q [B,T,HQ,D]``, ``k [B,T,HK,D]`` (bf16, fp16 or fp32; D 64, 128 or 256; views of a projection's output are read in
    place), weights ``[D]`` or ``None`` (ones). Entry ``f`` turns with ``f + rot_dim / 2`` by
    ``position * theta**(-2f / rot_dim)``; ``rot_dim`` (default D) is a multiple of 16, 0 for the norm alone.
    ``positions`` (int32 or int64, ``[B,T]`` or ``[T]``) are the tokens' places, for decoding the caches' lengths; without
    them they count from 0 in every batch row, or in every document of ``cu_seqlens`` (``B == 1``). fp32 inside, one
    rounding. Returns contiguous ``(q, k)``; differentiable in q, k and the weights.
    """
    name = "qk_norm_rope"
    _check_cuda(name, q, k, q_weight, k_weight, positions, cu_seqlens)
    if q.dim() != 4 or k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3]:
        raise ValueError(f"{name}: expected q [B,T,HQ,D] and k [B,T,HK,D], got {tuple(q.shape)}, {tuple(k.shape)}")
    if q.dtype != k.dtype:
        raise ValueError(f"{name}: q and k must share a dtype ({q.dtype}, {k.dtype})")
    _lib.dtype_code(q.dtype)
    b, t, hq, d = q.shape
    if not b or not hq or not k.shape[2]:
        raise ValueError(f"{name}: no batch or no heads in q {tuple(q.shape)}, k {tuple(k.shape)}")
    for w in (q_weight, k_weight):
        if w is not None and w.shape != (d,):
            raise ValueError(f"{name}: weights must be [{d}], got {tuple(w.shape)}")
    rot_dim = d if rot_dim is None else int(rot_dim)
    if d not in (64, 128, 256) or rot_dim < 0 or rot_dim > d or rot_dim % 16:
        raise NotImplementedError(f"{name}: D={d}, rot_dim={rot_dim} unsupported (D 64, 128 or 256, rot_dim a multiple of "
                                  "16 up to D)")
    if positions is not None:
        if cu_seqlens is not None:
            raise ValueError(f"{name}: positions and cu_seqlens exclude each other")
        if positions.dtype not in (torch.int32, torch.int64) or positions.shape not in ((b, t), (t,)):
            raise ValueError(f"{name}: positions must be int32 or int64 {(b, t)} or {(t,)}, got {positions.dtype} "
                             f"{tuple(positions.shape)}")
        if positions.dim() == 1:
            positions = positions.expand(b, t)
    n, flags = _cu_info(name, cu_seqlens, cu_seqlens_cpu, b, t)
    return rope_fwd_call(q, k, q_weight, k_weight, positions, cu_seqlens, rot_dim, float(theta), float(eps), flags, n)

"""Attention of decoder states over the Listener's features, beside ``Attention`` (one state per utterance, MLP keys): many states per
utterance, heads of keys and values, utterances of different lengths, fp32 / bf16 / fp16 (``las_cross_attention_fwd`` / ``_bwd``)."""
from __future__ import annotations

import functools
import math

import torch

from .. import _cabi
from .._cabi import DTYPES, SIZES_BELOW, CrossAttentionDesc, lib


def _aligned(t):
    return t if not t.data_ptr() & 15 else t.clone(memory_format=torch.contiguous_format)


def _refuse(query, key, value):
    """The first thing that is wrong with the operands."""
    for name, t in (("query", query), ("key", key), ("value", value)):
        if not t.is_cuda:
            raise RuntimeError("the LAS HIP path needs CUDA(ROCm) tensors; there is no CPU fallback")
        if t.dim() != 4:
            raise RuntimeError(f"cross_attention: {name} must be (batch, length, heads, head size), got {tuple(t.shape)}")
        if t.dtype != query.dtype or t.device != query.device:
            raise RuntimeError("cross_attention: query, key and value must share one type and device")
    if query.dtype not in DTYPES:
        raise RuntimeError(f"cross_attention computes in fp32, bf16 or fp16; got {query.dtype}")
    B, _U, H, D = query.shape
    if key.shape != value.shape or key.shape[0] != B or key.shape[3] != D:
        raise RuntimeError(f"cross_attention: query {tuple(query.shape)}, key {tuple(key.shape)}, value {tuple(value.shape)} do not go together")
    Hkv = key.shape[2]
    if max(B, _U, key.shape[1], H) >= SIZES_BELOW:
        raise RuntimeError(f"cross_attention: sizes below 2^30 are needed, got query {tuple(query.shape)}, key {tuple(key.shape)}")
    if H < 1 or Hkv < 1 or H % Hkv:
        raise RuntimeError(f"cross_attention: {H} query heads do not share {Hkv} key heads evenly")
    raise RuntimeError(f"cross_attention: the head size must be a multiple of {4 if query.dtype == torch.float32 else 8} and at most 128, got {D}")


def _lengths(key_lengths, B, T, device):
    if key_lengths.shape != (B,) or key_lengths.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"cross_attention: key_lengths must be ({B},) int32 or int64, got {tuple(key_lengths.shape)} {key_lengths.dtype}")
    if key_lengths.device != device:
        raise RuntimeError("cross_attention: key_lengths must be on the device of the query")
    if key_lengths.dtype != torch.int32:
        key_lengths = key_lengths.clamp(0, T).to(torch.int32)
    return key_lengths.contiguous()


@functools.lru_cache(maxsize=1024)
def _plan(qs, ks, vs, q_strides, k_strides, v_strides, dtype, scale):
    """What a call's shapes and strides settle, so that a decode loop settles it once: whether they go together at all, which operands have to be
    copied to contiguous rows, the library's descriptor, and the workspaces of the forward and the backward.  (Read by the library, never written.)"""
    code = DTYPES.get(dtype)
    if code is None or len(qs) != 4 or len(ks) != 4 or ks != vs:
        return None
    B, U, H, D = qs
    T, Hkv = ks[1], ks[2]
    per16 = 4 if code == 0 else 8
    if max(B, U, T, H) >= SIZES_BELOW or ks[0] != B or ks[3] != D or Hkv < 1 or H < 1 or H % Hkv or not 0 < D <= 128 or D % per16:
        return None
    copied, strides = [], []
    for shape, (sb, st, sh, sd) in ((qs, q_strides), (ks, k_strides), (ks, v_strides)):
        fits = sd == 1 and not (sb | st | sh) % per16
        copied.append(not fits)
        strides += (sb, st, sh) if fits else (shape[1] * shape[2] * D, shape[2] * D, D)
    d = CrossAttentionDesc(B, U, T, H, Hkv, D, code, 1.0 / math.sqrt(D) if scale is None else scale, *strides)
    return d, copied, lib().las_cross_attention_workspace_floats(d), lib().las_cross_attention_bwd_workspace_floats(d)


def _forward(query, key, value, key_lengths, scale, want_lse):
    device, dtype, qs, ks = query.device, query.dtype, query.shape, key.shape
    plan = _plan(qs, ks, value.shape, query.stride(), key.stride(), value.stride(), dtype, scale)
    if plan is None or not query.is_cuda or key.dtype != dtype or value.dtype != dtype or key.device != device or value.device != device:
        _refuse(query, key, value)
    d, copied, n, n_bwd = plan
    if key_lengths is not None:
        key_lengths = _lengths(key_lengths, qs[0], ks[1], device)
    d, q, k, v = _addressed(d, copied, query, key, value)
    out = torch.empty(qs, device=device, dtype=dtype)
    lse = torch.empty(qs[:3], device=device, dtype=torch.float32) if want_lse else None
    work = torch.empty(n, device=device, dtype=torch.float32) if n else None
    _cabi.call_on(device, lib().las_cross_attention_fwd, d, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                  None if key_lengths is None else key_lengths.data_ptr(), out.data_ptr(), None if lse is None else lse.data_ptr(),
                  None if work is None else work.data_ptr())
    return d, n_bwd, q, k, v, key_lengths, out, lse


def _addressed(d, copied, q, k, v):
    """Operands whose rows the library can address, and the descriptor of them: what the plan says has to be copied is copied, as is what starts
    between 16-byte pieces."""
    if True in copied:
        q, k, v = (x.contiguous() if c else x for x, c in zip((q, k, v), copied))
    if (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15:
        q, k, v = _aligned(q), _aligned(k), _aligned(v)
        strides = [0 if n == 1 else s for x in (q, k, v) for n, s in zip(x.shape[:3], x.stride())]      # (a dimension of one may claim any stride)
        d = CrossAttentionDesc(d.B, d.U, d.T, d.H, d.Hkv, d.D, d.dtype, d.scale, *strides)
    return d, q, k, v


class _CrossAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value, key_lengths, scale):
        ctx.desc, ctx.work, *saved = _forward(query, key, value, key_lengths, scale, True)
        ctx.save_for_backward(*saved)
        ctx.scale, ctx.strides = scale, [x.stride() for x in saved[:3]]
        return saved[4]

    @staticmethod
    @_cabi.differentiable_once
    def backward(ctx, dout):
        q, k, v, key_lengths, out, lse = ctx.saved_tensors
        d, device = ctx.desc, q.device
        dout, out, lse = _aligned(dout.contiguous()), _aligned(out.contiguous()), lse.contiguous()
        if key_lengths is not None:
            key_lengths = key_lengths.contiguous()
        # saved tensors may have been elsewhere in between (hooks that keep them on the host, say) and come back in another layout
        if [q.stride(), k.stride(), v.stride()] != ctx.strides or (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15:
            d, q, k, v = _addressed(*_plan(q.shape, k.shape, v.shape, q.stride(), k.stride(), v.stride(), q.dtype, ctx.scale)[:2], q, k, v)
        dq = dk = dv = None
        need_q, need_k, need_v = ctx.needs_input_grad[:3]
        if need_q:
            dq = torch.empty_like(out)
        if need_k or need_v:
            dk = torch.empty_like(k, memory_format=torch.contiguous_format)
            dv = torch.empty_like(dk)
        work = torch.empty(ctx.work, device=device, dtype=torch.float32) if ctx.work else None
        _cabi.call_on(device, lib().las_cross_attention_bwd, d, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                      None if key_lengths is None else key_lengths.data_ptr(), out.data_ptr(), lse.data_ptr(), dout.data_ptr(),
                      None if dq is None else dq.data_ptr(), None if dk is None else dk.data_ptr(), None if dv is None else dv.data_ptr(),
                      None if work is None else work.data_ptr())
        return dq, dk, dv, None, None


def cross_attention(query, key, value, key_lengths=None, scale=None):
    """``softmax(scale * query key^T) value`` of decoder states over an encoder's states.

    ``query`` (B, U, H, D), ``key`` / ``value`` (B, T, Hkv, D) of one type (fp32, bf16, fp16), any strides; H a multiple of Hkv (query head
    ``h`` reads key head ``h // (H // Hkv)``); D a multiple of 16 bytes, at most 128.  ``key_lengths`` (B,) int32 / int64 on the device: the
    utterances' valid frames (clamped to [0, T]); the frames behind them are never read and get zero gradients, and an utterance without
    any gives zeros.  ``scale`` (positive) defaults to ``D ** -0.5``.  Returns (B, U, H, D), contiguous; differentiable (once,
    in reverse mode) in query, key and value.
    Scores, softmax statistics and sums are fp32 whatever the type.  In bf16 and fp16 the probabilities and their gradients are rounded to the type for the
    matrix products that take them (2^-8, 2^-11 of each; in fp16 at a scale that follows the largest), and the backward's inner product of output and its gradient
    takes the rounded output: about 1.4 times the error of one rounding at the end.  What is infinite or NaN in a valid place shows (keys whose scores are all -inf give NaN).  U = 1 is one decode step: the key
    range is split over the GPU where the batch alone does not fill it.  Gradients that nobody asks for are not formed.  Rows that are not
    contiguous or not 16-byte aligned are copied first."""
    if scale is not None:
        scale = float(scale)
        if not 0.0 < scale < math.inf:
            raise RuntimeError(f"cross_attention: scale must be positive, got {scale}")
    _cabi.refuse_tangents("cross_attention", query, key, value)
    if torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad):
        return _CrossAttentionFn.apply(query, key, value, key_lengths, scale)
    return _forward(query, key, value, key_lengths, scale, False)[6]

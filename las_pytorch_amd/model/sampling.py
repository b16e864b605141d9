"""Drawing tokens from logits with temperature, top-k, top-p and min-p (``las_sample_tokens``), for callers that drive
``Speller.forward_step`` themselves; ``Speller.sample`` is such a loop."""
from __future__ import annotations

import functools

import torch

from .. import _cabi
from .._cabi import DTYPES, SIZES_BELOW, lib


def _limit(name, value, B, device, whole=False):
    """(scalar, address of a value per row or None, the tensor that must stay alive)."""
    if not torch.is_tensor(value):
        return (int(value) if whole else float(value)), None, None
    if value.shape != (B,) or value.device != device or value.is_floating_point() == whole or value.is_complex() or value.dtype == torch.bool:
        raise RuntimeError(f"sample_tokens: {name} must be a number or a ({B},) tensor of {'integers' if whole else 'floating numbers'} on the device of the "
                           f"logits, got {tuple(value.shape)} {value.dtype} on {value.device}")
    if whole and value.dtype != torch.int32:
        value = value.to(torch.int64).clamp(0, 2 ** 31 - 1).to(torch.int32)      # (narrower types do not hold the bound)
    value = (value if whole else value.to(torch.float32)).contiguous()
    return 0, value.data_ptr(), value


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(B, V):
    return lib().las_sample_workspace_bytes(B, V)


def sample_tokens(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One token per row: ``(tokens (B,) int64, logprob (B,) fp32)``.

    ``logits`` (B, V) fp32 / bf16 / fp16 logits or log-probs, any row stride; ``uniforms`` (B,) fp32 random numbers in [0, 1).  With
    ``w = exp((logits - max) / temperature)`` and candidates in falling order (equal ones by lower index) kept are the first ``top_k``
    (0: all), of those the ones before which less than ``top_p`` of their mass lies (1: all), of those the ones with ``w >= min_p`` (0:
    all).  The token is the first kept index, in vocabulary order, at which the cumulated mass exceeds ``uniforms`` times the kept
    mass; ``logprob`` is the log of its share.  Each limit is a number or a (B,) tensor on the device (tensors are not read on the host: values
    outside their range count as its nearer end, NaN as off).  ``temperature`` 0 or NaN gives the arg-max.  NaN and -inf logits are never drawn; a row of nothing else gives
    token -1 and logprob -inf.  The same inputs give the same tokens, always.  No derivative: ``logprob`` is cut off from the graph of ``logits``."""
    if not logits.is_cuda:
        raise RuntimeError("the LAS HIP path needs CUDA(ROCm) tensors; there is no CPU fallback")
    if logits.dim() != 2 or logits.shape[1] < 1 or logits.dtype not in DTYPES:
        raise RuntimeError(f"sample_tokens: logits must be (B,V) in fp32, bf16 or fp16, got {tuple(logits.shape)} {logits.dtype}")
    B, V = logits.shape
    if max(B, V) >= SIZES_BELOW:
        raise RuntimeError(f"sample_tokens: sizes below 2^30 are needed, got {tuple(logits.shape)}")
    dev = logits.device
    if uniforms.shape != (B,) or uniforms.dtype != torch.float32 or uniforms.device != dev:
        raise RuntimeError(f"sample_tokens: uniforms must be ({B},) fp32 on the device of the logits, got {tuple(uniforms.shape)} {uniforms.dtype}")
    t, tr, keep_t = _limit("temperature", temperature, B, dev)
    k, kr, keep_k = _limit("top_k", top_k, B, dev, whole=True)
    p, pr, keep_p = _limit("top_p", top_p, B, dev)
    m, mr, keep_m = _limit("min_p", min_p, B, dev)
    if tr is None and not 0.0 <= t < float("inf"):
        raise RuntimeError(f"sample_tokens: temperature must not be negative, got {t}")
    if kr is None and k < 0:
        raise RuntimeError(f"sample_tokens: top_k must not be negative, got {k}")
    if pr is None and not 0.0 <= p <= 1.0:
        raise RuntimeError(f"sample_tokens: top_p must lie in [0, 1], got {p}")
    if mr is None and not 0.0 <= m <= 1.0:
        raise RuntimeError(f"sample_tokens: min_p must lie in [0, 1], got {m}")
    logits = logits.detach()
    if logits.stride(1) != 1 and V > 1:
        logits = logits.contiguous()
    uniforms = uniforms.contiguous()
    tokens = torch.empty(B, device=dev, dtype=torch.int64)
    logprob = torch.empty(B, device=dev, dtype=torch.float32)
    n = _workspace_bytes(B, V)
    work = torch.empty(n, device=dev, dtype=torch.uint8) if n else None
    _cabi.call_on(dev, lib().las_sample_tokens, logits.data_ptr(), logits.stride(0), DTYPES[logits.dtype], B, V, uniforms.data_ptr(), t, min(k, 2 ** 31 - 1), p, m,
                  tr, kr, pr, mr, tokens.data_ptr(), logprob.data_ptr(), None if work is None else work.data_ptr())
    return tokens, logprob

"""Operators around a training generation, as hand-written HIP kernels behind the C ABI (include/az_engine.h): choosing moves from
scores (``sample_actions``).

Tensors live on the GPU; every call is asynchronous on torch's current stream of the tensors' device and may be captured into a
HIP graph.  There is no CPU path: a tensor elsewhere, or a shape or type a kernel does not cover, raises ``EngineError``."""
from __future__ import annotations

import ctypes as C

import torch

from .engine import EngineError, _NN_DTYPES, _ptr, load_library


def _check(rc: int) -> None:
    if rc != 0:
        raise EngineError(f"az call failed ({rc}): {load_library().az_tower_last_error().decode()}")


def _stream(device: torch.device) -> C.c_void_p:
    return C.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _on_gpu(t: torch.Tensor, name: str, dtypes=None, device=None) -> None:
    if not isinstance(t, torch.Tensor):
        raise EngineError(f"{name}: expected a tensor, got {type(t).__name__}")
    if dtypes is not None and t.dtype not in dtypes:
        raise EngineError(f"{name}: dtype {t.dtype} is not one of {', '.join(str(d) for d in dtypes)}")
    if t.layout != torch.strided:
        raise EngineError(f"{name}: expected a strided tensor")
    if device is not None and t.device != device:
        raise EngineError(f"{name}: on {t.device}, expected {device}")
    if t.device.type != "cuda":
        raise EngineError(f"{name}: on {t.device}; the operators have no CPU path")


def _per_row(v, name: str, rows: int, dtype: torch.dtype, device: torch.device):
    """-> (tensor or None, the number to pass beside it)"""
    if isinstance(v, torch.Tensor):
        if tuple(v.shape) != (rows,) or not v.is_contiguous():
            raise EngineError(f"{name}: expected a number or a contiguous {dtype} tensor of shape ({rows},)")
        _on_gpu(v, name, (dtype,), device)
        return v, 0
    return None, v


def sample_actions(scores: torch.Tensor, uniforms: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                   legal: torch.Tensor | None = None, return_logprobs: bool = False):
    """One action per row of ``scores`` (rows, n; f32 / bf16 / f16, unit stride along n, 1 <= n <= 524,288), drawn with
    ``uniforms`` (rows,) f32 in [0, 1) -> int32 (rows,), -1 for a row with nothing legal; with ``return_logprobs`` also the
    natural logarithm of the drawn action's probability, f32 (rows,) (-inf beside -1).

    The weights exp(score / temperature) are cut to the ``top_k`` largest scores (0: all), to the shortest prefix of those in
    descending order that holds ``top_p`` of their mass, and to weights of at least ``min_p`` of the largest; equal scores are
    ordered by index.  The action is then the first index, in index order, at which the kept mass exceeds ``uniforms`` of it.
    temperature 0 takes the first of the largest.  ``legal`` (rows, n) bool: scores outside it, NaN and -inf do not count; scores
    of +inf share the whole mass.  temperature, top_p, min_p (f32) and top_k (i32) may be tensors of (rows,).

    For moves from a search: scores = log(visits) makes the weights visits ** (1 / temperature) (training/self_play.py:73-74)."""
    _on_gpu(scores, "scores", tuple(_NN_DTYPES))
    if scores.dim() != 2 or scores.shape[1] < 1 or scores.shape[1] > 524288 or scores.shape[0] > 0x7FFFFFFF:
        raise EngineError(f"scores: expected (rows, n) with 1 <= n <= 524,288, got {tuple(scores.shape)}")
    dev, (rows, n) = scores.device, scores.shape
    if n > 1 and scores.stride(1) != 1:
        raise EngineError("scores: expected unit stride along the actions")
    _on_gpu(uniforms, "uniforms", (torch.float32,), dev)
    if tuple(uniforms.shape) != (rows,) or not uniforms.is_contiguous():
        raise EngineError(f"uniforms: expected a contiguous tensor of shape ({rows},)")
    if legal is not None:
        _on_gpu(legal, "legal", (torch.bool,), dev)
        if legal.shape != scores.shape or (n > 1 and legal.stride(1) != 1):
            raise EngineError(f"legal: expected {tuple(scores.shape)} with unit stride along the actions")
    t_t, t_v = _per_row(temperature, "temperature", rows, torch.float32, dev)
    k_t, k_v = _per_row(top_k, "top_k", rows, torch.int32, dev)
    p_t, p_v = _per_row(top_p, "top_p", rows, torch.float32, dev)
    m_t, m_v = _per_row(min_p, "min_p", rows, torch.float32, dev)
    if not (t_v >= 0 and k_v >= 0 and p_v >= 0 and 0 <= m_v <= 1) or k_v != int(k_v):
        raise EngineError("temperature >= 0, top_k >= 0 (a whole number), top_p >= 0 and 0 <= min_p <= 1")
    with torch.cuda.device(dev):
        actions = torch.empty(rows, dtype=torch.int32, device=dev)
        logp = torch.empty(rows, dtype=torch.float32, device=dev) if return_logprobs else None
        _check(load_library().az_sample_actions(
            _NN_DTYPES[scores.dtype], rows, n, _ptr(scores), scores.stride(0), _ptr(legal), legal.stride(0) if legal is not None else 0,
            _ptr(uniforms), _ptr(t_t), float(t_v), _ptr(k_t), min(int(k_v), n), _ptr(p_t), float(p_v), _ptr(m_t), float(m_v),
            _ptr(actions), _ptr(logp), _stream(dev)))
    return (actions, logp) if return_logprobs else actions

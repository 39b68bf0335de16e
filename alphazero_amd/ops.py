"""Operators around a training generation, as hand-written HIP kernels behind the C ABI (include/az_engine.h): choosing moves from
scores (``sample_actions``), the normalisation layer of a residual tower with its gradient (``group_norm_act``) and the orthogonalised
weight update (``orthogonalize``).

Tensors live on the GPU; every call is asynchronous on torch's current stream of the tensors' device and may be captured into a
HIP graph (group_norm_act's backward pass under the condition that stands there).  There is no CPU path: a tensor elsewhere, or a shape or type a kernel does not cover, raises ``EngineError``."""
from __future__ import annotations

import ctypes as C
import functools

import torch

from .engine import EngineError, _NN_DTYPES, _ptr, load_library


def _check(rc: int) -> None:
    if rc != 0:
        raise EngineError(f"az call failed ({rc}): {load_library().az_tower_last_error().decode()}")


# The stream and the device without the Python objects around them: 8 us less a call in autograd's thread.  (Looked up in the call: a torch
# without GPU support has neither, and this module is imported there too.)
def _stream(device: torch.device) -> C.c_void_p:
    return C.c_void_p(torch._C._cuda_getCurrentRawStream(device.index))


class _on:
    """the device current for the allocations inside, without a switch where it is current already"""

    def __init__(self, device: torch.device):
        self.guard = None if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


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

    Not differentiable: the log-probability carries no autograd graph, whether the scores require a gradient or not.

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
    if not (t_v >= 0 and 0 <= k_v < float("inf") and p_v >= 0 and 0 <= m_v <= 1) or k_v != int(k_v):
        raise EngineError("temperature >= 0, top_k >= 0 (a whole number), top_p >= 0 and 0 <= min_p <= 1")
    with _on(dev):
        actions = torch.empty(rows, dtype=torch.int32, device=dev)
        logp = torch.empty(rows, dtype=torch.float32, device=dev) if return_logprobs else None
        _check(load_library().az_sample_actions(
            _NN_DTYPES[scores.dtype], rows, n, _ptr(scores), scores.stride(0), _ptr(legal), legal.stride(0) if legal is not None else 0,
            _ptr(uniforms), _ptr(t_t), float(t_v), _ptr(k_t), min(int(k_v), n), _ptr(p_t), float(p_v), _ptr(m_t), float(m_v),
            _ptr(actions), _ptr(logp), _stream(dev)))
    return (actions, logp) if return_logprobs else actions


ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2}


def _dense(t: torch.Tensor) -> torch.Tensor:
    """the tensor as dense channels-last samples (a copy where it is not)"""
    return t.contiguous(memory_format=torch.channels_last)


def _empty_like(x: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(x, memory_format=torch.channels_last)


@functools.lru_cache(maxsize=256)
def _norm_workspace(backward: int, n: int, hw: int, c: int, groups: int) -> int:
    size = load_library().az_group_norm_workspace(backward, n, hw, c, groups)
    if size < 0:
        _check(-1)
    return max(int(size), 16)


# torch keeps one node per leaf (the one that accumulates its gradient) for as long as any autograd graph of the leaf lives, and the node keeps
# the stream it was made under: a backward pass hands gradients over to that stream and waits for it.  Under capture a side stream is drawn
# into the capture by that and joined again; the default stream may not take part in one (torch's warning of a mismatched stream
# of such a node says as much), and the error ends the process, not the call.  So every graph of group_norm_act whose leaves' nodes may be the default stream's is known by its leaves while it lives, and a differentiable
# call under capture is refused where such a graph shares a leaf.
class _Graph:
    """held by the autograd node of one eager call: its leaves (ids of tensors that live as long as the node) stand in ``alive`` until it ends"""

    __slots__ = ()
    alive: dict = {}

    def __init__(self, leaves):
        self.alive[id(self)] = leaves

    def __del__(self):
        self.alive.pop(id(self), None)

    @classmethod
    def holds(cls, leaves) -> bool:
        return any(i in held for held in list(cls.alive.values()) for i in leaves)


def _capturing() -> bool:
    return torch.cuda.is_current_stream_capturing()


def _on_default_stream(device: torch.device) -> bool:
    return torch._C._cuda_getCurrentRawStream(device.index) == 0


def _enter_graph(tensors) -> _Graph | None:
    """what the node of a call with these tensors holds; refuses a capture beside an eager default-stream graph of the same leaves"""
    leaves = [id(t) for t in tensors if t.requires_grad and t.is_leaf] if torch.is_grad_enabled() else None
    if not leaves:
        return None
    if not _capturing():
        # (on a side stream too, beside a graph that is known: it shares that one's nodes, and may outlive it)
        return _Graph(leaves) if _on_default_stream(tensors[0].device) or _Graph.holds(leaves) else None
    if _Graph.holds(leaves):
        raise EngineError("group_norm_act under graph capture: an eager autograd graph of the same parameters, made on the default stream, is alive; "
                          "drop its outputs and losses first, or make it on a side stream")
    return None


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, groups, eps, act, graph):
        n, c, h, w = x.shape
        x = _dense(x)
        residual = _dense(residual) if residual is not None else None
        weight = weight.contiguous() if weight is not None else None
        bias = bias.contiguous() if bias is not None else None
        pd = weight.dtype if weight is not None else bias.dtype if bias is not None else torch.float32
        with _on(x.device):
            y = _empty_like(x)
            size = _norm_workspace(0, n, h * w, c, groups)
            stats = torch.empty(n * groups * 2 + size // 8, dtype=torch.float64, device=x.device)  # the workspace behind the statistics
            ws = stats.data_ptr() + n * groups * 16
            _check(load_library().az_group_norm_forward(
                _NN_DTYPES[x.dtype], _NN_DTYPES[pd], n, h * w, c, groups, act, float(eps), _ptr(x), _ptr(residual), _ptr(weight), _ptr(bias),
                _ptr(y), _ptr(stats), ws, size, _stream(x.device)))
        ctx.save_for_backward(x, weight, bias, residual, stats)
        ctx.groups, ctx.act, ctx.pd, ctx.graph = groups, act, pd, graph
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, residual, stats = ctx.saved_tensors
        n, c, h, w = x.shape
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dy = _dense(dy)
        with _on(x.device):
            dx = _empty_like(x) if need_x else None
            dw = torch.empty(c, dtype=ctx.pd, device=x.device) if need_w else None
            db = torch.empty(c, dtype=ctx.pd, device=x.device) if need_b else None
            dr = _empty_like(x) if need_r and ctx.act else None
            size = _norm_workspace(1, n, h * w, c, ctx.groups)
            ws = torch.empty(size, dtype=torch.uint8, device=x.device)
            if need_x or need_w or need_b or dr is not None:
                _check(load_library().az_group_norm_backward(
                    _NN_DTYPES[x.dtype], _NN_DTYPES[ctx.pd], n, h * w, c, ctx.groups, ctx.act, _ptr(x), _ptr(residual), _ptr(weight), _ptr(bias),
                    _ptr(dy), _ptr(stats), _ptr(dx), _ptr(dr), _ptr(dw), _ptr(db), _ptr(ws), size, _stream(x.device)))
        if need_r and dr is None:
            dr = dy  # (no activation: the sum passes the gradient on)
        return dx, dw, db, dr, None, None, None, None


def group_norm_act(x: torch.Tensor, num_groups: int, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
                   eps: float = 1e-5, activation: str = "relu", residual: torch.Tensor | None = None) -> torch.Tensor:
    """``act(group_norm(x) * weight + bias (+ residual))`` with its gradient, for x (N, C, H, W) f32 / bf16 / f16 whose memory is
    channels last (other layouts are copied into it first; the result is channels last).  ``activation``: "none", "relu" or
    "silu".  weight and bias (C,) are f32 or of x's dtype, both alike; ``residual`` is like x.  Statistics are held in f64, the
    rest in f32, and each output is rounded once.  Differentiable once, in every tensor argument.

    Forward and backward may be captured into a HIP graph, the backward pass only while no eager autograd graph of the same leaves
    (parameters) that was made on the default stream is alive: a kept output or loss of such a step keeps its graph.  A differentiable
    call under capture raises ``EngineError`` beside such a graph of this operator's own that shares a leaf; graphs of the same leaves that
    run through other operators alone are not seen, and capturing a backward pass beside one ends the process.
    ``torch.cuda.make_graphed_callables``, which warms up on a side stream, works."""
    _on_gpu(x, "x", tuple(_NN_DTYPES))
    if x.dim() != 4:
        raise EngineError(f"x: expected (N, C, H, W), got {tuple(x.shape)}")
    n, c, h, w = x.shape
    if activation not in ACTIVATIONS:
        raise EngineError(f"activation: one of {', '.join(ACTIVATIONS)}, got {activation!r}")
    if not isinstance(num_groups, int) or num_groups < 1 or c < 1 or c % num_groups or c > 16384 or num_groups > 1024:
        raise EngineError(f"{c} channels in {num_groups} groups: expected 1 .. 16,384 channels, a multiple of 1 .. 1,024 groups")
    if h * w > 1 << 28 or n * num_groups >= 1 << 24:
        raise EngineError("at most 2^24 - 1 groups in all samples, 2^28 pixels a sample")
    if not eps >= 0.0:
        raise EngineError("eps >= 0")
    dtypes = {x.dtype, torch.float32}
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            _on_gpu(t, name, tuple(dtypes), x.device)
            if tuple(t.shape) != (c,):
                raise EngineError(f"{name}: expected ({c},), got {tuple(t.shape)}")
            dtypes = {t.dtype}  # (the second one like the first)
    if residual is not None:
        _on_gpu(residual, "residual", (x.dtype,), x.device)
        if residual.shape != x.shape:
            raise EngineError(f"residual: expected {tuple(x.shape)}, got {tuple(residual.shape)}")
    graph = _enter_graph([t for t in (x, weight, bias, residual) if t is not None])
    return _GroupNormAct.apply(x, weight, bias, residual, num_groups, eps, ACTIVATIONS[activation], graph)


@torch.no_grad()
def orthogonalize(matrices, *, steps: int = 5, coefficients=(3.4445, -4.7750, 2.0315), eps: float = 1e-7):
    """Newton-Schulz orthogonalisation: ``X = M / (|M|_F + eps)``, then ``steps`` times ``A = X X^T; X = a X + (b A + c A A) X`` on
    the shorter side, which moves every singular value towards 1 (with these coefficients, into about 0.7 .. 1.2).

    ``matrices``: a tensor (rows, cols), a batch (n, rows, cols), or a sequence of (rows, cols) tensors of any sizes, all f32, all
    bf16 or all f16, on one GPU -> new dense tensors of the same shapes and type (a sequence gives a list).  A whole network's
    matrices in one call share their launches.  Sums are f32; factors hold 22 bits (errors like those of f32 products, within
    a factor of two), of bf16 matrices with a short side beyond 64 they hold 11 (1.2 to 1.7 times the error of the result's own rounding
    in all).  A matrix whose norm is far below ``eps`` loses accuracy: entries of X below 2^-16 keep fewer bits.  A matrix's result does not
    depend on the others of the call, but for those of at most 64 x 768, which alone take another kernel than beside larger ones: the
    two results differ by their rounding errors.  A matrix that holds an infinity or a NaN gives NaN.  Not differentiable."""
    single = isinstance(matrices, torch.Tensor)
    if single and matrices.dim() not in (2, 3):
        raise EngineError(f"matrices: expected (rows, cols) or (n, rows, cols), got {tuple(matrices.shape)}")
    if not single and not isinstance(matrices, (list, tuple)):
        raise EngineError(f"matrices: expected a tensor or a sequence of tensors, got {type(matrices).__name__}")
    ms = list(matrices) if not single else [matrices] if matrices.dim() == 2 else list(matrices.unbind(0))
    if not isinstance(steps, int) or not 1 <= steps <= 64:
        raise EngineError("steps: 1 .. 64")
    try:
        a, b, c = (float(v) for v in coefficients)
    except (TypeError, ValueError) as exc:
        raise EngineError("coefficients: three numbers") from exc
    if single:
        _on_gpu(matrices, "matrices", tuple(_NN_DTYPES))
    for i, m in enumerate(ms):
        _on_gpu(m, f"matrices[{i}]", tuple(_NN_DTYPES) if i == 0 else (ms[0].dtype,), ms[0].device if isinstance(ms[0], torch.Tensor) and i else None)
        if m.dim() != 2 or max(m.shape) > 65536:
            raise EngineError(f"matrices[{i}]: expected (rows, cols) with sides up to 65,536, got {tuple(m.shape)}")
    if not ms:
        return torch.empty_like(matrices) if single else []
    lib, dev, n = load_library(), ms[0].device, len(ms)
    with _on(dev):
        src = [m.contiguous() for m in ms]
        out = torch.empty(matrices.shape, dtype=matrices.dtype, device=dev) if single else [torch.empty(m.shape, dtype=m.dtype, device=dev) for m in ms]
        dst = out if not single else [out] if matrices.dim() == 2 else list(out.unbind(0))
        dt, rows, cols = _NN_DTYPES[ms[0].dtype], (C.c_int32 * n)(*[m.shape[0] for m in ms]), (C.c_int32 * n)(*[m.shape[1] for m in ms])
        size = lib.az_orthogonalize_workspace(dt, n, rows, cols)
        if size < 0:
            _check(-1)
        ws = torch.empty(max(int(size), 256), dtype=torch.uint8, device=dev)
        _check(lib.az_orthogonalize(dt, n, (C.c_void_p * n)(*[m.data_ptr() for m in src]), (C.c_void_p * n)(*[m.data_ptr() for m in dst]),
                                    rows, cols, steps, a, b, c, float(eps), _ptr(ws), ws.numel(), _stream(dev)))
    return out

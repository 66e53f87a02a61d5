"""Operators on rows of candidate logits: sampling, a teacher's top logits, distillation, scores by class.

A row holds the logits of one slot's candidate window (what the generator takes its fan-ins from), or any other row of
logits; its first ``counts[r]`` places are valid, and a valid place holds nothing when its logit is ``-inf``.  Logits are
``[rows, width]`` tensors on a HIP device in float32, float16 or bfloat16 with unit stride inside a row and any stride
between rows; ``width`` is at most 131072.  All work is enqueued on the current stream of the logits' device.

* ``sample_rows``: temperature, top-k, top-p and min-p, from given random numbers, without replacement;
* ``top_rows``: the largest logits with their places and the row's log-sum-exp - what is kept of a teacher;
* ``distill_loss`` (differentiable) and ``distill_loss_and_grad`` (both in one pass over the logits);
* ``class_scores`` (differentiable): candidate logits looked up in a table over (kind of row, class of candidate).

The reference has none of these: its generator takes ``torch.topk`` of a row (models/generator.py:162-168) and never
receives a gradient (train.py:297-299).
"""
from __future__ import annotations

import contextlib
import ctypes as C
import math
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _abi

MAX_WIDTH = 131072
MAX_DRAWS = 8
MAX_TOP = 256
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


class Sampling(NamedTuple):
    """Settings of a draw.  Each is a number, or a tensor with one value a row (for ``sample_rows``)."""
    temperature: Union[float, torch.Tensor] = 1.0
    top_k: Union[int, torch.Tensor] = 0
    top_p: Union[float, torch.Tensor] = 1.0
    min_p: Union[float, torch.Tensor] = 0.0


class TopRows(NamedTuple):
    """What ``top_rows`` keeps of a teacher's rows; ``temperature`` is the one ``lse`` was taken at (None: not known)."""
    values: torch.Tensor
    index: torch.Tensor
    lse: Optional[torch.Tensor]
    temperature: Optional[float] = None


class ScoreWindows(NamedTuple):
    """Candidate windows for ``class_scores``: ``cand`` [rows, width] node ids, ``counts`` [rows] or None, ``cls`` [nodes]
    a node's class, ``row_kind`` [rows], ``by_kind`` [rows] the rows in the order of their kinds and ``kind_start``
    [kinds + 1] where each kind begins in it (``ScoreWindows.of`` makes the last two).  All int32."""
    cand: torch.Tensor
    counts: Optional[torch.Tensor]
    cls: torch.Tensor
    row_kind: torch.Tensor
    by_kind: torch.Tensor
    kind_start: torch.Tensor

    @staticmethod
    def of(cand: torch.Tensor, counts: Optional[torch.Tensor], cls: torch.Tensor, row_kind: torch.Tensor, kinds: int) -> "ScoreWindows":
        kind, by_kind = torch.sort(row_kind, stable=True)
        start = torch.searchsorted(kind, torch.arange(kinds + 1, dtype=kind.dtype, device=kind.device))
        return ScoreWindows(cand, counts, cls, row_kind, by_kind.to(torch.int32), start.to(torch.int32))


# ------------------------------------------------------------------ checks
def _rows_of(logits: torch.Tensor, what: str) -> Tuple[int, int, int, int]:
    if not torch.is_tensor(logits) or not logits.is_cuda:
        raise _abi.AigAbiError(f"{what} needs the logits on a HIP device (no CPU path exists)")
    if logits.dim() != 2 or logits.dtype not in _DTYPES:
        raise _abi.AigAbiError(f"{what} takes logits [rows, width] in float32, float16 or bfloat16, got {logits.dtype} {tuple(logits.shape)}")
    rows, width = int(logits.size(0)), int(logits.size(1))
    if not 1 <= width <= MAX_WIDTH:
        raise _abi.AigAbiError(f"{what} takes rows of 1 to {MAX_WIDTH} logits, got {width}")
    if width > 1 and rows > 0 and logits.stride(1) != 1:
        raise _abi.AigAbiError(f"{what} takes rows of adjacent logits, got strides {logits.stride()}")
    return rows, width, int(logits.stride(0)) if rows > 1 else width, _DTYPES[logits.dtype]


def _side(t: Optional[torch.Tensor], shape: tuple, dtype: torch.dtype, like: torch.Tensor, what: str):
    """Pointer of an operand beside the logits (None stays NULL)."""
    if t is None:
        return None
    if not torch.is_tensor(t) or t.device != like.device or t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous():
        got = f"{t.dtype} {tuple(t.shape)} on {t.device}" if torch.is_tensor(t) else type(t).__name__
        raise _abi.AigAbiError(f"{what} must be a contiguous {dtype} tensor of shape {shape} on {like.device}, got {got}")
    return C.c_void_p(t.data_ptr())


def _on(t: torch.Tensor):
    """The tensor's device as the current one, where it is not already."""
    return contextlib.nullcontext() if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


def _data(t: torch.Tensor):
    return C.c_void_p(t.data_ptr())


# ------------------------------------------------------------------ sampling
def sampling_arg(how: Sampling, rows: int, like: torch.Tensor) -> _abi.Sampling:
    """The argument block of a draw's settings; tensors must outlive the call that takes it."""
    a = _abi.Sampling()
    for name, dtype in (("temperature", torch.float32), ("top_k", torch.int32), ("top_p", torch.float32), ("min_p", torch.float32)):
        v = getattr(how, name)
        if torch.is_tensor(v):
            setattr(a, name + "_rows", _side(v, (rows,), dtype, like, name))
            continue
        v = int(v) if name == "top_k" else float(v)
        if v != v or v < 0:
            raise ValueError(f"{name} must not be negative, got {v}")
        if name in ("top_p", "min_p") and v > 1:
            raise ValueError(f"{name} is a share of 1, got {v}")
        setattr(a, name, min(v, 2 ** 31 - 1) if name == "top_k" else v)
    return a


@torch.no_grad()
def sample_rows(logits: torch.Tensor, u: torch.Tensor, counts: Optional[torch.Tensor] = None, want: Optional[torch.Tensor] = None,
                temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> torch.Tensor:
    """Draws ``u.size(1)`` (1 to 8) places of each row without replacement: int32 ``[rows, draws]``, -1 where nothing is
    left to draw or a row wants fewer (``want``, int32 ``[rows]``).

    Weights are ``exp((logit - largest) / temperature)`` in whole multiples of 2^-36 of the row's largest.  In the order
    of the logits (equal ones: lowest place first) ``top_k`` keeps the first k (0: all), ``top_p`` those in front of which
    less than that share of what is kept so far lies (the first always; 1: all), ``min_p`` those with at least that
    share of the largest weight.  ``u`` (float32 ``[rows, draws]`` in [0, 1)) is a place on the sum of the weights left,
    laid out by place.  ``temperature`` 0 takes the largest logit, then the next, whatever the filters.  The four settings
    are numbers or tensors with one value a row (float32; ``top_k`` int32; values outside their range count as the
    nearest inside)."""
    rows, width, ld, dtype = _rows_of(logits, "sample_rows")
    if not torch.is_tensor(u) or u.dim() != 2 or not 1 <= int(u.size(1)) <= MAX_DRAWS:
        raise _abi.AigAbiError(f"sample_rows takes u as [rows, 1 to {MAX_DRAWS} draws]")
    draws = int(u.size(1))
    u_ptr = _side(u, (rows, draws), torch.float32, logits, "u")
    counts_ptr = _side(counts, (rows,), torch.int32, logits, "counts")
    want_ptr = _side(want, (rows,), torch.int32, logits, "want")
    how = sampling_arg(Sampling(temperature, top_k, top_p, min_p), rows, logits)
    out = torch.empty((rows, draws), dtype=torch.int32, device=logits.device)
    with _on(logits):
        _abi.check(_abi.timed("aig_sample_rows", _abi.lib().aig_sample_rows, rows, width, ld, dtype, _data(logits), counts_ptr,
                              want_ptr, C.byref(how), draws, u_ptr, _data(out), _abi.stream(), meta=(rows, width)),
                   "aig_sample_rows")
    return out


# ------------------------------------------------------------------ a teacher's top logits
@torch.no_grad()
def top_rows(logits: torch.Tensor, m: int, counts: Optional[torch.Tensor] = None, temperature: float = 1.0) -> TopRows:
    """The ``m`` (1 to 256) largest logits of each row, largest first, equal ones by lowest place: ``values`` float32 and
    ``index`` int32 ``[rows, m]`` (absent entries ``-inf`` and -1), and ``lse``, float32 ``[rows]``, the log-sum-exp of the
    row at ``temperature`` (``-inf`` for a row without a valid place)."""
    rows, width, ld, dtype = _rows_of(logits, "top_rows")
    m, temperature = int(m), float(temperature)
    if not 1 <= m <= MAX_TOP:
        raise ValueError(f"top_rows keeps 1 to {MAX_TOP} logits a row, got {m}")
    if not 0 < temperature < math.inf:
        raise ValueError(f"the temperature must be positive and finite, got {temperature}")
    counts_ptr = _side(counts, (rows,), torch.int32, logits, "counts")
    values = torch.empty((rows, m), dtype=torch.float32, device=logits.device)
    index = torch.empty((rows, m), dtype=torch.int32, device=logits.device)
    lse = torch.empty(rows, dtype=torch.float32, device=logits.device)
    with _on(logits):
        _abi.check(_abi.timed("aig_top_rows", _abi.lib().aig_top_rows, rows, width, ld, dtype, _data(logits), counts_ptr, m, temperature,
                              _data(values), _data(index), _data(lse), _abi.stream(), meta=(rows, width)), "aig_top_rows")
    return TopRows(values, index, lse, temperature)


# ------------------------------------------------------------------ distillation
class _Teacher(NamedTuple):
    values: torch.Tensor
    index: torch.Tensor
    lse: Optional[torch.Tensor]
    counts: Optional[torch.Tensor]
    weight: Optional[torch.Tensor]
    temperature: float


def _teacher(logits, top, counts, weight, temperature, tail) -> _Teacher:
    rows, width, _, _ = _rows_of(logits, "distill_loss")
    temperature = float(temperature)
    if not 0 < temperature < math.inf:
        raise ValueError(f"the temperature must be positive and finite, got {temperature}")
    values, index, lse = top[0], top[1], top[2]
    if not torch.is_tensor(values) or values.dim() != 2 or not 1 <= int(values.size(1)) <= MAX_TOP:
        raise _abi.AigAbiError(f"a teacher's values are [rows, 1 to {MAX_TOP}]")
    if values.dtype in (torch.float16, torch.bfloat16):       # (kept in half precision: widened here)
        values = values.float()
    m = int(values.size(1))
    if tail:
        if lse is None:
            raise ValueError("tail=True needs the teacher's log-sum-exp (top.lse)")
        taken_at = getattr(top, "temperature", None)
        if taken_at is not None and taken_at != temperature:
            raise ValueError(f"the teacher's log-sum-exp was taken at temperature {taken_at}, the loss is asked for at {temperature}")
    else:
        lse = None
    for name, t, shape, dtype in (("values", values, (rows, m), torch.float32), ("index", index, (rows, m), torch.int32),
                                  ("lse", lse, (rows,), torch.float32), ("counts", counts, (rows,), torch.int32),
                                  ("weight", weight, (rows,), torch.float32)):
        _side(t, shape, dtype, logits, name)
    return _Teacher(values.detach(), index, None if lse is None else lse.detach(), counts,
                    None if weight is None else weight.detach(), temperature)


def _distill(logits: torch.Tensor, t: _Teacher, loss: Optional[torch.Tensor], grad: Optional[torch.Tensor],
             upstream: Optional[torch.Tensor] = None) -> None:
    rows, width, ld, dtype = _rows_of(logits, "distill_loss")
    a = _abi.Distill()
    a.rows, a.width, a.ld, a.m = rows, width, ld, int(t.values.size(1))
    a.dtype, a.temperature = dtype, t.temperature
    a.logits = logits.data_ptr()
    for name in ("counts", "values", "index", "lse", "weight"):
        v = getattr(t, name)
        setattr(a, name, None if v is None else v.data_ptr())
    with _on(logits):
        _abi.check(_abi.timed("aig_distill_rows", _abi.lib().aig_distill_rows, C.byref(a), None if loss is None else _data(loss),
                              None if grad is None else _data(grad), width, None if upstream is None else _data(upstream),
                              0 if upstream is None or upstream.numel() == 1 else 1, _abi.stream(), meta=(rows, width)),
                   "aig_distill_rows")


def _sum_rows(v: torch.Tensor, factor: float) -> torch.Tensor:
    lib = _abi.lib()
    out = torch.empty((), dtype=torch.float32, device=v.device)
    need = lib.aig_sum_rows_ws_bytes(v.numel())
    ws = _abi.workspace(need, v.device) if need else None
    with _on(v):
        _abi.check(lib.aig_sum_rows(v.numel(), _data(v), factor, _data(out), None if ws is None else _data(ws), need, _abi.stream()),
                   "aig_sum_rows")
    return out


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher, factor):
        rows = int(logits.size(0))
        loss = torch.empty(rows, dtype=torch.float32, device=logits.device)
        _distill(logits, teacher, loss, None)
        ctx.save_for_backward(logits, *(v for v in teacher[:5] if v is not None))
        ctx.present, ctx.temperature, ctx.factor = [v is not None for v in teacher[:5]], teacher.temperature, factor
        return loss if factor is None else _sum_rows(loss, factor)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        logits, *rest = ctx.saved_tensors
        rest = iter(rest)
        teacher = _Teacher(*(next(rest) if here else None for here in ctx.present), ctx.temperature)
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        g = g.float().contiguous()
        if ctx.factor is not None and ctx.factor != 1.0:
            g = g * ctx.factor
        _distill(logits, teacher, None, grad, g)
        return grad, None, None


def distill_loss(logits: torch.Tensor, top: TopRows, counts: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None,
                 temperature: float = 1.0, tail: bool = True, reduction: str = "mean") -> torch.Tensor:
    """Distillation of a teacher's top logits into a student's rows, differentiable in ``logits``.

    With ``y = logits / T`` over a row's valid places, ``p = softmax(y)`` and the teacher's listed logits ``t_j`` at places
    ``i_j``, ``q_j = exp(t_j / T - lse)``, the loss of a row is ``T^2`` times (``weight`` [rows] times, where given)

        sum_j q_j (log q_j - log p[i_j])  +  q_R (log q_R - log p_R)

    ``tail`` True: ``lse`` is the teacher's own (``top.lse``, taken at the same temperature) and R stands for all places that
    are not listed, as one outcome with the teacher's remaining probability.  False: ``q`` is normalised over the listed
    entries and the second term is left out.  Entries whose place is not one of the student row's valid places (-1 among
    them) are left out; a row without valid places or without entries has loss 0 and gradient 0.  ``reduction`` is "none"
    (float32 ``[rows]``), "sum" or "mean" (over the rows)."""
    if reduction not in ("none", "sum", "mean"):
        raise ValueError(f"reduction is 'none', 'sum' or 'mean', got {reduction!r}")
    t = _teacher(logits, top, counts, weight, temperature, tail)
    rows = int(logits.size(0))
    if reduction == "mean" and rows == 0:
        raise ValueError("the mean over no rows")
    return _DistillLoss.apply(logits, t, None if reduction == "none" else 1.0 if reduction == "sum" else 1.0 / rows)


@torch.no_grad()
def distill_loss_and_grad(logits: torch.Tensor, top: TopRows, counts: Optional[torch.Tensor] = None,
                          weight: Optional[torch.Tensor] = None, temperature: float = 1.0,
                          tail: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """``distill_loss`` of every row (float32 ``[rows]``) and the gradient of their sum w.r.t. the logits (in the logits'
    type), in one pass over the logits and without an autograd graph: what a training step needs, and what a HIP graph
    can record.  A mean over rows, or any other weighting, goes into ``weight``."""
    t = _teacher(logits, top, counts, weight, temperature, tail)
    loss = torch.empty(int(logits.size(0)), dtype=torch.float32, device=logits.device)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    _distill(logits, t, loss, grad)
    return loss, grad


# ------------------------------------------------------------------ scores by class
def _windows_arg(table: torch.Tensor, w: ScoreWindows) -> _abi.ScoreWindowsArg:
    if not torch.is_tensor(table) or not table.is_cuda:
        raise _abi.AigAbiError("class_scores needs the table on a HIP device (no CPU path exists)")
    if table.dim() != 2 or table.dtype != torch.float32 or not table.is_contiguous():
        raise _abi.AigAbiError(f"class_scores takes a contiguous float32 table [kinds, classes], got {table.dtype} {tuple(table.shape)}")
    if w.cand.dim() != 2 or w.cls.dim() != 1:
        raise _abi.AigAbiError("class_scores takes cand [rows, width] and cls [nodes]")
    a = _abi.ScoreWindowsArg()
    a.rows, a.width, a.nodes = int(w.cand.size(0)), int(w.cand.size(1)), int(w.cls.size(0))
    a.kinds, a.classes = int(table.size(0)), int(table.size(1))
    i32 = torch.int32
    for name, shape in (("cand", (a.rows, a.width)), ("counts", (a.rows,)), ("cls", (a.nodes,)), ("row_kind", (a.rows,)),
                        ("by_kind", (a.rows,)), ("kind_start", (a.kinds + 1,))):
        setattr(a, name, _side(getattr(w, name), shape, i32, table, name))
    return a


class _ClassScores(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, windows):
        a = _windows_arg(table, windows)
        out = torch.empty((a.rows, a.width), dtype=torch.float32, device=table.device)
        with _on(table):
            _abi.check(_abi.timed("aig_class_scores", _abi.lib().aig_class_scores, C.byref(a), _data(table), _data(out), _abi.stream(),
                                  meta=(int(a.rows), int(a.width))), "aig_class_scores")
        ctx.windows, ctx.shape = windows, tuple(table.shape)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        return class_scores_grad(g.float().contiguous(), ctx.windows, *ctx.shape), None


@torch.no_grad()
def class_scores_grad(grad: torch.Tensor, windows: ScoreWindows, kinds: int, classes: int) -> torch.Tensor:
    """The gradient of ``class_scores``' table for a gradient of its output (float32 ``[rows, width]``): float32
    ``[kinds, classes]``, the sum over the rows of a kind and their places of a class - sums in a fixed order."""
    lib = _abi.lib()
    out = torch.empty((kinds, classes), dtype=torch.float32, device=grad.device)
    a = _windows_arg(out, windows)
    g_ptr = _side(grad, (int(a.rows), int(a.width)), torch.float32, out, "grad")
    need = lib.aig_class_scores_bwd_ws_bytes(a.rows, kinds, classes)
    ws = _abi.workspace(need, grad.device)
    with _on(grad):
        _abi.check(_abi.timed("aig_class_scores_bwd", lib.aig_class_scores_bwd, C.byref(a), g_ptr, _data(out), _data(ws), ws.numel(),
                              _abi.stream(), meta=(int(a.rows), int(a.width))), "aig_class_scores_bwd")
    return out


def class_scores(table: torch.Tensor, windows: ScoreWindows) -> torch.Tensor:
    """Logits ``[rows, width]`` looked up in ``table`` (float32 ``[kinds, classes]``) by the kind of the row and the class of
    the candidate, differentiable in the table: nodes with equal feature rows score alike, so a template's candidate
    logits are a table of a few entries.  Places past a row's count, and candidates, classes or kinds outside their range,
    are ``-inf``."""
    return _ClassScores.apply(table, windows)

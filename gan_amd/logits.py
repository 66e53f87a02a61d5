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

import ctypes as C
import functools
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _abi

MAX_WIDTH = 131072
MAX_DRAWS = 8
MAX_TOP = 256
NARROW = 1024          # rows up to this width are held in registers and keep no sums for their gradient
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


class Sampling(NamedTuple):
    """Settings of a draw.  Each is a number, or a tensor with one value a row (for ``sample_rows``)."""
    temperature: Union[float, torch.Tensor] = 1.0
    top_k: Union[int, torch.Tensor] = 0
    top_p: Union[float, torch.Tensor] = 1.0
    min_p: Union[float, torch.Tensor] = 0.0


class _TopRows(NamedTuple):
    values: torch.Tensor
    index: torch.Tensor
    lse: Optional[torch.Tensor]


class TopRows(_TopRows):
    """What ``top_rows`` keeps of a teacher's rows: the three tensors ``values``, ``index`` and ``lse``.  ``temperature``, an
    attribute beside them, is the one ``lse`` was taken at (None: not known)."""
    temperature: Optional[float] = None

    def __new__(cls, values, index, lse, temperature=None):
        self = super().__new__(cls, values, index, lse)
        self.temperature = temperature
        return self

    def _replace(self, **fields):
        temperature = fields.pop("temperature", self.temperature)
        return TopRows(*super()._replace(**fields), temperature)


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
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise _abi.AigAbiError(f"{what} needs the logits on a HIP device (no CPU path exists)")
    dtype = _DTYPES.get(logits.dtype)
    if dtype is None or logits.dim() != 2:
        raise _abi.AigAbiError(f"{what} takes logits [rows, width] in float32, float16 or bfloat16, got {logits.dtype} {tuple(logits.shape)}")
    (rows, width), (ld, step) = logits.shape, logits.stride()
    if not 1 <= width <= MAX_WIDTH:
        raise _abi.AigAbiError(f"{what} takes rows of 1 to {MAX_WIDTH} logits, got {width}")
    if step != 1 and width > 1 and rows > 0:
        raise _abi.AigAbiError(f"{what} takes rows of adjacent logits, got strides {logits.stride()}")
    return rows, width, ld if rows > 1 else width, dtype


def _side(t: Optional[torch.Tensor], shape: tuple, dtype: torch.dtype, device: torch.device, what: str) -> Optional[int]:
    """Address of an operand beside the logits (None stays NULL)."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.shape != shape or t.device != device or not t.is_contiguous():
        got = f"{t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
        raise _abi.AigAbiError(f"{what} must be a contiguous {dtype} tensor of shape {shape} on {device}, got {got}")
    return t.data_ptr()


_entry: dict = {}      # entry points by name, once looked up


def _call(name: str, device: torch.device, *args, meta=None) -> None:
    """An entry point of the library on the current stream of ``device`` (the last argument of all of them)."""
    fn = _entry.get(name)
    if fn is None:
        fn = _entry[name] = getattr(_abi.lib(), name)
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _abi.check(_abi.timed(name, fn, *args, _abi.stream(), meta=meta), name)
    t = _abi.timeline
    if t.enabled or t.sizes_of is not None:
        rc = _abi.timed(name, fn, *args, _abi.stream(), meta=meta)
    else:
        rc = fn(*args, _abi.stream())
    if rc:
        _abi.check(rc, name)


# ------------------------------------------------------------------ sampling
def _setting(name: str, v):
    v = int(v) if name == "top_k" else float(v)
    if v != v or v < 0:
        raise ValueError(f"{name} must not be negative, got {v}")
    if name in ("top_p", "min_p") and v > 1:
        raise ValueError(f"{name} is a share of 1, got {v}")
    return min(v, 2 ** 31 - 1) if name == "top_k" else v


@functools.lru_cache(maxsize=64)
def _settings_of_all(temperature, top_k, top_p, min_p) -> _abi.Sampling:
    return _abi.Sampling(temperature=_setting("temperature", temperature), top_k=_setting("top_k", top_k),
                         top_p=_setting("top_p", top_p), min_p=_setting("min_p", min_p))


_SETTING_TYPES = (("temperature", torch.float32), ("top_k", torch.int32), ("top_p", torch.float32), ("min_p", torch.float32))


def sampling_arg(how: Sampling, rows: int, device: torch.device) -> _abi.Sampling:
    """The argument block of a draw's settings; tensors among them must outlive the call that takes it."""
    if not any(isinstance(v, torch.Tensor) for v in how):
        return _settings_of_all(*how)
    a = _abi.Sampling()
    for (name, dtype), v in zip(_SETTING_TYPES, how):
        if isinstance(v, torch.Tensor):
            setattr(a, name + "_rows", _side(v, (rows,), dtype, device, name))
        else:
            setattr(a, name, _setting(name, v))
    return a


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
    device = logits.device
    if not isinstance(u, torch.Tensor) or u.dim() != 2 or not 1 <= u.size(1) <= MAX_DRAWS:
        raise _abi.AigAbiError(f"sample_rows takes u as [rows, 1 to {MAX_DRAWS} draws]")
    draws = u.size(1)
    how = sampling_arg(Sampling(temperature, top_k, top_p, min_p), rows, device)
    u_ptr = _side(u, (rows, draws), torch.float32, device, "u")
    counts_ptr, want_ptr = (_side(v, (rows,), torch.int32, device, what) for v, what in ((counts, "counts"), (want, "want")))
    out = torch.empty((rows, draws), dtype=torch.int32, device=device)
    _call("aig_sample_rows", device, rows, width, ld, dtype, logits.data_ptr(), counts_ptr, want_ptr, C.byref(how), draws, u_ptr,
          out.data_ptr(), meta=(rows, width))
    return out


# ------------------------------------------------------------------ a teacher's top logits
def top_rows(logits: torch.Tensor, m: int, counts: Optional[torch.Tensor] = None, temperature: float = 1.0) -> TopRows:
    """The ``m`` (1 to 256) largest logits of each row, largest first, equal ones by lowest place: ``values`` float32 and
    ``index`` int32 ``[rows, m]`` (absent entries ``-inf`` and -1), and ``lse``, float32 ``[rows]``, the log-sum-exp of the
    row at ``temperature`` (``-inf`` for a row without a valid place)."""
    rows, width, ld, dtype = _rows_of(logits, "top_rows")
    m, temperature = int(m), float(temperature)
    if not 1 <= m <= MAX_TOP:
        raise ValueError(f"top_rows keeps 1 to {MAX_TOP} logits a row, got {m}")
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"the temperature must be within 1e-6 and 1e6, got {temperature}")
    device = logits.device
    counts_ptr = _side(counts, (rows,), torch.int32, device, "counts")
    values = torch.empty((rows, m), dtype=torch.float32, device=device)
    index = torch.empty((rows, m), dtype=torch.int32, device=device)
    lse = torch.empty(rows, dtype=torch.float32, device=device)
    _call("aig_top_rows", device, rows, width, ld, dtype, logits.data_ptr(), counts_ptr, m, temperature, values.data_ptr(),
          index.data_ptr(), lse.data_ptr(), meta=(rows, width))
    return TopRows(values, index, lse, temperature)


# ------------------------------------------------------------------ distillation
def _teacher(logits, top, counts, weight, temperature, tail, scale=1.0):
    """The argument block of a distillation, and the tensors it points to (they must outlive the calls that take it)."""
    rows, width, ld, dtype = _rows_of(logits, "distill_loss")
    temperature = float(temperature)
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"the temperature must be within 1e-6 and 1e6, got {temperature}")
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
    device, one, i32, f32 = logits.device, (rows,), torch.int32, torch.float32
    a = _abi.Distill(rows, width, ld, m, dtype, temperature, scale, logits.data_ptr(), _side(counts, one, i32, device, "counts"),
                     _side(values, (rows, m), f32, device, "values"), _side(index, (rows, m), i32, device, "index"),
                     _side(lse, one, f32, device, "lse"), _side(weight, one, f32, device, "weight"))
    return a, (counts, values, index, lse, weight)


_HELD = ("counts", "values", "index", "lse", "weight")


_OPERANDS = {"counts": (("rows",), torch.int32), "values": (("rows", "m"), torch.float32), "index": (("rows", "m"), torch.int32),
             "lse": (("rows",), torch.float32), "weight": (("rows",), torch.float32), "cand": (("rows", "width"), torch.int32),
             "cls": (("nodes",), torch.int32), "row_kind": (("rows",), torch.int32), "by_kind": (("rows",), torch.int32),
             "kind_start": ((), torch.int32)}


def _handed_back(a, names, tensors, device) -> list:
    """Saved operands where an argument block looks for them, and the tensors that must outlive the launch.  (Hooks on saved
    tensors may hand out copies, which are checked as the operands themselves were.)"""
    out = list(tensors)
    for i, (name, v) in enumerate(zip(names, tensors)):
        sizes, dtype = _OPERANDS[name]
        if v is not None and (v.data_ptr() != getattr(a, name) or v.dtype is not dtype or not v.is_contiguous()):
            out[i] = v.contiguous()
            shape = (a.kinds + 1,) if name == "kind_start" else tuple(getattr(a, n) for n in sizes)
            setattr(a, name, _side(out[i], shape, dtype, device, "saved " + name))
    return out


def _distill(device, a: _abi.Distill, loss, grad, upstream=None) -> None:
    _call("aig_distill_rows", device, C.byref(a), None if loss is None else loss.data_ptr(), None if grad is None else grad.data_ptr(),
          a.width, None if upstream is None else upstream.data_ptr(), 0 if upstream is None or upstream.numel() == 1 else 1,
          meta=(a.rows, a.width))


def _sum_rows(v: torch.Tensor) -> torch.Tensor:
    out = torch.empty((), dtype=torch.float32, device=v.device)
    need = _abi.lib().aig_sum_rows_ws_bytes(v.numel())
    ws = _abi.workspace(need, v.device) if need else None
    _call("aig_sum_rows", v.device, v.numel(), v.data_ptr(), 1.0, out.data_ptr(), None if ws is None else ws.data_ptr(), need)
    return out


def _refuse_recording(t: torch.Tensor, what: str, instead: str) -> None:
    """A recorded backward pass accumulates into its leaves on the stream that they were first used on; where an eager graph of
    the same leaves lives, that is not the recording's, and the runtime ends the process."""
    if t.requires_grad and torch.is_grad_enabled() and torch.cuda.is_current_stream_capturing():
        raise _abi.AigAbiError(f"{what} builds an autograd graph, which is not recorded into a HIP graph: record {instead}, which needs none")


def _check_backward(what: str) -> None:
    if torch.cuda.is_current_stream_capturing():
        raise _abi.AigAbiError(f"the backward pass of {what} is not recorded into a HIP graph")
    if torch.is_grad_enabled():        # (a backward pass runs with it on only when its own graph is asked for)
        raise RuntimeError(f"{what} can be differentiated once: call backward without create_graph")


def _save(ctx, tensors) -> None:
    """Operands for the backward pass.  (Torch refuses to save what was made in inference mode, as a teacher's rows may well
    be: that is kept beside.)"""
    ctx.beside = None
    for v in tensors:
        if v is not None and v.is_inference():
            ctx.beside = [v if v is not None and v.is_inference() else None for v in tensors]
            tensors = [v if b is None else None for v, b in zip(tensors, ctx.beside)]
            break
    ctx.save_for_backward(*tensors)


def _saved(ctx):
    return ctx.saved_tensors if ctx.beside is None else [v if b is None else b for v, b in zip(ctx.saved_tensors, ctx.beside)]


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, arg, held, reduce):
        loss = torch.empty(arg.rows, dtype=torch.float32, device=logits.device)
        if ctx.needs_input_grad[0] and arg.width > NARROW:
            ctx.stats = torch.empty((arg.rows, 8), dtype=torch.float32, device=logits.device)
            arg.stats = ctx.stats.data_ptr()
        _distill(logits.device, arg, loss, None)
        _save(ctx, (logits, *held))
        ctx.arg, ctx.stride, ctx.dtype = arg, logits.stride(), logits.dtype
        return _sum_rows(loss) if reduce else loss

    @staticmethod
    def backward(ctx, g):
        _check_backward("distill_loss")
        logits, *held = _saved(ctx)
        a = _abi.Distill.from_buffer_copy(ctx.arg)
        if logits.data_ptr() != a.logits or logits.stride() != ctx.stride or logits.dtype is not ctx.dtype:
            # (a hook's copy has strides of its own)
            logits = logits if logits.stride(1) == 1 else logits.contiguous()
            if logits.dtype is not ctx.dtype or logits.shape != (a.rows, a.width) or logits.device != g.device:
                raise _abi.AigAbiError(f"saved logits must be {ctx.dtype} {(a.rows, a.width)} on {g.device}, got {logits.dtype} "
                                       f"{tuple(logits.shape)} on {logits.device}")
            a.logits, a.ld = logits.data_ptr(), _rows_of(logits, "distill_loss")[2]
        held = _handed_back(a, _HELD, held, logits.device)
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        if g.dtype != torch.float32 or not g.is_contiguous():
            g = g.float().contiguous()
        _distill(logits.device, a, None, grad, g)
        return grad, None, None, None


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
    (float32 ``[rows]``), "sum" or "mean" (over the rows).  ``temperature`` is within 1e-6 and 1e6.  Differentiable once; into a
    HIP graph, record ``distill_loss_and_grad``."""
    if reduction not in ("none", "sum", "mean"):
        raise ValueError(f"reduction is 'none', 'sum' or 'mean', got {reduction!r}")
    rows = int(logits.size(0)) if torch.is_tensor(logits) and logits.dim() else 0
    if reduction == "mean" and rows == 0:
        raise ValueError("the mean over no rows")
    arg, held = _teacher(logits, top, counts, weight, temperature, tail, 1.0 / rows if reduction == "mean" else 1.0)
    _refuse_recording(logits, "distill_loss of logits that require a gradient", "distill_loss_and_grad")
    return _DistillLoss.apply(logits, arg, held, reduction != "none")


def distill_loss_and_grad(logits: torch.Tensor, top: TopRows, counts: Optional[torch.Tensor] = None,
                          weight: Optional[torch.Tensor] = None, temperature: float = 1.0,
                          tail: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """``distill_loss`` of every row (float32 ``[rows]``) and the gradient of their sum w.r.t. the logits (in the logits'
    type), in one pass over the logits and without an autograd graph: what a training step needs, and what a HIP graph
    can record.  A mean over rows, or any other weighting, goes into ``weight``."""
    arg, held = _teacher(logits, top, counts, weight, temperature, tail)
    loss = torch.empty(arg.rows, dtype=torch.float32, device=logits.device)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    _distill(logits.device, arg, loss, grad)
    return loss, grad


# ------------------------------------------------------------------ scores by class
def _windows_arg(like: torch.Tensor, kinds: int, classes: int, w: ScoreWindows) -> _abi.ScoreWindowsArg:
    if not torch.is_tensor(like) or not like.is_cuda:
        raise _abi.AigAbiError("class_scores needs its tensors on a HIP device (no CPU path exists)")
    if not torch.is_tensor(w.cand) or not torch.is_tensor(w.cls) or w.cand.dim() != 2 or w.cls.dim() != 1:
        raise _abi.AigAbiError("class_scores takes cand [rows, width] and cls [nodes]")
    (rows, width), (nodes,), device, i32 = w.cand.shape, w.cls.shape, like.device, torch.int32
    return _abi.ScoreWindowsArg(rows, width, nodes, kinds, classes, _side(w.cand, (rows, width), i32, device, "cand"),
                                _side(w.counts, (rows,), i32, device, "counts"), _side(w.cls, (nodes,), i32, device, "cls"),
                                _side(w.row_kind, (rows,), i32, device, "row_kind"), _side(w.by_kind, (rows,), i32, device, "by_kind"),
                                _side(w.kind_start, (kinds + 1,), i32, device, "kind_start"))


class _ClassScores(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, windows, a):
        out = torch.empty((a.rows, a.width), dtype=torch.float32, device=table.device)
        _call("aig_class_scores", table.device, C.byref(a), table.data_ptr(), out.data_ptr(), meta=(a.rows, a.width))
        _save(ctx, windows)
        ctx.arg = a
        return out

    @staticmethod
    def backward(ctx, g):
        _check_backward("class_scores")
        a = _abi.ScoreWindowsArg.from_buffer_copy(ctx.arg)
        held = _handed_back(a, ScoreWindows._fields, _saved(ctx), g.device)
        if g.dtype != torch.float32 or not g.is_contiguous():
            g = g.float().contiguous()
        return _table_grad(g, a), None, None


def _table_grad(g: torch.Tensor, a: _abi.ScoreWindowsArg) -> torch.Tensor:
    out = torch.empty((a.kinds, a.classes), dtype=torch.float32, device=g.device)
    need = _abi.lib().aig_class_scores_bwd_ws_bytes(a.rows, a.width, a.kinds, a.classes)
    ws = _abi.workspace(need, g.device)
    _call("aig_class_scores_bwd", g.device, C.byref(a), g.data_ptr(), out.data_ptr(), ws.data_ptr(), ws.numel(), meta=(a.rows, a.width))
    return out


def class_scores_grad(grad: torch.Tensor, windows: ScoreWindows, kinds: int, classes: int) -> torch.Tensor:
    """The gradient of ``class_scores``' table for a gradient of its output (float32 ``[rows, width]``): float32
    ``[kinds, classes]``, the sum over the rows of a kind and their places of a class - sums in a fixed order.  What of
    ``grad`` lies past a row's count is not read as a value."""
    a = _windows_arg(grad, kinds, classes, windows)
    _side(grad, (a.rows, a.width), torch.float32, windows.cand.device, "grad")
    return _table_grad(grad, a)


def class_scores(table: torch.Tensor, windows: ScoreWindows) -> torch.Tensor:
    """Logits ``[rows, width]`` looked up in ``table`` (float32 ``[kinds, classes]``) by the kind of the row and the class of
    the candidate, differentiable (once) in the table: nodes with equal feature rows score alike, so a template's candidate
    logits are a table of a few entries.  Places past a row's count, and candidates, classes or kinds outside their range,
    are ``-inf``."""
    if not torch.is_tensor(table) or not table.is_cuda:
        raise _abi.AigAbiError("class_scores needs the table on a HIP device (no CPU path exists)")
    if table.dim() != 2 or table.dtype != torch.float32 or not table.is_contiguous():
        raise _abi.AigAbiError(f"class_scores takes a contiguous float32 table [kinds, classes], got {table.dtype} {tuple(table.shape)}")
    _refuse_recording(table, "class_scores of a table that requires a gradient", "class_scores(table.detach()) and class_scores_grad")
    return _ClassScores.apply(table, windows, _windows_arg(table, int(table.size(0)), int(table.size(1)), windows))

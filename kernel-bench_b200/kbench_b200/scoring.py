"""What rows of log values say about their columns: log probabilities of given columns, entropy, the
best alternatives, and the gradient of these with respect to the rows.

The solver's rows are such rows: a root row holds, in log2 and up to a common factor, the probability
of the family's origin in every species column (the loss is minus its log-sum-exp), a clade row that
of the clade's placement.  Rows in nats (``base="e"``) and in 16-bit storage are taken as well.
There is no reference counterpart.

    loss, saved = runtime.run_forward(static, theta, col_weights)
    s = scoring.score_rows(saved["root_rows"], observed, top=5)
    cot = scoring.score_rows_backward(saved["root_rows"], s.stats, s.entropy, observed, grad_given=-w)
    grads = runtime.run_backward(static, theta, col_weights, saved, root_cotangent=cot)

:func:`score_rows` and :func:`score_rows_backward` enqueue one launch each on the current stream.
Impossible columns are -inf; a row of nothing else has log mass and log probabilities -inf, entropy 0
and gradient 0; a row with NaN or +inf scores NaN and has no alternatives (column -1).
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib

MAX_GIVEN = 32
MAX_TOP = 32
MAX_COLS = 1 << 30
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class RowScores(NamedTuple):
    """Per row, in units of the base's logarithm (bits or nats), fp32."""

    log_mass: torch.Tensor                  # [R] log of the row's sum
    entropy: torch.Tensor                   # [R]
    given_log_prob: Optional[torch.Tensor]  # as ``given``: log probability of each given column
    top_log_prob: Optional[torch.Tensor]    # [R, top], best first, -inf past the last column
    top_column: Optional[torch.Tensor]      # [R, top] int64, -1 past the last column
    stats: torch.Tensor                     # [R, 2]: largest entry and sum relative to it


def _natural(base) -> int:
    if base == 2 or base == "2":
        return 0
    if base == "e":
        return 1
    raise ValueError(f"base must be 2 or 'e' (got {base!r})")


def _check_rows(name: str, rows) -> torch.Tensor:
    if rows.device.type != "cuda":
        raise RuntimeError(f"{name} requires CUDA tensors")
    if rows.dtype not in _DTYPES:
        raise RuntimeError(f"{name} supports fp32, bf16 and fp16 rows only (got {rows.dtype})")
    if rows.ndim != 2:
        raise ValueError(f"rows must be [R, S] (got {tuple(rows.shape)})")
    if rows.shape[1] > MAX_COLS:  # the C entry point's length has 32 bits
        raise ValueError(f"at most {MAX_COLS} columns (got {rows.shape[1]})")
    return rows if rows.stride(1) == 1 or rows.shape[1] <= 1 else rows.contiguous()


def _check_given(given, rows):
    """``given`` as a contiguous int64 tensor and its columns a row."""
    if given is None:
        return None, 0
    if given.device != rows.device:
        raise RuntimeError("given must be on the rows' device")
    if given.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"given must be int64 or int32 (got {given.dtype})")
    if given.ndim not in (1, 2) or given.shape[0] != rows.shape[0]:
        raise ValueError(f"given must be [R] or [R, T] with R = {rows.shape[0]} (got {tuple(given.shape)})")
    n = 1 if given.ndim == 1 else int(given.shape[1])
    if n > MAX_GIVEN:
        raise ValueError(f"at most {MAX_GIVEN} given columns a row (got {n})")
    if given.dtype != torch.int64:
        given = given.to(torch.int64)
    return given.contiguous(), n


def _check_f32(name: str, t, shape, device):
    if t is None:
        return None
    if t.device != device:
        raise RuntimeError(f"{name} must be on the rows' device")
    if t.dtype != torch.float32:
        raise RuntimeError(f"{name} must be fp32 (got {t.dtype})")
    if t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)} (got {tuple(t.shape)})")
    return t if t.is_contiguous() else t.contiguous()


def score_rows(rows, given=None, *, top: int = 0, base=2) -> RowScores:
    """Scores of ``rows`` [R, S <= 2^30] (fp32, bf16 or fp16; any row stride), without an autograd graph.

    ``given`` int64 or int32 [R] or [R, T <= 32]: the columns whose log probabilities are asked for;
    one outside [0, S) stands for none and scores 0.  ``top`` <= 32: how many of the largest entries
    are listed (equal entries by the lower column)."""
    top = int(top)
    if 0 <= top <= MAX_TOP:  # the extension takes a C int
        out = _lib.call_host("score_rows", "kb_score_rows", rows.device, rows, given, top, _natural(base))
        if out is not None:
            return RowScores(*out)
    rows = _check_rows("score_rows", rows)
    if not 0 <= top <= MAX_TOP:
        raise ValueError(f"top must be in [0, {MAX_TOP}] (got {top})")
    natural = _natural(base)
    columns, n_given = _check_given(given, rows)
    R, S = rows.shape
    log_mass, entropy, given_lp, top_lp, top_column, stats = out = _lib.host().score_outputs(rows, given, top)
    _lib.call_on(rows.device, "kb_score_rows", rows.data_ptr(), rows.stride(0), _DTYPES[rows.dtype], R, S, natural,
                 _lib.ptr(columns), n_given, top, log_mass.data_ptr(), entropy.data_ptr(), _lib.ptr(given_lp),
                 _lib.ptr(top_lp), _lib.ptr(top_column), stats.data_ptr())
    return RowScores(*out)


def score_rows_backward(rows, stats, entropy, given=None, *, grad_log_mass=None, grad_given=None, grad_entropy=None,
                        base=2, out=None):
    """Gradient of :func:`score_rows` with respect to ``rows``, in their dtype.

    ``stats`` [R, 2] and ``entropy`` [R] (needed with ``grad_entropy`` alone) are the forward's;
    ``grad_log_mass`` [R], ``grad_given`` (shaped as ``given``) and ``grad_entropy`` [R] the cotangents
    (``None``: zero).  To differentiate listed alternatives pass their columns as ``given``.  The
    gradient is 0 at impossible columns.  ``out``: a buffer [R, S] to write to, whose address range does not
    meet that of ``rows``."""
    natural = _natural(base)
    got = _lib.call_host("score_rows_backward", "kb_score_rows_backward", rows.device, rows, stats, entropy, given,
                         grad_log_mass, grad_given, grad_entropy, natural, out)
    if got is not None:
        return got
    rows = _check_rows("score_rows_backward", rows)
    R, S = rows.shape
    dev = rows.device
    stats = _check_f32("stats", stats, (R, 2), dev)
    if stats is None:
        raise ValueError("stats is needed (score_rows(...).stats)")
    entropy = _check_f32("entropy", entropy, (R,), dev)
    if grad_entropy is not None and entropy is None:
        raise ValueError("grad_entropy needs the forward's entropy")
    if grad_given is not None and given is None:
        raise ValueError("grad_given needs the given columns")
    columns, n_given = _check_given(given, rows)
    grad_log_mass = _check_f32("grad_log_mass", grad_log_mass, (R,), dev)
    grad_given = _check_f32("grad_given", grad_given, None if given is None else given.shape, dev)
    grad_entropy = _check_f32("grad_entropy", grad_entropy, (R,), dev)
    if out is None:
        out = torch.empty((R, S), device=dev, dtype=rows.dtype)
    elif out.device != dev or out.dtype != rows.dtype:
        raise RuntimeError("out must have the rows' device and dtype")
    elif out.shape != rows.shape or (S > 1 and out.stride(1) != 1) or (R > 1 and out.stride(0) < S):
        raise ValueError("out must be [R, S] with unit column stride and rows that do not overlap")
    elif _overlap(out, rows):
        raise ValueError("out must not overlap rows")
    _lib.call_on(dev, "kb_score_rows_backward", rows.data_ptr(), rows.stride(0), _DTYPES[rows.dtype], R, S, natural,
                 stats.data_ptr(), _lib.ptr(entropy), _lib.ptr(columns), n_given, _lib.ptr(grad_log_mass),
                 _lib.ptr(grad_given), _lib.ptr(grad_entropy), out.data_ptr(), out.stride(0))
    _lib.host().written([out])
    return out


def _overlap(a, b) -> bool:
    """Whether the address ranges of two row matrices meet (storages do not tell: one imported by another
    library's view of the same memory starts elsewhere)."""
    def span(t):
        if t.numel() == 0:
            return 0, 0
        last = (t.shape[0] - 1) * t.stride(0) + t.shape[1]
        return t.data_ptr(), t.data_ptr() + last * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1

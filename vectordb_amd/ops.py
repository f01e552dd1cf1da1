"""Operators on row tables and score rows: torch tensors on the GPU, through the C ABI of libvdbcore.so.

A table is a matrix of rows: a model's embeddings, or the vectors of a collection (a ``RowStore`` keeps its rows on the
device and can be looked up in directly).  A score row holds one value for every row of a table: the logits of a
position, or a query's distances.

    lookup, lookup_grad                    rows by number, scaled, and the gradient of the table
    distill, distill_grad, distill_step    a score row's divergence from a teacher's top scores, its gradient, both at once
    sample                                 one row number drawn from each score row

The reference has no counterpart.  The teacher's lists and the row numbers have the form of a search result: (score,
row) slots with row -1 where there is nothing.  Scores are better the larger they are, so a search's distances are negated for a
teacher's list; ``sample`` takes distances as they are with ``distances=True``.  Its filters are the packed row masks of searches.

Every function enqueues on the current torch stream and returns without waiting; inputs made on another stream have to
be ordered by the caller, as for any torch operation.  Nothing is allocated but the outputs (or none, with ``out=``) and a
workspace from torch's allocator, so the calls can be captured into a graph.  Autograd does not record them: gradients are
the functions named ``*_grad``, which a ``torch.autograd.Function`` calls, and a tensor that requires a gradient is refused
where gradients are recorded (so call them under ``torch.no_grad()`` or in such a function).  An ``out`` shares no memory with the
inputs but where it is said; writing to it counts as an in-place change of that tensor.  Values are float32, bfloat16 or float16, sums
are taken in 32 bits or more, and equal inputs give equal bits.  Arguments that do not fit raise ``ValueError``.  Tensors lie on the
library's device, which every call makes the current one of its thread.
"""

from __future__ import annotations

import ctypes as C
import functools
from typing import Optional, Tuple, Union

import torch

from . import _native

VALUE_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

# What a call needs of the library and the device, looked up once: small calls are bound by what happens on the host.
_lib = None
_device_no = -1
_where: Optional[torch.device] = None


def _fail(text: str):
    raise ValueError(text)


def _start() -> None:
    global _lib, _device_no, _where
    _native.init()
    _device_no = _native.current_device() or 0
    _where = torch.device("cuda", _device_no)
    _lib = _native.load()


def _on_gpu(t, what: str) -> None:
    if not isinstance(t, torch.Tensor):
        _fail(f"{what} must be a torch tensor, got {type(t).__name__}")
    if t.requires_grad and torch.is_grad_enabled():
        _fail(f"{what} requires a gradient, which this call would not record: call it under torch.no_grad() or in a torch.autograd.Function, "
              f"with the *_grad functions for the gradients")
    if _lib is None or t.get_device() != _device_no:
        if not t.is_cuda:
            _fail(f"{what} must be on the GPU, it is on {t.device}")
        if _lib is None:
            _start()
        if t.get_device() != _device_no:
            _fail(f"{what} must be on GPU {_device_no}, the library's device; it is on {t.device}")


def _matrix(t, what: str) -> Tuple[int, int, int, int]:
    """(value type, rows, columns, leading dimension) of a matrix whose rows are contiguous."""
    _on_gpu(t, what)
    code = VALUE_TYPES.get(t.dtype)
    if code is None:
        _fail(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")
    if t.dim() != 2:
        _fail(f"{what} must have two dimensions, got shape {tuple(t.shape)}")
    n, d = t.shape
    ld, step = t.stride()
    if step != 1 and d > 1 and n > 0:
        _fail(f"the rows of {what} must be contiguous, its strides are {t.stride()}")
    return code, n, d, ld if n > 1 else d


def _vector(t, what: str, n: int, dtype: torch.dtype) -> None:
    _on_gpu(t, what)
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        _fail(f"{what} must be a contiguous {dtype} vector of {n}, got {t.dtype} of shape {tuple(t.shape)}, strides {t.stride()}")


def _row_numbers(t, what: str) -> torch.Tensor:
    _on_gpu(t, what)
    if t.dtype != torch.int64 or not t.is_contiguous():
        _fail(f"{what} must be contiguous int64 row numbers, got {t.dtype} of shape {tuple(t.shape)}, strides {t.stride()}")
    return t


def _output(out, what: str, shape, dtype: torch.dtype) -> torch.Tensor:
    """A new contiguous output, or the caller's, whose rows must not share memory."""
    if out is None:
        return torch.empty(shape, device=_where, dtype=dtype)
    _on_gpu(out, what)
    if out.dtype != dtype or tuple(out.shape) != tuple(shape):
        _fail(f"{what} must be {dtype} of shape {tuple(shape)}, got {out.dtype} of shape {tuple(out.shape)}")
    if out.dim() == 2 and out.numel() > 0 and ((out.shape[1] > 1 and out.stride(1) != 1) or (out.shape[0] > 1 and out.stride(0) < out.shape[1])):
        _fail(f"the rows of {what} must be contiguous and apart, its strides are {out.stride()}")
    return out


def _written(given: Optional[torch.Tensor]) -> None:
    """What was written to a caller's tensor is seen by autograd, which may have kept it for a backward pass."""
    if given is not None:
        torch.autograd.graph.increment_version(given)


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _stream() -> int:
    return torch.cuda.current_stream(_device_no).cuda_stream


_current_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
if _current_raw_stream is not None:
    def _stream() -> int:                                   # noqa: F811 - the same number without a Stream object around it
        return _current_raw_stream(_device_no)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(fn: str, *sizes) -> int:
    need = C.c_int64(0)
    _native.check(getattr(_native.load(), fn)(*sizes, C.byref(need)))
    return need.value


def _workspace(fn: str, *sizes):
    """(tensor that holds the workspace, its address, its size); the tensor may be dropped once the call is enqueued."""
    need = _workspace_bytes(fn, *sizes)
    if not need:
        return None, None, 0
    t = torch.empty(need, device=_where, dtype=torch.uint8)
    return t, t.data_ptr(), need


# ---------------------------------------------------------------- lookup
def lookup(table: Union[torch.Tensor, "_native.RowStore"], rows: torch.Tensor, scale: float = 1.0, dtype: Optional[torch.dtype] = None,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``scale * table[rows]``, shape ``rows.shape + (dim,)``, in ``dtype`` (the table's unless given; a store's rows come
    as float32).  A row number outside the table, such as the -1 of an unfilled result slot, gives a row of zeros."""
    rows = _row_numbers(rows, "rows")
    n = rows.numel()
    store = table if isinstance(table, _native.RowStore) else None
    if store is not None:
        dim, natural = store.dim, torch.float32
    else:
        code, n_rows, dim, ld = _matrix(table, "table")
        natural = table.dtype
        if dim < 1:
            _fail("the rows of table must have at least one value")
    dtype = dtype or (out.dtype if out is not None else natural)
    if dtype not in VALUE_TYPES:
        _fail(f"dtype must be float32, bfloat16 or float16, got {dtype}")
    shape = tuple(rows.shape) + (dim,)
    given, out = out, _output(out, "out", shape, dtype)
    if out.dim() != 2 and not out.is_contiguous():
        _fail("out must be contiguous unless rows is a vector")
    ld_out = out.stride(0) if out.dim() == 2 and n > 1 else dim
    if store is not None:
        _native.check(_lib.vdb_rows_lookup_dev(store.h, _p(rows), n, scale, _p(out), VALUE_TYPES[dtype], ld_out, _stream()))
    else:
        _native.check(_lib.vdb_lookup_dev(_p(table), code, n_rows, dim, ld, _p(rows), n, scale, _p(out), VALUE_TYPES[dtype], ld_out, _stream()))
    _written(given)
    return out


def lookup_grad(grad: torch.Tensor, rows: torch.Tensor, n_rows: int, scale: float = 1.0, dtype: Optional[torch.dtype] = None,
                out: Optional[torch.Tensor] = None, accumulate: bool = False) -> torch.Tensor:
    """Gradient of the table of a ``lookup``: ``out[r] = scale * sum of grad[i] with rows[i] == r``, shape ``(n_rows, dim)``, in
    ``dtype`` (``grad``'s unless given).  ``grad`` has the shape of the lookup's result.  ``accumulate`` adds to ``out`` and touches
    the named rows alone.  Row numbers outside the table contribute nothing."""
    rows = _row_numbers(rows, "rows")
    n = rows.numel()
    if not isinstance(grad, torch.Tensor) or grad.dim() != rows.dim() + 1 or tuple(grad.shape[:-1]) != tuple(rows.shape):
        _fail(f"grad must have the shape {tuple(rows.shape)} + (dim,), got {tuple(getattr(grad, 'shape', ()))}")
    if grad.dim() != 2:
        if not grad.is_contiguous():
            _fail("grad must be contiguous unless rows is a vector")
        grad = grad.view(n, grad.shape[-1])
    code, _, dim, ld = _matrix(grad, "grad")
    if dim < 1 or n_rows < 0:
        _fail(f"bad sizes for a lookup gradient: {n_rows} rows of {dim} values")
    if accumulate and out is None:
        _fail("accumulate needs the tensor to add to (out)")
    dtype = dtype or (out.dtype if out is not None else grad.dtype)
    if dtype not in VALUE_TYPES:
        _fail(f"dtype must be float32, bfloat16 or float16, got {dtype}")
    given, out = out, _output(out, "out", (n_rows, dim), dtype)
    keep, work, size = _workspace("vdb_lookup_grad_workspace", n, n_rows, dim)
    _native.check(_lib.vdb_lookup_grad_dev(_p(grad), code, ld, _p(rows), n, scale, _p(out), VALUE_TYPES[dtype], n_rows, dim,
                                                     out.stride(0) if n_rows > 1 else dim, int(accumulate), work, size, _stream()))
    _written(given)
    return out


# ---------------------------------------------------------------- distillation
def _distill_args(scores, teacher, rows, temperature, teacher_lse):
    code, n, vocab, ld = _matrix(scores, "scores")
    if vocab < 1:
        _fail("a score row must have at least one value")
    _on_gpu(teacher, "teacher")
    _on_gpu(rows, "rows")
    if teacher.dtype != torch.float32 or rows.dtype != torch.int64:
        _fail(f"teacher must be float32 and rows int64, got {teacher.dtype} and {rows.dtype}")
    if teacher.dim() != 2 or teacher.shape[0] != n or teacher.shape != rows.shape:
        _fail(f"teacher and rows must have the shape ({n}, k), got {tuple(teacher.shape)} and {tuple(rows.shape)}")
    k = teacher.shape[1]
    for t, what in ((teacher, "teacher"), (rows, "rows")):
        if k > 1 and n > 0 and t.stride(1) != 1:
            _fail(f"the lists of {what} must be contiguous, its strides are {t.stride()}")
    if teacher_lse is not None:
        _vector(teacher_lse, "teacher_lse", n, torch.float32)
    return (_p(scores), code, n, vocab, ld, _p(teacher), _p(rows), k, teacher.stride(0) if n > 1 else k, rows.stride(0) if n > 1 else k,
            _p(teacher_lse), float(temperature))


def distill(scores: torch.Tensor, teacher: torch.Tensor, rows: torch.Tensor, temperature: float = 1.0,
            teacher_lse: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Divergence of every score row from the teacher's k best scores of it -> (loss [n], stats [n, 2]).

    ``teacher`` [n, k] float32 are the teacher's scores, ``rows`` [n, k] int64 the places they belong to (outside the row: unfilled).
    With tau = ``temperature``, q = softmax(scores / tau) and p = softmax of a row's filled slots / tau, or
    exp(teacher / tau - teacher_lse) where the log-sum-exp over the teacher's whole row is given:
    ``loss = tau^2 * sum_j p_j (log p_j - log q[rows_j])``.  A row without filled slots has loss 0.  ``stats`` is what
    ``distill_grad`` needs of this pass.  A search's distances go in negated.  The logarithms are float32: of a loss that a large
    temperature makes a small difference of them, times tau^2, less is left."""
    args = _distill_args(scores, teacher, rows, temperature, teacher_lse)
    n, vocab = scores.shape
    loss = torch.empty(n, device=_where, dtype=torch.float32)
    stats = torch.empty((n, 2), device=_where, dtype=torch.float32)
    keep, work, size = _workspace("vdb_distill_workspace", n, vocab)
    _native.check(_lib.vdb_distill_dev(*args, _p(loss), _p(stats), work, size, _stream()))
    return loss, stats


def distill_grad(scores: torch.Tensor, teacher: torch.Tensor, rows: torch.Tensor, stats: torch.Tensor, grad_loss: torch.Tensor,
                 temperature: float = 1.0, teacher_lse: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of ``sum(grad_loss * loss)`` of ``distill`` for the scores, in their type.  ``out`` may be ``scores`` itself; rows whose
    ``grad_loss`` is 0 get zeros whatever they hold."""
    args = _distill_args(scores, teacher, rows, temperature, teacher_lse)
    n, vocab = scores.shape
    _on_gpu(stats, "stats")
    if stats.dtype != torch.float32 or tuple(stats.shape) != (n, 2) or not stats.is_contiguous():
        _fail(f"stats must be contiguous float32 of shape ({n}, 2), got {stats.dtype} of shape {tuple(stats.shape)}")
    _vector(grad_loss, "grad_loss", n, torch.float32)
    given, out = out, _output(out, "out", (n, vocab), scores.dtype)
    _native.check(_lib.vdb_distill_grad_dev(*args, _p(stats), _p(grad_loss), _p(out), out.stride(0) if n > 1 else vocab, _stream()))
    _written(given)
    return out


def distill_step(scores: torch.Tensor, teacher: torch.Tensor, rows: torch.Tensor, grad_loss: torch.Tensor, temperature: float = 1.0,
                 teacher_lse: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``distill`` and ``distill_grad`` in one call, for weights ``grad_loss`` [n] that are known beforehand -> (loss [n], gradient)."""
    args = _distill_args(scores, teacher, rows, temperature, teacher_lse)
    n, vocab = scores.shape
    _vector(grad_loss, "grad_loss", n, torch.float32)
    loss = torch.empty(n, device=_where, dtype=torch.float32)
    given, out = out, _output(out, "out", (n, vocab), scores.dtype)
    keep, work, size = _workspace("vdb_distill_workspace", n, vocab)
    _native.check(_lib.vdb_distill_step_dev(*args, _p(grad_loss), _p(loss), None, _p(out), out.stride(0) if n > 1 else vocab,
                                                      work, size, _stream()))
    _written(given)
    return loss, out


# ---------------------------------------------------------------- sampling
def sample(scores: torch.Tensor, uniforms: torch.Tensor, temperature: Union[float, torch.Tensor] = 1.0,
           top_k: Union[None, int, torch.Tensor] = None, top_p: Union[None, float, torch.Tensor] = None,
           min_p: Union[None, float, torch.Tensor] = None, mask_words: Optional[torch.Tensor] = None,
           distances: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """One row number drawn from each score row -> (rows [n] int64, log-probabilities [n] float32).

    The settings are one value for all rows or a vector [n] (float32; ``top_k`` int32), applied in this order:
    ``temperature`` (0 = the best row), ``top_k`` (0 or None = off), ``top_p`` (1 or None = off) of what that leaves, ``min_p`` (0 or
    None = off) relative to the best row.  The draw is the first remaining row, in ascending row number, at which the running
    sum of the probabilities exceeds ``uniforms`` [n] (float32 in [0, 1)).  Equal scores rank by row number.
    ``mask_words``: packed row filter, int32 or uint32 words, one per row of ``scores`` or one for all; rows whose bit is 0, scores of
    -inf and NaN are never drawn.  ``distances``: smaller scores are better.  Where nothing can be drawn: (-1, -inf).

    Weights exp((score - best) / temperature) below 2^-40 count as nothing, and the others are summed as multiples of 2^-s, s =
    min(52, 62 - ceil(log2 of the row's length)): sums are exact, and a border or a draw is that of weights which are off by at most
    2^-(s+1) each (2^-46 at 131072 scores).  The log-probability is of the drawn row's own weight, not rounded."""
    code, n, vocab, ld = _matrix(scores, "scores")
    if vocab < 1:
        _fail("a score row must have at least one value")
    _vector(uniforms, "uniforms", n, torch.float32)

    def setting(v, what, off, dtype):
        if v is None:
            return None, off
        if isinstance(v, torch.Tensor):
            _vector(v, what, n, dtype)
            return _p(v), off
        if isinstance(v, bool) or not isinstance(v, (int, float)) or (dtype == torch.int32 and not isinstance(v, int)):
            _fail(f"{what} must be a number or a vector of {n}, got {v!r}")
        if dtype == torch.int32:
            return None, max(0, min(int(v), 2 ** 31 - 1))
        return None, float(v)

    t, tv = setting(temperature, "temperature", 1.0, torch.float32)
    k, kv = setting(top_k, "top_k", 0, torch.int32)
    p, pv = setting(top_p, "top_p", 1.0, torch.float32)
    m, mv = setting(min_p, "min_p", 0.0, torch.float32)
    mask_ld = 0
    if mask_words is not None:
        _on_gpu(mask_words, "mask_words")
        words = (vocab + 31) // 32
        ok = mask_words.element_size() == 4 and not mask_words.is_floating_point() and mask_words.dim() in (1, 2)
        ok = ok and mask_words.shape[-1] >= words and (mask_words.shape[-1] == 1 or mask_words.stride(-1) == 1)
        if not ok or (mask_words.dim() == 2 and mask_words.shape[0] != n):
            _fail(f"a filter over {vocab} scores takes {words} contiguous 32-bit words, for all rows or for each of {n}; got "
                  f"{mask_words.dtype} of shape {tuple(mask_words.shape)}")
        mask_ld = mask_words.stride(0) if mask_words.dim() == 2 and n > 1 else 0
    out = torch.empty(n, device=_where, dtype=torch.int64)
    logp = torch.empty(n, device=_where, dtype=torch.float32)
    # short rows with a top-k need none
    keep, work, size = (None, None, 0) if vocab <= 32768 and (k is not None or kv > 0) else _workspace("vdb_sample_workspace", n, vocab)
    _native.check(_lib.vdb_sample_dev(_p(scores), code, n, vocab, ld, int(distances), _p(uniforms), t, tv, k, kv, p, pv, m, mv,
                                                _p(mask_words), mask_ld, _p(out), _p(logp), work, size, _stream()))
    return out, logp

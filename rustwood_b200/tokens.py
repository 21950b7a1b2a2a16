"""Token operators on torch CUDA tensors (the rw_*_device token calls of include/rwgpu.h):

  embed, embed_grad            embedding lookup with scaling; its gradient by sorted ids
  dropout                      from a counter-based generator; its own gradient
  logprobs, logprobs_grad      log-probabilities of given classes, entropy and the top
                               alternatives from margins; their gradient

Every call takes a Context and tensors on its GPU, works on torch's current stream there
without synchronising, and can be captured into a CUDA graph. Element types are float32,
bfloat16 and float16; ids and targets int32 or int64. Inputs may have any strides (rows
that are not contiguous are copied first); an `out` tensor has to be usable in place. The
gradients are explicit calls: autograd does not see through these functions.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import NamedTuple, Optional

import torch

from . import _native as N
from .booster import Context

__all__ = ["LogProbs", "embed", "embed_grad", "dropout", "logprobs", "logprobs_grad"]

_ELEM = {torch.float32: N.RW_F32, torch.bfloat16: N.RW_BF16, torch.float16: N.RW_F16}
_MASK64 = (1 << 64) - 1
_INDEX = {torch.int32: N.RW_I32, torch.int64: N.RW_I64}


def _elem(what: str, dtype: torch.dtype) -> int:
    t = _ELEM.get(dtype)
    if t is None:
        raise TypeError(f"{what} is {dtype}: float32, bfloat16 or float16 is needed")
    return t


def _on_gpu(ctx: Context, what: str, t: torch.Tensor) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} is not a torch tensor")
    if t.get_device() != ctx.gpu:
        raise ValueError(f"{what} is on {t.device}, the context on cuda:{ctx.gpu}")
    return t


def _usable(t: torch.Tensor) -> bool:
    """Whether a 2-D tensor's rows are contiguous and do not overlap."""
    rows, cols = t.shape
    return (cols <= 1 or t.stride(1) == 1) and (rows <= 1 or t.stride(0) >= max(cols, 1))


def _matrix(ctx: Context, what: str, t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """t as [rows][last dimension] with contiguous rows, and their distance."""
    _on_gpu(ctx, what, t)
    if t.dim() != 2:
        if t.dim() == 0:
            raise ValueError(f"{what} has no dimension")
        t = t.reshape(_rows_of(t), t.shape[-1])
    if t.is_contiguous():
        return t, t.shape[1]
    if not _usable(t):
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _rows_of(t: torch.Tensor) -> int:
    return t.numel() // t.shape[-1] if t.shape[-1] else t.shape[:-1].numel()


def _vector(ctx: Context, what: str, t: torch.Tensor, n: int, dtype=None) -> torch.Tensor:
    _on_gpu(ctx, what, t)
    if t.numel() != n:
        raise ValueError(f"{what} has {t.numel()} elements: {n} are needed")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{what} is {t.dtype}: {dtype} is needed")
    return t if t.is_contiguous() else t.contiguous()


def _index(ctx: Context, what: str, t: torch.Tensor, n: Optional[int] = None) -> tuple[torch.Tensor, int]:
    kind = _INDEX.get(t.dtype) if isinstance(t, torch.Tensor) else None
    if kind is None:
        raise TypeError(f"{what} is not an int32 or int64 tensor")
    return _vector(ctx, what, t, t.numel() if n is None else n), kind


def _output(ctx: Context, out: Optional[torch.Tensor], shape, dtype: torch.dtype,
            device: torch.device) -> tuple[torch.Tensor, int]:
    """The output tensor and the distance of its rows."""
    if out is None:
        return torch.empty(*shape, dtype=dtype, device=device), shape[-1]
    _on_gpu(ctx, "out", out)
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype:
        raise ValueError(f"out is {tuple(out.shape)} {out.dtype}: {tuple(shape)} {dtype} is needed")
    if out.is_contiguous():
        return out, shape[-1]
    if out.dim() != 2 or not _usable(out):
        raise ValueError("out has rows that are not contiguous")
    return out, out.stride(0) if out.shape[0] > 1 else out.shape[1]


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


# the handle of torch's current stream on a device, without a Stream object around it
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda gpu: torch.cuda.current_stream(gpu).cuda_stream)


@functools.lru_cache(maxsize=256)
def _bytes_needed(query: str, *sizes: int) -> int:
    """A workspace query's answer, which depends on the sizes alone."""
    need = C.c_uint64()
    N.check(getattr(N.lib, query)(None, *sizes, C.byref(need)))
    return need.value


def embed(ctx: Context, table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0,
          dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """scale * table[ids], rounded once to dtype (the table's unless given): [*ids.shape, d].
    An id outside the table gives a row of zeros."""
    if isinstance(table, torch.Tensor) and table.dim() != 2:
        raise ValueError("table is not [vocab][d]")
    table, ld = _matrix(ctx, "table", table)
    flat, kind = _index(ctx, "ids", ids)
    vocab, d = table.shape
    dtype = dtype or (out.dtype if out is not None else table.dtype)
    table_type, out_type = _elem("table", table.dtype), _elem("dtype", dtype)
    out, out_ld = _output(ctx, out, (*ids.shape, d), dtype, table.device)
    ctx.check(N.lib.rw_embed_device(ctx.h, table.data_ptr(), table_type, vocab, ld, flat.data_ptr(),
                                    kind, flat.numel(), d, scale, out.data_ptr(), out_type, out_ld,
                                    _stream(ctx.gpu)))
    return out


def embed_grad(ctx: Context, grad: torch.Tensor, ids: torch.Tensor, vocab: int,
               scale: float = 1.0, dtype: Optional[torch.dtype] = None,
               out: Optional[torch.Tensor] = None, accumulate: bool = False) -> torch.Tensor:
    """The gradient of embed with respect to its table, from grad [*ids.shape, d]: row v is
    scale times the sum of grad's rows whose id is v. [vocab, d] in dtype (float32 unless
    given). With accumulate, the sums are added to `out` and its other rows stay as they
    are. The sums do not depend on timing: the same inputs give the same bits."""
    grad, ld = _matrix(ctx, "grad", grad)
    n, d = grad.shape
    flat, kind = _index(ctx, "ids", ids, n)
    if accumulate and out is None:
        raise ValueError("accumulate needs out")
    dtype = dtype or (out.dtype if out is not None else torch.float32)
    grad_type, out_type = _elem("grad", grad.dtype), _elem("dtype", dtype)
    out, out_ld = _output(ctx, out, (vocab, d), dtype, grad.device)
    need = _bytes_needed("rw_embed_grad_workspace", n, d, vocab)
    ws = torch.empty(need, dtype=torch.uint8, device=grad.device)
    ctx.check(N.lib.rw_embed_grad_device(ctx.h, grad.data_ptr(), grad_type, ld, flat.data_ptr(), kind,
                                         n, d, vocab, scale, accumulate, out.data_ptr(), out_type,
                                         out_ld, ws.data_ptr(), need, _stream(ctx.gpu)))
    return out


def dropout(ctx: Context, x: torch.Tensor, p: float, seed: int, sequence: int = 0,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x / (1 - p) where kept and 0 elsewhere, p rounded to a multiple of 2^-16. What is kept
    depends on (seed, sequence), each 64 bits, and an element's index in x (row-major): the
    same call on the gradient is the gradient. out may be x."""
    rows, ld = _matrix(ctx, "x", x)
    kind = _elem("x", rows.dtype)
    out, out_ld = _output(ctx, out, x.shape, rows.dtype, rows.device)
    n, d = rows.shape
    ctx.check(N.lib.rw_dropout_device(ctx.h, rows.data_ptr(), kind, n, d, ld, p, seed & _MASK64,
                                      sequence & _MASK64, out.data_ptr(), out_ld, _stream(ctx.gpu)))
    return out


class LogProbs(NamedTuple):
    """Per row of margins (all float32, top_index int64); see rw_logprobs_device."""
    row_max: torch.Tensor
    log_sum: torch.Tensor
    lse: torch.Tensor               # scale * row_max + log_sum
    logp: Optional[torch.Tensor]    # of the targets; None without targets
    entropy: torch.Tensor
    top_logp: torch.Tensor          # [..., top_k]
    top_index: torch.Tensor         # [..., top_k]


def logprobs(ctx: Context, x: torch.Tensor, targets: Optional[torch.Tensor] = None,
             scale: float = 1.0, top_k: int = 0) -> LogProbs:
    """Log-probabilities of the targets, entropy and the top_k <= 32 most likely classes of
    softmax(scale * x) over the last dimension, in one pass over x."""
    rows, ld = _matrix(ctx, "x", x)
    kind = _elem("x", rows.dtype)
    n, classes = rows.shape
    shape, device = x.shape[:-1], rows.device
    t, target_kind = (None, N.RW_I64) if targets is None else _index(ctx, "targets", targets, n)
    need = _bytes_needed("rw_logprobs_workspace", n, classes, kind, top_k)
    row = torch.empty(5, *shape, dtype=torch.float32, device=device)
    top_logp = torch.empty(*shape, top_k, dtype=torch.float32, device=device)
    top_index = torch.empty(*shape, top_k, dtype=torch.int64, device=device)
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    at, step = row.data_ptr(), 4 * n
    ctx.check(N.lib.rw_logprobs_device(
        ctx.h, rows.data_ptr(), kind, n, classes, ld, scale, _ptr(t), target_kind, top_k, at, at + step,
        at + 2 * step, None if t is None else at + 3 * step, at + 4 * step, top_logp.data_ptr(),
        top_index.data_ptr(), _ptr(ws), need, _stream(ctx.gpu)))
    row_max, log_sum, lse, logp, entropy = row.unbind(0)
    return LogProbs(row_max, log_sum, lse, None if t is None else logp, entropy, top_logp, top_index)


def logprobs_grad(ctx: Context, x: torch.Tensor, targets: Optional[torch.Tensor],
                  row_max: torch.Tensor, log_sum: torch.Tensor, entropy: Optional[torch.Tensor],
                  grad_logp: Optional[torch.Tensor], grad_entropy: Optional[torch.Tensor] = None,
                  scale: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient with respect to x of sum(grad_logp * logp + grad_entropy * entropy), from
    logprobs' row_max, log_sum and entropy of the same x and scale; either gradient may be
    None. In x's type and shape; out may be x."""
    rows, ld = _matrix(ctx, "x", x)
    kind = _elem("x", rows.dtype)
    n, classes = rows.shape
    row_max = _vector(ctx, "row_max", row_max, n, torch.float32)
    log_sum = _vector(ctx, "log_sum", log_sum, n, torch.float32)
    t = g = e = h = None
    target_kind = N.RW_I64
    if grad_logp is not None:
        if targets is None:
            raise ValueError("grad_logp needs targets")
        t, target_kind = _index(ctx, "targets", targets, n)
        g = _vector(ctx, "grad_logp", grad_logp, n, torch.float32)
    if grad_entropy is not None:
        if entropy is None:
            raise ValueError("grad_entropy needs entropy")
        e = _vector(ctx, "grad_entropy", grad_entropy, n, torch.float32)
        h = _vector(ctx, "entropy", entropy, n, torch.float32)
    out, out_ld = _output(ctx, out, x.shape, rows.dtype, rows.device)
    ctx.check(N.lib.rw_logprobs_grad_device(
        ctx.h, rows.data_ptr(), kind, n, classes, ld, scale, _ptr(t), target_kind, row_max.data_ptr(),
        log_sum.data_ptr(), _ptr(h), _ptr(g), _ptr(e), out.data_ptr(), out_ld, _stream(ctx.gpu)))
    return out

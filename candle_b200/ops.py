"""Front ends with the names, argument meaning and error behaviour of candle's own.

``rms_norm`` / ``layer_norm`` mirror ``candle_nn::ops::{rms_norm, layer_norm}``
(candle-nn/src/ops.rs:641-652, 896-909) plus the checks their ``cuda_fwd`` performs
(:536-543, 770-781); ``index_select`` mirrors ``Tensor::index_select``
(candle-core/src/tensor.rs:1568-1589).  The optional ``residual`` argument fuses the
``(x + residual)?`` the models compute just before the norm
(candle-transformers/src/models/llama.rs:446-450, bert.rs:301).
"""
from __future__ import annotations

import ctypes
import struct
from functools import lru_cache

import torch

from . import _cabi
from ._cabi import FLAG_FAST_SUM, FLAG_FORCE_GENERIC, FLAG_FORCE_LANEROW, FLAG_FORCE_REPLAY  # noqa: F401
from .errors import CandleError, InvalidIndex

_DTYPES = {torch.float32: _cabi.DTYPE_F32, torch.float16: _cabi.DTYPE_F16, torch.bfloat16: _cabi.DTYPE_BF16}
_DTYPE_NAMES = {torch.float32: "F32", torch.float16: "F16", torch.bfloat16: "BF16"}
_ID_DTYPES = {
    torch.uint8: _cabi.ID_U8,
    torch.uint32: _cabi.ID_U32,
    torch.int32: _cabi.ID_U32,  # the bit pattern is read as u32: negative values fail the bounds check
    torch.int64: _cabi.ID_I64,
}


def _dims(t: torch.Tensor) -> str:
    return str(list(t.shape))


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _stream(t: torch.Tensor):
    return torch.cuda.current_stream(t.device).cuda_stream


def _same_device(*ts: torch.Tensor) -> None:
    first = ts[0]
    if not first.is_cuda:
        raise CandleError("candle_b200 runs on Device::Cuda only: there is no CPU fallback")
    for t in ts[1:]:
        if t is not None and t.device != first.device:
            raise CandleError(f"device mismatch in op, lhs: {first.device}, rhs: {t.device}")


def new_status(device) -> torch.Tensor:
    """A zeroed ``cb200_status`` record (4 x int64 = 32 bytes) in device memory."""
    return torch.zeros(4, dtype=torch.int64, device=device)


def raise_for_status(status: torch.Tensor, op: str = "index-select") -> None:
    """Synchronises on the status record and raises what candle's CPU backend would have raised."""
    code_word, position, index, size = status.cpu().tolist()
    code = code_word & 0xFFFFFFFF
    if code == _cabi.STATUS_INVALID_INDEX:
        raise InvalidIndex(index & (2**64 - 1), size, op, position)
    if code == _cabi.STATUS_WAIT_TIMEOUT:
        raise CandleError(f"device-side wait timed out at row {position} in {op}")


def _norm_checks(name: str, xs: torch.Tensor, params: list[tuple[str, torch.Tensor]], residual):
    if xs.dtype not in _DTYPES or any(p.dtype != xs.dtype for _, p in params):
        raise CandleError(f"unsupported dtype for rmsnorm {_DTYPE_NAMES.get(xs.dtype, xs.dtype)}")
    if not xs.is_contiguous():
        raise CandleError("input has to be contiguous")
    for pname, p in params:
        if not p.is_contiguous():
            raise CandleError(f"{pname} has to be contiguous")
    if residual is not None:
        if residual.shape != xs.shape or residual.dtype != xs.dtype:
            raise CandleError(f"shape mismatch in binary op add, lhs: {_dims(xs)}, rhs: {_dims(residual)}")
        if not residual.is_contiguous():
            raise CandleError("input has to be contiguous")
    _same_device(xs, *[p for _, p in params], residual)


def _out_check(out: torch.Tensor | None, xs: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty_like(xs)
    if out.shape != xs.shape or out.dtype != xs.dtype or out.device != xs.device or not out.is_contiguous():
        raise CandleError(f"out must be a contiguous tensor like the input, got {_dims(out)} for {_dims(xs)}")
    return out


def rms_norm(xs: torch.Tensor, alpha: torch.Tensor, eps: float, *, residual: torch.Tensor | None = None,
             return_sum: bool = False, flags: int = 0, out: torch.Tensor | None = None,
             status: torch.Tensor | None = None):
    """``candle_nn::ops::rms_norm(xs, alpha, eps)``; with ``residual`` the norm of ``xs + residual``.

    Returns ``y`` (``out`` when given), or ``(y, xs + residual)`` when ``return_sum`` is set.  A
    ``status`` record (``new_status``) receives device-side problems (a bounded wait that ran out).
    """
    if xs.dim() == 0:
        raise CandleError("unexpected rank, expected: at least 1, got: 0")
    if alpha.dim() != 1:
        raise CandleError(f"unexpected rank, expected: 1, got: {alpha.dim()} ({_dims(alpha)})")
    if xs.shape[-1] != alpha.shape[0]:
        raise CandleError(f"shape mismatch in rms-norm {_dims(xs)} {_dims(alpha)}")
    _norm_checks("rms-norm", xs, [("alpha", alpha)], residual)
    cols = xs.shape[-1]
    rows = xs.numel() // cols if cols else 0
    y = _out_check(out, xs)
    h = torch.empty_like(xs) if return_sum else None
    _cabi.call("cb200_rms_norm_checked", _ptr(xs), _ptr(residual), _ptr(alpha), _ptr(y), _ptr(h), rows, cols,
               float(eps), _DTYPES[xs.dtype], flags, _ptr(status), _stream(xs))
    return (y, h) if return_sum else y


def layer_norm(xs: torch.Tensor, alpha: torch.Tensor, beta: torch.Tensor, eps: float, *,
               residual: torch.Tensor | None = None, return_sum: bool = False, flags: int = 0,
               out: torch.Tensor | None = None, status: torch.Tensor | None = None):
    """``candle_nn::ops::layer_norm(xs, alpha, beta, eps)``; with ``residual`` the norm of ``xs + residual``."""
    if xs.dim() == 0:
        raise CandleError("unexpected rank, expected: at least 1, got: 0")
    if alpha.dim() != 1 or beta.dim() != 1:
        bad = alpha if alpha.dim() != 1 else beta
        raise CandleError(f"unexpected rank, expected: 1, got: {bad.dim()} ({_dims(bad)})")
    if xs.shape[-1] != alpha.shape[0] or xs.shape[-1] != beta.shape[0]:
        raise CandleError(f"shape mismatch in layer-norm src: {_dims(xs)} alpha: {_dims(alpha)} beta: {_dims(beta)}")
    _norm_checks("layer-norm", xs, [("alpha", alpha), ("beta", beta)], residual)
    cols = xs.shape[-1]
    rows = xs.numel() // cols if cols else 0
    y = _out_check(out, xs)
    h = torch.empty_like(xs) if return_sum else None
    _cabi.call("cb200_layer_norm_checked", _ptr(xs), _ptr(residual), _ptr(alpha), _ptr(beta), _ptr(y), _ptr(h), rows,
               cols, float(eps), _DTYPES[xs.dtype], flags, _ptr(status), _stream(xs))
    return (y, h) if return_sum else y


def _norm_slow(xs: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, eps: float, remove_mean: bool):
    """candle's composite norm chain (candle-nn/src/layer_norm.rs:115-135) in one launch."""
    if xs.dim() == 0:
        raise CandleError("unexpected rank, expected: at least 1, got: 0")
    if xs.dtype not in _DTYPES:
        raise CandleError(f"unsupported dtype for rmsnorm {_DTYPE_NAMES.get(xs.dtype, xs.dtype)}")
    cols = xs.shape[-1]
    for p in (weight, bias):
        if p is None:
            continue
        if p.dtype != xs.dtype:
            raise CandleError(f"dtype mismatch in mul, lhs: {_DTYPE_NAMES[xs.dtype]}, rhs: {_DTYPE_NAMES.get(p.dtype, p.dtype)}")
        if p.dim() != 1 or p.shape[0] != cols:
            raise CandleError(f"shape mismatch in broadcast_mul, lhs: {_dims(xs)}, rhs: {_dims(p)}")
    _same_device(xs, weight, bias)
    # the chain starts with to_dtype, which reads a strided input into a contiguous tensor
    xs = xs if xs.is_contiguous() else xs.contiguous()
    weight = weight if weight.is_contiguous() else weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    rows = xs.numel() // cols if cols else 0
    y = torch.empty_like(xs)
    _cabi.call("cb200_layer_norm_slow", _ptr(xs), _ptr(weight), _ptr(bias), _ptr(y), rows, cols, float(eps),
               _DTYPES[xs.dtype], 1 if remove_mean else 0, _stream(xs))
    return y


def rms_norm_slow(x: torch.Tensor, alpha: torch.Tensor, eps: float) -> torch.Tensor:
    """``candle_nn::ops::rms_norm_slow`` (candle-nn/src/ops.rs:628-639)."""
    return _norm_slow(x, alpha, None, eps, False)


def layer_norm_slow(x: torch.Tensor, alpha: torch.Tensor, beta: torch.Tensor, eps: float) -> torch.Tensor:
    """``candle_nn::ops::layer_norm_slow`` (candle-nn/src/ops.rs:876-894)."""
    return _norm_slow(x, alpha, beta, eps, True)


def _ids_checks(ids: torch.Tensor) -> torch.Tensor:
    if ids.dim() != 1:
        raise CandleError(f"unexpected number of dims: expected 1, got {ids.dim()}, shape {_dims(ids)}")
    if ids.dtype not in _ID_DTYPES:
        raise CandleError(f"unsupported dtype {ids.dtype} for index-select ids (expected U8, U32 or I64)")
    return ids if ids.is_contiguous() else ids.contiguous()  # the CPU op honours an ids stride


def index_select(t: torch.Tensor, ids: torch.Tensor, dim: int, *, check: bool = True,
                 status: torch.Tensor | None = None) -> torch.Tensor:
    """``Tensor::index_select(ids, dim)``.  With ``check`` the call synchronises and raises
    ``InvalidIndex`` like the CPU backend; pass ``check=False`` and a ``status`` record to defer."""
    if not t.is_contiguous():
        raise CandleError("index-select requires contiguous tensors")
    ids = _ids_checks(ids)
    _same_device(t, ids)
    dim = dim if dim >= 0 else dim + t.dim()
    if not 0 <= dim < t.dim():
        raise CandleError(f"dim out of range in index-select: {dim} for shape {_dims(t)}")
    shape = list(t.shape)
    left = 1
    for d in shape[:dim]:
        left *= d
    right = 1
    for d in shape[dim + 1:]:
        right *= d
    src_dim = shape[dim]
    shape[dim] = ids.shape[0]
    out = torch.empty(shape, dtype=t.dtype, device=t.device)
    st = status if status is not None else (new_status(t.device) if check else None)
    _cabi.call("cb200_index_select", _ptr(t), _ptr(ids), _ptr(out), left, src_dim, right, ids.shape[0],
               t.element_size(), _ID_DTYPES[ids.dtype], _ptr(st), _stream(t))
    if check:
        raise_for_status(st)
    return out


def embedding_rms_norm(table: torch.Tensor, ids: torch.Tensor, alpha: torch.Tensor, eps: float, *,
                       return_gathered: bool = False, flags: int = 0, check: bool = True,
                       status: torch.Tensor | None = None):
    """``rms_norm(Embedding::forward(ids), alpha, eps)`` in one launch (ids of any shape)."""
    if table.dim() != 2 or not table.is_contiguous():
        raise CandleError("index-select requires contiguous tensors")
    if alpha.dim() != 1 or alpha.shape[0] != table.shape[1]:
        raise CandleError(f"shape mismatch in rms-norm {list(ids.shape) + [table.shape[1]]} {_dims(alpha)}")
    _norm_checks("rms-norm", table, [("alpha", alpha)], None)
    flat = _ids_checks(ids.reshape(-1))
    _same_device(table, flat, alpha)
    vocab, hidden = table.shape
    final = list(ids.shape) + [hidden]
    y = torch.empty(final, dtype=table.dtype, device=table.device)
    g = torch.empty(final, dtype=table.dtype, device=table.device) if return_gathered else None
    st = status if status is not None else (new_status(table.device) if check else None)
    _cabi.call("cb200_embedding_rms_norm", _ptr(table), _ptr(flat), _ptr(alpha), _ptr(y), _ptr(g), vocab, hidden,
               flat.shape[0], float(eps), _DTYPES[table.dtype], _ID_DTYPES[flat.dtype], flags, _ptr(st),
               _stream(table))
    if check:
        raise_for_status(st)
    return (y, g) if return_gathered else y


def qembedding_rms_norm(qtensor, ids: torch.Tensor, alpha: torch.Tensor, eps: float, *,
                        return_gathered: bool = False, flags: int = 0, check: bool = True,
                        status: torch.Tensor | None = None, vocab_range: tuple[int, int] | None = None,
                        vocab: int | None = None):
    """Rows ``ids`` of a block-quantised table decoded to ``alpha.dtype`` and RMS-normalised: one launch
    for Q4_0 / Q8_0 and the K-quant formats at the usual row lengths, lookup followed by the norm otherwise."""
    from .quantized import QTensor  # local import: quantized imports this module

    if not isinstance(qtensor, QTensor) or len(qtensor.shape) != 2:
        raise CandleError("qembedding expects a rank-2 QTensor")
    if alpha.dtype not in _DTYPES:
        raise CandleError(f"unsupported dtype for rmsnorm {alpha.dtype}")
    local_vocab, hidden = qtensor.shape
    if alpha.dim() != 1 or alpha.shape[0] != hidden or not alpha.is_contiguous():
        raise CandleError(f"shape mismatch in rms-norm {list(ids.shape) + [hidden]} {_dims(alpha)}")
    flat = _ids_checks(ids.reshape(-1))
    _same_device(qtensor.data, flat, alpha)
    begin, end = vocab_range if vocab_range is not None else (0, local_vocab)
    total = vocab if vocab is not None else end
    if end - begin != local_vocab:
        raise CandleError(f"vocab shard [{begin}, {end}) does not match the table's {local_vocab} rows")
    final = list(ids.shape) + [hidden]
    y = torch.empty(final, dtype=alpha.dtype, device=alpha.device)
    g = torch.empty(final, dtype=alpha.dtype, device=alpha.device) if return_gathered else None
    st = status if status is not None else (new_status(alpha.device) if check else None)
    _cabi.call("cb200_qembedding_rms_norm", _ptr(qtensor.data), qtensor.dtype.value, _ptr(flat), _ptr(alpha), _ptr(y),
               _ptr(g), total, hidden, flat.shape[0], float(eps), _DTYPES[alpha.dtype], _ID_DTYPES[flat.dtype],
               begin, end, flags, _ptr(st), _stream(alpha))
    if check:
        raise_for_status(st)
    return (y, g) if return_gathered else y


def qembedding_rms_norm_owner(qtensor, ids: torch.Tensor, alpha: torch.Tensor, eps: float, dst_ptrs, *,
                              vocab_range: tuple[int, int], vocab: int, flags: int = 0,
                              status: torch.Tensor | None = None) -> None:
    """Owner-writes-to-all step of a vocabulary-sharded lookup + RMS norm: the ids inside
    ``vocab_range`` are decoded from this rank's slice ``qtensor``, normalised, and stored into every
    buffer of ``dst_ptrs`` (device addresses of ``[ids.numel(), hidden]`` buffers of ``alpha.dtype``:
    this rank's own first, then the peers' mapped ones).  Ids owned by other ranks are skipped; the
    caller synchronises the ranks before reading.  Invalid ids are recorded in ``status``."""
    import ctypes

    from .quantized import QTensor  # local import: quantized imports this module

    if not isinstance(qtensor, QTensor) or len(qtensor.shape) != 2:
        raise CandleError("qembedding expects a rank-2 QTensor")
    if alpha.dtype not in _DTYPES:
        raise CandleError(f"unsupported dtype for rmsnorm {alpha.dtype}")
    local_vocab, hidden = qtensor.shape
    if alpha.dim() != 1 or alpha.shape[0] != hidden or not alpha.is_contiguous():
        raise CandleError(f"shape mismatch in rms-norm {list(ids.shape) + [hidden]} {_dims(alpha)}")
    flat = _ids_checks(ids.reshape(-1))
    _same_device(qtensor.data, flat, alpha)
    begin, end = vocab_range
    if end - begin != local_vocab:
        raise CandleError(f"vocab shard [{begin}, {end}) does not match the table's {local_vocab} rows")
    ptrs = [int(p) for p in dst_ptrs]
    arr = (ctypes.c_void_p * len(ptrs))(*ptrs)
    _cabi.call("cb200_qembedding_rms_norm_owner", _ptr(qtensor.data), qtensor.dtype.value, _ptr(flat), _ptr(alpha),
               ctypes.cast(arr, ctypes.c_void_p), len(ptrs), vocab, hidden, flat.shape[0], float(eps),
               _DTYPES[alpha.dtype], _ID_DTYPES[flat.dtype], begin, end, flags, _ptr(status), _stream(alpha))


def qembedding_rms_norm_row_owner(qtensor, ids: torch.Tensor, alpha: torch.Tensor, eps: float, dst_ptrs, row_bounds, *,
                                  vocab_range: tuple[int, int], vocab: int, flags: int = 0,
                                  status: torch.Tensor | None = None) -> None:
    """Row-owner step of a vocabulary-sharded lookup + RMS norm: the ids inside ``vocab_range`` are
    decoded from this rank's slice ``qtensor`` and normalised, and each finished row is stored into
    the one buffer whose block of token rows contains it.  ``dst_ptrs[r]`` is the device address of
    rank r's ``[row_bounds[r + 1] - row_bounds[r], hidden]`` buffer (rank order; peers' buffers mapped
    into this process), ``row_bounds`` the ``len(dst_ptrs) + 1`` block limits from 0 to ``ids.numel()``.
    Ids owned by other ranks are skipped; the caller synchronises the ranks before reading."""
    import ctypes

    from .quantized import QTensor  # local import: quantized imports this module

    if not isinstance(qtensor, QTensor) or len(qtensor.shape) != 2:
        raise CandleError("qembedding expects a rank-2 QTensor")
    if alpha.dtype not in _DTYPES:
        raise CandleError(f"unsupported dtype for rmsnorm {alpha.dtype}")
    local_vocab, hidden = qtensor.shape
    if alpha.dim() != 1 or alpha.shape[0] != hidden or not alpha.is_contiguous():
        raise CandleError(f"shape mismatch in rms-norm {list(ids.shape) + [hidden]} {_dims(alpha)}")
    flat = _ids_checks(ids.reshape(-1))
    _same_device(qtensor.data, flat, alpha)
    begin, end = vocab_range
    if end - begin != local_vocab:
        raise CandleError(f"vocab shard [{begin}, {end}) does not match the table's {local_vocab} rows")
    ptrs = [int(p) for p in dst_ptrs]
    bounds = [int(b) for b in row_bounds]
    if len(bounds) != len(ptrs) + 1:
        raise CandleError(f"{len(ptrs)} destinations need {len(ptrs) + 1} row bounds, got {len(bounds)}")
    arr = (ctypes.c_void_p * len(ptrs))(*ptrs)
    barr = (ctypes.c_int64 * len(bounds))(*bounds)
    _cabi.call("cb200_qembedding_rms_norm_row_owner", _ptr(qtensor.data), qtensor.dtype.value, _ptr(flat), _ptr(alpha),
               ctypes.cast(arr, ctypes.c_void_p), len(ptrs), ctypes.cast(barr, ctypes.c_void_p), vocab, hidden,
               flat.shape[0], float(eps), _DTYPES[alpha.dtype], _ID_DTYPES[flat.dtype], begin, end, flags, _ptr(status),
               _stream(alpha))


def softmax_last_dim(xs: torch.Tensor) -> torch.Tensor:
    """``candle_nn::ops::softmax_last_dim`` (candle-nn/src/ops.rs:289-435)."""
    if xs.dtype not in _DTYPES:
        raise CandleError(f"unsupported dtype for softmax {_DTYPE_NAMES.get(xs.dtype, xs.dtype)}")
    if not xs.is_contiguous():
        raise CandleError("input has to be contiguous")
    _same_device(xs)
    if xs.dim() == 0:
        raise CandleError("unexpected rank, expected: at least 1, got: 0")
    cols = xs.shape[-1]
    rows = xs.numel() // cols if cols else 0
    y = torch.empty_like(xs)
    _cabi.call("cb200_softmax_last_dim", _ptr(xs), _ptr(y), rows, cols, _DTYPES[xs.dtype], _stream(xs))
    return y


def _rope(variant: int, name: str, xs: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    # the checks of rotary_emb.rs:203-228 (rope_i), 457-482 (rope), 706-731 (rope_thd)
    if xs.dim() != 4:
        raise CandleError(f"unexpected rank, expected: 4, got: {xs.dim()} ({_dims(xs)})")
    if cos.dim() != 2 or sin.dim() != 2:
        bad = cos if cos.dim() != 2 else sin
        raise CandleError(f"unexpected rank, expected: 2, got: {bad.dim()} ({_dims(bad)})")
    if variant == _cabi.ROPE_THD:
        b, seq_len, h, n_embd = xs.shape
    else:
        b, h, seq_len, n_embd = xs.shape
    if cos.shape[1] * 2 != n_embd or sin.shape[1] * 2 != n_embd or seq_len > cos.shape[0] or seq_len > sin.shape[0]:
        raise CandleError(f"inconsistent last dim size in rope {_dims(xs)} {_dims(cos)} {_dims(sin)}")
    if not xs.is_contiguous():
        raise CandleError("xs has to be contiguous in rope")
    if not cos.is_contiguous():
        raise CandleError("cos has to be contiguous in rope")
    if not sin.is_contiguous():
        raise CandleError("sin has to be contiguous in rope")
    if xs.dtype not in _DTYPES or cos.dtype != xs.dtype or sin.dtype != xs.dtype:
        raise CandleError(f"unsupported dtype for rope {xs.dtype} {cos.dtype} {sin.dtype}")
    _same_device(xs, cos, sin)
    dst = torch.empty_like(xs)
    _cabi.call("cb200_rope", _ptr(xs), _ptr(cos), _ptr(sin), _ptr(dst), b, h, seq_len, n_embd, _DTYPES[xs.dtype], variant,
               _stream(xs))
    return dst


def rope_i(xs: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """``candle_nn::rotary_emb::rope_i``: interleaved pairs, ``xs`` is ``[b, h, t, d]``."""
    return _rope(_cabi.ROPE_INTERLEAVED, "rope-i", xs, cos, sin)


def rope(xs: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """``candle_nn::rotary_emb::rope``: pairs ``(x[k], x[k + d/2])``, ``xs`` is ``[b, h, t, d]``."""
    return _rope(_cabi.ROPE_HALF, "rope", xs, cos, sin)


def rope_thd(xs: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """``candle_nn::rotary_emb::rope_thd``: as ``rope`` for ``xs`` laid out ``[b, t, h, d]``."""
    return _rope(_cabi.ROPE_THD, "rope-thd", xs, cos, sin)


def rms_norm_rows(xs: torch.Tensor, rows: torch.Tensor, alpha: torch.Tensor, eps: float, *, check: bool = True,
                  status: torch.Tensor | None = None) -> torch.Tensor:
    """RMS norm of the selected rows only: ``rms_norm(xs, alpha, eps).index_select(rows, 0)`` without
    normalising the rows nobody reads.  The final norm of a decoder is followed by a slice that keeps
    the last token of each sequence (candle-transformers/src/models/quantized_llama.rs:507-508: norm of
    all rows, then ``x.i((.., seq_len - 1, ..))``); with ``rows`` = those positions in the flattened
    ``[b * t, hidden]`` activations this reads and writes ``b`` rows instead of ``b * t``.  Rows are
    independent, so the values are the same."""
    if xs.dim() != 2:
        raise CandleError(f"unexpected rank, expected: 2, got: {xs.dim()} ({_dims(xs)})")
    return embedding_rms_norm(xs, rows, alpha, eps, check=check, status=status)


def qembedding_route_rows(qtensor, ids: torch.Tensor, dst_ptrs, row_bounds, *, vocab_range: tuple[int, int], vocab: int,
                          status: torch.Tensor | None = None) -> None:
    """Routing step of a vocabulary-sharded lookup with row-sharded consumers: for every id inside
    ``vocab_range`` the raw block row of this rank's slice ``qtensor`` is copied into the staging buffer
    of the rank whose block of token rows holds the id's position (``dst_ptrs`` in rank order,
    ``row_bounds`` the block limits).  After the ranks' barrier each staging buffer is a
    ``[rows_r, hidden]`` table of blocks in token order, ready for a local lookup + norm."""
    import ctypes

    from .quantized import QTensor  # local import: quantized imports this module

    if not isinstance(qtensor, QTensor) or len(qtensor.shape) != 2:
        raise CandleError("qembedding expects a rank-2 QTensor")
    local_vocab, hidden = qtensor.shape
    flat = _ids_checks(ids.reshape(-1))
    _same_device(qtensor.data, flat)
    begin, end = vocab_range
    if end - begin != local_vocab:
        raise CandleError(f"vocab shard [{begin}, {end}) does not match the table's {local_vocab} rows")
    ptrs = [int(p) for p in dst_ptrs]
    bounds = [int(b) for b in row_bounds]
    if len(bounds) != len(ptrs) + 1:
        raise CandleError(f"{len(ptrs)} destinations need {len(ptrs) + 1} row bounds, got {len(bounds)}")
    arr = (ctypes.c_void_p * len(ptrs))(*ptrs)
    barr = (ctypes.c_int64 * len(bounds))(*bounds)
    _cabi.call("cb200_qembedding_route_rows", _ptr(qtensor.data), qtensor.dtype.value, _ptr(flat),
               ctypes.cast(arr, ctypes.c_void_p), len(ptrs), ctypes.cast(barr, ctypes.c_void_p), vocab, hidden,
               flat.shape[0], _ID_DTYPES[flat.dtype], begin, end, _ptr(status), _stream(flat))


# ---- training and serving operators beside the path -------------------------------------------------
# f32 inside with one rounding to the output's type; the sums of gradients are held in f32 and have an order that
# shapes, ids, alignment and strides fix, so equal inputs laid out alike give equal bits.  Scratch memory comes from
# torch's allocator, one piece per call.


_COUNT_LIMIT = 1 << 29  # columns of a row, heads of a token: the kernels count them in 32 bits


def _check_columns(op: str, columns: int) -> None:
    if columns >= _COUNT_LIMIT:
        raise CandleError(f"rows of {columns} columns in {op}, they must be fewer than 2^29")


def _stream_of(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


# The current stream's handle without a Stream object around it: a launch of a few microseconds feels the difference.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
if _raw_stream is not None:
    def _stream_of(device: torch.device) -> int:  # noqa: F811
        return _raw_stream(device.index)

# and the current device's number: every call has a tensor of the device, so there is nothing to initialise
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _launch(device: torch.device, name: str, *args) -> None:
    """The entry point `name` on `device`'s current stream, whichever device is current."""
    if device.index == _current_device():
        _cabi.call(name, *args, _stream_of(device))
    else:
        with torch.cuda.device(device):
            _cabi.call(name, *args, _stream_of(device))


@lru_cache(maxsize=512)
def _workspace_bytes(device: torch.device, name: str, *args) -> int:
    n = ctypes.c_int64(0)
    with torch.cuda.device(device):
        _cabi.call(name, *args, ctypes.addressof(n))
    return n.value


def _workspace(device: torch.device, name: str, *args) -> tuple[torch.Tensor, int]:
    n = _workspace_bytes(device, name, *args)
    return torch.empty(n, dtype=torch.uint8, device=device), n


def _span(t: torch.Tensor) -> tuple[int, int]:
    """First and one-past-last byte address of a tensor with non-negative strides."""
    n = t.numel()
    if n == 0:
        return 0, 0
    if t.is_contiguous():
        at = t.data_ptr()
        return at, at + n * t.element_size()
    last = sum((n - 1) * st for n, st in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _interleaved(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two views of one buffer, such as q and k of a packed projection, share no element: for a stride S that
    both have and whose multiples all their larger strides are, their pieces lie apart within [0, S)."""
    if a.dtype != b.dtype:
        return False
    size = a.element_size()
    for step in set(a.stride()) & set(b.stride()) - {0}:  # a broadcast dimension sets nothing apart
        inner = []
        for t in (a, b):
            dims = [(n, st) for n, st in zip(t.shape, t.stride()) if n > 1]
            if any(st >= step and st % step for _, st in dims):
                break
            inner.append(1 + sum((n - 1) * st for n, st in dims if st < step))
        at, rest = divmod((b.data_ptr() - a.data_ptr()) % (step * size), size)
        if len(inner) == 2 and rest == 0 and inner[0] <= at and at + inner[1] <= step:
            return True
    return False


def _check_apart(op: str, out: torch.Tensor, *others: torch.Tensor | None, same: bool = True) -> None:
    """Refuses an output that overlaps one of `others`, unless (with `same`) it is that very view."""
    lo, hi = _span(out)
    for t in others:
        if t is None:
            continue
        a, b = _span(t)
        if hi <= a or b <= lo:
            continue
        if same and t.data_ptr() == out.data_ptr() and t.shape == out.shape and t.dtype == out.dtype and all(
                x == y for n, x, y in zip(t.shape, t.stride(), out.stride()) if n > 1):
            continue
        if not _interleaved(out, t):
            raise CandleError(f"the output of {op} overlaps another tensor of the call")


def embedding_scaled(table: torch.Tensor, ids: torch.Tensor, scale: float, *, out: torch.Tensor | None = None,
                     check: bool = True, status: torch.Tensor | None = None) -> torch.Tensor:
    """``scale * Embedding::forward(ids)`` in one launch, rounded once: the lookup of models that multiply the
    embedding by a constant such as ``sqrt(hidden)``.  ids of any shape; the row of a bad id is left unwritten and
    reported as by ``index_select``.  (candle multiplies in the table's type with the scale rounded to it.)"""
    if table.dim() != 2 or not table.is_contiguous():
        raise CandleError("index-select requires contiguous tensors")
    if table.dtype not in _DTYPES:
        raise CandleError(f"unsupported dtype {table.dtype} for embedding")
    flat = _ids_checks(ids if ids.dim() == 1 else ids.reshape(-1))
    vocab, hidden = table.shape
    _check_columns("embedding", hidden)
    _same_device(table, flat, out)
    final = [*ids.shape, hidden]
    if out is None:
        out = torch.empty(final, dtype=table.dtype, device=table.device)
    else:
        if list(out.shape) != final or out.dtype != table.dtype or not out.is_contiguous():
            raise CandleError(f"out must be a contiguous tensor of shape {final}, got {_dims(out)}")
        _check_apart("embedding", out, table, flat, same=False)
    st = status if status is not None else (new_status(table.device) if check else None)
    _launch(table.device, "cb200_embedding_scaled", _ptr(table), _ptr(flat), _ptr(out), vocab, hidden, flat.shape[0],
            float(scale), _DTYPES[table.dtype], _ID_DTYPES[flat.dtype], _ptr(st))
    if check:
        raise_for_status(st)
    return out


def embedding_backward(grad: torch.Tensor, ids: torch.Tensor, vocab: int, *, scale: float = 1.0,
                       out: torch.Tensor | None = None, accumulate: bool = False, out_dtype: torch.dtype | None = None,
                       padding_id: int | None = None, check: bool = True,
                       status: torch.Tensor | None = None) -> torch.Tensor:
    """Gradient of ``scale * Embedding::forward(ids)`` with respect to the ``[vocab, hidden]`` table: row v is
    ``scale`` times the sum of the rows of ``grad`` whose id is v, in f32 and in a fixed order (that of the tokens up to
    63 of them; longer runs are added in parts).

    ``grad`` is ``[*ids.shape, hidden]`` (rows may be strided).  The result is a fresh tensor of ``out_dtype``
    (``grad``'s, or f32) or ``out``; every row is written, zeros where no id points.  With ``accumulate`` the sums are
    added to ``out`` and the other rows are not touched.  Tokens whose id is ``padding_id``, a row
    of the table, contribute nothing."""
    if grad.dtype not in _DTYPES:
        raise CandleError(f"unsupported dtype {grad.dtype} for embedding-backward")
    shape = grad.shape
    if len(shape) == 0 or shape[:-1] != ids.shape:
        raise CandleError(f"shape mismatch in embedding-backward {_dims(grad)} {_dims(ids)}")
    hidden = shape[-1]
    _check_columns("embedding-backward", hidden)
    flat = _ids_checks(ids if ids.dim() == 1 else ids.reshape(-1))
    n = flat.shape[0]
    try:
        rows = grad if len(shape) == 2 else grad.view(n, hidden)
    except RuntimeError:
        raise CandleError("the rows of grad must have one stride in embedding-backward") from None
    row_stride, column_stride = rows.stride()
    if hidden > 1 and column_stride != 1:
        raise CandleError("the last dimension of grad has to be contiguous in embedding-backward")
    vocab = int(vocab)
    if vocab < 0:
        raise CandleError(f"the table of embedding-backward has {vocab} rows")
    if padding_id is not None and not 0 <= padding_id < vocab:
        raise CandleError(f"padding_id {padding_id} is no row of the table of embedding-backward, which has {vocab} rows")
    if out_dtype is None:
        out_dtype = grad.dtype if out is None else out.dtype
    if out_dtype != grad.dtype and out_dtype != torch.float32:
        raise CandleError(f"unsupported dtype {out_dtype} for the result of embedding-backward of {grad.dtype}")
    _same_device(grad, flat, out)
    if out is None:
        if accumulate:
            raise CandleError("embedding-backward accumulates into `out`, which is missing")
        out = torch.empty(vocab, hidden, dtype=out_dtype, device=grad.device)
    else:
        if out.shape != (vocab, hidden) or out.dtype != out_dtype or not out.is_contiguous():
            raise CandleError(f"out must be a contiguous {out_dtype} tensor of shape {[vocab, hidden]}, got {out.dtype} {_dims(out)}")
        _check_apart("embedding-backward", out, rows, flat, same=False)
    ws, ws_bytes = _workspace(grad.device, "cb200_embedding_backward_workspace", vocab, hidden, n)
    st = status if status is not None else (new_status(grad.device) if check else None)
    _launch(grad.device, "cb200_embedding_backward", _ptr(rows), row_stride if n > 1 else hidden, _ptr(flat), _ptr(out),
            vocab, hidden, n, float(scale), -1 if padding_id is None else int(padding_id), 1 if accumulate else 0,
            _DTYPES[grad.dtype], _DTYPES[out_dtype], _ID_DTYPES[flat.dtype], _ptr(ws), ws_bytes, _ptr(st))
    if check:
        raise_for_status(st)
    return out


def _rms_backward_refuse(grad, xs, alpha, grad_sum) -> None:
    """Raises what is wrong with the arguments of the RMS norm's gradient."""
    if xs.dim() == 0:
        raise CandleError("unexpected rank, expected: at least 1, got: 0")
    if alpha.dim() != 1:
        raise CandleError(f"unexpected rank, expected: 1, got: {alpha.dim()} ({_dims(alpha)})")
    if xs.shape[-1] != alpha.shape[0]:
        raise CandleError(f"shape mismatch in rms-norm {_dims(xs)} {_dims(alpha)}")
    _check_columns("rms-norm-backward", alpha.shape[0])
    for g in (grad, grad_sum):
        if g is None:
            continue
        if g.shape != xs.shape or g.dtype != xs.dtype:
            raise CandleError(f"shape mismatch in rms-norm-backward, xs: {_dims(xs)} {xs.dtype}, gradient: {_dims(g)} {g.dtype}")
        if not g.is_contiguous():
            raise CandleError("the gradient has to be contiguous")
    _norm_checks("rms-norm", xs, [("alpha", alpha)], None)
    _same_device(xs, grad, grad_sum)


def rms_norm_backward(grad: torch.Tensor, xs: torch.Tensor, alpha: torch.Tensor, eps: float, *,
                      grad_sum: torch.Tensor | None = None, out: torch.Tensor | None = None):
    """Gradient of ``rms_norm(xs, alpha, eps)``: ``(dxs, dalpha)`` for the gradient ``grad`` of its result, ``dalpha`` in
    f32.  After ``rms_norm(x, alpha, eps, residual=r, return_sum=True)`` pass the returned sum as ``xs`` and the gradient
    that reaches that sum on the residual stream as ``grad_sum``, which is added: ``dxs`` is then the gradient of both
    ``x`` and ``r``.  ``out`` may be ``grad``, ``xs`` or ``grad_sum``."""
    t, shape, dev = xs.dtype, xs.shape, xs.get_device()
    if not (
        t in _DTYPES and len(shape) > 0 and alpha.shape == shape[-1:] and shape[-1] < _COUNT_LIMIT and alpha.dtype == t and grad.shape == shape and grad.dtype == t
        and xs.is_contiguous() and alpha.is_contiguous() and grad.is_contiguous()
        and dev >= 0 and alpha.get_device() == dev and grad.get_device() == dev
        and (grad_sum is None or grad_sum.shape == shape and grad_sum.dtype == t and grad_sum.is_contiguous()
             and grad_sum.get_device() == dev)
    ):
        _rms_backward_refuse(grad, xs, alpha, grad_sum)
    dx = _out_check(out, xs)
    if out is not None:
        _check_apart("rms-norm-backward", out, grad, xs, grad_sum)
        _check_apart("rms-norm-backward", out, alpha, same=False)
    cols = xs.shape[-1]
    rows = xs.numel() // cols if cols else 0
    dalpha = torch.empty(cols, dtype=torch.float32, device=xs.device)
    ws, ws_bytes = _workspace(xs.device, "cb200_rms_norm_backward_workspace", rows, cols)
    _launch(xs.device, "cb200_rms_norm_backward", _ptr(grad), _ptr(xs), _ptr(alpha), _ptr(grad_sum), _ptr(dx), _ptr(dalpha),
            rows, cols, float(eps), _DTYPES[xs.dtype], _ptr(ws), ws_bytes)
    return dx, dalpha


_HEADS = struct.Struct("=qqqqii")  # cb200_heads
_QK_ARGS = struct.Struct("=qqqqqqqqiifiiiii")  # cb200_qk_args


def _fresh(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _heads(t: torch.Tensor, rank: int, heads: int) -> bytes:
    if rank == 4:
        batch, token, head, _ = t.stride()
        return _HEADS.pack(t.data_ptr(), batch, token, head, heads, 0)
    token, head, _ = t.stride()
    return _HEADS.pack(t.data_ptr(), 0, token, head, heads, 0)


def _qk_refuse(op: str, q, k, q_weight, k_weight, cos, sin, positions, more) -> None:
    """Raises what is wrong with the arguments of the head norms with rotation or their gradient."""
    if q.dim() not in (3, 4) or k.dim() != q.dim():
        raise CandleError(f"unexpected rank in {op}, expected: [tokens, heads, dim] or [batch, tokens, heads, dim], got: "
                          f"{_dims(q)} {_dims(k)}")
    d = q.shape[-1]
    if k.shape[-1] != d or k.shape[:-2] != q.shape[:-2]:
        raise CandleError(f"shape mismatch in {op} {_dims(q)} {_dims(k)}")
    _check_columns(op, d)
    if q.shape[-2] + k.shape[-2] >= _COUNT_LIMIT:
        raise CandleError(f"{q.shape[-2]} + {k.shape[-2]} heads in {op}, they must be fewer than 2^29")
    if q.dtype not in _DTYPES or any(t.dtype != q.dtype for t in (k, q_weight, k_weight)):
        raise CandleError(f"unsupported dtype for {op} {q.dtype} {k.dtype} {q_weight.dtype} {k_weight.dtype}")
    for w in (q_weight, k_weight):
        if w.dim() != 1 or w.shape[0] != d:
            raise CandleError(f"shape mismatch in {op}, heads of {d} columns, weight: {_dims(w)}")
        if not w.is_contiguous():
            raise CandleError("the weight has to be contiguous")
    if cos.dim() != 2 or sin.shape != cos.shape or not 0 < 2 * cos.shape[1] <= d:
        raise CandleError(f"inconsistent last dim size in rope {_dims(q)} {_dims(cos)} {_dims(sin)}")
    if not cos.is_contiguous():
        raise CandleError("cos has to be contiguous in rope")
    if not sin.is_contiguous():
        raise CandleError("sin has to be contiguous in rope")
    if sin.dtype != cos.dtype or cos.dtype not in (q.dtype, torch.float32):
        raise CandleError(f"unsupported dtype for rope {q.dtype} {cos.dtype} {sin.dtype}")
    for t, like in ((q, q), (k, k), *more):
        if t.shape != like.shape or t.dtype != q.dtype:
            raise CandleError(f"shape mismatch in {op} {_dims(like)} {like.dtype}, {_dims(t)} {t.dtype}")
        if t.stride(-1) != 1 and d > 1:
            raise CandleError(f"the last dimension has to be contiguous in {op}")
    if positions is None:
        if q.shape[-3] > cos.shape[0]:
            raise CandleError(f"inconsistent last dim size in rope {_dims(q)} {_dims(cos)} {_dims(sin)}")
    else:
        if positions.shape != q.shape[:-2]:
            raise CandleError(f"shape mismatch in {op} {_dims(q)}, positions: {_dims(positions)}")
        if positions.dtype not in _ID_DTYPES:
            raise CandleError(f"unsupported dtype {positions.dtype} for positions (expected U8, U32 or I64)")
        if not positions.is_contiguous():
            raise CandleError(f"positions have to be contiguous in {op}")
    _same_device(q, k, q_weight, k_weight, cos, sin, positions, *(t for t, _ in more))


def _qk_args(op: str, q, k, q_weight, k_weight, eps, cos, sin, positions, interleaved, more=()):
    """The checked arguments that the head norms with rotation and their gradient share, packed, and (rank, q heads,
    k heads, dim, device).  `more` are tensors that have to be like q or k: (tensor, like).  What is right is decided
    by one chain of comparisons, since a decoding step's kernel takes less time than its checks; `_qk_refuse` then
    says what is wrong."""
    qs, ks, cs, t, ct, dev = q.shape, k.shape, cos.shape, q.dtype, cos.dtype, q.get_device()
    rank = len(qs)
    if not (
        (rank == 4 or rank == 3) and len(ks) == rank and len(cs) == 2 and sin.shape == cs
        and qs[-1] == ks[-1] and qs[:-2] == ks[:-2] and 0 < 2 * cs[1] <= qs[-1] < _COUNT_LIMIT
        and qs[-2] + ks[-2] < _COUNT_LIMIT
        and t in _DTYPES and k.dtype == t and q_weight.dtype == t and k_weight.dtype == t
        and (ct == t or ct == torch.float32) and sin.dtype == ct
        and q_weight.shape == k_weight.shape == (qs[-1],)
        and q_weight.is_contiguous() and k_weight.is_contiguous() and cos.is_contiguous() and sin.is_contiguous()
        and q.stride(-1) == 1 and k.stride(-1) == 1
        and all(m.shape == like.shape and m.dtype == t and m.get_device() == dev and m.stride(-1) == 1 for m, like in more)
        and (qs[-3] <= cs[0] if positions is None else positions.shape == qs[:-2] and positions.dtype in _ID_DTYPES
             and positions.is_contiguous() and positions.get_device() == dev)
        and dev >= 0 and k.get_device() == dev and q_weight.get_device() == dev and k_weight.get_device() == dev
        and cos.get_device() == dev and sin.get_device() == dev
    ):
        _qk_refuse(op, q, k, q_weight, k_weight, cos, sin, positions, more)
    args = _QK_ARGS.pack(
        q_weight.data_ptr(), k_weight.data_ptr(), cos.data_ptr(), sin.data_ptr(),
        0 if positions is None else positions.data_ptr(), qs[0] if rank == 4 else 1, qs[-3], cs[0], qs[-1], 2 * cs[1], eps,
        1 if interleaved else 0, _DTYPES[t], _DTYPES[ct], _cabi.ID_I64 if positions is None else _ID_DTYPES[positions.dtype], 0)
    return args, rank, qs[-2], ks[-2], qs[-1], q.device


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, eps: float,
                 cos: torch.Tensor, sin: torch.Tensor, *, positions: torch.Tensor | None = None,
                 interleaved: bool = False, out: tuple[torch.Tensor, torch.Tensor] | None = None, check: bool = True,
                 status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every query and key head followed by its rotation, in one pass: ``rope(rms_norm(q, q_weight, eps))`` and
    the same of k, computed in f32 and rounded once.

    q is ``[batch, tokens, q_heads, dim]`` or ``[tokens, q_heads, dim]``, k the same with its own number of heads; any
    strides but a contiguous last dimension, so views of a packed projection and ``[b, h, t, d]`` tensors seen through
    ``transpose(1, 2)`` need no copy.  cos / sin are ``[positions, rotary / 2]`` in the heads' type or f32: the first
    ``rotary`` columns are rotated, as ``rope`` does or (``interleaved``) as ``rope_i``.  ``positions`` has the shape of
    the tokens; without it a token's position is its index in the sequence.  ``out`` may be (q, k) themselves.
    The heads of a token whose position the tables do not have are left unwritten and reported."""
    more = () if out is None else ((out[0], q), (out[1], k))
    args, rank, q_heads, k_heads, _, device = _qk_args("qk-norm-rope", q, k, q_weight, k_weight, eps, cos, sin, positions,
                                                       interleaved, more)
    if out is None:
        q_out, k_out = _fresh(q), _fresh(k)
    else:
        q_out, k_out = out
        _check_apart("qk-norm-rope", q_out, q)
        _check_apart("qk-norm-rope", k_out, k)
        _check_apart("qk-norm-rope", q_out, k, k_out, q_weight, k_weight, cos, sin, positions, same=False)
        _check_apart("qk-norm-rope", k_out, q, q_weight, k_weight, cos, sin, positions, same=False)
    check = check and positions is not None
    st = status if status is not None else (new_status(device) if check else None)
    _launch(device, "cb200_qk_norm_rope", _heads(q, rank, q_heads), _heads(k, rank, k_heads), _heads(q_out, rank, q_heads),
            _heads(k_out, rank, k_heads), args, _ptr(st))
    if check:
        raise_for_status(st, "qk-norm-rope")
    return q_out, k_out


def qk_norm_rope_backward(grad_q: torch.Tensor, grad_k: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                          q_weight: torch.Tensor, k_weight: torch.Tensor, eps: float, cos: torch.Tensor,
                          sin: torch.Tensor, *, positions: torch.Tensor | None = None, interleaved: bool = False,
                          out: tuple[torch.Tensor, torch.Tensor] | None = None, check: bool = True,
                          status: torch.Tensor | None = None):
    """Gradient of ``qk_norm_rope``: ``(dq, dk, dq_weight, dk_weight)`` from the gradients of its two results and its
    inputs (the same q, k, weights, cos, sin and positions), the weights' gradients in f32.  ``out`` receives (dq, dk)
    and may be the gradients or (q, k) themselves."""
    more = [(grad_q, q), (grad_k, k)]
    if out is not None:
        more += [(out[0], q), (out[1], k)]
    op = "qk-norm-rope-backward"
    args, rank, q_heads, k_heads, dim, device = _qk_args(op, q, k, q_weight, k_weight, eps, cos, sin, positions, interleaved,
                                                         more)
    if out is None:
        dq, dk = _fresh(q), _fresh(k)
    else:
        dq, dk = out
        _check_apart(op, dq, q, grad_q)
        _check_apart(op, dk, k, grad_k)
        _check_apart(op, dq, k, grad_k, dk, q_weight, k_weight, cos, sin, positions, same=False)
        _check_apart(op, dk, q, grad_q, q_weight, k_weight, cos, sin, positions, same=False)
    dw = torch.empty(2, dim, dtype=torch.float32, device=device)
    ws, ws_bytes = _workspace(device, "cb200_qk_norm_rope_backward_workspace", dim)
    check = check and positions is not None
    st = status if status is not None else (new_status(device) if check else None)
    dq_weight, dk_weight = dw.unbind(0)
    _launch(device, "cb200_qk_norm_rope_backward", _heads(grad_q, rank, q_heads), _heads(grad_k, rank, k_heads),
            _heads(q, rank, q_heads), _heads(k, rank, k_heads), _heads(dq, rank, q_heads), _heads(dk, rank, k_heads),
            _ptr(dq_weight), _ptr(dk_weight), args, _ptr(ws), ws_bytes, _ptr(st))
    if check:
        raise_for_status(st, op)
    return dq, dk, dq_weight, dk_weight

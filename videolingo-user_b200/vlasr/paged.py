"""Paged KV cache and beam search over libvlasr.so.

The reference engine decodes greedily over one contiguous cache per chunk
(VideoLingo-user native/asr/src/decoder.cu:1372-1800); these operators are
what a beam search over pages that beams share needs instead.  They have no
counterpart there.

=====================  ==========================================================
paged_rope_append      rotate q and k, store k and v through the page tables
paged_attention        causal attention of each sequence's new tokens (one, a
                       few or a long chunk) over its pages
beam_select            the best continuations over beams and vocabulary
paged_beam_reorder     page tables of the chosen parents; pages that two beams
                       would write are split by copying
=====================  ==========================================================

Common arguments: caches [num_pages, page_size, kv_heads, head_dim] (the
pages may be strided), q_start int32 [batch + 1], kv_len int32 [batch],
page_table int32 [batch, max_pages] (rows may be strided).  Sequence b's new
tokens are the packed rows q_start[b] .. q_start[b + 1] - 1, the last of its
kv_len[b] positions; position p lies in row p % page_size of page
page_table[b, p // page_size].  Packed rows behind the last sequence are left
as they were, and what they hold does not matter (they may be read).  What is
out of range on the device is skipped and sets VL_STATUS_BAD_PAGE in `status`
(an int32 tensor), if given.
"""

from __future__ import annotations

import ctypes
import functools
import inspect

import torch

from . import _lib
from ._lib import VL_BF16, VL_F16, VL_F32, VlasrInputError, check
from .ops import LAUNCH_PDL

BEAM_MAX = 32

_CODES = {torch.float32: VL_F32, torch.float16: VL_F16, torch.bfloat16: VL_BF16}
_I32, _I64, _F32, _BOOL, _U8 = (torch.int32, torch.int64, torch.float32, torch.bool, torch.uint8)

# A decode step makes these calls once per layer, so the checks are written to
# cost as few tensor-attribute reads as they can.
try:
    from torch._C import _cuda_getCurrentRawStream as _raw_stream
    from torch._C import _cuda_getDevice as _current_device
except ImportError:      # a build of torch without them
    def _raw_stream(device: int) -> int:
        return torch.cuda.current_stream(device).cuda_stream

    _current_device = torch.cuda.current_device


def _operator(fn):
    """Launches go to the tensors' device, whatever the current one is (the
    first CUDA tensor among the arguments names it), and an argument that is
    no tensor is an input error."""
    signature = inspect.signature(fn)
    # what a parameter must be: True a tensor, False a tensor or None
    tensors = {name: "None" not in p.annotation for name, p in signature.parameters.items()
               if "torch.Tensor" in str(p.annotation)}

    @functools.wraps(fn)
    def call(*args, **kwargs):
        try:
            try:
                return fn(*args, **kwargs)
            except _OtherDevice as e:
                with torch.cuda.device(e.device):
                    return fn(*args, **kwargs)
        except AttributeError:
            for name, value in signature.bind(*args, **kwargs).arguments.items():
                if name in tensors and not isinstance(value, torch.Tensor) and (
                        tensors[name] or value is not None):
                    raise VlasrInputError(
                        f"{fn.__name__}: {name} is not a torch.Tensor") from None
            raise
    return call


class _OtherDevice(Exception):
    def __init__(self, device: int):
        self.device = device


def _lead(t: torch.Tensor, name: str) -> tuple[int, torch.dtype, int]:
    """dtype code, dtype and device of the tensor the others must match."""
    dev = t.get_device()
    if dev < 0:
        raise VlasrInputError(f"{name} must be a CUDA tensor (there is no CPU path)")
    dt = t.dtype
    code = _CODES.get(dt)
    if code is None:
        raise VlasrInputError(f"unsupported dtype {dt}; expected float32/float16/bfloat16")
    if dev != _current_device():
        raise _OtherDevice(dev)
    return code, dt, dev


def _like(t: torch.Tensor, dt: torch.dtype, dev: int, name: str) -> None:
    if t.dtype is not dt or t.get_device() != dev:
        raise VlasrInputError(f"{name} must match dtype/device {dt}/cuda:{dev}")


def _packed(t: torch.Tensor, dt: torch.dtype, dev: int, name: str) -> None:
    if t.dtype is not dt or t.get_device() != dev:
        raise VlasrInputError(f"{name} must be {dt} on cuda:{dev}")
    if not t.is_contiguous():
        raise VlasrInputError(f"{name} must be contiguous")


def _status_ptr(status: torch.Tensor | None, dev: int) -> int | None:
    if status is None:
        return None
    _packed(status, _I32, dev, "status")
    if status.numel() < 1:
        raise VlasrInputError("status must hold one int32")
    return status.data_ptr()


def _head_rows(t: torch.Tensor, head_dim: int, name: str) -> tuple[int, int, int]:
    """[tokens, heads, head_dim] or [tokens, heads * head_dim] -> tokens, heads, row stride."""
    shape, stride = t.shape, t.stride()
    if len(shape) == 2:
        tokens, width = shape
        if width % head_dim or stride[1] != 1:
            raise VlasrInputError(f"{name} must be [tokens, heads * {head_dim}] with contiguous rows")
    elif len(shape) == 3:
        tokens, heads, hd = shape
        if hd != head_dim or stride[2] != 1 or (stride[1] != head_dim and heads != 1):
            raise VlasrInputError(f"{name} must be [tokens, heads, {head_dim}] with packed heads")
        width = heads * hd
    else:
        raise VlasrInputError(f"{name} must be [tokens, heads, head_dim] or [tokens, heads * head_dim]")
    # one row may carry any stride
    return tokens, width // head_dim, stride[0] if tokens > 1 else max(stride[0], width)


def _cache_pages(k_cache: torch.Tensor, v_cache: torch.Tensor) -> tuple[int, int, int, int, int]:
    """num_pages, page_size, kv_heads, head_dim, page stride of both caches."""
    shape, stride = k_cache.shape, k_cache.stride()
    if len(shape) != 4 or v_cache.shape != shape or v_cache.stride() != stride:
        raise VlasrInputError("k_cache and v_cache must be [num_pages, page_size, kv_heads, "
                              "head_dim] of the same shape and strides")
    num_pages, page_size, heads, hd = shape
    if hd == 0:
        raise VlasrInputError("the caches' head_dim must be positive")
    if stride[3] != 1 or (stride[2] != hd and heads != 1) or stride[1] != heads * hd:
        raise VlasrInputError("the rows of a cache page must be contiguous")
    return num_pages, page_size, heads, hd, stride[0] if num_pages > 1 else max(
        stride[0], page_size * heads * hd)


def _batch(dev, q_start, kv_len, page_table) -> tuple[int, int, int]:
    """batch, max_pages and row stride of the page table."""
    _packed(q_start, _I32, dev, "q_start")
    _packed(kv_len, _I32, dev, "kv_len")
    batch = kv_len.numel()
    if q_start.numel() != batch + 1 or kv_len.dim() != 1 or q_start.dim() != 1:
        raise VlasrInputError("q_start must be [batch + 1] and kv_len [batch]")
    shape = page_table.shape
    if (page_table.dtype is not _I32 or page_table.get_device() != dev or len(shape) != 2
            or shape[0] != batch or page_table.stride(1) != 1):
        raise VlasrInputError("page_table must be int32 [batch, max_pages] with contiguous rows")
    max_pages = shape[1]
    return batch, max_pages, page_table.stride(0) if batch > 1 else max(page_table.stride(0),
                                                                        max_pages)


@_operator
def paged_rope_append(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor,
                      k_cache: torch.Tensor, v_cache: torch.Tensor, q_start: torch.Tensor,
                      kv_len: torch.Tensor, page_table: torch.Tensor, *,
                      head_dim: int | None = None, rotary_dim: int | None = None,
                      base: float = 10000.0, interleaved: bool = False,
                      position_scale: float = 1.0, q_out: torch.Tensor | None = None,
                      status: torch.Tensor | None = None) -> torch.Tensor | None:
    """Rotary embedding of q and k and the append of k and v to the pages
    (vl_paged_rope_append); returns the rotated q.

    q [tokens, heads * head_dim] (or [tokens, heads, head_dim]; a row stride is
    allowed, e.g. a column slice of a packed qkv buffer) is not modified unless
    q_out is q; k and v never are.  The first rotary_dim dims of a head rotate
    (0: none) in pairs (d, d + rotary_dim/2), or (2d, 2d + 1) with interleaved,
    by position * position_scale * base^(-2d/rotary_dim).  q None only
    appends."""
    code, dt, dev = _lead(k, "k")
    _like(v, dt, dev, "v")
    _like(k_cache, dt, dev, "k_cache")
    _like(v_cache, dt, dev, "v_cache")
    num_pages, page_size, kvh, hd, page_stride = _cache_pages(k_cache, v_cache)
    if head_dim is not None and head_dim != hd:
        raise VlasrInputError(f"head_dim {head_dim} is not the cache's ({hd})")
    tokens, kh, ks = _head_rows(k, hd, "k")
    vt, vh, vs = _head_rows(v, hd, "v")
    if kh != kvh or vh != kvh or vt != tokens:
        raise VlasrInputError("k and v must have one row per token and the cache's heads")
    batch, max_pages, table_stride = _batch(dev, q_start, kv_len, page_table)
    nq = qs = os_ = 0
    q_ptr = out_ptr = None
    if q is not None:
        _like(q, dt, dev, "q")
        qt, nq, qs = _head_rows(q, hd, "q")
        if q_out is None:
            ot, oh, os_ = tokens, nq, nq * hd
            q_out = torch.empty(tokens, os_, dtype=dt, device=q.device)
        else:
            _like(q_out, dt, dev, "q_out")
            ot, oh, os_ = _head_rows(q_out, hd, "q_out")
        if qt != tokens or ot != tokens or oh != nq:
            raise VlasrInputError("q and q_out must have one row per token and the same heads")
        q_ptr, out_ptr = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise VlasrInputError("q_out needs q")
    rc = _lib.load().vl_paged_rope_append(
        q_ptr, k.data_ptr(), v.data_ptr(), out_ptr, k_cache.data_ptr(), v_cache.data_ptr(),
        q_start.data_ptr(), kv_len.data_ptr(), page_table.data_ptr(), tokens, batch, max_pages,
        table_stride, nq, kvh, hd, hd if rotary_dim is None else rotary_dim,
        1 if interleaved else 0, base, position_scale, qs, ks, vs, os_, num_pages, page_size,
        page_stride, code, _status_ptr(status, dev), _raw_stream(dev))
    if rc:
        check(rc, "vl_paged_rope_append")
    return q_out


def paged_attention_workspace_bytes(tokens: int, batch: int, max_q_len: int, n_q_heads: int,
                                    n_kv_heads: int, head_dim: int,
                                    dtype: torch.dtype = torch.bfloat16) -> int:
    return int(_lib.load().vl_paged_attention_workspace_bytes(
        tokens, batch, max_q_len, n_q_heads, n_kv_heads, head_dim, _CODES[dtype]))


def _workspace(device: torch.device, dev: int, workspace: torch.Tensor | None,
               need: int) -> tuple[torch.Tensor, int]:
    """The caller's workspace and its bytes, or one of the call's own from the
    allocator (stream-ordered, and inside a capture the graph's)."""
    if workspace is None:
        return torch.empty(max(need, 16), dtype=_U8, device=device), need
    if workspace.get_device() != dev or not workspace.is_contiguous():
        raise VlasrInputError(f"workspace must be a contiguous tensor on cuda:{dev}")
    return workspace, workspace.numel() * workspace.element_size()


@_operator
def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    q_start: torch.Tensor, kv_len: torch.Tensor, page_table: torch.Tensor, *,
                    max_q_len: int, scale: float = 0.0, out: torch.Tensor | None = None,
                    workspace: torch.Tensor | None = None, status: torch.Tensor | None = None,
                    pdl: bool = False) -> torch.Tensor:
    """Causal attention of each sequence's new tokens over its pages
    (vl_paged_attention).

    q [tokens, heads * head_dim] (or 3-D; a row stride is allowed), rotated
    already, its k and v appended already; out the same (it may be q).
    max_q_len bounds the new tokens of a sequence and picks the kernel: pass 1
    for a decode step.  scale 0 means 1/sqrt(head_dim).  Without `workspace`
    the call takes its own.  pdl=True launches it as a programmatic dependent
    of the previous kernel on the stream (VL_LAUNCH_PDL): that kernel must
    not write q_start, kv_len or page_table."""
    code, dt, dev = _lead(q, "q")
    _like(k_cache, dt, dev, "k_cache")
    _like(v_cache, dt, dev, "v_cache")
    num_pages, page_size, kvh, hd, page_stride = _cache_pages(k_cache, v_cache)
    tokens, nq, qs = _head_rows(q, hd, "q")
    batch, max_pages, table_stride = _batch(dev, q_start, kv_len, page_table)
    device = q.device
    if out is None:
        out = torch.empty(tokens, nq * hd, dtype=dt, device=device)
    else:
        _like(out, dt, dev, "out")
    ot, oh, os_ = _head_rows(out, hd, "out")
    if ot != tokens or oh != nq:
        raise VlasrInputError("out must have q's rows and heads")
    lib = _lib.load()
    ws, ws_bytes = _workspace(device, dev, workspace, lib.vl_paged_attention_workspace_bytes(
        tokens, batch, max_q_len, nq, kvh, hd, code))
    rc = lib.vl_paged_attention(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), q_start.data_ptr(),
        kv_len.data_ptr(), page_table.data_ptr(), tokens, batch, max_q_len, max_pages,
        table_stride, nq, kvh, hd, scale, qs, os_, num_pages, page_size, page_stride,
        out.data_ptr(), code, ws.data_ptr(), ws_bytes, _status_ptr(status, dev),
        LAUNCH_PDL if pdl else 0, _raw_stream(dev))
    if rc:
        check(rc, "vl_paged_attention")
    return out


def beam_select_workspace_bytes(batch: int, beams: int, vocab: int) -> int:
    return int(_lib.load().vl_beam_select_workspace_bytes(batch, beams, vocab))


@_operator
def beam_select(logits: torch.Tensor, scores: torch.Tensor, *,
                finished: torch.Tensor | None = None, eos_ids=(), pad_id: int = 0,
                tokens: torch.Tensor | None = None, parents: torch.Tensor | None = None,
                scores_out: torch.Tensor | None = None,
                finished_out: torch.Tensor | None = None,
                workspace: torch.Tensor | None = None, status: torch.Tensor | None = None):
    """One step's selection of beam search (vl_beam_select).

    logits [batch * beams, vocab] (a row stride is allowed), scores float32
    [batch, beams] the beams' summed log-probabilities (start with 0, -inf,
    -inf, ...), finished bool/uint8 [batch, beams].  A live beam offers every
    token at score + log-softmax, a finished one pad_id at its own score; the
    best `beams` values of an entry are taken, ties to the lower
    beam * vocab + token.  Returns (tokens int64, parents int32, scores
    float32, finished bool), each [batch, beams]; scores_out may be scores and
    finished_out may be finished.  A wait that ran out inside the kernel makes
    its beam offer nothing and sets VL_STATUS_TIMEOUT in `status`."""
    code, _, dev = _lead(logits, "logits")
    if logits.dim() != 2 or logits.stride(1) != 1:
        raise VlasrInputError("logits must be a 2-D tensor with contiguous rows")
    _packed(scores, _F32, dev, "scores")
    shape = scores.shape
    if len(shape) != 2:
        raise VlasrInputError("scores must be [batch, beams]")
    batch, beams = shape
    rows, vocab = logits.shape
    if rows != batch * beams:
        raise VlasrInputError("logits must have batch * beams rows")
    def place(t, name, dtype):
        _packed(t, _U8 if dtype is _BOOL and t.dtype is _U8 else dtype, dev, name)
        if t.shape != shape:
            raise VlasrInputError(f"{name} must be [batch, beams]")

    if finished is not None:
        place(finished, "finished", _BOOL)
    # (empty_like takes half of torch.empty's time)
    if tokens is None:
        tokens = torch.empty_like(scores, dtype=_I64)
    else:
        place(tokens, "tokens", _I64)
    if parents is None:
        parents = torch.empty_like(scores, dtype=_I32)
    else:
        place(parents, "parents", _I32)
    if scores_out is None:
        scores_out = torch.empty_like(scores)
    else:
        place(scores_out, "scores_out", _F32)
    if finished_out is None:
        finished_out = torch.empty_like(scores, dtype=_BOOL)
    else:
        place(finished_out, "finished_out", _BOOL)
    n_eos = len(eos_ids)
    eos = (ctypes.c_int64 * n_eos)(*eos_ids) if n_eos else None
    lib = _lib.load()
    ws, ws_bytes = _workspace(logits.device, dev, workspace,
                              lib.vl_beam_select_workspace_bytes(batch, beams, vocab))
    rc = lib.vl_beam_select_status(
        logits.data_ptr(), batch, beams, vocab,
        logits.stride(0) if rows > 1 else max(logits.stride(0), vocab), scores.data_ptr(),
        None if finished is None else finished.data_ptr(), eos, n_eos, pad_id,
        tokens.data_ptr(), parents.data_ptr(), scores_out.data_ptr(), finished_out.data_ptr(),
        code, ws.data_ptr(), ws_bytes, _status_ptr(status, dev), _raw_stream(dev))
    if rc:
        check(rc, "vl_beam_select")
    return tokens, parents, scores_out, finished_out


@_operator
def paged_beam_reorder(page_table: torch.Tensor, parents: torch.Tensor, kv_len: torch.Tensor,
                       pool_start: torch.Tensor, pool_pages: int, k_cache: torch.Tensor,
                       v_cache: torch.Tensor, *, out: torch.Tensor | None = None,
                       kv_len_out: torch.Tensor | None = None,
                       status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Page tables after a selection (vl_paged_beam_reorder) -> (tables, kv_len).

    page_table int32 [batch * beams, max_pages], parents int32 [batch, beams]
    (beam_select's), kv_len int32 [batch * beams] the positions each row
    holds, caches [layers, num_pages, page_size, kv_heads, head_dim] (or one
    layer, 4-D).  Row (e, i) shares the whole pages of row
    (e, parents[e, i]); the page of its next position becomes its own: kept by
    the lowest row that can, else taken from the entry's range
    pool_start[e] .. + pool_pages - 1 with the rows so far copied in every
    layer.  The old tables are only read; `out` and `kv_len_out` must be other
    tensors."""
    _, dt, dev = _lead(k_cache, "k_cache")
    _like(v_cache, dt, dev, "v_cache")
    shape, stride = k_cache.shape, k_cache.stride()
    if v_cache.shape != shape or v_cache.stride() != stride or len(shape) not in (4, 5):
        raise VlasrInputError("k_cache and v_cache must be [layers, num_pages, page_size, "
                              "kv_heads, head_dim] of the same shape and strides")
    if len(shape) == 4:
        shape, stride = (1, *shape), (0, *stride)
    layers, num_pages, page_size, kvh, hd = shape
    row = kvh * hd
    if stride[4] != 1 or (stride[3] != hd and kvh != 1) or stride[2] != row:
        raise VlasrInputError("the rows of a cache page must be contiguous")
    _packed(parents, _I32, dev, "parents")
    if parents.dim() != 2:
        raise VlasrInputError("parents must be [batch, beams]")
    batch, beams = parents.shape
    rows = batch * beams
    _packed(kv_len, _I32, dev, "kv_len")
    _packed(pool_start, _I32, dev, "pool_start")
    if kv_len.numel() != rows or pool_start.numel() != batch:
        raise VlasrInputError("kv_len must be [batch * beams] and pool_start [batch]")

    def row_stride(t, name):
        if (t.dtype is not _I32 or t.get_device() != dev or t.dim() != 2 or t.shape[0] != rows
                or t.stride(1) != 1):
            raise VlasrInputError(f"{name} must be int32 [batch * beams, max_pages] with "
                                  "contiguous rows")
        return t.stride(0) if rows > 1 else max(t.stride(0), t.shape[1])

    table_stride = row_stride(page_table, "page_table")
    max_pages = page_table.shape[1]
    if out is None:
        out = torch.empty_like(page_table, memory_format=torch.contiguous_format)
        out_stride = max_pages
    else:
        out_stride = row_stride(out, "out")
        if out.shape[1] != max_pages:
            raise VlasrInputError("out must have page_table's shape")
    if kv_len_out is None:
        kv_len_out = torch.empty_like(kv_len)
    else:
        _packed(kv_len_out, _I32, dev, "kv_len_out")
        if kv_len_out.numel() != rows:
            raise VlasrInputError("kv_len_out must be [batch * beams]")
    es = k_cache.element_size()
    page_stride = stride[1] if num_pages > 1 else max(stride[1], page_size * row)
    rc = _lib.load().vl_paged_beam_reorder(
        page_table.data_ptr(), parents.data_ptr(), kv_len.data_ptr(), pool_start.data_ptr(),
        pool_pages, batch, beams, max_pages, table_stride, out.data_ptr(), out_stride,
        kv_len_out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), layers, num_pages,
        page_size, row * es, page_stride * es, stride[0] * es, _status_ptr(status, dev),
        _raw_stream(dev))
    if rc:
        check(rc, "vl_paged_beam_reorder")
    return out, kv_len_out

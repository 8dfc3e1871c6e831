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
as they were.  What is out of range on the device is skipped and sets
VL_STATUS_BAD_PAGE in `status` (an int32 tensor), if given.
"""

from __future__ import annotations

import contextlib
import ctypes

import torch

from . import _lib
from ._lib import VL_BF16, VL_F16, VL_F32, VlasrInputError, check
from .ops import LAUNCH_PDL

BEAM_MAX = 32

_CODES = {torch.float32: VL_F32, torch.float16: VL_F16, torch.bfloat16: VL_BF16}


def _code(t: torch.Tensor, name: str) -> int:
    if not isinstance(t, torch.Tensor):
        raise VlasrInputError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise VlasrInputError(f"{name} must be a CUDA tensor (there is no CPU path)")
    code = _CODES.get(t.dtype)
    if code is None:
        raise VlasrInputError(f"unsupported dtype {t.dtype}; expected float32/float16/bfloat16")
    return code


def _like(ref: torch.Tensor, t: torch.Tensor, name: str) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype != ref.dtype or t.device != ref.device:
        raise VlasrInputError(f"{name} must match dtype/device {ref.dtype}/{ref.device}")


def _ints(ref: torch.Tensor, t: torch.Tensor, name: str, dtype=torch.int32) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != ref.device:
        raise VlasrInputError(f"{name} must be {dtype} on {ref.device}")
    if not t.is_contiguous():
        raise VlasrInputError(f"{name} must be contiguous")


def _on(device: torch.device):
    """Launches go to the tensors' device, whatever the current one is."""
    if device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _status_ptr(ref: torch.Tensor, status: torch.Tensor | None) -> int | None:
    if status is None:
        return None
    _ints(ref, status, "status")
    if status.numel() < 1:
        raise VlasrInputError("status must hold one int32")
    return status.data_ptr()


def _head_rows(t: torch.Tensor, head_dim: int, name: str) -> tuple[int, int, int]:
    """[tokens, heads, head_dim] or [tokens, heads * head_dim] -> tokens, heads, row stride."""
    shape, stride = t.shape, t.stride()
    if len(shape) == 3:
        if shape[2] != head_dim or stride[2] != 1 or (stride[1] != head_dim and shape[1] != 1):
            raise VlasrInputError(f"{name} must be [tokens, heads, {head_dim}] with packed heads")
        tokens, heads = shape[0], shape[1]
    elif len(shape) == 2:
        if shape[1] % head_dim or stride[1] != 1:
            raise VlasrInputError(f"{name} must be [tokens, heads * {head_dim}] with contiguous rows")
        tokens, heads = shape[0], shape[1] // head_dim
    else:
        raise VlasrInputError(f"{name} must be [tokens, heads, head_dim] or [tokens, heads * head_dim]")
    # one row may carry any stride
    return tokens, heads, stride[0] if tokens > 1 else max(stride[0], heads * head_dim)


def _cache_pages(k_cache: torch.Tensor, v_cache: torch.Tensor) -> tuple[int, int, int, int, int]:
    """num_pages, page_size, kv_heads, head_dim, page stride of both caches."""
    shape, stride = k_cache.shape, k_cache.stride()
    if len(shape) != 4 or v_cache.shape != shape or v_cache.stride() != stride:
        raise VlasrInputError("k_cache and v_cache must be [num_pages, page_size, kv_heads, "
                              "head_dim] of the same shape and strides")
    num_pages, page_size, heads, hd = shape
    if stride[3] != 1 or (stride[2] != hd and heads != 1) or stride[1] != heads * hd:
        raise VlasrInputError("the rows of a cache page must be contiguous")
    return num_pages, page_size, heads, hd, stride[0] if num_pages > 1 else max(
        stride[0], page_size * heads * hd)


def _batch(ref, q_start, kv_len, page_table) -> tuple[int, int, int]:
    """batch, max_pages and row stride of the page table."""
    _ints(ref, q_start, "q_start")
    _ints(ref, kv_len, "kv_len")
    batch = kv_len.numel()
    if kv_len.dim() != 1 or q_start.dim() != 1 or q_start.numel() != batch + 1:
        raise VlasrInputError("q_start must be [batch + 1] and kv_len [batch]")
    if (not isinstance(page_table, torch.Tensor) or page_table.dtype != torch.int32
            or page_table.device != ref.device or page_table.dim() != 2
            or page_table.shape[0] != batch or page_table.stride(1) != 1):
        raise VlasrInputError("page_table must be int32 [batch, max_pages] with contiguous rows")
    max_pages = page_table.shape[1]
    return batch, max_pages, page_table.stride(0) if batch > 1 else max(page_table.stride(0),
                                                                        max_pages)


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
    code = _code(k, "k")
    for name, t in (("v", v), ("k_cache", k_cache), ("v_cache", v_cache)):
        _like(k, t, name)
    num_pages, page_size, kvh, hd, page_stride = _cache_pages(k_cache, v_cache)
    if head_dim is not None and head_dim != hd:
        raise VlasrInputError(f"head_dim {head_dim} is not the cache's ({hd})")
    tokens, kh, ks = _head_rows(k, hd, "k")
    vt, vh, vs = _head_rows(v, hd, "v")
    if kh != kvh or vh != kvh or vt != tokens:
        raise VlasrInputError("k and v must have one row per token and the cache's heads")
    batch, max_pages, table_stride = _batch(k, q_start, kv_len, page_table)
    nq = qs = os_ = 0
    q_ptr = out_ptr = None
    if q is not None:
        _like(k, q, "q")
        qt, nq, qs = _head_rows(q, hd, "q")
        if q_out is None:
            q_out = torch.empty((tokens, nq * hd), dtype=q.dtype, device=q.device)
        _like(k, q_out, "q_out")
        ot, oh, os_ = _head_rows(q_out, hd, "q_out")
        if qt != tokens or ot != tokens or oh != nq:
            raise VlasrInputError("q and q_out must have one row per token and the same heads")
        q_ptr, out_ptr = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise VlasrInputError("q_out needs q")
    if rotary_dim is None:
        rotary_dim = hd
    with _on(k.device):
        check(_lib.load().vl_paged_rope_append(
            q_ptr, k.data_ptr(), v.data_ptr(), out_ptr, k_cache.data_ptr(), v_cache.data_ptr(),
            q_start.data_ptr(), kv_len.data_ptr(), page_table.data_ptr(), tokens, batch,
            max_pages, table_stride, nq, kvh, hd, rotary_dim, 1 if interleaved else 0, base,
            position_scale, qs, ks, vs, os_, num_pages, page_size, page_stride, code,
            _status_ptr(k, status), torch.cuda.current_stream().cuda_stream),
            "vl_paged_rope_append")
    return q_out


def paged_attention_workspace_bytes(tokens: int, batch: int, max_q_len: int, n_q_heads: int,
                                    n_kv_heads: int, head_dim: int,
                                    dtype: torch.dtype = torch.bfloat16) -> int:
    return int(_lib.load().vl_paged_attention_workspace_bytes(
        tokens, batch, max_q_len, n_q_heads, n_kv_heads, head_dim, _CODES[dtype]))


def _workspace(ref: torch.Tensor, workspace: torch.Tensor | None, need: int) -> torch.Tensor:
    """The caller's workspace, or one of the call's own from the allocator
    (stream-ordered, and inside a capture the graph's)."""
    if workspace is None:
        return torch.empty(max(need, 16), dtype=torch.uint8, device=ref.device)
    if (not isinstance(workspace, torch.Tensor) or workspace.device != ref.device
            or not workspace.is_contiguous()):
        raise VlasrInputError(f"workspace must be a contiguous tensor on {ref.device}")
    return workspace


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
    code = _code(q, "q")
    _like(q, k_cache, "k_cache")
    _like(q, v_cache, "v_cache")
    num_pages, page_size, kvh, hd, page_stride = _cache_pages(k_cache, v_cache)
    tokens, nq, qs = _head_rows(q, hd, "q")
    batch, max_pages, table_stride = _batch(q, q_start, kv_len, page_table)
    if out is None:
        out = torch.empty((tokens, nq * hd), dtype=q.dtype, device=q.device)
    _like(q, out, "out")
    ot, oh, os_ = _head_rows(out, hd, "out")
    if ot != tokens or oh != nq:
        raise VlasrInputError("out must have q's rows and heads")
    lib = _lib.load()
    with _on(q.device):
        need = lib.vl_paged_attention_workspace_bytes(tokens, batch, max_q_len, nq, kvh, hd, code)
        ws = _workspace(q, workspace, need)
        check(lib.vl_paged_attention(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), q_start.data_ptr(),
            kv_len.data_ptr(), page_table.data_ptr(), tokens, batch, max_q_len, max_pages,
            table_stride, nq, kvh, hd, scale, qs, os_, num_pages, page_size, page_stride,
            out.data_ptr(), code, ws.data_ptr(), ws.numel() * ws.element_size(),
            _status_ptr(q, status), LAUNCH_PDL if pdl else 0,
            torch.cuda.current_stream().cuda_stream), "vl_paged_attention")
    return out


def beam_select_workspace_bytes(batch: int, beams: int, vocab: int) -> int:
    return int(_lib.load().vl_beam_select_workspace_bytes(batch, beams, vocab))


def beam_select(logits: torch.Tensor, scores: torch.Tensor, *,
                finished: torch.Tensor | None = None, eos_ids=(), pad_id: int = 0,
                tokens: torch.Tensor | None = None, parents: torch.Tensor | None = None,
                scores_out: torch.Tensor | None = None,
                finished_out: torch.Tensor | None = None,
                workspace: torch.Tensor | None = None):
    """One step's selection of beam search (vl_beam_select).

    logits [batch * beams, vocab] (a row stride is allowed), scores float32
    [batch, beams] the beams' summed log-probabilities (start with 0, -inf,
    -inf, ...), finished bool/uint8 [batch, beams].  A live beam offers every
    token at score + log-softmax, a finished one pad_id at its own score; the
    best `beams` values of an entry are taken, ties to the lower
    beam * vocab + token.  Returns (tokens int64, parents int32, scores
    float32, finished bool), each [batch, beams]; scores_out may be scores and
    finished_out may be finished."""
    code = _code(logits, "logits")
    if logits.dim() != 2 or logits.stride(1) != 1:
        raise VlasrInputError("logits must be a 2-D tensor with contiguous rows")
    _ints(logits, scores, "scores", torch.float32)
    if scores.dim() != 2:
        raise VlasrInputError("scores must be [batch, beams]")
    shape = scores.shape
    batch, beams = shape
    rows, vocab = logits.shape
    if rows != batch * beams:
        raise VlasrInputError("logits must have batch * beams rows")
    dev = logits.device

    def place(t, name, dtype):
        if t is None:
            return torch.empty(shape, dtype=dtype, device=dev)
        if dtype is torch.bool and isinstance(t, torch.Tensor) and t.dtype == torch.uint8:
            dtype = torch.uint8
        _ints(logits, t, name, dtype)
        if t.shape != shape:
            raise VlasrInputError(f"{name} must be [batch, beams]")
        return t

    if finished is not None:
        place(finished, "finished", torch.bool)
    tokens = place(tokens, "tokens", torch.int64)
    parents = place(parents, "parents", torch.int32)
    scores_out = place(scores_out, "scores_out", torch.float32)
    finished_out = place(finished_out, "finished_out", torch.bool)
    n_eos = len(eos_ids)
    eos = (ctypes.c_int64 * max(n_eos, 1))(*eos_ids)
    lib = _lib.load()
    with _on(dev):
        ws = _workspace(logits, workspace, lib.vl_beam_select_workspace_bytes(batch, beams, vocab))
        check(lib.vl_beam_select(
            logits.data_ptr(), batch, beams, vocab,
            logits.stride(0) if rows > 1 else max(logits.stride(0), vocab), scores.data_ptr(),
            None if finished is None else finished.data_ptr(), eos, n_eos, pad_id,
            tokens.data_ptr(), parents.data_ptr(), scores_out.data_ptr(),
            finished_out.data_ptr(), code, ws.data_ptr(), ws.numel() * ws.element_size(),
            torch.cuda.current_stream().cuda_stream), "vl_beam_select")
    return tokens, parents, scores_out, finished_out


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
    _code(k_cache, "k_cache")
    _like(k_cache, v_cache, "v_cache")
    shape, stride = k_cache.shape, k_cache.stride()
    if len(shape) == 4:
        shape, stride = (1,) + tuple(shape), (0,) + tuple(stride)
    if len(shape) != 5 or v_cache.shape != k_cache.shape or v_cache.stride() != k_cache.stride():
        raise VlasrInputError("k_cache and v_cache must be [layers, num_pages, page_size, "
                              "kv_heads, head_dim] of the same shape and strides")
    layers, num_pages, page_size, kvh, hd = shape
    row = kvh * hd
    if stride[4] != 1 or (stride[3] != hd and kvh != 1) or stride[2] != row:
        raise VlasrInputError("the rows of a cache page must be contiguous")
    _ints(k_cache, parents, "parents")
    if parents.dim() != 2:
        raise VlasrInputError("parents must be [batch, beams]")
    batch, beams = parents.shape
    rows = batch * beams
    _ints(k_cache, kv_len, "kv_len")
    _ints(k_cache, pool_start, "pool_start")
    if kv_len.numel() != rows or pool_start.numel() != batch:
        raise VlasrInputError("kv_len must be [batch * beams] and pool_start [batch]")

    def table(t, name):
        if (not isinstance(t, torch.Tensor) or t.dtype != torch.int32
                or t.device != k_cache.device or t.dim() != 2 or t.shape[0] != rows
                or t.stride(1) != 1):
            raise VlasrInputError(f"{name} must be int32 [batch * beams, max_pages] with "
                                  "contiguous rows")
        return t.stride(0) if rows > 1 else max(t.stride(0), t.shape[1])

    table_stride = table(page_table, "page_table")
    max_pages = page_table.shape[1]
    if out is None:
        out = torch.empty((rows, max_pages), dtype=torch.int32, device=k_cache.device)
    out_stride = table(out, "out")
    if out.shape[1] != max_pages:
        raise VlasrInputError("out must have page_table's shape")
    if kv_len_out is None:
        kv_len_out = torch.empty(rows, dtype=torch.int32, device=k_cache.device)
    _ints(k_cache, kv_len_out, "kv_len_out")
    if kv_len_out.numel() != rows:
        raise VlasrInputError("kv_len_out must be [batch * beams]")
    es = k_cache.element_size()
    page_stride = stride[1] if num_pages > 1 else max(stride[1], page_size * row)
    with _on(k_cache.device):
        check(_lib.load().vl_paged_beam_reorder(
            page_table.data_ptr(), parents.data_ptr(), kv_len.data_ptr(), pool_start.data_ptr(),
            pool_pages, batch, beams, max_pages, table_stride, out.data_ptr(), out_stride,
            kv_len_out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), layers, num_pages,
            page_size, row * es, page_stride * es, stride[0] * es,
            _status_ptr(k_cache, status), torch.cuda.current_stream().cuda_stream),
            "vl_paged_beam_reorder")
    return out, kv_len_out

"""Op-level wrappers of the sm_100a kernels, mirroring the reference's kernel wrappers.

Like the reference (``dryft/engine/kernels/*.py``) each wrapper validates its
inputs (``ValueError`` on contract violations), allocates and returns new
outputs, never mutates inputs (except the KV cache written in place by
``rope_attention``), and launches on the current CUDA stream. Every call runs
the CUDA library; there is no PyTorch or CPU fallback.
"""
from __future__ import annotations

import threading

import torch
from torch.autograd import forward_ad

from . import _lib

BF16 = torch.bfloat16
_scratch = {}
_scratch_lock = threading.RLock()  # making the memory may run a finalizer that makes a call of its own
_workspaces = {}


def _op_scratch(device) -> torch.Tensor:
    """Zero-initialised per-device scratch for the split-KV and argmax partials.
    The kernels restore their counters to zero, so it is reused across calls
    (calls on different streams must not overlap)."""
    key = torch.device(device).index
    buf = _scratch.get(key)
    if buf is None:
        with _scratch_lock:  # threads that come here together get the same one
            buf = _scratch.get(key)
            if buf is None:
                n = int(_lib.load().qb_op_scratch_bytes())
                buf = torch.zeros(n, dtype=torch.uint8, device=device)
                if not torch.cuda.is_current_stream_capturing():
                    torch.cuda.current_stream(device).synchronize()  # zero before a call on another stream uses it
                _scratch[key] = buf
    return buf


def _require(cond: bool, msg: str):
    if not cond:
        raise ValueError(msg)


def _bf16_cuda(*ts):
    for t in ts:
        if t is None:
            continue
        _require(t.is_cuda and t.dtype == BF16 and t.is_contiguous(),
                 "expected contiguous bf16 CUDA tensors")


def check_device_errors(device=None) -> None:
    """Synchronise with the current stream and raise if an op-level kernel reported
    a device error (calls on other streams report once they have run)."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    with torch.cuda.device(device):
        buf = _op_scratch(torch.device("cuda", torch.cuda.current_device()))
        try:
            _lib.check(_lib.load().qb_op_check(buf.data_ptr(), _lib.stream_handle()))
        except Exception:
            _workspaces.clear()  # a kernel that gave up may have left its tickets mid-count
            raise


def norm_projection(x, gain, weight, eps=1e-6, *, swiglu=False):
    """RMSNorm(x) (skipped when gain is None) fused with W.x; with ``swiglu`` the
    weight is ``[2N, K]`` gate/up-interleaved and the result is SwiGLU [N].
    ``dryft/engine/kernels/projection.py:36-53``."""
    _bf16_cuda(x, gain, weight)
    _require(x.numel() == x.shape[-1], "the batch-one path requires one hidden row")
    rows, k = weight.shape
    _require(x.shape[-1] == k and (gain is None or gain.numel() == k), "incompatible projection dimensions")
    if swiglu:
        _require(rows % 2 == 0, "packed gate/up width must be even")
    n = rows // 2 if swiglu else rows
    out = torch.empty((*x.shape[:-1], n), dtype=BF16, device=x.device)
    _lib.check(_lib.load().qb_norm_projection(x.data_ptr(), _lib.ptr(gain), weight.data_ptr(), out.data_ptr(),
                                              k, rows, float(eps), int(bool(swiglu)), _lib.stream_handle()))
    return out


def output_projection_residual(x, weight, residual):
    """bf16(bf16(W.x) + residual): ``dryft/engine/kernels/projection.py:70-83``."""
    _bf16_cuda(x, weight, residual)
    n, k = weight.shape
    _require(x.numel() == k and residual.numel() == n, "output projection requires one activation and residual row")
    out = torch.empty_like(residual)
    _lib.check(_lib.load().qb_projection_residual(x.data_ptr(), weight.data_ptr(), residual.data_ptr(),
                                                  out.data_ptr(), k, n, _lib.stream_handle()))
    return out


def projection_residual_peer(x, weight, residual, recv_words, rank, epoch, sublayer=0, parity=0):
    """One rank's share of a tensor-parallel o-proj / down projection with the
    cross-rank reduction in its epilogue: bf16(bf16(sum_r W_r.x_r) + residual),
    partials added in rank order (``dryft/engine/kernels/projection.py:70-83``
    with the sum spread over ranks). ``recv_words``: one uint64-viewable CUDA
    tensor (or raw device address) per rank, each ``[2, size, N]`` words;
    ``epoch``: CUDA int64 [1] (token base). Device-side wait timeouts surface
    through ``check_device_errors``."""
    _bf16_cuda(x, weight, residual)
    n, k = weight.shape
    _require(x.numel() == k and residual.numel() == n, "projection requires one activation and residual row")
    size = len(recv_words)
    _require(1 <= size <= 8 and 0 <= rank < size, "1..8 ranks, rank in range")
    _require(epoch.is_cuda and epoch.dtype == torch.int64 and epoch.numel() >= 1, "epoch must be CUDA int64")
    ptrs = []
    for t in recv_words:
        if isinstance(t, int):
            ptrs.append(t)
        else:
            _require(t.is_cuda and t.numel() * t.element_size() >= 2 * size * n * 8, "receive buffer too small")
            ptrs.append(t.data_ptr())
    arr = (_lib.c_void_p * size)(*ptrs)
    out = torch.empty_like(residual)
    scratch = _op_scratch(x.device)
    _lib.check(_lib.load().qb_projection_residual_peer(x.data_ptr(), weight.data_ptr(), residual.data_ptr(),
                                                       out.data_ptr(), k, n, arr, rank, size, sublayer, parity,
                                                       epoch.data_ptr(), scratch.data_ptr(), _lib.stream_handle()))
    return out


def down_residual(x, weight, residual):
    """Down projection + residual with one rounding before the add:
    ``dryft/engine/kernels/down.py:288-296``."""
    return output_projection_residual(x, weight, residual)


def greedy_token(x, weight, gain=None, eps=1e-6, return_logits=False):
    """(Optional final RMSNorm +) LM head + argmax of the bf16 logits with the
    lowest index on ties: ``dryft/engine/kernels/greedy.py:45-60``."""
    _bf16_cuda(x, weight, gain)
    _require(x.numel() == x.shape[-1], "the batch-one head takes one hidden row")
    v, k = weight.shape
    _require(x.shape[-1] == k, "incompatible head dimensions")
    token = torch.empty(1, dtype=torch.int64, device=x.device)
    logits = torch.empty(v, dtype=BF16, device=x.device) if return_logits else None
    scratch = _op_scratch(x.device)
    _lib.check(_lib.load().qb_norm_greedy_head(x.data_ptr(), _lib.ptr(gain), weight.data_ptr(), k, v, float(eps),
                                               _lib.ptr(logits), token.data_ptr(), scratch.data_ptr(),
                                               scratch.numel(), _lib.stream_handle()))
    return (token, logits) if return_logits else token


def grouped_attention(q, keys, values, positions):
    """Split-KV GQA attention. q ``[Q, Hq, D]`` (normalised, rotated), keys/values
    ``[Hkv, cap, D]``, positions int64 ``[Q]`` (consecutive) -> ``[Q, Hq, D]``.
    ``dryft/engine/kernels/attention.py:213-237`` (batch one)."""
    _bf16_cuda(q, keys, values)
    _require(q.dim() == 3 and keys.dim() == 3 and keys.shape == values.shape, "expected q [Q,Hq,D], kv [Hkv,cap,D]")
    Q, hq, d = q.shape
    hkv, cap, _ = keys.shape
    _require(d == 128 and keys.shape[2] == 128, "head_dim must be 128")
    _require(positions.is_cuda and positions.dtype == torch.int64 and positions.numel() == Q,
             "positions must be a CUDA int64 tensor with one entry per query")
    out = torch.empty_like(q)
    scratch = _op_scratch(q.device)
    _lib.check(_lib.load().qb_grouped_attention(q.data_ptr(), keys.data_ptr(), values.data_ptr(), hq, hkv, cap, Q,
                                                positions.data_ptr(), out.data_ptr(), scratch.data_ptr(),
                                                scratch.numel(), _lib.stream_handle()))
    return out


def rope_attention(qkv, q_norm, k_norm, cos, sin, keys, values, position, eps=1e-6, n_heads=None):
    """Decode attention with q/k RMSNorm + RoPE + KV append fused in.
    qkv packed ``[Hq*D + 2*Hkv*D]``; keys/values ``[Hkv, cap, D]`` updated at
    ``position`` (int64 [1] CUDA); cos/sin ``[cap, D]`` -> ``[Hq, D]``.
    ``dryft/engine/kernels/fused.py:153-165`` + ``attention.py:213-237``."""
    _bf16_cuda(qkv, q_norm, k_norm, cos, sin, keys, values)
    hkv, cap, d = keys.shape
    _require(d == 128, "head_dim must be 128")
    width = qkv.numel()
    hq = n_heads if n_heads is not None else width // d - 2 * hkv
    _require(width == (hq + 2 * hkv) * d, "packed qkv width does not match the cache heads")
    _require(cos.shape[0] >= cap and sin.shape[0] >= cap, "rope tables shorter than the cache")
    out = torch.empty((hq, d), dtype=BF16, device=qkv.device)
    scratch = _op_scratch(qkv.device)
    _lib.check(_lib.load().qb_rope_attention(qkv.data_ptr(), q_norm.data_ptr(), k_norm.data_ptr(), cos.data_ptr(),
                                             sin.data_ptr(), float(eps), keys.data_ptr(), values.data_ptr(), hq, hkv,
                                             cap, position.data_ptr(), out.data_ptr(), scratch.data_ptr(),
                                             scratch.numel(), _lib.stream_handle()))
    return out


# ------------------------------------------------------ paged K/V cache, sampling
# These calls run on the device their tensors are on (current or not), on its
# current stream, and may overlap on different streams: each stream has its own
# workspace, and a call made while a graph is captured takes one from the
# graph's own memory, so graphs share none either. Threads may share a stream: a
# call's launches, which pass their pieces through the workspace, are made under
# its lock. A stream's workspace is kept at the largest size it was asked for (39 MB
# above 16 query rows per KV head, and 512 bytes a row and head with a prefix).
# ``out`` must not overlap an input.

I32 = torch.int32
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", torch.cuda.is_current_stream_capturing)
_workspace_bytes = {}


_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _status(index: int) -> int:
    """Address of the device error word that ``check_device_errors`` reads."""
    buf = _scratch.get(index)
    if buf is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("call an operator once on this device before capturing a graph")
        buf = _op_scratch(torch.device("cuda", index))
    return buf.data_ptr()


class _Workspace:
    """A stream's memory for paged calls, and the lock under which one call after
    the other takes it and launches into it (re-entrant: making the memory may
    run a finalizer that makes a call of its own)."""

    __slots__ = ("lock", "memory", "nbytes", "address")

    def __init__(self):
        self.lock = threading.RLock()
        self.memory = None
        self.nbytes = self.address = 0


def _workspace(index: int, stream: int, max_queries: int, hq: int, hkv: int, prefix_tokens: int):
    """(workspace, its size in bytes) of a paged call. Its lock is held: the caller releases it after the launches."""
    key = (index, max_queries, hq, hkv, prefix_tokens)
    nbytes = _workspace_bytes.get(key)
    if nbytes is None:
        n = _lib.c_size_t()
        _lib.check(_lib.load().qb_paged_workspace_bytes(max_queries, hq, hkv, prefix_tokens, _lib.ctypes.byref(n)))
        if len(_workspace_bytes) > 4096:
            _workspace_bytes.clear()
        nbytes = _workspace_bytes[key] = n.value
    ws = _Workspace() if _capturing() else _workspaces.get((index, stream))
    if ws is None:
        ws = _workspaces.setdefault((index, stream), _Workspace())
    ws.lock.acquire()
    if ws.nbytes < nbytes:
        try:
            memory = torch.empty(nbytes, dtype=torch.uint8, device=torch.device("cuda", index))
            memory[:_lib.load().qb_paged_zero_bytes()].zero_()
            ws.memory, ws.nbytes, ws.address = memory, nbytes, memory.data_ptr()
        except BaseException:
            ws.lock.release()
            raise
    return ws, nbytes


def _no_grad(*ts):
    """These operators have no backward pass and no forward-mode derivative:
    refuse what would silently lose a gradient or a tangent."""
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                raise ValueError("this operator has no backward pass: use it under torch.no_grad()")
    if getattr(forward_ad, "_current_level", -1) >= 0:
        for t in ts:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError("this operator has no forward-mode derivative")


def _is_bf16(t, index: int) -> bool:
    return t.dtype is BF16 and t.get_device() == index and t.is_contiguous()


def _is_i32(t, index: int) -> bool:
    return t.dtype is I32 and t.get_device() == index and t.is_contiguous()


def _batch(index: int, k_pages, v_pages, page_table, q_start, kv_lens):
    """Checked (pages, Hkv, page, table width, sequences) of a paged batch."""
    shape, table, seqs = k_pages.shape, page_table.shape, kv_lens.shape
    if len(shape) != 4 or shape[3] != 128 or shape[1] < 1 or v_pages.shape != shape:
        raise ValueError("expected k_pages and v_pages [pages, Hkv, page, 128]")
    if index < 0 or not (_is_bf16(k_pages, index) and _is_bf16(v_pages, index)):
        raise ValueError("expected contiguous bf16 pools on the device of the queries")
    if not (_is_i32(page_table, index) and _is_i32(q_start, index) and _is_i32(kv_lens, index)):
        raise ValueError("page_table, q_start and kv_lens must be contiguous int32 tensors on the device of the queries")
    if len(table) != 2 or len(seqs) != 1 or table[0] != seqs[0] or q_start.shape != (seqs[0] + 1,):
        raise ValueError("expected page_table [B, P], q_start [B + 1], kv_lens [B]")
    if table[0] >= 1 << 31 or table[1] >= 1 << 31:  # the C call takes 32 bits
        raise ValueError("at most 1024 sequences, and tables of 2^30 keys")
    return shape[0], shape[1], shape[2], table[1], seqs[0]


def _rows_out(out, shape, like):
    if out is None:
        return torch.empty(shape, dtype=BF16, device=like.device)
    if not _is_bf16(out, like.get_device()) or out.shape != shape:
        raise ValueError("out must be a contiguous bf16 tensor of the result's shape on the device of the queries")
    return out


def _queries(q, hkv: int, index: int, max_queries):
    """Checked (rows, query heads, bound of a sequence's rows)."""
    shape = q.shape
    if not _is_bf16(q, index) or len(shape) != 3 or shape[2] != 128 or shape[1] < 1 or shape[1] % hkv:
        raise ValueError("expected contiguous bf16 CUDA queries [T, Hq, 128], Hq a multiple of Hkv")
    tokens = shape[0]
    return tokens, shape[1], tokens if max_queries is None else min(int(max_queries), tokens)


def rope_paged_append(qkv, q_norm, k_norm, cos, sin, k_pages, v_pages, page_table, q_start, kv_lens, eps=1e-6,
                      n_heads=None, first_position=0, out=None):
    """Per-head q/k RMSNorm and RoPE of packed rows, K and V appended to a paged cache.

    qkv ``[T, (Hq + 2 Hkv) 128]``; q_norm/k_norm ``[128]`` or None (no norm);
    cos/sin ``[positions, 128]``; k_pages/v_pages ``[pages, Hkv, page, 128]``
    written in place; page_table int32 ``[B, P]``, q_start int32 ``[B + 1]``,
    kv_lens int32 ``[B]`` (keys of each sequence once its rows are appended)
    -> rotated q ``[T, Hq, 128]``. Row i of sequence b, rows ``q_start[b]`` to
    ``q_start[b + 1]``, goes to slot ``kv_lens[b] - n + i`` and is turned by
    the angle of ``first_position`` more (the length of a shared prefix). Rows
    from ``q_start[B]`` on are left as they are in ``out``. Page ids, lengths
    or positions out of range are skipped and raise in ``check_device_errors``.
    ``dryft/engine/kernels/fused.py:9-30,47-82`` for a ragged batch."""
    _no_grad(qkv, q_norm, k_norm, cos, sin, k_pages, v_pages, out)
    index = qkv.get_device()
    if not (_is_bf16(qkv, index) and _is_bf16(cos, index) and _is_bf16(sin, index)
            and (q_norm is None or _is_bf16(q_norm, index)) and (k_norm is None or _is_bf16(k_norm, index))):
        raise ValueError("expected contiguous bf16 CUDA tensors on one device")
    pages, hkv, page, width, seqs = _batch(index, k_pages, v_pages, page_table, q_start, kv_lens)
    rows, table = qkv.shape, cos.shape
    if len(rows) != 2 or rows[1] % 128:
        raise ValueError("expected qkv [T, (Hq + 2 Hkv) 128]")
    hq = n_heads if n_heads is not None else rows[1] // 128 - 2 * hkv
    if hq < 1 or rows[1] != (hq + 2 * hkv) * 128:
        raise ValueError("packed qkv width does not match the cache heads")
    if len(table) != 2 or table[1] != 128 or sin.shape != table:
        raise ValueError("expected cos and sin [positions, 128]")
    if (q_norm is not None and q_norm.numel() != 128) or (k_norm is not None and k_norm.numel() != 128):
        raise ValueError("norm gains must have 128 entries")
    if not 0 <= first_position < 1 << 30:
        raise ValueError("first_position must lie in 0..2^30")
    if _current_device() != index:
        with torch.cuda.device(index):
            return rope_paged_append(qkv, q_norm, k_norm, cos, sin, k_pages, v_pages, page_table, q_start, kv_lens, eps,
                                     n_heads, first_position, out)
    out = _rows_out(out, (rows[0], hq, 128), qkv)
    if seqs == 0:
        return out  # every row is one of no sequence
    rc = _lib.load().qb_rope_paged_append(
        qkv.data_ptr(), _lib.ptr(q_norm), _lib.ptr(k_norm), cos.data_ptr(), sin.data_ptr(), table[0], eps,
        k_pages.data_ptr(), v_pages.data_ptr(), pages, page, page_table.data_ptr(), width, q_start.data_ptr(),
        kv_lens.data_ptr(), seqs, rows[0], first_position, hq, hkv, out.data_ptr(), _status(index), _raw_stream(index))
    if rc:
        _lib.check(rc)
    return out


def paged_attention(q, k_pages, v_pages, page_table, q_start, kv_lens, window=0, sinks=0, max_queries=None, out=None):
    """Causal GQA attention of packed query rows over a paged cache.

    q ``[T, Hq, 128]`` (normalised, rotated), the rest as in
    ``rope_paged_append`` -> ``[T, Hq, 128]``. The query at position p sees
    key c iff ``c <= p`` and (``window == 0`` or ``c > p - window`` or ``c <
    sinks``). Pages without a key that some row sees are not read, so they may
    have been given back (any id in the table). ``max_queries`` bounds the query
    rows of a sequence (default T; a tight bound picks the faster kernel); a
    longer sequence raises in ``check_device_errors``. Rows from ``q_start[B]``
    on are left as they are in ``out``; a row that sees no key gives 0. A value
    that is not finite in a key that one row of a sequence sees may reach that
    sequence's other rows. ``dryft/engine/kernels/attention.py:200-237`` for a
    ragged batch."""
    _no_grad(q, k_pages, v_pages, out)
    index = q.get_device()
    pages, hkv, page, width, seqs = _batch(index, k_pages, v_pages, page_table, q_start, kv_lens)
    tokens, hq, max_queries = _queries(q, hkv, index, max_queries)
    window, sinks = min(int(window), 1 << 30), min(int(sinks), 1 << 30)  # beyond any sequence
    if window < 0 or sinks < 0:
        raise ValueError("window and sinks must not be negative")
    if _current_device() != index:
        with torch.cuda.device(index):
            return paged_attention(q, k_pages, v_pages, page_table, q_start, kv_lens, window, sinks, max_queries, out)
    out = _rows_out(out, q.shape, q)
    if seqs == 0:
        return out
    stream, status = _raw_stream(index), _status(index)
    ws, need = _workspace(index, stream, max_queries, hq, hkv, 0)
    try:
        rc = _lib.load().qb_paged_attention(
            q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), pages, page, page_table.data_ptr(), width,
            q_start.data_ptr(), kv_lens.data_ptr(), seqs, tokens, max_queries, hq, hkv, window, sinks, out.data_ptr(),
            ws.address, need, status, stream)
    finally:
        ws.lock.release()
    if rc:
        _lib.check(rc)
    return out


def shared_prefix_attention(q, k_pages, v_pages, prefix_table, prefix_len, page_table, q_start, kv_lens,
                            max_queries=None, out=None):
    """``paged_attention`` (without a window) of a batch whose sequences all
    begin with the same ``prefix_len`` keys, held once in the pages
    ``prefix_table`` (int32 ``[n]``): one pass over them serves every sequence.
    Each query sees the whole prefix and its sequence's own keys up to its
    position; ``kv_lens`` and ``page_table`` count and place the own keys only
    (append them with ``first_position=prefix_len``)."""
    _no_grad(q, k_pages, v_pages, out)
    index = q.get_device()
    pages, hkv, page, width, seqs = _batch(index, k_pages, v_pages, page_table, q_start, kv_lens)
    tokens, hq, max_queries = _queries(q, hkv, index, max_queries)
    if not _is_i32(prefix_table, index) or prefix_table.dim() != 1:
        raise ValueError("prefix_table must be a contiguous int32 tensor [n] on the device of q")
    if not 0 <= prefix_len <= min(prefix_table.shape[0] * page, 1 << 30) or prefix_table.shape[0] >= 1 << 31:
        raise ValueError("prefix_len must lie in 0..prefix_table's keys, and not above 2^30")
    if _current_device() != index:
        with torch.cuda.device(index):
            return shared_prefix_attention(q, k_pages, v_pages, prefix_table, prefix_len, page_table, q_start, kv_lens,
                                           max_queries, out)
    out = _rows_out(out, q.shape, q)
    if seqs == 0:
        return out
    stream, status = _raw_stream(index), _status(index)
    ws, need = _workspace(index, stream, max_queries, hq, hkv, tokens)
    try:
        rc = _lib.load().qb_shared_prefix_attention(
            q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), pages, page, prefix_table.data_ptr(),
            prefix_table.shape[0], prefix_len, page_table.data_ptr(), width, q_start.data_ptr(), kv_lens.data_ptr(),
            seqs, tokens, max_queries, hq, hkv, out.data_ptr(), ws.address, need, status, stream)
    finally:
        ws.lock.release()
    if rc:
        _lib.check(rc)
    return out


def _setting(value, name, rows, dtype, index, lo, hi):
    """(device address or None, number) of a sampling setting: one number for all rows, or a tensor [rows]."""
    if isinstance(value, torch.Tensor):
        if value.dtype is not dtype or value.get_device() != index or value.numel() != rows or not value.is_contiguous():
            raise ValueError(f"{name} must be a number or a contiguous {dtype} tensor [rows] on the device of the logits")
        return value.data_ptr(), 0
    if not lo <= value <= hi:
        raise ValueError(f"{name} must lie in [{lo}, {hi}]")
    return None, value


def sample_token(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None, status=None):
    """Draw one token per row: temperature, then top-k, top-p and min-p, from given uniform numbers.

    logits ``[R, V]`` (or ``[V]``) bf16 or fp32, V at most 262144; uniforms
    fp32 ``[R]`` in [0, 1) -> int64 ``[R]``. Every setting is a number or a
    tensor ``[R]`` (fp32; top_k int32). Tokens rank by falling logit, then
    rising index; ``top_k`` > 0 keeps the first ranks, ``top_p`` < 1 of these
    the ones before which less than ``top_p`` of their mass lies, ``min_p`` > 0
    of these the ones with at least ``min_p`` of the largest weight; the token
    is the first, by index, at which the kept mass passes ``uniform`` times the
    whole. Temperature 0 takes the largest logit, lowest index on ties, as
    ``greedy_token``; infinity weighs every kept token the same. A row without a logit
    above -inf gives -1 and raises in ``check_device_errors``, or, with
    ``status`` (int32 ``[1]``, zero), is reported there. The sampled counterpart of
    ``dryft/engine/kernels/greedy.py:45-60``."""
    _no_grad(logits)
    index, shape = logits.get_device(), logits.shape
    fp32 = logits.dtype is torch.float32
    if index < 0 or not (fp32 or logits.dtype is BF16) or len(shape) not in (1, 2) or not logits.is_contiguous():
        raise ValueError("expected contiguous bf16 or fp32 CUDA logits [R, V]")
    vocab = shape[-1]
    rows = 1 if len(shape) == 1 else shape[0]
    if vocab > 1 << 18 or rows > 1 << 24:  # before the C call's 32 bits
        raise ValueError("expected at most 2^24 rows of at most 262144 logits")
    if (uniforms.dtype is not torch.float32 or uniforms.get_device() != index or uniforms.numel() != rows
            or not uniforms.is_contiguous()):
        raise ValueError("uniforms must be a contiguous fp32 tensor [R] on the device of the logits")
    t, t_all = _setting(temperature, "temperature", rows, torch.float32, index, 0.0, float("inf"))
    k, k_all = _setting(top_k, "top_k", rows, I32, index, 0, 2 ** 31 - 1)
    p, p_all = _setting(top_p, "top_p", rows, torch.float32, index, 0.0, 1.0)
    m, m_all = _setting(min_p, "min_p", rows, torch.float32, index, 0.0, 1.0)
    if _current_device() != index:
        with torch.cuda.device(index):
            return sample_token(logits, uniforms, temperature, top_k, top_p, min_p, out, status)
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=logits.device)
    elif out.dtype is not torch.int64 or out.get_device() != index or out.numel() != rows or not out.is_contiguous():
        raise ValueError("out must be a contiguous int64 tensor [R] on the device of the logits")
    if status is not None and not (_is_i32(status, index) and status.numel() == 1):
        raise ValueError("status must be an int32 tensor [1] on the device of the logits")
    rc = _lib.load().qb_sample_token(logits.data_ptr(), fp32, rows, vocab, uniforms.data_ptr(), t, t_all, k, k_all, p,
                                     p_all, m, m_all, out.data_ptr(),
                                     _status(index) if status is None else status.data_ptr(), _raw_stream(index))
    if rc:
        _lib.check(rc)
    return out

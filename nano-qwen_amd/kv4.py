"""Paged KV caches held in 4 bits, and eviction from paged caches by attention weight.

``kv4_append`` stores rows in 4-bit pages, ``kv4_gather`` reads them back,
``attention_decode_kv4`` attends them: 17/64 of a bf16 cache's bytes, which is what a
decode step reads.  ``attention_key_weights`` gives the attention weight that each cached
key got, ``select_keys`` the keys worth keeping, ``kv_compact`` moves them to other pages;
these take 4-bit and plain pages.  ``PagedKVCache4`` and ``PagedKVCache.evict`` are made
of them.

A row is held in blocks of 32 elements: codes {0, 1/2, 1, 3/2, 2, 3, 4, 6} with a sign (E2M1)
and a power of two per block (E8M0), 4.25 bits an element.  A pool is uint8 (num_pages, Hkv,
page_size, 17 D / 16); its last two axes hold a page's K codes, V codes, K scales and V
scales one after the other, not row by row.

The calls take no part in autograd and refuse tensors that do.  They allocate through torch
and record no memset, so they may be captured in graphs.  Host tensors raise: there is no
CPU path.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional, Tuple, Union

import torch

from . import _lib, ops
from .losses import _PROXY, _before_dispatch, _dispatch_mode, _is_tracing, _memory

__all__ = ["kv4_empty_pool", "kv4_append", "kv4_gather", "attention_decode_kv4",
           "attention_key_weights", "select_keys", "kv_compact"]

_HEAD_DIMS = {17 * d // 16: d for d in (32, 64, 128)}  # bytes of a row -> head_dim
_MOST = 2 ** 31 - 1  # the C entries' int, to which ctypes cuts a larger number without a word
_MOST_REACH = 2 ** 30  # elements that 256 query rows of the key weights span, by their strides
_MOST_KEYS = 2 ** 30  # of a sequence: the kernels count them, rounded up to their steps, in ints


class _DeviceCall(ops.KernelCall):
    """A KernelCall that launches on its tensors' device, whichever is current."""

    __slots__ = ("device",)

    def __init__(self, t, fn, args, name, keep, result):
        super().__init__(fn, (*args, ops._stream(t)), len(args), name, keep, result)
        self.device = t.get_device()

    def launch(self, stream: Optional[torch.cuda.Stream] = None):
        if self.device == torch._C._cuda_getDevice():
            return super().launch(stream)
        with torch.cuda.device(self.device):
            return super().launch(stream)


def _launch(plan: bool, t, fn, args, name, keep, result):
    """The planned call, or the result of launching it now on t's device and its current stream.

    A recording of tensor operations would hold the outputs' allocation without the launch
    that fills them: it is refused."""
    if _is_tracing() or _dispatch_mode(_PROXY) is not None or _before_dispatch.get(0) is not None:
        raise RuntimeError(f"{name}: a trace of tensor operations cannot hold this kernel")
    if plan:
        return _DeviceCall(t, fn, args, name, keep, result)
    device = t.get_device()
    if device == torch._C._cuda_getDevice():
        _lib.check(fn(*args, torch._C._cuda_getCurrentRawStream(device)), name)
    else:
        with torch.cuda.device(device):
            _lib.check(fn(*args, torch._C._cuda_getCurrentRawStream(device)), name)
    return result


def _check(name: str, first: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    """Device tensors of one device that want no gradient."""
    ops._require_device(first)
    index, grad, dual = first.get_device(), torch.is_grad_enabled(), ops._forward_ad._current_level >= 0
    for t in (first, *others):
        if t is None:
            continue
        if t.get_device() != index:
            ops._require_device(t)
            raise ValueError(f"{name}: the operands lie on different devices: {first.device} and {t.device}")
        if dual or (grad and t.requires_grad):
            _check_gradient(name, t)


def _check_gradient(name: str, t: Optional[torch.Tensor]) -> None:
    if t is None:
        return
    if torch.is_grad_enabled() and t.requires_grad:
        raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad() or give it detached tensors")
    if ops._forward_ad._current_level >= 0 and ops._forward_ad.unpack_dual(t).tangent is not None:
        raise RuntimeError(f"{name} has no forward-mode gradient: give it the primal tensors")


def _pool4(pool: torch.Tensor):
    """(pages, Hkv, page_size, head_dim), (address, {page, head} strides) of a 4-bit pool."""
    shape = pool.shape
    if pool.dtype is not torch.uint8 or len(shape) != 4 or shape[3] not in _HEAD_DIMS:
        raise ValueError("a 4-bit pool is uint8 (pages, Hkv, page_size, 17 D / 16) with D 32, 64 or 128, "
                         f"got {pool.dtype} {tuple(shape)}")
    n, H, P, row = shape
    if P <= 0 or P % 32:
        raise ValueError(f"page_size must be a positive multiple of 32, got {P}")
    page, head, step, one = pool.stride()
    at = pool.data_ptr()
    if one != 1 or step != row or (page | head | at) & 15:
        raise ValueError("a page's head must be contiguous and all of them 16-byte aligned")
    return (n, H, P, _HEAD_DIMS[row]), (at, _int64s(page, head))


@lru_cache(maxsize=1024)  # of a program's few layouts: making one takes as long as a launch's other arguments
def _int64s(*values: int) -> ctypes.Array:
    return (ctypes.c_int64 * len(values))(*values)


def _strides2(t: torch.Tensor):
    return _int64s(*t.stride()[:2])


_OUTER = {torch.bfloat16: 7, torch.float32: 3}  # strides of which are whole 16 bytes


def _rows(t: torch.Tensor, out: Optional[str] = None):
    """(tensor, address, outer strides) of rows as the kernels read them, a copy where t's own
    are not; of an output, ``out`` its name, an error."""
    *outer, last = t.stride()
    at, odd = t.data_ptr(), 0
    for s in outer:
        odd |= s
    if last != 1 or at & 15 or odd & _OUTER[t.dtype]:
        if out is not None:
            ops._rows_out(t, out)
        t = t.clone(memory_format=torch.contiguous_format)  # (contiguous() gives t itself where only its address is off)
        at, outer = t.data_ptr(), t.stride()[:-1]
    return t, at, _int64s(*outer)


def _i32(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype is torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()


def _table(table: torch.Tensor, B: int):
    """(tensor, address, stride, columns)"""
    shape = table.shape
    if len(shape) != 2 or shape[0] != B:
        raise ValueError(f"a block table must be (B={B}, pages per sequence), got {tuple(shape)}")
    if shape[1] > _MOST:
        raise ValueError(f"a block table has fewer than 2^31 columns, got {shape[1]}")
    table = _i32(table)
    return table, table.data_ptr(), table.stride(0), shape[1]


def _lens(lens: torch.Tensor, B: int, name: str = "lens") -> torch.Tensor:
    lens = _i32(lens)
    if lens.numel() != B:
        raise ValueError(f"{name} must hold one number per sequence ({B}), got shape {tuple(lens.shape)}")
    return lens


def _overlap(t: torch.Tensor, out: torch.Tensor) -> bool:
    """Whether numbers t, read where they lie (not by a copy of them), share memory with out."""
    if t.dtype is not torch.int32 or not t.is_contiguous():
        return False
    a, b = t.data_ptr(), out.data_ptr()
    return a < b + out.nbytes and b < a + t.nbytes


def _at(t: Optional[torch.Tensor]):
    """The address of an operand that may be left out."""
    return None if t is None else _memory(t)


def _sizes(name: str, *sizes: int) -> None:
    n = 1
    for s in sizes:
        n *= s
    if n > _MOST:
        raise ValueError(f"{name}: more than 2^31 - 1 rows in one call")


def kv4_empty_pool(num_pages: int, num_kv_heads: int, page_size: int, head_dim: int, device="cuda") -> torch.Tensor:
    """An uninitialised 4-bit pool (num_pages, num_kv_heads, page_size, 17 head_dim / 16)."""
    if 17 * head_dim // 16 not in _HEAD_DIMS or head_dim % 32:
        raise ValueError(f"head_dim must be 32, 64 or 128, got {head_dim}")
    pool = torch.empty(num_pages, num_kv_heads, page_size, 17 * head_dim // 16, dtype=torch.uint8, device=device)
    _pool4(pool)
    return pool


def kv4_append(k: torch.Tensor, v: torch.Tensor, pool: torch.Tensor, block_table: torch.Tensor, *,
               q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
               q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
               eps: float = 1e-6, cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
               position_ids: Optional[torch.Tensor] = None, pos_offset: int = 0,
               pos_base: Optional[torch.Tensor] = None, pos_shift: Optional[torch.Tensor] = None,
               row_offset: int = 0, row_base: Optional[torch.Tensor] = None,
               lens_out: Optional[torch.Tensor] = None, plan: bool = False):
    """Store K (QK-Norm + RoPE of k) and V rows in 4-bit pages; q's rows in the same launch.

    k/v: (B, Hkv, S, D) bf16 or fp32, any (b, h, s) strides.  Token s of sequence b is row
    ``row_base[b] + s`` (else ``row_offset + s``).  k_weight None skips the norm, cos/sin
    None the rotation.  Positions: ``position_ids``, else ``pos_base[b] + s``, else
    ``pos_offset + s``, plus ``pos_shift[b]`` where given (rows evicted so far).  q: (B, Hq,
    S, D), normed with q_weight and rotated alike into ``q_out`` (by default fresh), the
    operand of ``attention_decode_kv4``.  ``lens_out`` (int32 (B,), none of the inputs)
    receives ``row_base[b] + S``.  Everything up to the codes is fp32: a row is rounded once.

    A sequence whose rows lie outside its table's pages stores nothing and keeps its length
    in ``lens_out``; rows whose page is not one of the pool's are not stored.
    Returns q_out (None without q), or with ``plan=True`` a KernelCall.
    """
    _check("kv4_append", k, v, pool, block_table, q, q_out, pos_base, pos_shift, row_base, lens_out)
    if torch.is_grad_enabled() or ops._forward_ad._current_level >= 0:
        for t in (q_weight, k_weight, cos, sin):  # which may lie on other devices
            _check_gradient("kv4_append", t)
    (n, H, P, D), pages = _pool4(pool)
    shape = k.shape
    if len(shape) != 4 or shape != v.shape or shape[1] != H or shape[3] != D:
        raise ValueError(f"k {tuple(shape)} and v {tuple(v.shape)} must be (B, {H}, S, {D}), as the pool")
    if k.dtype is not v.dtype or (q is not None and q.dtype is not k.dtype):
        raise TypeError("k, v and q must share one dtype")
    dt = ops._code(k)
    B, _, S, _ = shape
    Hq, q_rows, q_to = 0, (None, None, None), (None, None, None)
    if q is None and (q_out is not None or q_weight is not None):
        raise ValueError("q_out and q_weight go with q")
    if q is not None:
        if q.dim() != 4 or (q.shape[0], q.shape[2], q.shape[3]) != (B, S, D):
            raise ValueError(f"q must be (B={B}, Hq, S={S}, D={D}), got {tuple(q.shape)}")
        Hq = q.shape[1]
        if q_out is None:
            q_out = torch.empty(B, S, Hq, D, dtype=q.dtype, device=q.device).transpose(1, 2)
        elif q_out.shape != q.shape or q_out.dtype != q.dtype:
            raise ValueError("q_out must match q in shape and dtype")
        q_rows, q_to = _rows(q), _rows(q_out, "q_out")
    bt, bt_at, bt_stride, cols = _table(block_table, B)
    if row_base is None and not 0 <= row_offset <= min(cols * P, _MOST) - S:
        raise ValueError(f"rows {row_offset} .. {row_offset + S - 1} lie outside the block table's {min(cols * P, _MOST)}")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    if lens_out is not None:
        if row_base is None:
            raise ValueError("lens_out goes with row_base")
        if lens_out.dtype != torch.int32 or not lens_out.is_contiguous() or lens_out.numel() != B:
            raise ValueError("lens_out must be a contiguous int32 tensor of B elements")
        if B and any(t is not None and _overlap(t, lens_out) for t in (row_base, pos_base, pos_shift)):
            raise ValueError("lens_out must not share memory with row_base, pos_base or pos_shift")
    for w, what in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None and w.numel() != D:
            raise ValueError(f"{what} must hold {D} elements, got {tuple(w.shape)}")
    cos_t = sin_t = pos = qw = kw = None
    max_pos = 0
    if cos is not None:
        dev = k.device
        cos_t, sin_t, max_pos = ops._tables(cos, sin, dev)
        if cos_t.shape[1] != D // 2:
            raise ValueError(f"the tables must be (max_pos, {D // 2}), got {tuple(cos_t.shape)}")
        pos = ops._positions(position_ids, pos_offset, pos_base, B, S, max_pos, dev)  # a shift only adds to them
    if B == 0 or S == 0:
        return q_out
    _sizes("kv4_append", B, S, Hq + 2 * H)
    pb = None if pos_base is None else _lens(pos_base, B, "pos_base")
    ps = None if pos_shift is None else _lens(pos_shift, B, "pos_shift")
    rb = None if row_base is None else _lens(row_base, B, "row_base")
    if q_weight is not None:
        qw, flag = ops._norm_weight(q_weight, k.device, dt, _lib.NQ_QWEIGHT_BF16, plan)
        dt |= flag
    if k_weight is not None:
        kw, flag = ops._norm_weight(k_weight, k.device, dt & ~_lib.NQ_QWEIGHT_BF16, _lib.NQ_KWEIGHT_BF16, plan)
        dt |= flag
    k_rows, v_rows = _rows(k), _rows(v)
    args = (*k_rows[1:], *v_rows[1:], *q_rows[1:], *q_to[1:], *pages, n, bt_at, bt_stride, cols, P, B, S, Hq, H, D, dt,
            _at(qw), _at(kw), float(eps), _at(cos_t), _at(sin_t), max_pos, _at(pos), _at(pb), _at(ps),
            int(pos_offset), _at(rb), int(row_offset), _at(lens_out))
    return _launch(plan, k, _lib.load().nq_kv4_append, args, "nq_kv4_append",
                   (k_rows[0], v_rows[0], q_rows[0], pool, bt, qw, kw, cos_t, sin_t, pos, pb, ps, rb, lens_out), q_out)


def kv4_gather(pool: torch.Tensor, block_table: torch.Tensor, *, S: int, row_offset: int = 0,
               row_base: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16,
               k_out: Optional[torch.Tensor] = None, v_out: Optional[torch.Tensor] = None, plan: bool = False):
    """Rows ``row_base[b] + s`` (else ``row_offset + s``), s < S, of 4-bit pages as (k, v).

    (B, Hkv, S, D) in ``dtype`` (bf16 or fp32, exact in both), by default fresh; ``k_out`` and
    ``v_out`` may be views of larger buffers.  Rows without a page come back as NaN.
    """
    _check("kv4_gather", pool, block_table, row_base, k_out, v_out)
    (n, H, P, D), pages = _pool4(pool)
    B = block_table.shape[0]
    bt, bt_at, bt_stride, cols = _table(block_table, B)
    if S < 0 or (row_base is None and not 0 <= row_offset <= min(cols * P, _MOST) - S):
        raise ValueError(f"rows {row_offset} .. {row_offset + S - 1} lie outside the block table's {min(cols * P, _MOST)}")
    if dtype not in _OUTER:
        raise TypeError(f"unsupported dtype {dtype}; rows are read back as bfloat16 or float32")
    shape = (B, H, S, D)
    for name, t in (("k_out", k_out), ("v_out", v_out)):
        if t is not None and (tuple(t.shape) != shape or t.dtype != dtype):
            raise ValueError(f"{name} must be {shape} in {dtype}, got {tuple(t.shape)} in {t.dtype}")
    k = torch.empty(B, H, S, D, dtype=dtype, device=pool.device) if k_out is None else k_out
    v = torch.empty_like(k, memory_format=torch.contiguous_format) if v_out is None else v_out
    k_rows, v_rows = _rows(k, "k_out"), _rows(v, "v_out")
    if 0 in shape:
        return k, v
    _sizes("kv4_gather", B, S, H)
    rb = None if row_base is None else _lens(row_base, B, "row_base")
    args = (*pages, n, bt_at, bt_stride, cols, P, *k_rows[1:], *v_rows[1:], B, S, H, D, ops._code(k), _at(rb),
            int(row_offset))
    return _launch(plan, pool, _lib.load().nq_kv4_gather, args, "nq_kv4_gather", (pool, bt, rb), (k, v))


def attention_decode_kv4(q: torch.Tensor, pool: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor, *,
                         max_len: int, sm_scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                         return_lse: bool = False, workspace: Optional[torch.Tensor] = None, plan: bool = False):
    """Single-token GQA attention over keys [0, lens[b]) of 4-bit pages.

    q: (B, Hq, D) or (B, Hq, 1, D) bf16 or fp32, normed and rotated (``kv4_append``'s q_out).
    ``max_len`` bounds the lengths; the block table must map every page up to it.  Returns
    (B, Hq, D) in q's type, with ``return_lse`` also the fp32 (B, Hq) log-sum-exp of the
    scaled scores.  A sequence without keys gives zeros and -inf, one whose length lies
    outside [0, max_len], or whose pages are not the pool's, NaN.  Products are exact in the
    stored values; bf16 q rounds the probabilities to bf16, fp32 q keeps 24 bits of both.
    ``workspace``: a contiguous buffer of ``nq_attn_decode_kv4_workspace_bytes``, for one call
    at a time; by default a fresh one where the call needs it.
    """
    _check("attention_decode_kv4", q, pool, block_table, lens, out, workspace)
    (n, H, P, D), pages = _pool4(pool)
    if q.dim() == 4 and q.shape[2] == 1:
        q = q[:, :, 0]
    shape = q.shape
    if len(shape) != 3 or shape[2] != D or shape[1] == 0 or shape[1] % H:
        raise ValueError(f"q must be (B, Hq, {D}) with Hq a multiple of the pool's {H} heads, got {tuple(shape)}")
    B, Hq, _ = shape
    dt = ops._code(q)
    bt, bt_at, bt_stride, cols = _table(block_table, B)
    if not 0 < max_len <= cols * P or max_len > _MOST_KEYS:
        raise ValueError(f"max_len must be in [1, {min(cols * P, _MOST_KEYS)}] (block table columns x page_size, 2^30), "
                         f"got {max_len}")
    dev = q.device
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != shape or out.dtype != q.dtype:
        raise ValueError(f"out must be {tuple(shape)} in {q.dtype}")
    out_rows = _rows(out, "out")
    lse = torch.empty(B, Hq, dtype=torch.float32, device=dev) if return_lse else None
    if B == 0:
        return (out, lse) if return_lse else out
    _sizes("attention_decode_kv4", B, H, -(-Hq // H // 16) + 1)
    lens_t = _lens(lens, B)
    q_rows = _rows(q)
    lib = _lib.load()
    if workspace is None:
        need = lib.nq_attn_decode_kv4_workspace_bytes(B, Hq, H, D, int(max_len))
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    elif not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    args = (*q_rows[1:], *pages, n, bt_at, bt_stride, cols, P, lens_t.data_ptr(), *out_rows[1:], ops._ptr(lse),
            _at(workspace), 0 if workspace is None else workspace.nbytes, B, Hq, H, D, int(max_len), dt, 0.0 if sm_scale is None else float(sm_scale))
    return _launch(plan, q, lib.nq_attn_decode_kv4, args, "nq_attn_decode_kv4", (q_rows[0], pool, bt, lens_t, workspace),
                   (out, lse) if return_lse else out)


def attention_key_weights(q: torch.Tensor, k_pool: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
                          lse: torch.Tensor, *, max_len: int, weights: Optional[torch.Tensor] = None,
                          causal: bool = True, sm_scale: Optional[float] = None, plan: bool = False):
    """The attention weight that each cached key got, (B, Hkv, max_len) fp32.

    Key t of sequence b and kv head h: the sum of ``exp(scale q . k_t - lse)`` over the query
    heads of h and the queries that see t.  q: (B, Hq, S, D) bf16 as attended (normed and
    rotated), the last S of the sequence's ``lens[b]`` tokens, ``causal`` or all seeing all;
    lse: the (B, Hq, S) (or, S = 1, (B, Hq)) fp32 log-sum-exp their attention returned (-inf:
    the query saw nothing and adds nothing, whatever it holds).  k_pool: 4-bit pages or bf16
    K pages (pages, Hkv, page_size, D).  Keys from lens[b] on get 0.  With ``weights`` the sums
    are added to its first max_len entries a head and it is returned.  More than 256 rows (queries
    times query heads of a kv head) take a workspace of 4 bytes a key, kv head and 256 of them:
    32768 queries over as many keys, 64/4 heads, 1.07 GB.
    """
    _check("attention_key_weights", q, k_pool, block_table, lens, lse, weights)
    four = k_pool.dtype is torch.uint8
    if four:
        (n, H, P, D), pages = _pool4(k_pool)
    else:
        ops._pool_check(k_pool, "k_pool")
        n, H, P, D = k_pool.shape
        if k_pool.dtype != torch.bfloat16:
            raise TypeError(f"k_pool must be bfloat16 or a 4-bit pool, got {k_pool.dtype}")
        if P <= 0 or P % 32:
            raise ValueError(f"page_size must be a positive multiple of 32, got {P}")
        pages = k_pool.data_ptr(), _int64s(*k_pool.stride()[:3])
    if q.dtype is not torch.bfloat16:
        raise TypeError(f"q must be bfloat16, got {q.dtype}")
    shape = q.shape
    if len(shape) != 4 or shape[3] != D or shape[1] == 0 or shape[1] % H:
        raise ValueError(f"q must be (B, Hq, S, {D}) with Hq a multiple of the pool's {H} heads, got {tuple(shape)}")
    B, Hq, S, _ = shape
    if lse.dtype is not torch.float32 or tuple(lse.shape) not in ((B, Hq, S), (B, Hq)) or lse.numel() != B * Hq * S:
        raise ValueError(f"lse must be fp32 {(B, Hq, S)}, got {lse.dtype} {tuple(lse.shape)}")
    bt, bt_at, bt_stride, cols = _table(block_table, B)
    if not 0 < max_len <= cols * P or max_len > _MOST_KEYS:
        raise ValueError(f"max_len must be in [1, {min(cols * P, _MOST_KEYS)}] (block table columns x page_size, 2^30), "
                         f"got {max_len}")
    add = weights is not None
    if not add:
        weights = torch.empty(B, H, max_len, dtype=torch.float32, device=q.device)
    else:
        _check_weights(weights, B, H, max_len)
        (s0, n0), (s1, n1) = sorted(((weights.stride(0), B), (weights.stride(1), H)))
        if (n0 > 1 and s0 < max_len) or (n1 > 1 and s1 < (s0 * (n0 - 1) + max_len if n0 > 1 else max_len)):
            raise ValueError("weights of one head must not be another's: they are added to at once")
    if B == 0 or S == 0:
        return weights if add else weights.zero_()
    _sizes("attention_key_weights", B, Hq, S)
    lens_t = _lens(lens, B)
    _, head, token, _ = q.stride()
    if head * (Hq // H) > _MOST_REACH or token * 257 > _MOST_REACH:  # tokens first: rows as near as they go
        q = q.transpose(1, 2).clone(memory_format=torch.contiguous_format).transpose(1, 2)
    q_rows, lse = _rows(q), lse.contiguous()
    lib = _lib.load()
    need = lib.nq_key_weights_workspace_bytes(B, Hq, H, S, int(max_len))
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    args = (*q_rows[1:], *pages, int(four), n, bt_at, bt_stride, cols, P, lens_t.data_ptr(), lse.data_ptr(),
            weights.data_ptr(), _strides2(weights), int(add), ops._ptr(ws), need, B, Hq, H, S, D, int(max_len),
            int(bool(causal)), 0.0 if sm_scale is None else float(sm_scale))
    return _launch(plan, q, lib.nq_key_weights, args, "nq_key_weights", (q_rows[0], k_pool, bt, lens_t, lse, ws), weights)


def _check_weights(weights: torch.Tensor, B: int, H: int, least: int) -> None:
    if (weights.dtype != torch.float32 or weights.dim() != 3 or tuple(weights.shape[:2]) != (B, H)
            or weights.shape[2] < least or (weights.shape[2] > 1 and weights.stride(2) != 1)):
        raise ValueError(f"weights must be fp32 ({B}, {H}, at least {least}) with contiguous keys, "
                         f"got {weights.dtype} {tuple(weights.shape)}")


def select_keys(weights: torch.Tensor, lens: torch.Tensor, *, keep: int, recent: int = 0, first: int = 0,
                plan: bool = False):
    """The cached rows that each kv head keeps, int32 (B, Hkv, keep) in ascending order.

    weights: (B, Hkv, W) fp32; lens: the sequences' lengths, at most W.  Kept are the first
    ``first`` rows, the last ``recent`` and, of those in between, the heaviest; equal weights
    by the lower index, NaN above every number.  A sequence of no more than ``keep`` rows keeps
    them all, with -1 behind them.
    """
    _check("select_keys", weights, lens)
    if weights.dim() != 3:
        raise ValueError(f"weights must be (B, Hkv, W), got {tuple(weights.shape)}")
    B, H, W = weights.shape
    _check_weights(weights, B, H, 1)
    if keep <= 0 or recent < 0 or first < 0 or recent + first > keep or max(keep, W) > _MOST_KEYS:
        raise ValueError(f"keep must be positive and hold first + recent, got {keep}, {first} and {recent}, "
                         f"and neither it nor the weights' {W} pass 2^30")
    lens_t = _lens(lens, B)
    kept = torch.empty(B, H, keep, dtype=torch.int32, device=weights.device)
    if B == 0 or H == 0:
        return kept
    _sizes("select_keys", B, H)
    args = (ops._ptr(weights), _strides2(weights), ops._ptr(lens_t), ops._ptr(kept), B, H, W, int(keep), int(recent),
            int(first))
    return _launch(plan, weights, _lib.load().nq_select_keys, args, "nq_select_keys", (weights, lens_t), kept)


def kv_compact(pools: Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]], block_table: torch.Tensor,
               new_table: torch.Tensor, kept: torch.Tensor, *, weights: Optional[torch.Tensor] = None,
               plan: bool = False):
    """Move row ``kept[b, h, i]`` of each sequence to row i of its new pages, in the same pool.

    pools: a 4-bit pool, or (k_pool, v_pool) of bf16 or fp32 pages.  The new pages must be none
    of those that any sequence's kept rows lie in (what they hold is overwritten while these
    are read), and each one's own.  ``kept`` as ``select_keys`` gives it; -1 moves nothing, and
    rows of the new pages behind the last one moved are left as they are.  With ``weights``
    (B, Hkv, W >= keep) returns a fresh tensor of that shape with the kept rows' weights and 0
    behind them, else None.
    """
    four = isinstance(pools, torch.Tensor)
    k_pool, v_pool = (pools, None) if four else pools
    _check("kv_compact", k_pool, v_pool, block_table, new_table, kept, weights)
    if four:
        (n, H, P, D), (_, ks) = _pool4(k_pool)
        vs, row = None, 0
    else:
        for name, pool in (("k_pool", k_pool), ("v_pool", v_pool)):
            ops._pool_check(pool, name)
            ops._code(pool)
        if k_pool.shape != v_pool.shape or k_pool.dtype != v_pool.dtype:
            raise ValueError(f"the pools differ: {tuple(k_pool.shape)} {k_pool.dtype} and {tuple(v_pool.shape)} {v_pool.dtype}")
        n, H, P, D = k_pool.shape
        if P <= 0 or P % 32:
            raise ValueError(f"page_size must be a positive multiple of 32, got {P}")
        e = k_pool.element_size()
        ks, vs = (_int64s(*(x * e for x in t.stride()[:3])) for t in (k_pool, v_pool))
        row = D * e
    if kept.dtype != torch.int32 or kept.dim() != 3 or kept.shape[1] != H:
        raise ValueError(f"kept must be int32 (B, {H}, keep), got {kept.dtype} {tuple(kept.shape)}")
    B, _, keep = kept.shape
    bt, bt_at, bt_stride, cols = _table(block_table, B)
    new, new_at, new_stride, new_cols = _table(new_table, B)
    if new_cols * P < keep:
        raise ValueError(f"the new table maps {new_cols * P} rows, {keep} are kept")
    if B and new_at == bt_at:
        raise ValueError("new_table must name other pages than block_table")
    out = None
    if weights is not None:
        _check_weights(weights, B, H, keep)
        _sizes("kv_compact", weights.shape[2])
        out = torch.empty_like(weights, memory_format=torch.contiguous_format)
        if weights.stride() != out.stride():
            weights = weights.contiguous()
    if 0 in kept.shape:
        return out if out is None or out.numel() == 0 else out.zero_()
    _sizes("kv_compact", B, H, keep)
    kept = kept.contiguous()
    args = (_at(k_pool), ks, _at(v_pool), vs, row, D, n, bt_at, bt_stride, cols, new_at, new_stride, new_cols, P, _at(kept),
            _at(weights), _at(out), None if out is None else _strides2(out),
            0 if out is None else out.shape[2], B, H, keep)
    return _launch(plan, k_pool, _lib.load().nq_kv_compact, args, "nq_kv_compact",
                   (k_pool, v_pool, bt, new, kept, weights), out)

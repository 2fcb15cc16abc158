"""Paged-KV cache writer: new latent KV rows -> the paged cache the forward
reads, through the same block tables.

The reference builds its paged caches on the host in its tests
(sparse_attn_sharedkv_tilelang/golden.py:315-408): row ``pos`` of batch ``b``
is stored in physical block ``block_table[b, pos // block_size]`` at offset
``pos % block_size``; ``-1`` marks an unused table entry. This module writes
rows into that layout on the GPU with ``sas_cache_write_v1``, either as a
bf16/fp16 copy or quantised into the 656-byte fp8 rows of
:mod:`dsv4_amd.paged` (``quantize_kv_fp8``'s format and rounding, bit for bit).
"""

from __future__ import annotations

import ctypes as C
import struct
from typing import Optional, Tuple

import torch

from . import _lib, rope

_DT = {torch.bfloat16: _lib.SAS_DT_BF16, torch.float16: _lib.SAS_DT_FP16}
FP8_ROW_BYTES = 656
# the current stream as a hipStream_t value, without a Stream object
_raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)


class PreparedCacheWrite:
    """Arguments of one cache write, validated once; :meth:`launch` runs the
    kernel on the current (or given) stream without host syncs."""

    def __init__(self, args: _lib.SasCacheWriteArgs, keep: list, device):
        self.args = args
        self._keep = keep
        self.device = device
        # the int32 / contiguous conversions were enqueued on this stream
        self._prep_stream = torch.cuda.current_stream(device)

    def launch(self, stream: Optional[torch.cuda.Stream] = None) -> None:
        st = stream if stream is not None else torch.cuda.current_stream(self.device)
        if st != self._prep_stream:
            # order the launch after the conversions, and keep every bound
            # tensor's memory from being reused by the caching allocator on
            # its own stream while the kernel on `st` may still touch it
            ev = torch.cuda.Event()
            ev.record(self._prep_stream)
            st.wait_event(ev)
            for t in self._keep:
                t.record_stream(st)
        _lib.check(_lib.lib().sas_cache_write_v1(C.byref(self.args), C.c_void_p(st.cuda_stream)),
                   "write_kv_cache")


def _i32(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype is torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()


def _bind(kv, cache, block_table, seq_ids, positions):
    """Validate and convert: (launch arguments in SasCacheWriteArgs' order,
    the tensors they point into, device)."""
    if kv.dim() != 2:
        raise ValueError(f"kv must be [N, D], got {tuple(kv.shape)}")
    if kv.dtype not in _DT:
        raise ValueError(f"kv dtype must be bf16 or fp16, got {kv.dtype}")
    if cache.dim() != 4 or cache.shape[2] != 1:
        raise ValueError(f"cache must be [num_blocks, block_size, 1, row], got {tuple(cache.shape)}")
    N, D = kv.shape
    fp8 = cache.dtype == torch.uint8
    if fp8:
        if cache.shape[-1] != FP8_ROW_BYTES or kv.dtype != torch.bfloat16 or D != 576:
            raise ValueError("fp8 cache rows need uint8 [..., 656] and bf16 kv with D = 576")
    elif cache.dtype != kv.dtype or cache.shape[-1] != D:
        raise ValueError("cache must hold rows of kv's dtype and width, or uint8 fp8 rows")
    if block_table.dim() != 2:
        raise ValueError("block_table must be [B, max_blocks]")
    if seq_ids.shape != (N,) or positions.shape != (N,):
        name, t = ("seq_ids", seq_ids) if seq_ids.shape != (N,) else ("positions", positions)
        raise ValueError(f"{name} must be [N] = [{N}], got {tuple(t.shape)}")
    dev = kv.device
    if cache.device != dev or block_table.device != dev or seq_ids.device != dev or positions.device != dev:
        raise ValueError("all tensors must be on kv's device")
    if kv.stride(1) != 1 or not cache.is_contiguous():
        raise ValueError("kv rows and cache must be contiguous")
    bt, sid, pos = _i32(block_table), _i32(seq_ids), _i32(positions)
    nb, bs = cache.shape[0], cache.shape[1]
    return ((kv.data_ptr(), sid.data_ptr(), pos.data_ptr(), bt.data_ptr(), cache.data_ptr(), N, bt.shape[0], D,
             kv.stride(0), bt.shape[1], bs, nb, _DT[kv.dtype],
             _lib.SAS_DT_FP8_E4M3_ROW656 if fp8 else _DT[kv.dtype]), (kv, cache, bt, sid, pos), dev)


def prepare_kv_cache_write(kv: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor,
                           seq_ids: torch.Tensor, positions: torch.Tensor) -> PreparedCacheWrite:
    """Validate the arguments of :func:`write_kv_cache` and bind them."""
    args, keep, dev = _bind(kv, cache, block_table, seq_ids, positions)
    return PreparedCacheWrite(_lib.SasCacheWriteArgs(*args), list(keep), dev)


# SasCacheWriteArgs as packed bytes (five pointers, seven int64, two int32):
# filling the ctypes structure field by field took a third of a small call
_ARGS = struct.Struct("@5Q7q2i")
assert _ARGS.size == C.sizeof(_lib.SasCacheWriteArgs)
_write_raw = None


def _write_bytes():
    """sas_cache_write_v1 taking its arguments as packed bytes."""
    global _write_raw
    if _write_raw is None:
        f = _lib.lib()["sas_cache_write_v1"]   # a function object of its own: other argument types
        f.argtypes = [C.c_char_p, C.c_void_p]
        f.restype = C.c_int
        _write_raw = f
    return _write_raw


def write_kv_cache(kv: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor,
                   seq_ids: torch.Tensor, positions: torch.Tensor,
                   stream: Optional[torch.cuda.Stream] = None) -> None:
    """Scatter ``kv [N, D]`` into ``cache`` on the GPU (no host sync).

    ``cache`` is ``[num_blocks, block_size, 1, D]`` in ``kv``'s dtype (rows
    copied) or uint8 ``[num_blocks, block_size, 1, 656]`` (bf16 ``kv`` with
    D = 576, quantised to fp8 rows). ``seq_ids`` / ``positions`` (int32
    ``[N]``) give each row's batch and logical position; rows whose position
    is negative, or whose block-table entry is -1 or missing, are skipped.
    The rows of one call must go to distinct cache rows.
    """
    if stream is not None or not kv.is_cuda:
        prepare_kv_cache_write(kv, cache, block_table, seq_ids, positions).launch(stream)
        return
    # on the current stream, as any conversion made by _bind
    args, keep, dev = _bind(kv, cache, block_table, seq_ids, positions)
    rc = _write_bytes()(_ARGS.pack(*args), torch.cuda.current_stream(dev).cuda_stream if _raw is None else _raw(dev.index))
    if rc:
        _lib.check(rc, "write_kv_cache")


# what SasCacheAppendArgs puts behind its rope arguments: four pointers, then what
# follows from the geometry
_APPEND_PTRS = struct.Struct("@4Q")
_APPEND_DIMS = struct.Struct("@4q2i")
assert C.sizeof(_lib.SasNormRopeArgs) + _APPEND_PTRS.size + _APPEND_DIMS.size == C.sizeof(_lib.SasCacheAppendArgs)


def append_kv_cache(
    kv: torch.Tensor,
    cache: torch.Tensor,
    block_table: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    seqused_kv: torch.Tensor,
    *,
    table: Optional[torch.Tensor] = None,
    positions: Optional[torch.Tensor] = None,
    norm_dim: Optional[int] = None,
    weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    interleaved: bool = True,
    q: Optional[torch.Tensor] = None,
    q_norm_dim: Optional[int] = None,
    q_weight: Optional[torch.Tensor] = None,
) -> Optional[torch.Tensor]:
    """Append a step's KV rows ``kv [T, D]`` to the paged ``cache``, normed and
    rotated on the way as :func:`dsv4_amd.rope.norm_rope` does it, and, where ``q``
    ``[T, H, D]`` is given, the step's queries in the same launch; returns the queries.

    Rows are packed as the attention's queries are: tokens ``cu_seqlens_q[b] ..
    cu_seqlens_q[b + 1]`` are the last ones of sequence ``b``, whose ``seqused_kv[b]``
    counts them already, so token ``i`` of its ``n`` is written at position
    ``seqused_kv[b] - n + i`` through ``block_table`` and
    :func:`~dsv4_amd.api.sparse_attn_sharedkv` takes the same two tensors next. The
    angles are those of that position, or of ``positions [T]`` (the depths of a
    draft tree's nodes). ``table``, ``norm_dim``, ``weight``, ``eps`` and
    ``interleaved`` are ``norm_rope``'s; so are ``q_norm_dim`` and ``q_weight``.

    ``cache`` is ``[num_blocks, block_size, 1, D]`` in ``kv``'s dtype, or uint8
    ``[num_blocks, block_size, 1, 656]`` (bf16 ``kv`` with D = 576), quantised from
    the fp32 values (NaN and infinities as :func:`dsv4_amd.paged.quantize_kv_fp8`
    has them: a group with one holds a NaN). Tokens behind the last sequence, at
    a negative position or at one outside ``table`` are padding: nothing of the
    cache is written for them and their queries come back as zeros; rows without a
    block are skipped, as by :func:`write_kv_cache`. The rows of one call must go
    to distinct cache rows. No host sync.
    """
    key = (rope._signature(2, q, kv, positions, table, q_norm_dim, q_weight, norm_dim, weight, eps, interleaved, False),
           cache.shape, cache.dtype, cache.get_device(), cache.is_contiguous(),
           block_table.shape, block_table.dtype, block_table.get_device(), block_table.is_contiguous(),
           cu_seqlens_q.shape, cu_seqlens_q.dtype, cu_seqlens_q.get_device(), cu_seqlens_q.is_contiguous(),
           seqused_kv.shape, seqused_kv.dtype, seqused_kv.get_device(), seqused_kv.is_contiguous())
    b = rope._sigs.get(key)
    if b is not None and rope._aligned(q, kv, table, q_weight, weight):
        out = None if q is None else rope._out(q, b.q_like)
        packed = rope._pack_ptrs(q, kv, q_weight, weight, positions, table, out, None)
        rope._launch("sas_cache_append_v1", packed + b.dims + _APPEND_PTRS.pack(
            cu_seqlens_q.data_ptr(), seqused_kv.data_ptr(), block_table.data_ptr(), cache.data_ptr()) + b.extra, b.dev,
            "append_kv_cache")
        return out
    if kv.dim() != 2 or (q is not None and (q.dim() != 3 or q.shape[0] != kv.shape[0] or q.shape[2] != kv.shape[1])):
        raise ValueError(f"kv must be [T, D] and q [T, H, D], got {tuple(kv.shape)}"
                         + ("" if q is None else f" and {tuple(q.shape)}"))
    b = rope._bind(q, kv, positions, table, q_norm_dim, q_weight, norm_dim, weight, eps, interleaved, False, False)
    dev, D = b.dev, kv.shape[1]
    fp8 = cache.dtype == torch.uint8
    if cache.dim() != 4 or cache.shape[2] != 1:
        raise ValueError(f"cache must be [num_blocks, block_size, 1, row], got {tuple(cache.shape)}")
    if fp8:
        if cache.shape[-1] != FP8_ROW_BYTES or kv.dtype != torch.bfloat16 or D != 576:
            raise ValueError("fp8 cache rows need uint8 [..., 656] and bf16 kv with D = 576")
    elif cache.dtype != kv.dtype or cache.shape[-1] != D:
        raise ValueError("cache must hold rows of kv's dtype and width, or uint8 fp8 rows")
    if not cache.is_contiguous():
        raise ValueError("cache must be contiguous")
    B = seqused_kv.numel()
    if seqused_kv.dim() != 1 or cu_seqlens_q.shape != (B + 1,) or block_table.dim() != 2 or block_table.shape[0] != B:
        raise ValueError(f"cu_seqlens_q [B + 1], seqused_kv [B] and block_table [B, max_blocks] must agree, got "
                         f"{tuple(cu_seqlens_q.shape)}, {tuple(seqused_kv.shape)}, {tuple(block_table.shape)}")
    for t in (cache, block_table, cu_seqlens_q, seqused_kv):
        if t.device != dev:
            raise ValueError("all tensors must be on kv's device")
    bt, cu, used = _i32(block_table), _i32(cu_seqlens_q), _i32(seqused_kv)
    out = None if q is None else rope._out(q, b.q_like)
    b.extra = _APPEND_DIMS.pack(B, bt.shape[1], cache.shape[1], cache.shape[0],
                                _lib.SAS_DT_FP8_E4M3_ROW656 if fp8 else _DT[kv.dtype], 0)
    if bt is block_table and cu is cu_seqlens_q and used is seqused_kv:
        rope._keep(key, b, q, kv, positions, table, q_weight, weight, (q_norm_dim, norm_dim, eps, interleaved))
    rope._launch("sas_cache_append_v1", b.ptrs(out, None) + b.dims + _APPEND_PTRS.pack(
        cu.data_ptr(), used.data_ptr(), bt.data_ptr(), cache.data_ptr()) + b.extra, dev, "append_kv_cache")
    return out


# SasCacheEvictArgs as packed bytes: six pointers, nine int64
_EVICT = struct.Struct("@6Q9q")
assert _EVICT.size == C.sizeof(_lib.SasCacheEvictArgs)


def evict_kv_cache(
    cache: torch.Tensor,
    weights: torch.Tensor,
    block_table: torch.Tensor,
    seqused_kv: torch.Tensor,
    *,
    budget: int,
    keep_first: int = 0,
    keep_recent: int = 0,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Cut every sequence of more than ``budget`` cache rows down to that many, in place:
    its first ``keep_first`` rows stay, its last ``keep_recent`` ones, and of the others
    the heaviest by ``weights`` (of equal ones those at the lowest positions; NaN counts
    as the least). Returns ``(seqused_kv, kept)``.

    ``cache [num_blocks, block_size, 1, row]`` holds rows of any type whose size is a
    multiple of 16 bytes; ``weights`` float64 ``[B, R]``
    (:func:`dsv4_amd.api.add_row_weights`), row ``b`` beside row ``b`` of ``block_table``;
    a cache row past ``R`` weighs 0. The rows that stay move together, in their order, to the
    sequence's first ``budget`` positions, their weights with them, and the weights behind
    become 0, ready for the rows that come next; the cache's bytes behind stay as they are. So
    the next step appends at position ``budget`` (:func:`append_kv_cache` with the
    ``positions`` that the tokens' angles belong to) and the attention reads the rows as
    one run (``ori_win_left`` at least the longest sequence), and blocks past the last
    row can be given back.

    ``seqused_kv`` int32 ``[B]`` is the new lengths, ``kept`` int32 ``[B, budget]`` the old
    positions of the rows that stay (-1 past the last): what else is kept by row moves by it.
    A row whose old or new place has no block is not moved. Sequences that share a block (a
    common prefix) must not be evicted from. No host sync.

    Beside compressed rows: the attention finds a token's compressed rows by its position,
    which ``seqused_kv`` gives it, so raw rows of a layer that has compressed ones are not to
    be evicted (their number in ``seqused_kv``'s place hides compressed rows; a window and
    ``ori_first`` bound them). Compressed rows may be, with their own lengths here
    (``seqused_kv // cmp_ratio``, later what the last eviction returned and the rows since):
    the attention goes on with ``seqused_kv`` as it was and ``cmp_sparse_indices`` that name
    rows by their new places (the old row ``kept[b, i]`` is ``i``). Places move forward, so
    the threshold no longer hides a call's own new rows from its earlier tokens: their lists
    leave those out. The attention's dense form, without lists, reads every row up to the
    threshold, also the bytes that an eviction leaves behind: after one, give lists of all
    rows that are left.
    """
    if cache.dim() != 4 or cache.shape[2] != 1 or not cache.is_contiguous():
        raise ValueError(f"cache must be contiguous [num_blocks, block_size, 1, row], got {tuple(cache.shape)}")
    row = cache.shape[3] * cache.element_size()
    B = seqused_kv.numel()
    if seqused_kv.dim() != 1 or block_table.dim() != 2 or block_table.shape[0] != B:
        raise ValueError(f"seqused_kv [B] and block_table [B, max_blocks] must agree, got {tuple(seqused_kv.shape)}, "
                         f"{tuple(block_table.shape)}")
    if weights.dtype is not torch.float64 or weights.dim() != 2 or weights.shape[0] != B or not weights.is_contiguous():
        raise ValueError(f"weights must be contiguous float64 [{B}, rows], got {weights.dtype} {tuple(weights.shape)}")
    for name, v in (("budget", budget), ("keep_first", keep_first), ("keep_recent", keep_recent)):
        if isinstance(v, bool) or not isinstance(v, int):
            raise ValueError(f"{name} must be an integer (got {v!r})")
    if not 1 <= budget <= 1 << 30 or keep_first < 0 or keep_recent < 0 or keep_first + keep_recent > budget:
        raise ValueError(f"budget must be at least 1, at most 2^30, and hold keep_first and keep_recent (got {budget}, {keep_first}, "
                         f"{keep_recent})")
    dev = cache.device
    if weights.device != dev or block_table.device != dev or seqused_kv.device != dev:
        raise ValueError("all tensors must be on cache's device")
    if not cache.is_cuda:
        raise ValueError("evict_kv_cache runs on the GPU: cache must be a device tensor")
    bt, used = _i32(block_table), _i32(seqused_kv)
    left = torch.empty_like(used)
    kept = used.new_empty((B, budget))
    rope._launch("sas_cache_evict_v1", _EVICT.pack(
        cache.data_ptr(), weights.data_ptr(), bt.data_ptr(), used.data_ptr(), left.data_ptr(), kept.data_ptr(), B, row,
        bt.shape[1], cache.shape[1], cache.shape[0], weights.shape[1], budget, keep_first, keep_recent), dev,
        "evict_kv_cache")
    return left, kept

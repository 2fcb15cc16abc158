"""Norms of queries and KV rows for each head with the rotation by position in
the same pass: what a layer does to its projections before
:func:`dsv4_amd.api.sparse_attn_sharedkv` reads them, and (``inverse``) to its
output after. The reference's operator starts from rows that are normed and
rotated already (sparse_attn_sharedkv_tilelang/api.py:129-153); here they can be
made by one kernel, differentiated, and with
:func:`dsv4_amd.cache.append_kv_cache` written straight into the paged cache.
"""

from __future__ import annotations

import ctypes as C
import struct
from typing import Optional, Tuple, Union

import torch

from . import _lib

_DT = {torch.bfloat16: _lib.SAS_DT_BF16, torch.float16: _lib.SAS_DT_FP16}
_raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)

# SasNormRopeArgs as packed bytes: eight pointers, then what follows from a call's
# geometry (seven int64, six int32, eps, reserved), kept per signature; the
# backward and the append put theirs behind it. (ctypes structures filled field by
# field, and every check made anew, took a small call 12.5 us of host time, 7.5 now.)
_PTRS = struct.Struct("@8Q")
_DIMS = struct.Struct("@7q6ifi")
_GRAD_PTRS = struct.Struct("@6QQQ")
_GRAD_STRIDES = struct.Struct("@3q")
assert _PTRS.size + _DIMS.size == C.sizeof(_lib.SasNormRopeArgs)
assert _PTRS.size + _DIMS.size + _GRAD_PTRS.size + _GRAD_STRIDES.size == C.sizeof(_lib.SasNormRopeBwdArgs)
_raw_fns = {}
_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _bytes_fn(name: str):
    """An entry point taking its arguments as packed bytes."""
    f = _raw_fns.get(name)
    if f is None:
        f = _lib.lib()[name]   # a function object of its own: other argument types
        f.argtypes = [C.c_char_p, C.c_void_p]
        f.restype = C.c_int
        _raw_fns[name] = f
    return f


def _launch(name: str, packed: bytes, dev: torch.device, what: str) -> None:
    """Queue a launch on ``dev``'s current stream."""
    f = _raw_fns.get(name) or _bytes_fn(name)
    index = dev.index
    stream = torch.cuda.current_stream(dev).cuda_stream if _raw is None else _raw(index)
    if index == _device():
        rc = f(packed, stream)
    else:
        with torch.cuda.device(dev):
            rc = f(packed, stream)
    if rc:
        _lib.check(rc, what)


def rope_table(num_positions: int, rope_dim: int = 64, base: float = 10000.0, *,
               device: Union[str, torch.device] = "cuda") -> torch.Tensor:
    """The (cos, sin) pairs of positions ``0 .. num_positions - 1``: fp32
    ``[num_positions, rope_dim / 2, 2]``, pair ``i`` of position ``p`` at the angle
    ``p / base^(2 i / rope_dim)``, computed in 64 bits. Any tensor of this shape
    serves as ``table`` (scaled or interpolated angles, say)."""
    if num_positions < 1 or rope_dim < 2 or rope_dim % 2:
        raise ValueError(f"rope_table needs num_positions >= 1 and an even rope_dim (got {num_positions}, {rope_dim})")
    f = float(base) ** (-torch.arange(0, rope_dim, 2, dtype=torch.float64, device=device) / rope_dim)
    a = torch.arange(num_positions, dtype=torch.float64, device=device)[:, None] * f
    return torch.stack([a.cos(), a.sin()], -1).to(torch.float32)


def _i32(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype is torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as the kernels take it: unit channel stride, rows on 16-byte
    boundaries (16-bit elements); a copy where it is not."""
    s = t.stride()
    if s[-1] == 1 and not t.data_ptr() % 16 and not any(x % 8 for x in s[:-1]):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _norm(name: str, n: Optional[int], w: Optional[torch.Tensor], x: torch.Tensor):
    """(norm channels, the weight as the kernels take it or None)."""
    n = x.shape[-1] if n is None else int(n)
    if w is not None:
        if w.shape != (n,):
            raise ValueError(f"{name}_weight must be [{n}], got {tuple(w.shape)}")
        if w.dtype is not torch.float32 and w.dtype is not x.dtype:
            raise ValueError(f"{name}_weight must be fp32 or {x.dtype}, got {w.dtype}")
        if w.device != x.device:
            raise ValueError("all tensors must be on one device")
        if n == 0:
            w = None
        elif not w.is_contiguous() or w.data_ptr() % 16:
            w = w.clone(memory_format=torch.contiguous_format)
    return n, w


def _table(table: Optional[torch.Tensor], positions: Optional[torch.Tensor], x: torch.Tensor, need_positions: bool):
    """(table, its rows, rotated channels, positions) checked against the rows ``x``."""
    if table is None:
        return None, 0, 0, None
    if table.dim() != 3 or table.shape[2] != 2 or table.dtype is not torch.float32 or table.shape[0] < 1:
        raise ValueError(f"table must be fp32 [num_positions, rope_dim / 2, 2], got {table.dtype} {tuple(table.shape)}")
    if table.device != x.device:
        raise ValueError("all tensors must be on one device")
    if not table.is_contiguous() or table.data_ptr() % 16:
        table = table.clone(memory_format=torch.contiguous_format)
    if positions is None:
        if need_positions:
            raise ValueError("positions are needed with a table")
    else:
        if positions.device != x.device:
            raise ValueError("all tensors must be on one device")
        if positions.dtype.is_floating_point or positions.dtype.is_complex or positions.dtype is torch.bool:
            raise ValueError(f"positions must be integers, got {positions.dtype}")
        if positions.dtype is torch.int64:   # (one past 32 bits stays outside the table)
            positions = positions.clamp(-1, 2 ** 31 - 1)
        positions = _i32(positions)
    return table, table.shape[0], 2 * table.shape[1], positions


class _Bound:
    """Checked arguments of one call: the tensors as the kernels take them, and
    what follows from their geometry, packed behind the pointers (``dims``)."""

    __slots__ = ("q", "kv", "qw", "kw", "table", "pos", "dims", "dev", "lead", "q_like", "kv_like", "extra")

    def ptrs(self, q_out, kv_out) -> bytes:
        return _pack_ptrs(self.q, self.kv, self.qw, self.kw, self.pos, self.table, q_out, kv_out)


def _pack_ptrs(q, kv, qw, kw, pos, table, q_out, kv_out) -> bytes:
    return _PTRS.pack(0 if q is None else q.data_ptr(), 0 if kv is None else kv.data_ptr(),
                      0 if qw is None else qw.data_ptr(), 0 if kw is None else kw.data_ptr(),
                      0 if pos is None else pos.data_ptr(), 0 if table is None else table.data_ptr(),
                      0 if q_out is None else q_out.data_ptr(), 0 if kv_out is None else kv_out.data_ptr())


# Resolutions of the signatures seen (geometry, types and scalars alone: no address, no
# tensor), of calls whose tensors are taken as given; dropped together when full.
_SIGS_MAX = 256
_sigs = {}


def _signature(what, q, kv, positions, table, q_norm_dim, q_weight, kv_norm_dim, kv_weight, eps, interleaved, inverse):
    return (what, None if q is None else (q.shape, q.stride(), q.dtype, q.get_device()),
            None if kv is None else (kv.shape, kv.stride(), kv.dtype, kv.get_device()),
            None if positions is None else (positions.shape, positions.dtype, positions.is_contiguous(), positions.get_device()),
            None if table is None else (table.shape, table.dtype, table.is_contiguous(), table.get_device()),
            q_norm_dim, kv_norm_dim,
            None if q_weight is None else (q_weight.shape, q_weight.dtype, q_weight.stride(), q_weight.get_device()),
            None if kv_weight is None else (kv_weight.shape, kv_weight.dtype, kv_weight.stride(), kv_weight.get_device()),
            eps, interleaved, inverse)


def _aligned(*tensors) -> bool:
    a = 0
    for t in tensors:
        if t is not None:
            a |= t.data_ptr()
    return not a & 15


_SCALARS = (int, float, bool, type(None))


def _keep(key, b: _Bound, q, kv, positions, table, q_weight, kv_weight, scalars) -> None:
    """Keep what a call's geometry gives, where its tensors were taken as given
    (positions too: without a table they were not looked at) and its scalars are
    plain ones (a tensor would be found again by its identity)."""
    if (b.q is not q or b.kv is not kv or b.table is not table or b.pos is not positions
            or b.qw is not q_weight or b.kw is not kv_weight or any(type(x) not in _SCALARS for x in scalars)):
        return
    if len(_sigs) >= _SIGS_MAX:
        _sigs.clear()
    kept = _Bound()
    kept.q = kept.kv = kept.qw = kept.kw = kept.table = kept.pos = None
    kept.dims, kept.dev, kept.lead, kept.q_like, kept.kv_like, kept.extra = b.dims, b.dev, b.lead, b.q_like, b.kv_like, b.extra
    _sigs[key] = kept


def _out(t: torch.Tensor, like: bool) -> torch.Tensor:
    """A new contiguous tensor of t's geometry."""
    return torch.empty_like(t) if like else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _bind(q, kv, positions, table, q_norm_dim, q_weight, kv_norm_dim, kv_weight, eps, interleaved, inverse,
          need_positions=True) -> _Bound:
    x = q if q is not None else kv
    if x is None:
        raise ValueError("q or kv is needed")
    if x.dtype not in _DT:
        raise ValueError(f"q and kv must be bf16 or fp16, got {x.dtype}")
    b = _Bound()
    b.dev = dev = x.device
    if dev.type != "cuda":
        raise ValueError("norm_rope runs on the GPU: q and kv must be device tensors")
    lead = tuple(q.shape[:-2]) if q is not None else tuple(kv.shape[:-1])
    b.lead = lead
    D = x.shape[-1]
    T = 1
    for n in lead:
        T *= n
    H = qt = qh = kt = 0
    if q is not None:
        if q.dim() < 3:
            raise ValueError(f"q must be [..., H, D], got {tuple(q.shape)}")
        H = q.shape[-2]
        if H < 1:
            raise ValueError("q needs at least one head")
        b.q = _rows(q if q.dim() == 3 else q.reshape(T, H, D))
        qt, qh, _ = b.q.stride()
    else:
        b.q = None
    if kv is not None:
        if kv.dtype is not x.dtype or kv.device != dev or kv.shape != (*lead, D):
            raise ValueError(f"kv must be {x.dtype} {(*lead, D)} on {dev}, got {kv.dtype} {tuple(kv.shape)} on {kv.device}")
        b.kv = _rows(kv if kv.dim() == 2 else kv.reshape(T, D))
        kt = b.kv.stride(0)
    else:
        b.kv = None
    qn = kn = 0
    b.qw = b.kw = None
    if q is not None:
        qn, b.qw = _norm("q", q_norm_dim, q_weight, x)
    if kv is not None:
        kn, b.kw = _norm("kv", kv_norm_dim, kv_weight, x)
    wf32 = True
    if b.qw is not None or b.kw is not None:
        a = b.qw if b.qw is not None else b.kw
        if b.qw is not None and b.kw is not None and b.qw.dtype is not b.kw.dtype:
            raise ValueError("q_weight and kv_weight must have one dtype")
        wf32 = a.dtype is torch.float32
    b.table, table_rows, R, b.pos = _table(table, positions, x, need_positions)
    if b.pos is not None and b.pos.shape != lead:
        raise ValueError(f"positions must be {lead}, got {tuple(b.pos.shape)}")
    b.q_like, b.kv_like = q is not None and q.is_contiguous(), kv is not None and kv.is_contiguous()
    b.extra = None
    b.dims = _DIMS.pack(T, H, D, qt, qh, kt, table_rows, R, qn, kn, _DT[x.dtype],
                        _lib.SAS_DT_FP32 if wf32 else _DT[x.dtype],
                        (0 if interleaved else _lib.SAS_ROPE_HALF) | (_lib.SAS_ROPE_INVERSE if inverse else 0), float(eps), 0)
    return b


def norm_rope(
    q: Optional[torch.Tensor],
    kv: Optional[torch.Tensor] = None,
    *,
    positions: Optional[torch.Tensor] = None,
    table: Optional[torch.Tensor] = None,
    q_norm_dim: Optional[int] = None,
    q_weight: Optional[torch.Tensor] = None,
    kv_norm_dim: Optional[int] = None,
    kv_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    interleaved: bool = True,
    inverse: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """RMS norms of the query heads and KV rows, and their rotation by position.

    ``q`` ``[..., H, D]`` and ``kv`` ``[..., D]`` (bf16 or fp16; either may be None)
    share their leading dims, ``positions``'s. Every head of ``q`` is a row. Its
    first ``q_norm_dim`` channels (None: all of them, 0: no norm) become
    ``x * rsqrt(mean(x^2) + eps) * q_weight``, then its last ``rope_dim`` channels
    are rotated by the angles of its position: ``table`` (see :func:`rope_table`)
    gives them, ``rope_dim`` being twice its second dim (None: no rotation).
    ``kv`` likewise with ``kv_norm_dim`` / ``kv_weight``. Pairs are adjacent channels,
    or with ``interleaved=False`` channels half of ``rope_dim`` apart;
    ``inverse`` rotates back (an attention output whose values were rotated:
    ``q_norm_dim=0``). Weights are fp32 or of the rows' dtype.

    Sums are fp32, results rounded once. Tokens whose position lies outside the
    table are padding: zeros. Rows may be strided (slices of one projection);
    rows whose channels are not contiguous or not on 16-byte boundaries are
    copied first. Returns contiguous ``q_out``, or ``(q_out, kv_out)`` where ``kv`` is
    given (``kv_out`` alone without ``q``).
    """
    key = _signature(0, q, kv, positions, table, q_norm_dim, q_weight, kv_norm_dim, kv_weight, eps, interleaved, inverse)
    b = _sigs.get(key)
    if b is not None and _aligned(q, kv, table, q_weight, kv_weight):
        qo = None if q is None else _out(q, b.q_like)
        ko = None if kv is None else _out(kv, b.kv_like)
        packed = _pack_ptrs(q, kv, q_weight, kv_weight, positions, table, qo, ko)
    else:
        b = _bind(q, kv, positions, table, q_norm_dim, q_weight, kv_norm_dim, kv_weight, eps, interleaved, inverse)
        qo = None if q is None else _out(q, b.q_like)
        ko = None if kv is None else _out(kv, b.kv_like)
        packed = b.ptrs(qo, ko)
        _keep(key, b, q, kv, positions, table, q_weight, kv_weight, (q_norm_dim, kv_norm_dim, eps, interleaved, inverse))
    _launch("sas_norm_rope_v1", packed + b.dims, b.dev, "norm_rope")
    return qo if kv is None else ko if q is None else (qo, ko)


def _grad_rows(name: str, g: Optional[torch.Tensor], x: Optional[torch.Tensor], lead_dims: int) -> Optional[torch.Tensor]:
    if x is None:
        return None
    if g is None or g.shape != x.shape or g.dtype is not x.dtype or g.device != x.device:
        raise ValueError(f"{name} must be {x.dtype} {tuple(x.shape)} on {x.device}")
    return _rows(g if g.dim() == lead_dims else g.reshape(-1, *g.shape[g.dim() - lead_dims + 1:]))


_plan = None


def _workspace_bytes(packed: bytes) -> int:
    """What sas_norm_rope_bwd_plan reports for packed arguments."""
    global _plan
    if _plan is None:
        f = _lib.lib()["sas_norm_rope_bwd_plan"]
        f.argtypes = [C.c_char_p, C.POINTER(C.c_size_t)]
        f.restype = C.c_int
        _plan = f
    n = C.c_size_t(0)
    _lib.check(_plan(packed, C.byref(n)), "norm_rope_backward")
    return n.value


def norm_rope_backward(
    dq_out: Optional[torch.Tensor],
    q: Optional[torch.Tensor],
    dkv_out: Optional[torch.Tensor] = None,
    kv: Optional[torch.Tensor] = None,
    *,
    positions: Optional[torch.Tensor] = None,
    table: Optional[torch.Tensor] = None,
    q_norm_dim: Optional[int] = None,
    q_weight: Optional[torch.Tensor] = None,
    kv_norm_dim: Optional[int] = None,
    kv_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    interleaved: bool = True,
    inverse: bool = False,
) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor], Optional[torch.Tensor], Optional[torch.Tensor]]:
    """Gradients of :func:`norm_rope` from those of its outputs, in the outputs'
    dtype and shapes; the other arguments are the forward's. Returns ``(dq, dkv,
    dq_weight, dkv_weight)``, None for what was not given; weight gradients in
    their weights' dtype, summed in fp32 over tokens and heads in a fixed order
    (the same call gives the same bits)."""
    key = (_signature(1, q, kv, positions, table, q_norm_dim, q_weight, kv_norm_dim, kv_weight, eps, interleaved, inverse),
           None if dq_out is None else (dq_out.shape, dq_out.stride(), dq_out.dtype, dq_out.get_device()),
           None if dkv_out is None else (dkv_out.shape, dkv_out.stride(), dkv_out.dtype, dkv_out.get_device()))
    b = _sigs.get(key)
    hit = b is not None and _aligned(q, kv, table, q_weight, kv_weight, dq_out, dkv_out)
    if hit:
        gq, gk, qw, kw = dq_out, dkv_out, q_weight, kv_weight
        strides, need = b.extra
    else:
        b = _bind(q, kv, positions, table, q_norm_dim, q_weight, kv_norm_dim, kv_weight, eps, interleaved, inverse)
        gq, gk = _grad_rows("dq_out", dq_out, q, 3), _grad_rows("dkv_out", dkv_out, kv, 2)
        qw, kw = b.qw, b.kw
        strides = _GRAD_STRIDES.pack(0 if gq is None else gq.stride(0), 0 if gq is None else gq.stride(1),
                                     0 if gk is None else gk.stride(0))
    dq = None if q is None else _out(q, b.q_like)
    dkv = None if kv is None else _out(kv, b.kv_like)
    dqw = None if qw is None else torch.empty_like(qw, dtype=torch.float32)
    dkw = None if kw is None else torch.empty_like(kw, dtype=torch.float32)

    def p(t):
        return 0 if t is None else t.data_ptr()

    grads = (p(gq), p(gk), p(dq), p(dkv), p(dqw), p(dkw))
    head = (_pack_ptrs(q, kv, qw, kw, positions, table, None, None) if hit else b.ptrs(None, None)) + b.dims
    if not hit:
        with torch.cuda.device(b.dev):   # (the plan counts its compute units)
            need = _workspace_bytes(head + _GRAD_PTRS.pack(*grads, 0, 0) + strides)
        b.extra = strides, need
        if gq is dq_out and gk is dkv_out:
            _keep(key, b, q, kv, positions, table, q_weight, kv_weight, (q_norm_dim, kv_norm_dim, eps, interleaved, inverse))
    # the partial sums of the weights' gradients, from the caching allocator: under
    # capture from the graph's own pool
    ws = torch.empty(need, dtype=torch.uint8, device=b.dev) if need else None
    _launch("sas_norm_rope_bwd_v1", head + _GRAD_PTRS.pack(*grads, p(ws), need) + strides, b.dev, "norm_rope_backward")

    def like(g, w):
        if w is None:
            return None
        if g is None:   # no normed channel
            return torch.zeros_like(w)
        return g if w.dtype is torch.float32 else g.to(w.dtype)

    return dq, dkv, like(dqw, q_weight if q is not None else None), like(dkw, kv_weight if kv is not None else None)


class _NormRopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, kv, q_weight, kv_weight, kw):
        out = norm_rope(q, kv, q_weight=q_weight, kv_weight=kv_weight, **kw)
        ctx.save_for_backward(q, kv, q_weight, kv_weight, kw.get("positions"), kw.get("table"))
        ctx.kw = {k: v for k, v in kw.items() if k not in ("positions", "table")}
        return (out, None) if kv is None else (None, out) if q is None else out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq_out, dkv_out):
        q, kv, q_weight, kv_weight, positions, table = ctx.saved_tensors
        dq, dkv, dqw, dkw = norm_rope_backward(dq_out if q is not None else None, q, dkv_out if kv is not None else None,
                                               kv, q_weight=q_weight, kv_weight=kv_weight, positions=positions,
                                               table=table, **ctx.kw)
        return dq, dkv, dqw, dkw, None


def norm_rope_autograd(q: Optional[torch.Tensor], kv: Optional[torch.Tensor] = None, *,
                       q_weight: Optional[torch.Tensor] = None, kv_weight: Optional[torch.Tensor] = None, **kwargs):
    """:func:`norm_rope` recorded for autograd: gradients flow to ``q``, ``kv`` and
    the weights through :func:`norm_rope_backward` (not to ``table``). Other
    arguments and the result as for :func:`norm_rope`. To capture a training step
    while an eager graph of the same leaves lives, capture ``torch.autograd.grad``
    or :func:`norm_rope_backward`: PyTorch ends the process where a captured
    ``backward()`` accumulates into such leaves."""
    qo, ko = _NormRopeFn.apply(q, kv, q_weight, kv_weight, kwargs)
    return qo if kv is None else ko if q is None else (qo, ko)

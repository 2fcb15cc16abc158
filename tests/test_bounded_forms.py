"""Bounded caches, further forms of the calls that tests/test_bounded.py covers: what is
refused, lists of compressed rows each side of the planner's limits, evictions of compressed
rows. Tolerances are that
file's."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from dsv4_amd import _lib
from test_bounded import Case, _check_grads, _fwd_args, _grads, _refused, _run


def test_calls_without_first_rows_refuse_them():
    """ori_first is an argument of the calls with first rows alone; the others name it as
    unknown and run nothing."""
    from dsv4_amd import api
    q = torch.zeros(3, 16, 512, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    kv = torch.zeros(1, 16, 1, 512, dtype=torch.bfloat16)
    kw = dict(ori_kv=kv, ori_block_table=i[:1, None], cu_seqlens_q=i, seqused_kv=i[:1], softmax_scale=1.0, sinks=torch.zeros(16))
    lse = torch.zeros(3, 16)
    for first in (0, 4, None):
        for call in (lambda: api.sparse_attn_sharedkv(q, ori_first=first, **kw),
                     lambda: api.sparse_attn_sharedkv_autograd(q, ori_first=first, **kw),
                     lambda: api.sparse_attn_sharedkv_backward(q, q, q, lse, ori_first=first, **kw),
                     lambda: api.prepare_sparse_attn_sharedkv_backward(q, q, q, lse, ori_first=first, **kw)):
            with pytest.raises(TypeError, match="ori_first"):
                call()


def test_abi_key_major_sums_of_first_rows_are_refused_where_there_are_none():
    """SAS_BWD_WINDOW_KEYS with first rows: 16 and 48 heads, an odd address, a split count, no
    workspace."""
    L, fake = _lib.lib(), 1 << 20
    mk = lambda dout=fake, **kw: _lib.SasBwdFirstArgs(_lib.SasBwdArgs(  # noqa: E731
        fwd=_fwd_args(**dict(dict(T=4096, flags=_lib.SAS_BWD_WINDOW_KEYS), **kw)), dout=dout, dq=fake, d_ori_kv=fake, d_sinks=fake), 4)
    direct, ws = C.c_int32(0), C.c_size_t(1)
    for kw in (dict(H=16), dict(H=48), dict(q=fake + 8), dict(dout=fake + 8), dict(num_splits=2)):
        assert L.sas_bwd_first_plan(C.byref(mk(**kw)), C.byref(direct), C.byref(ws)) == _lib.SAS_OK and ws.value == 0
        _refused(L.sas_bwd_first_v1, mk(**kw), "SAS_BWD_WINDOW_KEYS with first rows")
    assert L.sas_bwd_first_plan(C.byref(mk()), C.byref(direct), C.byref(ws)) == _lib.SAS_OK and ws.value > 0
    _refused(L.sas_bwd_first_v1, mk(), "or without it")


# ---------------------------------------------------------------------------
# GPU: gradients
# ---------------------------------------------------------------------------

GRAD = {
    # 1525 compressed rows: below 14 times lists of 128, past 7 times lists of 144 (7 times
    # those of 256 again not)
    "topk_128": dict(kind="scfa", H=32, D=512, ql=[70], kl=[6100], K=128, F=9, win=70),
    "topk_144": dict(kind="scfa", H=32, D=512, ql=[70], kl=[6100], K=144, F=9, win=70),
    "topk_256": dict(kind="scfa", dt="fp16", H=96, D=576, ql=[70], kl=[6100], K=256, F=9, win=70),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(GRAD))
def test_gpu_first_backward(name):
    c = Case(**GRAD[name])
    kw = c.kwargs()
    out, lse = _run(c, **kw)
    _check_grads(c, _grads(c, out, lse, kw), out, lse)


# ---------------------------------------------------------------------------
# GPU: evictions of compressed rows
# ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dense", [False, True])
def test_gpu_evicted_compressed_rows(dense):
    """Compressed rows cut down to a budget by their own lengths, then attended by lists of
    their new places (of all of them after a dense call), lengths as before: what lists of the
    old places give over the whole cache, weights too."""
    from dsv4_amd.api import add_row_weights, sparse_attn_sharedkv
    from dsv4_amd.cache import evict_kv_cache
    budget, ratio = 40, 4
    c = Case(kind="cfa" if dense else "scfa", H=32, D=576, ql=[1, 2, 1], kl=[600, 410, 90], K=60, ratio=ratio, win=64)
    kw, q = c.kwargs(first=False), c.q.cuda()
    out, lse = sparse_attn_sharedkv(q, return_softmax_lse=True, **kw)
    weights = torch.zeros(3, c.ctable.shape[1] * c.bs, dtype=torch.float64, device="cuda")
    add_row_weights(q, lse, cmp_weights=weights, **kw)
    cut = kw["cmp_kv"].clone()
    rows, kept = evict_kv_cache(cut, weights, kw["cmp_block_table"], kw["seqused_kv"] // ratio, budget=budget, keep_recent=4)
    assert rows.tolist() == [budget, budget, 22]
    seq = torch.tensor([0, 1, 1, 2], device="cuda")
    new = torch.arange(budget, dtype=torch.int32, device="cuda").expand(4, budget)
    new = torch.where(new < rows[seq][:, None], new, -1)
    if not dense:
        new = new[:, torch.randperm(budget, generator=torch.Generator().manual_seed(5))[:25].cuda()]
    old = torch.where(new >= 0, kept[seq].gather(1, new.clamp(min=0).long()), -1)
    # (of two tokens the earlier may not see the last row: lists hold what both see)
    thr = torch.tensor([600, 409, 410, 90], device="cuda")[:, None] // ratio
    new = torch.where(old < thr, new, -1)
    lists = lambda x: dict(kw, cmp_sparse_indices=x.unsqueeze(1).contiguous())  # noqa: E731
    want, want_lse = sparse_attn_sharedkv(q, return_softmax_lse=True, **lists(old))
    got, got_lse = sparse_attn_sharedkv(q, return_softmax_lse=True, **dict(lists(new), cmp_kv=cut))
    assert torch.equal(got, want) and torch.equal(got_lse, want_lse)
    a, b = torch.zeros_like(weights), torch.zeros_like(weights)
    add_row_weights(q, got_lse, cmp_weights=a, **dict(lists(new), cmp_kv=cut))
    add_row_weights(q, want_lse, cmp_weights=b, **lists(old))
    for i, n in enumerate(rows.tolist()):
        assert torch.equal(a[i, :n], b[i, kept[i, :n].long()]) and not bool(a[i, n:].any())

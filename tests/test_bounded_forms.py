"""Bounded caches, further forms of the calls that tests/test_bounded.py covers: what is
refused, lists of compressed rows each side of the planner's limits. Tolerances are that
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

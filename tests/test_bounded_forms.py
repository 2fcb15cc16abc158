"""Bounded caches, further forms of the calls that tests/test_bounded.py covers: what is
refused."""

from __future__ import annotations

import pytest
import torch


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

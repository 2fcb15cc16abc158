"""Bounded caches, further forms of the calls that tests/test_bounded.py covers: what is
refused, lists of compressed rows each side of the planner's limits, evictions of compressed
rows; slots in several passes and splits, every length of segment, more than 64 sequences.

Tolerances are that file's, whose counts of fp32 adds hold here as follows. A cache row's
gradient is summed over a segment of at most 96 tokens of 32 heads in a chain (96 matrix
instructions of 32 products each), then over at most 13 segments of 5 head groups by
atomic adds: a term takes part in at most 96 + 32 + 65 roundings, below 2^-16 of the terms'
sum (0.13 h is 2^-11 in bf16, 2^-14 in fp16). Splits of dq add 64 more at most. d_sinks: 700
adds of 2^-24 beside Delta's 512 and the exponential's 2^-20, below 2^-13 still; of 4550
tokens a thread of the sink kernel sums 8, then 3 and 256 adds join them. A row weight's
chain is at most 64 tokens of 4 tiles of heads."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from dsv4_amd import _lib
from oracle import bounded_ref as R
from test_bounded import Case, _check_grads, _evict, _evict_case, _fwd_args, _grads, _refused, _run, _same, _weights, _zeros


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
    # more slots than a workgroup resolves (1280): two passes that divide the first rows (one
    # sequence has none in the second), or the window; three, two of them without raw rows
    "passes_first": dict(H=32, D=512, ql=[80, 70], kl=[1700, 70], F=1000, win=400),
    "passes_window": dict(dt="fp16", H=32, D=576, ql=[70], kl=[1600], F=20, win=1300),
    "passes_three": dict(kind="cfa", H=64, D=576, ql=[90], kl=[4000], ratio=2, F=300, win=700),
    # slots in splits: a top-k prompt past 1280, decode steps
    "splits_topk": dict(kind="scfa", H=32, D=512, ql=[70], kl=[1500], K=40, F=700, win=700),
    "splits_decode": dict(H=64, D=576, ql=[1, 2], kl=[900, 700], F=100, win=300),
    "splits_h16": dict(kind="scfa", dt="fp16", H=16, D=512, ql=[1, 1], kl=[1300, 100], K=200, F=150, win=200),
    "sequences": dict(H=32, D=512, ql=[64 + i % 3 for i in range(70)], kl=[64 + (i * 37) % 90 + i % 3 for i in range(70)],
                      F=5, win=20),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(GRAD))
def test_gpu_first_backward(name):
    c = Case(**GRAD[name])
    kw = c.kwargs()
    out, lse = _run(c, **kw)
    _check_grads(c, _grads(c, out, lse, kw), out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("splits", [2, 5, 64])
def test_gpu_first_backward_in_given_splits(splits):
    c = Case(kind="scfa", H=32, D=576, ql=[2, 66], kl=[600, 330], K=100, F=50, win=150)
    kw = c.kwargs()
    out, lse = _run(c, **kw)
    _check_grads(c, _grads(c, out, lse, dict(kw, num_splits=splits)), out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("first", [128, 129, 1 << 20, (1 << 31) - 1])
def test_gpu_more_first_rows_than_the_table_holds(first):
    """Every row is a first row; those past the block table's end are not there, and cost no
    slots."""
    from dsv4_amd.api import add_row_weights, sparse_attn_sharedkv_first
    c = Case(kind="scfa", H=32, D=512, ql=[70], kl=[110], F=128, K=20, win=16)
    kw, q = c.kwargs(), c.q.cuda()
    out, lse = sparse_attn_sharedkv_first(q, return_softmax_lse=True, **dict(kw, ori_first=first))
    c.check(out, lse)
    again, _ = sparse_attn_sharedkv_first(q, return_softmax_lse=True, **dict(kw, ori_first=first))
    assert torch.equal(again, out)
    _check_grads(c, _grads(c, out, lse, dict(kw, ori_first=first)), out, lse)
    w, ref = _zeros(c)[0], _zeros(c)[0]
    add_row_weights(q, lse, ori_weights=w, **dict(kw, ori_first=first))
    add_row_weights(q, lse, ori_weights=ref, **kw)
    assert torch.equal(w, ref)


def _segment(c, win, cus):
    """plan_prefill's tokens a segment, without compressed rows."""
    for seg in (96, 64, 32, 24):
        if c.T / seg * (c.H // 32) * ((win - 1 + seg) / 64 + 1) >= 2.75 * cus:
            break
    return seg


@pytest.mark.gpu
@pytest.mark.parametrize("F, dt, D", [(4, "bf16", 512), (70, "fp16", 576)])
@pytest.mark.parametrize("seg, ql, kl", [(96, [430, 270], [2300, 1500]), (64, [201, 299], [1300, 2000]), (32, [300], [1777])])
def test_gpu_first_backward_segments(seg, ql, kl, F, dt, D):
    """Segments of 32 to 96 tokens, the last ones partly filled, with narrow and wide tiles of
    first rows (the cases of tests/test_bounded.py take 24)."""
    c = Case(dt=dt, H=160, D=D, ql=ql, kl=kl, F=F, win=1100)
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    assert cus != 256 or _segment(c, 1100, cus) == seg
    kw = c.kwargs()
    out, lse = _run(c, **kw)
    _check_grads(c, _grads(c, out, lse, kw), out, lse)


@pytest.mark.gpu
def test_gpu_first_of_many_sequences():
    c = Case(kind="scfa", H=32, D=576, ql=[(i * 7) % 3 for i in range(150)], kl=[2 + (i * 41) % 300 for i in range(150)], K=40, F=9,
             win=60, bs=16)
    out, lse = _run(c)
    c.check(out, lse)
    _check_grads(c, _grads(c, out, lse, c.kwargs()), out, lse)


# ---------------------------------------------------------------------------
# weights
# ---------------------------------------------------------------------------

WEIGHTS = {
    # segments of 64, 32, 16 and 8 tokens by the planner's rule on 256 CUs (`row_tiles`: its count of
    # 128-row tiles), the last ones partly filled; tests/test_bounded.py's cases all take 4
    "segment_64": (64, dict(H=64, D=576, ql=[150, 70, 0, 1, 129] + [(i * 5) % 4 for i in range(65)],
                            kl=[600, 700, 5, 100, 130] + [3 + (i * 31) % 690 for i in range(65)], win=1000, F=0)),
    "segment_32": (32, dict(H=16, D=512, ql=[130], kl=[10000], win=20000, F=0)),
    "segment_16": (16, dict(dt="fp16", H=32, D=576, ql=[130], kl=[6000], win=7000, F=0)),
    "segment_8": (8, dict(dt="fp8", H=16, D=576, ql=[130], kl=[3000], win=4000, F=0)),
    # more than 64 sequences, with first and compressed rows, by rows and by slots
    "sequences_by_rows": (4, dict(kind="cfa", H=16, D=512, ql=[(i * 5) % 13 for i in range(150)],
                                  kl=[12 + (i * 41) % 500 for i in range(150)], ratio=4, F=150, win=20, bs=16)),
    "sequences_by_slot": (0, dict(kind="scfa", H=16, D=576, ql=[(i * 7) % 3 for i in range(150)],
                                  kl=[2 + (i * 41) % 300 for i in range(150)], K=40, F=9, win=60, bs=16, tail=3)),
}


def _weight_segment(c, win, cus):
    """weights_impl's tokens a segment of a tile's rows, 0: slots of one token."""
    B = len(c.ql)
    if c.T < 4 * B:
        return 0
    up = lambda n, d: -(-n // d)  # noqa: E731
    cap, mean = c.table.shape[1] * c.bs, max(1, c.T // B)
    ncmp = min(c.ctable.shape[1] * c.bs, max(c.kl) // c.ratio) if c.kind == "cfa" else 0
    row_tiles = B * (up(min(cap, mean + min(win - 1, cap)), 128) + up(ncmp, 128))
    seg = 64
    while seg > 4 and 2 * row_tiles * up(min(mean, win - 1 + 128), seg) < 3 * cus:
        seg //= 2
    return seg


def _all_weights(c, lse):
    """R.weights() with a row of adds at a time."""
    z = lambda t: torch.zeros(len(c.ql), 1 if t is None else t.shape[1] * c.bs, dtype=torch.float64)  # noqa: E731
    w, wc = z(c.table), z(c.ctable)
    for t in range(c.T):
        if c.keys.seq[t] < 0:
            continue
        p = torch.exp(c.q[t].double() @ R._k(c.keys, t, c.rows, c.crows).t() * c.scale - lse[t].double()[:, None]).mean(0)
        n = len(c.keys.raw[t][0])
        for to, at, part in ((w, c.keys.raw[t][0], p[:n]), (wc, c.keys.cmp[t][0], p[n:])):
            to[c.keys.seq[t]].index_add_(0, torch.tensor(at, dtype=torch.long), part)
    return w, wc


def test_oracle_weights_by_rows_of_adds():
    c = Case(kind="scfa", H=16, D=512, ql=[3, 0, 2], kl=[90, 4, 33], K=9, F=3, win=20, bs=8, tail=2)
    lse = c.attention()[1]
    for x, y in zip(_all_weights(c, lse), c.weights(lse)):
        torch.testing.assert_close(x, y, atol=1e-13, rtol=1e-12)


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(WEIGHTS))
def test_gpu_weights(name):
    seg, case = WEIGHTS[name]
    c = Case(**case)
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    assert cus != 256 or _weight_segment(c, c.win, cus) == seg
    lse = c.attention()[1].float().cuda()
    got = _zeros(c)
    _weights(c, lse, *got)
    for x, ref in zip(got, _all_weights(c, lse.cpu())):
        if x is None:
            continue
        x = x.cpu()
        assert bool(((x - ref).abs() <= 2.0 ** -12 * ref + 2.0 ** -37 * c.T).all())
        assert bool((x[ref == 0] == 0).all()) and torch.equal(torch.round(x * 2.0 ** 36), x * 2.0 ** 36)
    again = _zeros(c)
    _weights(c, lse, *again)
    assert torch.equal(again[0], got[0]) and (got[1] is None or torch.equal(again[1], got[1]))


@pytest.mark.gpu
def test_gpu_weights_of_two_calls_at_once():
    """Calls on two streams that add to the same rows."""
    c = Case(kind="scfa", H=32, D=576, ql=[5, 40], kl=[600, 300], K=64)
    kw, q, lse = c.kwargs(), c.q.cuda(), c.attention()[1].float().cuda()
    one, got = _zeros(c), _zeros(c)
    _weights(c, lse, *one, kw=kw, q=q)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                _weights(c, lse, *got, kw=kw, q=q)
    torch.cuda.synchronize()
    assert torch.equal(got[0], 8 * one[0]) and torch.equal(got[1], 8 * one[1])


@pytest.mark.gpu
def test_gpu_calls_without_tokens():
    """No query token in any sequence: empty outputs, no gradient, no weight."""
    for kind in ("swa", "cfa", "scfa"):
        c = Case(kind="swa" if kind == "swa" else "cfa", H=32, D=512, ql=[0, 0], kl=[90, 0])
        kw = c.kwargs()
        if kind == "scfa":
            kw["cmp_sparse_indices"] = torch.zeros(0, 1, 9, dtype=torch.int32, device="cuda")
        out, lse = _run(c, **kw)
        assert out.shape == (0, 32, 512) and lse.shape == (0, 32)
        dq, *rest = _grads(c, out, lse, kw)
        assert dq.shape == (0, 32, 512) and not any(bool(x.any()) for x in rest if x is not None)
        got = _zeros(c)
        _weights(c, lse, *got, kw=kw)
        assert not any(bool(x.any()) for x in got if x is not None)


# ---------------------------------------------------------------------------
# GPU: long evictions
# ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("budget, zero", [(4096, 0.3), (118000, 0.3), (60000, 0.9)])
def test_gpu_evict_of_131072_rows(budget, zero):
    """A divided key among the heaviest, among rows without any weight, and all but one."""
    for b in (budget, 131071):
        a = _evict_case([131072, 33000, 100], b, 4, 64, bs=64, row=8, zero=zero)
        _same(_evict(*a), R.evict(*a))


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

"""Caches that stay bounded: attention with first rows that stay visible
(sparse_attn_sharedkv_first) and its gradients, the weights of cache rows
(add_row_weights), evictions (evict_kv_cache). The CPU oracle pinned, argument errors
without a device, the kernels against the oracle.

Tolerances, with h half a step of the query's dtype (bf16 2^-8, fp16 2^-11). A score is
a sum of 576 fp32 products whose partial sums stay below 100: off by at most 576 x 2^-24 x
100 x scale = 2^-12.8, which its P is off relatively (0.28 h in fp16).
 Outputs: P is rounded once, the output once, a split's partial to fp16 under bf16
  outputs (h / 8): below 1.5 h (sum p |v| + |out|). fp16 P below 2^-14 rounds by 2^-25
  absolutely: at most 1300 keys x 2^-25 x max |v| (4.6), below 2^-12. LSE: 1e-3, as for
  the linear operator.
 Gradients: P and dS = P (dP - Delta) scale are rounded once (h), P is off by 0.28 h, and
  dP and Delta, 512 fp32 products each, by at most 512 x 2^-24 of their terms' sum: h / 16
  of it covers that in either type. The rows' sums run over at most 300 tokens of four
  head groups in fp32: 2^-14 of their terms, below 0.13 h. Together below 1.5 h of the
  terms' sizes; dq is rounded once more. d_sinks: 512 x 2^-24 for Delta, 2^-20 for the
  exponential, 300 adds: below 2^-13 of the terms.
 Weights: P's 2^-12.8, the fp32 sums' (tokens x heads) x 2^-24 for up to 2^10 terms in a
  chain, and half a grid step of 2^-36 an added value: below 2^-12 of the weight + 2^-37
  an added value.
 Evictions move bytes: equal."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from dsv4_amd import _lib, cases, paged
from oracle import backward_ref as BR
from oracle import bounded_ref as R


# ---------------------------------------------------------------------------
# oracle
# ---------------------------------------------------------------------------

def _known_positions(**kw):
    assert R.positions(9, 2, 4, **kw) == [0, 1, 6, 7, 8, 9]
    assert R.positions(5, 4, 4, **kw) == [0, 1, 2, 3, 4, 5]      # rows 2, 3 lie in the window


def test_oracle_known_positions():
    _known_positions()
    assert R.positions(3, 9, 1) == [0, 1, 2, 3]
    assert R.positions(0, 4, 4) == [0]
    assert R.positions(-1, 4, 4) == []
    assert R.positions(7, 0, 3) == [5, 6, 7]


def test_oracle_planted_second_count_fails():
    with pytest.raises(AssertionError):
        _known_positions(twice=True)


class Case:
    """Inputs on the CPU, drawn from `seed`."""

    def __init__(self, kind="swa", dt="bf16", H=16, D=512, ql=(1,), kl=(20,), F=4, K=0, ratio=4, win=128, bs=64, gap=False,
                 holes=False, tail=0, seed=3):
        g = torch.Generator().manual_seed(seed)
        self.kind, self.ql, self.kl, self.ratio, self.win, self.bs, self.H, self.D, self.F = (
            kind, ql, kl, ratio, win, bs, H, D, F)
        self.fp8 = dt == "fp8"
        self.dt = {"fp16": torch.float16, "f64": torch.float64}.get(dt, torch.bfloat16)
        self.half = torch.finfo(self.dt).eps / 2
        self.scale = D ** -0.5
        self.T = sum(ql) + tail
        self.q = torch.randn(self.T, H, D, generator=g).to(self.dt)
        self.dout = torch.randn(self.T, H, 512, generator=g).to(self.dt)
        self.sinks = torch.randn(H, generator=g)
        self.rows, self.cache, self.table = self._cache(kl, g)
        if gap:   # blocks that hold neither first rows nor a token's window are not there
            for b, (m, n) in enumerate(zip(ql, kl)):
                for blk in range(-(-F // bs), max(0, n - m - win + 1) // bs):
                    self.table[b, blk] = -1
        if holes:
            self.table[0, 0] = -1
            self.table[-1, -1] = -1
        self.crows = self.ccache = self.ctable = self.idx = None
        if kind != "swa":
            self.crows, self.ccache, self.ctable = self._cache([k // ratio for k in kl], g)
        if kind == "scfa":
            top = max(1, max(kl) // ratio + 2)   # a few beyond the threshold, -1 here and there, one twice
            self.idx = torch.stack([torch.randperm(max(top, K), generator=g)[:K] for _ in range(self.T)])
            self.idx = torch.where(self.idx < top, self.idx, -1).to(torch.int32).view(self.T, 1, K)
            if K > 1:
                self.idx[0, 0, 1] = self.idx[0, 0, 0]
        self.cu = torch.zeros(len(ql) + 1, dtype=torch.int32)
        self.cu[1:] = torch.tensor(ql).cumsum(0)
        self.used = torch.tensor(kl, dtype=torch.int32)
        self.keys = R.Keys(self.table, self.ctable, None if self.idx is None else self.idx[:, 0], ql, kl, F, win, bs, bs,
                           ratio, self.T)

    def _cache(self, lens, g):
        per = max(1, max(-(-max(x, 1) // self.bs) for x in lens))
        nb = per * len(lens) + 2
        table = torch.randperm(nb, generator=g)[:per * len(lens)].to(torch.int32).view(len(lens), per)
        rows = torch.randn(nb * self.bs, self.D, generator=g).to(self.dt)
        if self.fp8:
            cache = paged.quantize_kv_fp8(rows.view(nb, self.bs, 1, self.D))
            return paged.dequantize_kv_fp8(cache).view(nb * self.bs, self.D), cache, table
        return rows, rows.view(nb, self.bs, 1, self.D), table

    def kwargs(self, host_lens=False, sinks=True, first=True):
        mv = lambda t: None if t is None else t.cuda()  # noqa: E731
        lens = (lambda t: t) if host_lens else mv
        kw = dict(ori_kv=mv(self.cache), cmp_kv=mv(self.ccache), cmp_sparse_indices=mv(self.idx),
                  ori_block_table=mv(self.table), cmp_block_table=mv(self.ctable), cu_seqlens_q=lens(self.cu),
                  seqused_kv=lens(self.used), softmax_scale=self.scale,
                  cmp_ratio=self.ratio if self.kind != "swa" else None, ori_win_left=self.win - 1)
        if sinks:
            kw["sinks"] = mv(self.sinks)
        if first:
            kw["ori_first"] = self.F
        return kw

    def attention(self):
        return R.attention(self.keys, self.q, self.rows, self.crows, self.sinks, self.scale)

    def check(self, out, lse):
        ref, ref_lse, mag = self.attention()
        bound = 1.5 * self.half * (mag + ref.abs()) + (2.0 ** -12 if self.dt is torch.float16 else 2.0 ** -16)
        err = (out.cpu().double() - ref).abs()
        assert bool((err <= bound).all()), f"worst {float((err / bound).max()):.3g} of the bound"
        assert float((lse.cpu().double() - ref_lse).abs().max()) <= 1e-3
        assert bool((out.cpu()[sum(self.ql):] == 0).all()) and bool((lse.cpu()[sum(self.ql):] == 0).all())

    def gradients(self, out, lse, **kw):
        return R.gradients(self.keys, self.dout, self.q, out, lse, self.rows, self.crows, self.sinks, self.scale, self.half, **kw)

    def weights(self, lse, R_=None):
        B = len(self.ql)
        return R.weights(self.keys, self.q, lse, self.rows, self.crows, self.scale, B,
                         R_ or self.table.shape[1] * self.bs, 1 if self.ctable is None else self.ctable.shape[1] * self.bs)


TINY = dict(kind="scfa", dt="f64", H=2, D=576, ql=[3, 1], kl=[40, 23], F=3, K=6, win=16, bs=8)


def test_oracle_without_first_rows_is_the_linear_operator():
    c = Case(**dict(TINY, F=0))
    c.idx = cases.topk_indices(c.ql, c.kl, 6, c.ratio, torch.Generator().manual_seed(4))
    c.keys = R.Keys(c.table, c.ctable, c.idx[:, 0], c.ql, c.kl, 0, c.win, c.bs, c.bs, c.ratio, c.T)
    out, lse, _ = c.attention()
    kw = {k: v for k, v in dict(
        ori_kv=c.cache, ori_block_table=c.table, cu_seqlens_q=c.cu, seqused_kv=c.used, sinks=c.sinks.double(),
        softmax_scale=c.scale, cmp_kv=c.ccache, cmp_block_table=c.ctable, cmp_sparse_indices=c.idx, cmp_ratio=4,
        ori_win_left=c.win - 1).items()}
    ref = BR.backward_paged(c.q, c.dout, **kw)
    torch.testing.assert_close(out, ref["out"], atol=1e-10, rtol=1e-10)
    torch.testing.assert_close(lse, ref["lse"], atol=1e-10, rtol=1e-10)
    g, _ = c.gradients(out, lse)
    torch.testing.assert_close(g["dq"], ref["dq"], atol=1e-10, rtol=1e-9)
    torch.testing.assert_close(g["sinks"], ref["d_sinks"], atol=1e-10, rtol=1e-9)
    for name, key in (("rows", "d_ori"), ("crows", "d_cmp")):
        torch.testing.assert_close(g[name][ref[key][0]], ref[key][1], atol=1e-10, rtol=1e-9)


def _central_differences(**kw):
    c = Case(**TINY)
    out, lse, _ = c.attention()
    g, _ = c.gradients(out, lse, **kw)
    loss = lambda: float((c.attention()[0] * c.dout).sum())  # noqa: E731
    eps = 1e-5
    first = c.keys.raw[0][1][1]      # row 1 of sequence 0, behind the window
    spots = [(c.q, (0, 1, 7), "dq"), (c.q, (3, 0, 560), "dq"), (c.rows, (first, 30), "rows"), (c.rows, (first, 570), "rows"),
             (c.rows, (c.keys.raw[2][1][-1], 3), "rows"), (c.crows, (c.keys.cmp[0][1][0], 100), "crows")]
    for t, at, name in spots:
        x = t[at].item()
        t[at] = x + eps
        up = loss()
        t[at] = x - eps
        down = loss()
        t[at] = x
        assert abs((up - down) / (2 * eps) - float(g[name][at])) < 1e-6, (name, at)


def test_oracle_gradients_are_differences():
    _central_differences()


def test_oracle_planted_sign_fails():
    with pytest.raises(AssertionError):
        _central_differences(sign=-1.0)


def test_oracle_weights_are_what_the_sinks_leave():
    c = Case(**TINY)
    _, lse, _ = c.attention()
    w, wc = c.weights(lse)
    share = torch.exp(c.sinks.double() - lse)
    for b, toks in ((0, slice(0, 3)), (1, slice(3, 4))):
        left = (1 - share[toks]).mean(1).sum()
        assert abs(float(w[b].sum() + wc[b].sum() - left)) < 1e-9
    assert float(w[0, 0]) > 0 and float(w[0, 5]) == 0        # a first row; one between


def _known_evictions(**kw):
    cache = torch.arange(12).view(3, 4, 1, 1)
    w = torch.tensor([[9., 0., 5., 0., 5., 1., 2., 0.]], dtype=torch.float64)
    got, wn, n, kept = R.evict(cache, w, torch.tensor([[2, 0]]), torch.tensor([8]), 5, 1, 1, **kw)
    assert kept.tolist() == [[0, 2, 4, 6, 7]] and n.tolist() == [5]
    assert got[2].view(-1).tolist() == [8, 10, 0, 2] and got[0].view(-1).tolist() == [3, 1, 2, 3]
    assert wn.tolist() == [[9., 5., 5., 2., 0., 0., 0., 0.]]
    w[0] = 0                                                    # all equal: the lowest positions
    assert R.evict(cache, w, torch.tensor([[2, 0]]), torch.tensor([8]), 5, 1, 1, **kw)[3].tolist() == [[0, 1, 2, 3, 7]]


def test_oracle_known_evictions():
    _known_evictions()
    nan = torch.tensor([[float("nan"), -1., -float("inf"), 0.]], dtype=torch.float64)
    _, w, n, kept = R.evict(torch.zeros(1, 4, 1, 1), nan, torch.tensor([[0]]), torch.tensor([4]), 3, 0, 0)
    assert kept.tolist() == [[1, 2, 3]]
    assert R.evict(torch.zeros(1, 4, 1, 1), nan, torch.tensor([[0]]), torch.tensor([-3]), 2, 0, 0)[2:][1].tolist() == [[-1, -1]]


def test_oracle_planted_tie_fails():
    with pytest.raises(AssertionError):
        _known_evictions(high=True)


# ---------------------------------------------------------------------------
# argument errors (no device)
# ---------------------------------------------------------------------------

def _fwd_args(**kw):
    a = _lib.SasFwdArgs(T=4, B=1, H=64, D=576, DV=512, ori_block_size=64, ori_bt_stride=8, ori_num_blocks=8,
                        scenario=_lib.SAS_SWA, cmp_ratio=4, win_left=127, softmax_scale=0.04)
    fake = 1 << 20
    for f in ("q", "ori_kv", "ori_block_table", "q_prefix", "act_kv", "sinks", "out", "lse"):
        setattr(a, f, fake)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _refused(fn, args, needle, code=_lib.SAS_EINVAL):
    assert fn(C.byref(args), None) == code
    assert needle in _lib.lib().sas_last_error().decode()


def test_abi_first_refuses():
    L = _lib.lib()
    assert L.sas_fwd_first_v1(None, None) == _lib.SAS_EINVAL
    assert L.sas_fwd_first_plan(None, None, None) == _lib.SAS_EINVAL
    ns, ws = C.c_int32(0), C.c_size_t(0)
    for first in (-1, 1 << 31):
        _refused(L.sas_fwd_first_v1, _lib.SasFwdFirstArgs(_fwd_args(), first), "ori_first out of range")
        assert L.sas_fwd_first_plan(C.byref(_lib.SasFwdFirstArgs(_fwd_args(), first)), C.byref(ns), C.byref(ws)) == _lib.SAS_EINVAL
    _refused(L.sas_fwd_first_v1, _lib.SasFwdFirstArgs(_fwd_args(win_left=(1 << 31) - 1), (1 << 31) - 1), "key slots per token")
    _refused(L.sas_fwd_first_v1, _lib.SasFwdFirstArgs(_fwd_args(D=100), 4), "D must be")
    _refused(L.sas_fwd_first_v1, _lib.SasFwdFirstArgs(_fwd_args(num_splits=2), 4), "workspace", _lib.SAS_ENOWS)
    _refused(L.sas_fwd_first_v1, _lib.SasFwdFirstArgs(_fwd_args(q=None), 4), "null device pointer")
    assert L.sas_fwd_first_v1(C.byref(_lib.SasFwdFirstArgs(_fwd_args(T=0), 4)), None) == _lib.SAS_OK


def test_abi_first_plan_counts_first_rows():
    L = _lib.lib()
    ns, ws = C.c_int32(0), C.c_size_t(0)
    plans = {}
    for first in (0, 4, 1300):
        assert L.sas_fwd_first_plan(C.byref(_lib.SasFwdFirstArgs(_fwd_args(T=4096), first)), C.byref(ns), C.byref(ws)) == _lib.SAS_OK
        plans[first] = ns.value
    assert plans[0] == plans[4] == 1 and plans[1300] == 2     # a workgroup holds 1280 slots


def test_abi_first_backward_refuses():
    L = _lib.lib()
    assert L.sas_bwd_first_v1(None, None) == _lib.SAS_EINVAL and L.sas_bwd_first_plan(None, None, None) == _lib.SAS_EINVAL
    fake = 1 << 20
    b = _lib.SasBwdArgs(fwd=_fwd_args(), dout=fake, dq=fake, d_ori_kv=fake, d_sinks=fake)
    direct, ws = C.c_int32(0), C.c_size_t(0)
    for first in (-1, 1 << 31):
        _refused(L.sas_bwd_first_v1, _lib.SasBwdFirstArgs(b, first), "ori_first out of range")
        assert L.sas_bwd_first_plan(C.byref(_lib.SasBwdFirstArgs(b, first)), C.byref(direct), C.byref(ws)) == _lib.SAS_EINVAL
    b.dout = None
    _refused(L.sas_bwd_first_v1, _lib.SasBwdFirstArgs(b, 4), "null device pointer")
    b.dout = fake
    b.fwd.flags = _lib.SAS_BWD_DQ_DTYPE
    _refused(L.sas_bwd_first_v1, _lib.SasBwdFirstArgs(b, 4), "SAS_BWD_DQ_DTYPE")
    b.fwd.flags, b.fwd.T = 0, 0
    assert L.sas_bwd_first_v1(C.byref(_lib.SasBwdFirstArgs(b, 4)), None) == _lib.SAS_OK


def test_abi_weights_refuses():
    L, fake = _lib.lib(), 1 << 20
    mk = lambda first=0, ori=fake, cmp_=None, rows=8, crows=0, **kw: _lib.SasRowWeightsArgs(  # noqa: E731
        _fwd_args(sinks=None, out=None, **kw), first, ori, cmp_, rows, crows)
    fn = L.sas_row_weights_v1
    assert fn(None, None) == _lib.SAS_EINVAL
    _refused(fn, mk(ori=None), "neither raw nor compressed")
    _refused(fn, mk(cmp_=fake, crows=8), "without compressed rows")
    _refused(fn, mk(first=-1), "ori_first")
    _refused(fn, mk(first=1 << 31), "ori_first")
    _refused(fn, mk(rows=-1), "ori_rows")
    _refused(fn, mk(H=8), "H a multiple of 16")
    _refused(fn, mk(D=100), "D must be")
    _refused(fn, mk(win_left=-1), "win_left")
    _refused(fn, mk(lse=None), "null device pointer")
    _refused(fn, mk(lse=fake + 4), "16-byte aligned")
    _refused(fn, mk(q=fake + 8), "16-byte aligned")
    _refused(fn, mk(ori=fake + 4), "8-byte aligned")
    _refused(fn, mk(ori_kv=fake + 8), "ori_kv")
    _refused(fn, mk(ori_block_table=None), "ori_block_table")
    _refused(fn, mk(ori_num_blocks=1 << 30), "bad ori cache geometry")
    _refused(fn, mk(q_dtype=_lib.SAS_DT_FP16), "kv dtype")
    _refused(fn, mk(kv_dtype=_lib.SAS_DT_FP8_E4M3_ROW656, D=512), "fp8")
    _refused(fn, mk(cmp_=fake, crows=8, scenario=_lib.SAS_SCFA), "cmp_kv")
    geo = dict(scenario=_lib.SAS_SCFA, cmp_kv=fake, cmp_block_table=fake, cmp_block_size=64, cmp_bt_stride=2, cmp_num_blocks=4)
    _refused(fn, mk(cmp_=fake, crows=8, K=8, **geo), "cmp_indices")
    _refused(fn, mk(cmp_=fake, crows=8, K=8, **dict(geo, cmp_ratio=0)), "cmp_ratio")
    _refused(fn, mk(cmp_=fake, crows=8, K=8, **dict(geo, cmp_num_blocks=0, cmp_indices=fake)), "bad cmp cache geometry")
    assert fn(C.byref(mk(T=0)), None) == _lib.SAS_OK


def test_abi_evict_refuses():
    L, fake = _lib.lib(), 1 << 20
    base = dict(cache=fake, weights=fake, block_table=fake, act_kv=fake, act_kv_out=fake, kept=fake, B=2, row_bytes=1152,
                bt_stride=4, block_size=64, num_blocks=8, weight_rows=256, budget=16, keep_first=4, keep_recent=4)
    fn = L.sas_cache_evict_v1
    assert fn(None, None) == _lib.SAS_EINVAL
    for change, needle in ((dict(budget=0), "budget"), (dict(keep_first=-1), "keep_first"), (dict(keep_recent=13), "keep_recent"),
                           (dict(keep_first=17, keep_recent=0), "keep_first"), (dict(row_bytes=8), "16 bytes"),
                           (dict(row_bytes=1160), "16 bytes"), (dict(weight_rows=-1), "weight_rows"),
                           (dict(bt_stride=0), "geometry"), (dict(num_blocks=1 << 30), "geometry"), (dict(kept=None), "null"),
                           (dict(weights=None), "null"), (dict(cache=fake + 8), "16-byte"), (dict(weights=fake + 4), "8-byte"),
                           (dict(B=-1), "B must"), (dict(B=65536), "B must"),
                           (dict(budget=(1 << 30) + 1), "budget"), (dict(weight_rows=(1 << 30) + 1), "weight_rows")):
        _refused(fn, _lib.SasCacheEvictArgs(**dict(base, **change)), needle)
    assert fn(C.byref(_lib.SasCacheEvictArgs(**dict(base, B=0))), None) == _lib.SAS_OK


def test_python_refuses():
    from dsv4_amd.api import add_row_weights, sparse_attn_sharedkv_first, sparse_attn_sharedkv_first_backward
    from dsv4_amd.cache import evict_kv_cache
    q = torch.zeros(3, 16, 512, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    kw = dict(ori_kv=torch.zeros(1, 16, 1, 512, dtype=torch.bfloat16), ori_block_table=i[:1, None], cu_seqlens_q=i,
              seqused_kv=i[:1], softmax_scale=1.0)
    sinks = torch.zeros(16)
    for bad in (-1, 1.0, True, None, 1 << 31, 1 << 70):
        with pytest.raises(ValueError, match="ori_first"):
            sparse_attn_sharedkv_first(q, ori_first=bad, sinks=sinks, **kw)
        with pytest.raises(ValueError, match="ori_first"):
            sparse_attn_sharedkv_first_backward(q, q, q, sinks, ori_first=bad, sinks=sinks, **kw)
    with pytest.raises(ValueError, match="GPU"):
        sparse_attn_sharedkv_first(q, ori_first=4, sinks=sinks, **kw)
    lse, w = torch.zeros(3, 16), torch.zeros(1, 16, dtype=torch.float64)
    with pytest.raises(ValueError, match="needs ori_weights or cmp_weights"):
        add_row_weights(q, lse, **kw)
    with pytest.raises(ValueError, match="without cmp_kv"):
        add_row_weights(q, lse, cmp_weights=w, **kw)
    for bad in (w.float(), w[0], torch.zeros(2, 16, dtype=torch.float64), torch.zeros(1, 32, dtype=torch.float64)[:, ::2]):
        with pytest.raises(ValueError, match="ori_weights must be"):
            add_row_weights(q, lse, ori_weights=bad, **kw)
    for bad in (lse.double(), lse[:2], lse.view(-1)):
        with pytest.raises(ValueError, match="lse must be"):
            add_row_weights(q, bad, ori_weights=w, **kw)
    with pytest.raises(ValueError, match="GPU"):
        add_row_weights(q, lse, ori_weights=w, **kw)
    c, e = kw["ori_kv"], dict(budget=4)
    for bad in (c[0], c.expand(2, 16, 1, 512), torch.zeros(1, 16, 2, 512)):
        with pytest.raises(ValueError, match="cache must be"):
            evict_kv_cache(bad, w, i[:1, None], i[:1], **e)
    with pytest.raises(ValueError, match="must agree"):
        evict_kv_cache(c, w, i[:, None], i[:1], **e)
    for bad in (w.float(), w[0], torch.zeros(2, 16, dtype=torch.float64)):
        with pytest.raises(ValueError, match="weights must be"):
            evict_kv_cache(c, bad, i[:1, None], i[:1], **e)
    for bad in (dict(budget=0), dict(budget=4, keep_first=-1), dict(budget=4, keep_first=3, keep_recent=2),
                dict(budget=(1 << 30) + 1), dict(budget=1 << 70), dict(budget=4, keep_first=1 << 70)):
        with pytest.raises(ValueError, match="budget must be at least 1"):
            evict_kv_cache(c, w, i[:1, None], i[:1], **bad)
    with pytest.raises(ValueError, match="must be an integer"):
        evict_kv_cache(c, w, i[:1, None], i[:1], budget=4.0)
    with pytest.raises(ValueError, match="GPU"):
        evict_kv_cache(c, w, i[:1, None], i[:1], **e)


# ---------------------------------------------------------------------------
# GPU: attention with first rows
# ---------------------------------------------------------------------------

ATTN = {
    "one": dict(H=16, D=576, ql=[1], kl=[500]),
    "step": dict(kind="scfa", H=64, D=576, ql=[1, 1, 1], kl=[900, 130, 3], K=70, gap=True, tail=2),
    "no_first": dict(H=16, D=512, ql=[1, 5], kl=[300, 40], F=0),
    "all_first": dict(H=32, D=512, ql=[3], kl=[90], F=500, win=2),
    "in_the_window": dict(H=16, D=576, ql=[9], kl=[130], F=4),         # some tokens' windows hold first rows
    "one_visible": dict(H=64, D=512, ql=[20], kl=[600], F=1, win=1, bs=16),
    "wide": dict(dt="fp16", H=16, D=576, ql=[10, 6], kl=[900, 100], win=600, F=70),
    "many_first": dict(kind="scfa", dt="fp16", H=32, D=512, ql=[4], kl=[1500], F=1290, K=40, win=64, gap=True),
    "fp8": dict(kind="scfa", dt="fp8", H=32, D=576, ql=[16, 3], kl=[600, 70], K=256, ratio=8, F=8, gap=True),
    "fp8_h16": dict(dt="fp8", H=16, D=576, ql=[9], kl=[300]),
    "fp8_h128": dict(kind="cfa", dt="fp8", H=128, D=576, ql=[5], kl=[500], ratio=8, F=17),
    "cfa": dict(kind="cfa", H=64, D=576, ql=[9, 14], kl=[800, 90], ratio=8),
    "odd_heads": dict(H=48, D=576, ql=[7, 2], kl=[400, 33], F=5, win=100),
    "one_h32": dict(H=32, D=512, ql=[1], kl=[300]),
    "one_h80": dict(dt="fp16", H=80, D=576, ql=[1], kl=[200], F=60),
    "one_fp8_h48": dict(dt="fp8", H=48, D=576, ql=[1, 0, 1], kl=[300, 5, 1], F=9),
    "many_256": dict(H=64, D=576, ql=[50, 30, 20], kl=[500, 200, 20], F=7, win=249),
    "missing_rows": dict(kind="scfa", H=64, D=576, ql=[12, 70], kl=[5, 30], K=70),
    "holes": dict(H=64, D=576, ql=[4, 4], kl=[270, 290], holes=True),
    "empty_between": dict(H=64, D=512, ql=[4, 0, 5], kl=[270, 7, 190], gap=True),
    "long_topk": dict(kind="scfa", H=128, D=576, ql=[2], kl=[5000], K=1100, F=16),
    # runs of tokens
    "prompt": dict(H=64, D=576, ql=[300], kl=[300]),
    "prompt_512": dict(H=64, D=512, ql=[280], kl=[1000], gap=True, tail=5),
    "prompt_fp16": dict(dt="fp16", H=128, D=512, ql=[150, 3, 0, 90], kl=[400, 3, 9, 95], F=16, win=100, bs=16),
    "prompt_narrow": dict(H=64, D=576, ql=[200, 150], kl=[220, 800], F=8, win=3),
    "prompt_whole_first": dict(H=64, D=512, ql=[300], kl=[310], F=33, win=64),
    "prompt_holes": dict(H=64, D=576, ql=[150, 160], kl=[270, 290], holes=True),
    "prompt_missing": dict(H=64, D=576, ql=[300, 40], kl=[200, 900], F=6, win=20),
    "chunk_cfa": dict(kind="cfa", H=64, D=512, ql=[300], kl=[1300], ratio=64),
}


def _run(c, q=None, **kw):
    from dsv4_amd.api import sparse_attn_sharedkv_first
    return sparse_attn_sharedkv_first(c.q.cuda() if q is None else q, return_softmax_lse=True,
                                      **(kw if "ori_kv" in kw else dict(c.kwargs(), **kw)))


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(ATTN))
def test_gpu_first(name):
    c = Case(**ATTN[name])
    out, lse = _run(c)
    c.check(out, lse)
    again, lse2 = _run(c)                       # the kept resolution
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.gpu
def test_gpu_first_zero_is_the_attention():
    from dsv4_amd.api import sparse_attn_sharedkv
    c = Case(kind="scfa", H=64, D=576, ql=[3, 40], kl=[300, 90], F=0, K=64)
    out, lse = _run(c)
    ref, ref_lse = sparse_attn_sharedkv(c.q.cuda(), return_softmax_lse=True, **c.kwargs(first=False))
    assert torch.equal(out, ref) and torch.equal(lse, ref_lse)


@pytest.mark.gpu
def test_gpu_first_layouts_lengths_and_streams():
    """BSND queries, host-side lengths, another stream, out only."""
    c = Case(kind="scfa", H=32, D=576, ql=[5, 3], kl=[300, 90], K=64)
    ref, ref_lse = _run(c)
    out, lse = _run(c, **{k: v for k, v in c.kwargs(host_lens=True).items() if k in ("cu_seqlens_q", "seqused_kv")})
    assert torch.equal(out, ref) and torch.equal(lse, ref_lse)
    st = torch.cuda.Stream()
    kw, q = c.kwargs(), c.q.cuda()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        out, lse = _run(c, q, **kw)
    torch.cuda.synchronize()
    assert torch.equal(out, ref) and torch.equal(lse, ref_lse)
    qb = torch.zeros(2, 5, 32, 576, dtype=c.dt)
    ib = torch.full((2, 5, 1, 64), -1, dtype=torch.int32)
    qb[0], qb[1, :3], ib[0], ib[1, :3] = c.q[:5], c.q[5:], c.idx[:5], c.idx[5:]
    out, lse = _run(c, qb.cuda(), cmp_sparse_indices=ib.cuda(), layout_q="BSND")
    assert torch.equal(out[0], ref[:5]) and torch.equal(out[1, :3], ref[5:]) and bool((out[1, 3:] == 0).all())
    assert torch.equal(lse[1, :3], ref_lse[5:])


@pytest.mark.gpu
def test_gpu_first_masked_rows_are_not_read():
    """NaN in the rows between the first ones and the window, and in blocks of no
    sequence; an infinite sink logit of either sign."""
    c = Case(H=64, D=576, ql=[3], kl=[700], F=4, bs=64)
    ref, ref_lse = _run(c)
    kw = c.kwargs()
    flat = kw["ori_kv"].view(-1, 576)
    seen = torch.tensor(sorted({r for at in c.keys.raw for r in at[1]}))
    other = torch.ones(flat.shape[0], dtype=torch.bool)
    other[seen] = False
    flat[other.cuda()] = float("nan")
    out, lse = _run(c, **kw)
    assert torch.equal(out, ref) and torch.equal(lse, ref_lse)
    kw["sinks"] = torch.full((64,), -float("inf"), device="cuda")
    out, lse = _run(c, **kw)
    assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(lse).all())


@pytest.mark.gpu
def test_gpu_first_captured():
    """Captured and replayed with the program's own eager calls between."""
    c = Case(kind="scfa", H=32, D=576, ql=[1, 1], kl=[500, 90], K=64)
    kw, q = c.kwargs(), c.q.cuda()
    ref, ref_lse = _run(c, q, **kw)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = _run(c, q, **kw)
    for i in range(4):
        out.zero_()
        g.replay()
        eager, _ = _run(c, q, **kw)
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and torch.equal(lse, ref_lse) and torch.equal(eager, ref), i


# ---------------------------------------------------------------------------
# GPU: gradients
# ---------------------------------------------------------------------------

GRAD = {
    "one": dict(H=16, D=576, ql=[1], kl=[400]),
    "step": dict(kind="scfa", H=64, D=512, ql=[1, 2], kl=[500, 140], K=40, gap=True),
    "per_token": dict(kind="scfa", dt="fp16", H=16, D=576, ql=[70, 3], kl=[300, 20], K=30, win=40, F=5),
    "prompt": dict(H=64, D=576, ql=[200], kl=[260], win=64),
    "prompt_512": dict(H=32, D=512, ql=[90, 70], kl=[90, 400], F=16, gap=True, tail=3),
    "prompt_scfa": dict(kind="scfa", dt="fp16", H=32, D=512, ql=[130], kl=[500], K=20, F=70, win=50),
    "prompt_cfa": dict(kind="cfa", H=64, D=576, ql=[100], kl=[700], ratio=16, F=130, win=30, bs=16),
    "prompt_no_first": dict(H=32, D=576, ql=[100], kl=[150], F=0, win=64),
    "prompt_first_beyond": dict(H=32, D=512, ql=[100], kl=[100], F=1000, win=5),
    "prompt_two_tiles": dict(H=32, D=576, ql=[90, 60], kl=[90, 33], F=25, win=10, bs=16, holes=True),
    "prompt_32_rows": dict(dt="fp16", H=64, D=512, ql=[120], kl=[150], F=32, win=1),
    "prompt_33_rows": dict(dt="fp16", H=64, D=512, ql=[120], kl=[150], F=33, win=3),
    "prompt_missing": dict(H=32, D=576, ql=[100, 80], kl=[60, 300], F=6, win=20),
    "prompt_holes": dict(H=64, D=512, ql=[100, 80], kl=[260, 300], holes=True, F=6, win=20),
    "dense_32_heads": dict(kind="scfa", H=32, D=512, ql=[120], kl=[3300], K=64, F=9, win=70, ratio=4),   # 448 to 896 rows: key-major
    "sparse_32_heads": dict(kind="scfa", H=32, D=512, ql=[70], kl=[3700], K=64, F=9, win=70, ratio=4),   # past 896 rows: per token
    "sparse_beyond": dict(kind="scfa", H=64, D=576, ql=[90], kl=[900], K=6, F=9, win=70),   # tokens whose rows are added per token
}


def _grads(c, out, lse, kw, window_pass=None, dout=None, q=None):
    from dsv4_amd.api import sparse_attn_sharedkv_first_backward
    more = {} if window_pass is None else {"window_pass": window_pass}
    return sparse_attn_sharedkv_first_backward(c.dout.cuda() if dout is None else dout, c.q.cuda() if q is None else q, out, lse,
                                               **kw, **more)


def _check_grads(c, got, out, lse):
    g, e = c.gradients(out.cpu(), lse.cpu())
    dq, d_ori, d_cmp, d_sinks = got
    assert dq.dtype is c.dt and d_ori.dtype is torch.float32 and d_sinks.dtype is torch.float32
    pairs = [(dq, "dq"), (d_ori, "rows"), (d_sinks, "sinks")] + ([(d_cmp, "crows")] if c.crows is not None else [])
    for x, name in pairs:
        err, bound = (x.cpu().double().view_as(g[name]) - g[name]).abs(), e[name] + 2.0 ** -40
        assert bool((err <= bound).all()), f"{name}: worst {float((err / bound).max()):.3g} of the bound"
    assert d_cmp is None or c.crows is not None


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(GRAD))
def test_gpu_first_backward(name):
    c = Case(**GRAD[name])
    kw = c.kwargs()
    out, lse = _run(c, **kw)
    _check_grads(c, _grads(c, out, lse, kw), out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("first", [20, 40])
def test_gpu_first_backward_keeps_a_tokens_nan_to_its_rows(first):
    # a token at position 3 with a window of 2 attends rows 0 .. 3: a NaN in its query
    # leaves the gradients of every other row as if the token had none
    c = Case(H=32, D=512, ql=[70], kl=[70], F=first, win=2)
    kw = c.kwargs()
    quiet, dout = c.q.cuda().clone(), c.dout.cuda().clone()
    quiet[3] = 0
    dout[3] = 0
    out, lse = _run(c, quiet, **kw)
    want = _grads(c, out, lse, kw, dout=dout, q=quiet)[1]
    loud = quiet.clone()
    loud[3, 5, 7] = float("nan")
    out, lse = _run(c, loud, **kw)
    got = _grads(c, out, lse, kw, q=loud)[1]
    rows = want.view(-1, c.D)
    hit = torch.isnan(got.view(-1, c.D)).any(1)
    bt = kw["ori_block_table"][0].long()
    attended = torch.zeros(rows.shape[0], dtype=torch.bool, device="cuda")
    for j in range(4):
        attended[bt[j // c.bs] * c.bs + j % c.bs] = True
    assert torch.equal(hit, attended)
    # what is left differs by the order of the float32 adds: at most 69 tokens' terms, each below
    # the largest gradient times some tens
    err = (got.view(-1, c.D)[~hit] - rows[~hit]).abs().max()
    assert float(err) <= 69 * 69 * 2.0 ** -24 * 16 * float(rows.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("window_pass", [True, False])
def test_gpu_first_backward_both_ways(window_pass):
    c = Case(kind="scfa", H=64, D=576, ql=[80], kl=[200], K=20, F=5, win=40)
    kw = c.kwargs()
    out, lse = _run(c, **kw)
    _check_grads(c, _grads(c, out, lse, kw, window_pass), out, lse)


@pytest.mark.gpu
def test_gpu_first_autograd():
    from dsv4_amd.api import sparse_attn_sharedkv_first_autograd
    c = Case(kind="scfa", H=32, D=576, ql=[70], kl=[300], K=20, win=50)
    kw = c.kwargs()
    leaf = {k: kw.pop(k).requires_grad_() for k in ("ori_kv", "cmp_kv", "sinks")}
    q = c.q.cuda().requires_grad_()
    out, lse = sparse_attn_sharedkv_first_autograd(q, return_softmax_lse=True, **leaf, **kw)
    assert not lse.requires_grad
    out.backward(c.dout.cuda())
    want = _grads(c, out.detach(), lse, c.kwargs())
    assert torch.equal(q.grad, want[0])
    for x, w in zip(leaf.values(), want[1:]):
        # sums of atomic adds, in any order: fp32's rounding of at most 300 adds, then the leaf's type
        assert x.grad.dtype is x.dtype
        tol = (2.0 ** -15 if x.dtype is torch.float32 else c.half * 1.01) * (w.abs() + w.abs().max() * 2.0 ** -10)
        assert bool(((x.grad.double() - w.double()).abs() <= tol).all())


@pytest.mark.gpu
def test_gpu_first_backward_captured():
    c = Case(H=32, D=512, ql=[100], kl=[300], F=5, win=40)
    kw, q, dout = c.kwargs(), c.q.cuda(), c.dout.cuda()
    out, lse = _run(c, q, **kw)
    ref = _grads(c, out, lse, kw, dout=dout, q=q)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = _grads(c, out, lse, kw, dout=dout, q=q)
    for i in range(3):
        g.replay()
        _grads(c, out, lse, kw, dout=dout, q=q)
        torch.cuda.synchronize()
        assert torch.equal(got[0], ref[0]), i
        _check_grads(c, got, out, lse)


# ---------------------------------------------------------------------------
# GPU: weights
# ---------------------------------------------------------------------------

WEIGHTS = {
    "one": dict(H=16, D=512, ql=[1], kl=[500], win=1000, F=0),
    "one_row": dict(H=16, D=576, ql=[1, 1], kl=[1, 2]),
    "bounded": dict(H=64, D=576, ql=[1, 1, 1], kl=[700, 129, 128], win=2000, F=0, tail=2),
    "fp16_h128": dict(dt="fp16", H=128, D=512, ql=[2, 3], kl=[300, 31], win=4000, bs=16),
    "odd_heads": dict(H=48, D=576, ql=[3], kl=[200], win=400),
    "window": dict(H=64, D=576, ql=[1, 3], kl=[700, 90], gap=True),
    "fp8": dict(kind="scfa", dt="fp8", H=64, D=576, ql=[4, 1], kl=[900, 60], K=200, F=8, gap=True),
    "fp8_full": dict(dt="fp8", H=16, D=576, ql=[3], kl=[333], win=400),
    "scfa": dict(kind="scfa", H=32, D=512, ql=[5, 0, 9], kl=[600, 7, 200], K=130, ratio=2),
    "cfa": dict(kind="cfa", H=64, D=576, ql=[3, 9], kl=[800, 90], ratio=4, F=20, win=30),
    "missing_rows": dict(H=16, D=576, ql=[12, 70], kl=[5, 30], win=10),
    "holes": dict(H=64, D=576, ql=[4, 4], kl=[270, 290], holes=True, win=1000),
    # runs of tokens
    "prompt_end": dict(H=64, D=512, ql=[64], kl=[900], win=1000, F=0),
    "prompt_ends": dict(dt="fp16", H=16, D=576, ql=[33, 70, 5], kl=[400, 70, 1000], win=1000, bs=16, tail=3),
    "prompt_fp8": dict(dt="fp8", H=32, D=576, ql=[40], kl=[700], win=1000),
    "prompt_window": dict(H=32, D=512, ql=[200], kl=[300], win=60, F=5),
    "prompt_first": dict(H=32, D=576, ql=[90, 30], kl=[300, 200], win=20, F=150, holes=True),
    "prompt_cfa": dict(kind="cfa", H=64, D=512, ql=[100], kl=[900], ratio=4, F=4, win=64),
    "prompt_scfa": dict(kind="scfa", dt="fp8", H=32, D=576, ql=[60, 20], kl=[500, 100], K=40, F=4, win=64),
    "prompt_missing": dict(H=32, D=512, ql=[90], kl=[40], win=30, F=4),
}


def _weights(c, lse, ori, cmp_, kw=None, q=None):
    from dsv4_amd.api import add_row_weights
    add_row_weights(c.q.cuda() if q is None else q, lse, ori_weights=ori, cmp_weights=cmp_, **(kw or c.kwargs()))


def _zeros(c):
    z = lambda t: torch.zeros(len(c.ql), t.shape[1] * c.bs, dtype=torch.float64, device="cuda")  # noqa: E731
    return z(c.table), None if c.ctable is None else z(c.ctable)


def _check_weights(c, lse, ori, cmp_, calls=1):
    w, wc = c.weights(lse.cpu(), ori.shape[1])
    for x, ref in ((ori, w), (cmp_, wc)):
        if x is None:
            continue
        x, adds = x.cpu(), 2.0 ** -37 * calls * max(1, c.T)
        err = (x - calls * ref).abs()
        assert bool((err <= 2.0 ** -12 * calls * ref + adds).all()), float((err / (calls * ref + 1e-30)).max())
        assert bool((x[ref == 0] == 0).all())                       # rows that no token attends
        assert torch.equal(torch.round(x * 2.0 ** 36), x * 2.0 ** 36)   # the grid


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(WEIGHTS))
def test_gpu_weights(name):
    c = Case(**WEIGHTS[name])
    lse = c.attention()[1].float().cuda()
    ori, cmp_ = _zeros(c)
    _weights(c, lse, ori, cmp_)
    _check_weights(c, lse, ori, cmp_)
    one, onec = ori.clone(), None if cmp_ is None else cmp_.clone()
    _weights(c, lse, ori, cmp_)                                     # the kept resolution; the same bits
    assert torch.equal(ori, 2 * one) and (cmp_ is None or torch.equal(cmp_, 2 * onec))


def _odd(t):
    # the same values two or four bytes behind a 16-byte boundary
    room = torch.empty(t.numel() + 8, dtype=t.dtype, device="cuda")
    out = room[1:1 + t.numel()].view(t.shape)
    out.copy_(t)
    assert out.data_ptr() % 16 and out.is_contiguous()
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["q", "dout", "out", "all"])
def test_gpu_tensors_at_odd_addresses(which):
    c = Case(kind="scfa", H=32, D=576, ql=[70, 2], kl=[300, 90], K=20, F=5, win=40)
    kw, q, dout = c.kwargs(), c.q.cuda(), c.dout.cuda()
    out, lse = _run(c, q, **kw)
    ori, cmp_ = _zeros(c)
    _weights(c, lse, ori, cmp_, q=q)
    if which in ("q", "all"):
        q = _odd(q)
        got = _run(c, q, **kw)
        assert torch.equal(got[0], out) and torch.equal(got[1], lse)
    if which in ("dout", "all"):
        dout = _odd(dout)
    if which in ("out", "all"):
        out, lse = _odd(out), _odd(lse)
    _check_grads(c, _grads(c, out, lse, kw, dout=dout, q=q), out, lse)
    o, k = _zeros(c)
    _weights(c, lse, o, k, q=q)
    assert torch.equal(o, ori) and torch.equal(k, cmp_)


@pytest.mark.gpu
def test_gpu_weights_of_one_cache_alone():
    c = Case(**WEIGHTS["scfa"])
    lse = c.attention()[1].float().cuda()
    both, alone = _zeros(c), _zeros(c)
    _weights(c, lse, *both)
    _weights(c, lse, alone[0], None)
    _weights(c, lse, None, alone[1])
    assert torch.equal(both[0], alone[0]) and torch.equal(both[1], alone[1])


@pytest.mark.gpu
def test_gpu_weights_short_tensors():
    """Rows past the weights' rows are left out."""
    c = Case(H=16, D=512, ql=[40, 1], kl=[300, 30], win=1000)
    lse = c.attention()[1].float().cuda()
    full, short = _zeros(c)[0], torch.zeros(2, 77, dtype=torch.float64, device="cuda")
    _weights(c, lse, full, None)
    _weights(c, lse, short, None)
    assert torch.equal(short, full[:, :77])
    none = torch.zeros(2, 0, dtype=torch.float64, device="cuda")
    _weights(c, lse, none, None)


@pytest.mark.gpu
def test_gpu_weights_layouts_lengths_streams_capture():
    c = Case(kind="scfa", H=32, D=576, ql=[5, 3], kl=[300, 90], K=64)
    lse = c.attention()[1].float().cuda()
    ref = _zeros(c)
    _weights(c, lse, *ref)
    for _ in range(2):
        got = _zeros(c)
        _weights(c, lse, *got, kw=c.kwargs(host_lens=True))
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    qb, ib, lb = torch.zeros(2, 5, 32, 576, dtype=c.dt), torch.full((2, 5, 1, 64), -1, dtype=torch.int32), torch.zeros(2, 5, 32)
    qb[0], qb[1, :3], ib[0], ib[1, :3], lb[0], lb[1, :3] = c.q[:5], c.q[5:], c.idx[:5], c.idx[5:], lse[:5].cpu(), lse[5:].cpu()
    got = _zeros(c)
    _weights(c, lb.cuda(), *got, kw=dict(c.kwargs(), cmp_sparse_indices=ib.cuda(), layout_q="BSND"), q=qb.cuda())
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    kw, q = c.kwargs(), c.q.cuda()
    got, st = _zeros(c), torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        _weights(c, lse, *got, kw=kw, q=q)
    torch.cuda.synchronize()
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    got, g = _zeros(c), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _weights(c, lse, *got, kw=kw, q=q)
    for i in range(1, 4):
        g.replay()
        _weights(c, lse, *_zeros(c), kw=kw, q=q)
        torch.cuda.synchronize()
        assert torch.equal(got[0], i * ref[0]) and torch.equal(got[1], i * ref[1])


@pytest.mark.gpu
def test_gpu_weights_masked_rows_are_not_read():
    c = Case(H=32, D=576, ql=[40], kl=[500], F=4, win=30)
    lse = c.attention()[1].float().cuda()
    ref = _zeros(c)[0]
    _weights(c, lse, ref, None)
    kw = c.kwargs()
    flat = kw["ori_kv"].view(-1, 576)
    other = torch.ones(flat.shape[0], dtype=torch.bool)
    other[torch.tensor(sorted({r for at in c.keys.raw for r in at[1]}))] = False
    flat[other.cuda()] = float("nan")
    got = _zeros(c)[0]
    _weights(c, lse, got, None, kw=kw)
    assert torch.equal(got, ref)


@pytest.mark.gpu
def test_gpu_weights_of_nan():
    """A NaN row's weight is NaN, and no other's."""
    c = Case(H=16, D=512, ql=[3], kl=[90], win=1000, F=0)
    lse = c.attention()[1].float().cuda()
    kw = c.kwargs()
    kw["ori_kv"].view(-1, 512)[c.keys.raw[0][1][7]] = float("nan")
    got = _zeros(c)[0]
    _weights(c, lse, got, None, kw=kw)
    bad = torch.isnan(got[0]).nonzero().view(-1).tolist()
    assert bad == [7]


# ---------------------------------------------------------------------------
# GPU: evictions
# ---------------------------------------------------------------------------

def _evict_case(lens, budget, first=0, recent=0, bs=16, row=512, dt=torch.bfloat16, rows=None, seed=5, spare=0, zero=0.3):
    g = torch.Generator().manual_seed(seed)
    per = max(1, max(-(-max(n, 1) // bs) for n in lens)) + spare
    nb = per * len(lens) + 2
    table = torch.randperm(nb, generator=g)[:per * len(lens)].to(torch.int32).view(len(lens), per)
    cache = torch.randint(0, 256, (nb, bs, 1, row * dt.itemsize), generator=g, dtype=torch.uint8).view(dt)
    R_ = per * bs if rows is None else rows
    w = torch.randint(0, 1 << 30, (len(lens), R_), generator=g).double() * 2.0 ** -36
    w[torch.rand(w.shape, generator=g) < zero] = 0.0
    return cache, w, table, torch.tensor(lens, dtype=torch.int32), budget, first, recent


def _evict(cache, w, table, used, budget, first, recent):
    from dsv4_amd.cache import evict_kv_cache
    c, d = cache.cuda(), w.cuda()
    n, kept = evict_kv_cache(c, d, table.cuda(), used.cuda(), budget=budget, keep_first=first, keep_recent=recent)
    return c.cpu(), d.cpu(), n.cpu(), kept.cpu()


def _same(got, ref):
    assert got[2].tolist() == ref[2].tolist()
    assert torch.equal(got[3], ref[3])
    assert torch.equal(got[0].view(torch.uint8), ref[0].view(torch.uint8))
    assert torch.equal(got[1].nan_to_num(nan=-7.0, posinf=9.0, neginf=-9.0), ref[1].nan_to_num(nan=-7.0, posinf=9.0, neginf=-9.0))


EVICT = {
    "one_row_leaves": dict(lens=[65], budget=64, first=4, recent=8),
    "lengths": dict(lens=[0, 1, 40, 41, 42, 300, 39, 1000], budget=41, first=4, recent=16),
    "budget_of_one": dict(lens=[1, 2, 50], budget=1),
    "only_protected": dict(lens=[100, 33], budget=20, first=12, recent=8),
    "only_first": dict(lens=[100], budget=20, first=20),
    "only_recent": dict(lens=[100], budget=20, recent=20),
    "all_equal": dict(lens=[500, 77], budget=60, recent=3, zero=2.0),
    "long": dict(lens=[5000, 3000, 1025], budget=1100, first=3, recent=64, bs=64),
    "long_budget": dict(lens=[2500], budget=2499, first=1, recent=1, bs=128),
    "fp8_rows": dict(lens=[300, 400], budget=200, first=4, recent=10, row=656, dt=torch.uint8, bs=64),
    "wide_rows": dict(lens=[300], budget=100, row=576, dt=torch.float16, bs=7),
    "narrow_rows": dict(lens=[300, 20], budget=100, row=8, bs=3),
    "fp32_rows": dict(lens=[150], budget=100, row=4, dt=torch.float32, spare=3),
    "short_weights": dict(lens=[300, 90], budget=50, first=2, recent=5, rows=77),
    "no_weights": dict(lens=[300], budget=50, first=2, recent=5, rows=0),
    "many": dict(lens=[30 + 7 * i for i in range(70)], budget=100, first=4, recent=16),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(EVICT))
def test_gpu_evict(name):
    a = _evict_case(**EVICT[name])
    _same(_evict(*a), R.evict(*a))


@pytest.mark.gpu
def test_gpu_evict_odd_weights():
    """NaN below everything, infinities, zeros of both signs (equal), negative and tiny
    weights, neighbours in the last bit."""
    a = _evict_case([200], 90, 2, 3)
    w = a[1]
    w[0, 10:20] = float("nan")
    w[0, 20:25], w[0, 25:30] = float("inf"), -float("inf")
    w[0, 30:60:2], w[0, 31:60:2] = 0.0, -0.0
    w[0, 60:70] = -torch.rand(10, dtype=torch.float64)
    w[0, 70:75] = 5e-324
    w[0, 75:130] = 1.0 + 2.0 ** -52 * torch.arange(55, dtype=torch.float64).flip(0)
    for budget in (90, 7, 30, 60, 100, 150, 190, 196):
        b = (a[0], w, a[2], a[3], budget, 2, 3)
        _same(_evict(*b), R.evict(*b))


@pytest.mark.gpu
def test_gpu_evict_nan_beside_equal_weights():
    """Whole waves of NaN, others of one weight each side of them in the order."""
    for other in (-float("inf"), 5e-324, float("inf")):
        a = _evict_case([2000], 1200, 2, 3)
        a[1][:] = float("nan")
        a[1][0, 500:1300] = other
        _same(_evict(*a), R.evict(*a))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [4096, 4097, 32768, 32769, 40000])
def test_gpu_evict_long(n):
    """Each side of the lengths that the selection keeps in registers."""
    for budget, zero in ((n - 1, 0.3), (1000, 0.3), (n // 2, 0.9)):
        a = _evict_case([n, 50], budget, 4, 64, bs=64, row=8, zero=zero)
        _same(_evict(*a), R.evict(*a))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3000, 9000, 33000])
@pytest.mark.parametrize("spread", [50, 1 << 20, 1 << 45])
def test_gpu_evict_close_weights(n, spread):
    """Weights that differ in their last bits only, or in those and a few above, with NaN,
    zeros and infinities around them; the edge at each end and in the middle."""
    a = _evict_case([n], 10, 2, 3, bs=64, row=8)
    g = torch.Generator().manual_seed(2)
    a[1][:] = 1.0 + torch.randint(0, spread, a[1].shape, generator=g).double() * 2.0 ** -52
    a[1][0, 40:80], a[1][0, 100:300], a[1][0, 350:360] = float("nan"), 0.0, float("inf")
    a[1][0, 400:500] = -a[1][0, 400:500]
    for budget in (12, 16, 200, n // 2, n - 400, n - 200, n - 45, n - 20):
        b = a[:4] + (budget, 2, 3)
        _same(_evict(*b), R.evict(*b))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [4097, 20000, 32767, 32768])
@pytest.mark.parametrize("kind", ["few", "narrow", "squares", "below"])
def test_gpu_evict_distributions(n, kind):
    """Weights that fill their range unevenly: five values, a few thousand neighbouring ones
    of one binade, squares, all at or below 0."""
    a = _evict_case([n, 5000], 10, 4, 64, bs=64, row=8)
    g = torch.Generator().manual_seed(3)
    u = torch.rand(a[1].shape, generator=g, dtype=torch.float64)
    a[1][:] = {"few": (u * 5).floor() / 7, "narrow": 1 + (u * 4096).floor() * 2.0 ** -34, "squares": (u * u * 2 ** 20).round() * 2.0 ** -36,
               "below": -(u * 3).floor()}[kind]
    for budget in (100, n // 7, n // 2, n - 90):
        b = a[:4] + (budget, 4, 64)
        _same(_evict(*b), R.evict(*b))


@pytest.mark.gpu
def test_gpu_evict_rows_without_blocks():
    """A moved row needs both blocks; entries out of range count as none, nothing is
    read or written through them."""
    a = _evict_case([300, 310], 200, 4, 50)
    table = a[2]
    table[0, 3], table[0, 12], table[1, 5], table[1, 0] = -1, 1 << 30, a[0].shape[0], -7
    used = torch.tensor([300, 700], dtype=torch.int32)     # past the table's end
    b = (a[0], a[1], table, used, 200, 4, 50)
    _same(_evict(*b), R.evict(*b))


@pytest.mark.gpu
def test_gpu_evict_streams_and_capture():
    from dsv4_amd.cache import evict_kv_cache
    a = _evict_case([300, 20, 500], 100, 4, 16)
    ref = R.evict(*a)
    cache, w, table, used = (t.cuda() for t in a[:4])
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        n, kept = evict_kv_cache(cache, w, table, used, budget=100, keep_first=4, keep_recent=16)
    torch.cuda.synchronize()
    _same((cache.cpu(), w.cpu(), n.cpu(), kept.cpu()), ref)
    cache, w = a[0].cuda(), a[1].cuda()
    fresh = [cache.clone(), w.clone()]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.copy_(fresh[0])
        w.copy_(fresh[1])
        n, kept = evict_kv_cache(cache, w, table, used, budget=100, keep_first=4, keep_recent=16)
    for _ in range(3):
        g.replay()
        _evict(*a)
        torch.cuda.synchronize()
        _same((cache.cpu(), w.cpu(), n.cpu(), kept.cpu()), ref)


@pytest.mark.gpu
def test_gpu_evict_int64_lengths():
    a = _evict_case([300, 20], 100, 4, 16)
    ref = R.evict(*a)
    got = _evict(a[0], a[1], a[2].long(), a[3].long(), *a[4:])
    _same(got, ref)


# ---------------------------------------------------------------------------
# GPU: long caches
# ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("ql", [[3, 1], [70, 40]])
def test_gpu_rows_past_32_bit_offsets(ql):
    """A cache of more than 2^32 bytes whose blocks at the end hold the rows: what the
    small cache with the same blocks at its start gives."""
    from dsv4_amd.cache import evict_kv_cache
    c = Case(H=64, D=576, ql=ql, kl=[300, 200], F=6, win=64)
    kw = c.kwargs()
    small, table = kw["ori_kv"], kw["ori_block_table"]
    nb = small.shape[0]
    far = (5 << 30) // (c.bs * c.D * 2)
    big = torch.zeros(far + nb, c.bs, 1, c.D, dtype=c.dt, device="cuda")
    big[far:] = small
    there = dict(kw, ori_kv=big, ori_block_table=torch.where(table >= 0, table + far, table))
    (out, lse), (o2, l2) = _run(c, **kw), _run(c, **there)
    assert torch.equal(out, o2) and torch.equal(lse, l2)
    (w, _), (w2, _) = _zeros(c), _zeros(c)
    _weights(c, lse, w, None, kw)
    _weights(c, lse, w2, None, there)
    assert torch.equal(w, w2)
    g, g2 = _grads(c, out, lse, kw), _grads(c, out, lse, there)
    _check_grads(c, (g2[0], g2[1][far:].clone(), g2[2], g2[3]), out, lse)
    assert torch.equal(g[0], g2[0]) and not bool(g2[1][:far].any())
    del g2
    left = [evict_kv_cache(k["ori_kv"], x, k["ori_block_table"], k["seqused_kv"], budget=90, keep_first=4, keep_recent=20)
            for k, x in ((kw, w), (there, w2))]
    assert torch.equal(left[0][0], left[1][0]) and torch.equal(left[0][1], left[1][1]) and torch.equal(w, w2)
    assert torch.equal(small.view(torch.int16), big[far:].view(torch.int16)) and not bool(big[:far].view(torch.int16).any())


# ---------------------------------------------------------------------------
# GPU: a run of them together
# ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("D", [512, 576])
def test_gpu_bounded_decode(D):
    """Steps of append, attention over all rows, weights and, whenever a sequence is over
    its budget, eviction; every step against the oracle on the caches' own bytes."""
    from dsv4_amd.api import add_row_weights, sparse_attn_sharedkv_first
    from dsv4_amd.cache import append_kv_cache, evict_kv_cache
    from dsv4_amd.rope import rope_table
    g = torch.Generator().manual_seed(11)
    B, H, bs, budget = 3, 32, 16, 40
    per, cap = 4, 48
    nb = B * per + 1
    table = torch.randperm(nb, generator=g)[:B * per].to(torch.int32).view(B, per)
    cache = torch.zeros(nb, bs, 1, D, dtype=torch.bfloat16, device="cuda")
    weights = torch.zeros(B, per * bs, dtype=torch.float64, device="cuda")
    angles = rope_table(4096, 64)
    sinks = torch.randn(H, generator=g)
    used = torch.zeros(B, dtype=torch.int32, device="cuda")
    place = torch.zeros(B, dtype=torch.int32)          # the positions that angles belong to
    seen_eviction = 0
    for step in range(14):
        new = [5, 9, 2] if step % 3 == 0 else [1, 1, 1]
        T = sum(new)
        cu = torch.tensor([0, new[0], new[0] + new[1], T], dtype=torch.int32)
        pos = torch.cat([torch.arange(int(p), int(p) + m, dtype=torch.int32) for p, m in zip(place, new)])
        place += torch.tensor(new, dtype=torch.int32)
        used = used + torch.tensor(new, dtype=torch.int32, device="cuda")
        q = torch.randn(T, H, D, generator=g).to(torch.bfloat16).cuda()
        kv = torch.randn(T, D, generator=g).to(torch.bfloat16).cuda()
        q = append_kv_cache(kv, cache, table.cuda(), cu.cuda(), used, table=angles, positions=pos.cuda(), q=q)
        kw = dict(ori_kv=cache, ori_block_table=table.cuda(), cu_seqlens_q=cu.cuda(), seqused_kv=used, sinks=sinks.cuda(),
                  softmax_scale=D ** -0.5, ori_win_left=cap + 16, ori_first=0)
        out, lse = sparse_attn_sharedkv_first(q, return_softmax_lse=True, **kw)
        keys = R.Keys(table, None, None, new, used.tolist(), 0, cap + 17, bs, bs, 1, T)
        rows = cache.cpu().view(-1, D)
        ref, ref_lse, mag = R.attention(keys, q.cpu(), rows, None, sinks, D ** -0.5)
        assert bool(((out.cpu().double() - ref).abs() <= 1.5 * 2.0 ** -8 * (mag + ref.abs()) + 2.0 ** -16).all()), step
        assert float((lse.cpu().double() - ref_lse).abs().max()) <= 1e-3
        before = weights.cpu()
        add_row_weights(q, lse, ori_weights=weights, **kw)
        w = before + R.weights(keys, q.cpu(), lse.cpu(), rows, None, D ** -0.5, B, per * bs, 1)[0]
        assert bool(((weights.cpu() - w).abs() <= 2.0 ** -12 * w + T * 2.0 ** -37).all()), step
        if int(used.max()) > budget:
            seen_eviction += 1
            want = R.evict(cache.cpu(), weights.cpu(), table, used.cpu(), budget, 4, 8)
            used, kept = evict_kv_cache(cache, weights, table.cuda(), used, budget=budget, keep_first=4, keep_recent=8)
            _same((cache.cpu(), weights.cpu(), used.cpu(), kept.cpu()), want)
    assert seen_eviction >= 2

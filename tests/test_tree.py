"""Attention for trees of drafted tokens (sparse_attn_sharedkv_tree): the CPU
oracle pinned by known windows and the linear oracle, argument errors without a
device, and the kernels against the oracle.

Tolerances, with h half a step of the query's dtype: P is rounded once, the output
once, a split's partial to fp16 under bf16 outputs (h / 8). A score is a sum of 576
fp32 products whose partial sums stay below 100: off by at most 576 x 2^-24 x 100 x
scale = 2^-12.8, which its P is off relatively (0.28 h in fp16). Together below
1.5 h (sum p |v| + |out|). fp16 P below 2^-14 rounds by 2^-25 absolutely: at most 1300
keys x 2^-25 x max |v| (4.6) over a sum of at least 1, below 2^-12. LSE: the linear
operator's 1e-3."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from dsv4_amd import _lib, paged
from oracle import golden_ref as O
from oracle import tree_ref as R


# ---------------------------------------------------------------------------
# oracle
# ---------------------------------------------------------------------------

def _known_windows(**kw):
    # 10 committed rows, nodes 0 - 1 - 3 and 0 - 2: node 3 attends {0, 1, 3}
    assert R.window([0, 1, 3], 10, 4, 5, **kw) == ([8, 9, 10, 11, 13], 12)
    assert R.window([0, 2], 10, 4, 128, **kw) == (list(range(11)) + [12], 11)
    assert R.window([0, 1, 3], 10, 4, 2, **kw) == ([11, 13], 12)


def test_oracle_known_windows():
    _known_windows()
    assert R.window([], 10, 4, 3) == ([7, 8, 9], 9)
    assert R.window([0], 0, 4, 3) == ([0], 0)
    assert R.window([], 0, 4, 3) == ([], -1)
    assert R.window([0, 1, 2, 70], -2, 3, 8) == ([0], 0)     # nodes 0, 1 lie before position 0, 70 past the nodes


def test_oracle_planted_missing_self_fails():
    with pytest.raises(AssertionError):
        _known_windows(attend_self=False)


def test_mask_bits():
    m = R.mask_of([[[0, 63, 64, 130]]], 3)
    assert m.tolist() == [[(1 << 63) + 1 - (1 << 64), 1, 4]]


def test_oracle_chain_is_the_linear_operator():
    g = torch.Generator().manual_seed(1)
    ql, kl, D, H = [3, 1], [9, 20], 512, 16
    q = torch.randn(4, H, D, generator=g).to(torch.bfloat16)
    rows = torch.randn(64, D, generator=g).to(torch.bfloat16)
    cmp_rows = torch.randn(16, D, generator=g).to(torch.bfloat16)
    table, ctable = torch.tensor([[2, -1], [0, 3]]), torch.tensor([[1], [0]])
    idx = torch.randint(-1, 6, (4, 5), generator=g)
    sinks = torch.randn(H, generator=g)
    trees = [[list(range(i + 1)) for i in range(n)] for n in ql]
    out, lse, _ = R.attention(q, rows, cmp_rows, table, ctable, idx, trees, ql, kl, sinks, 0.04, 7, 16, 8, 4, 4)
    t = 0
    for b, (m, k) in enumerate(zip(ql, kl)):
        for s in range(m):
            sg = k - m + s
            win = [int(table[b, p // 16]) * 16 + p % 16 for p in range(max(0, sg - 6), sg + 1)]
            sel = [int(ctable[b, 0]) * 8 + int(i) for i in idx[t] if 0 <= i < (sg + 1) // 4]
            ref, ref_lse = O._attend(q[t].float(), [rows[win].float(), cmp_rows[sel].float()], sinks, 0.04,
                                     torch.bfloat16, 512, exact=True)
            assert torch.allclose(out[t], ref.double(), atol=1e-9) and torch.allclose(lse[t], ref_lse.double(), atol=1e-9)
            t += 1


# ---------------------------------------------------------------------------
# argument errors (no device)
# ---------------------------------------------------------------------------

def test_abi_refuses():
    L = _lib.lib()
    assert L.sas_fwd_tree_v1(None, None) == _lib.SAS_EINVAL
    a = _lib.SasFwdArgs(T=4, B=1, H=64, D=576, DV=512, ori_block_size=64, ori_bt_stride=8, ori_num_blocks=8,
                        scenario=_lib.SAS_SWA, cmp_ratio=4, win_left=127, softmax_scale=0.04)
    fake = 1 << 20
    for f in ("q", "ori_kv", "ori_block_table", "q_prefix", "act_kv", "sinks", "out", "lse"):
        setattr(a, f, fake)
    for mask, words, needle in ((None, 1, "tree_mask"), (fake + 4, 1, "tree_mask"), (fake, 0, "tree_words"),
                                (fake, 65, "tree_words"), (fake, -1, "tree_words")):
        t = _lib.SasFwdTreeArgs(fwd=a, tree_mask=mask, tree_words=words)
        assert L.sas_fwd_tree_v1(C.byref(t), None) == _lib.SAS_EINVAL
        assert needle in L.sas_last_error().decode()
    a.D = 100
    t = _lib.SasFwdTreeArgs(fwd=a, tree_mask=fake, tree_words=1)
    assert L.sas_fwd_tree_v1(C.byref(t), None) == _lib.SAS_EINVAL and "D must be" in L.sas_last_error().decode()
    a.D, a.num_splits = 576, 2
    t = _lib.SasFwdTreeArgs(fwd=a, tree_mask=fake, tree_words=1)
    assert L.sas_fwd_tree_v1(C.byref(t), None) == _lib.SAS_ENOWS
    a.T = 0
    t = _lib.SasFwdTreeArgs(fwd=a, tree_mask=None, tree_words=1)
    assert L.sas_fwd_tree_v1(C.byref(t), None) == _lib.SAS_OK


def test_python_refuses():
    from dsv4_amd.api import sparse_attn_sharedkv_tree
    q = torch.zeros(3, 16, 512, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    kw = dict(ori_kv=torch.zeros(1, 16, 1, 512, dtype=torch.bfloat16), ori_block_table=i[:1, None], cu_seqlens_q=i,
              seqused_kv=i[:1], sinks=torch.zeros(16), softmax_scale=1.0)
    for mask in (torch.zeros(3, 1, dtype=torch.int32), torch.zeros(2, 1, dtype=torch.int64), torch.zeros(3, dtype=torch.int64),
                 torch.zeros(3, 65, dtype=torch.int64), torch.zeros(3, 0, dtype=torch.int64)):
        with pytest.raises(ValueError, match="tree_mask must be int64"):
            sparse_attn_sharedkv_tree(q, tree_mask=mask, **kw)
    with pytest.raises(ValueError, match="GPU"):
        sparse_attn_sharedkv_tree(q, tree_mask=torch.zeros(3, 1, dtype=torch.int64), **kw)


def test_failed_call_of_a_kept_resolution_is_named(monkeypatch):
    from dsv4_amd import api
    r = api._Cached.__new__(api._Cached)
    r.out_shape, r.lse_shape, r.tail, r.ws_bytes, r.host_names = (1, 16, 512), (1, 16), b"", 0, []
    monkeypatch.setattr(api, "_tree_raw", lambda packed, stream: _lib.SAS_EINVAL)
    monkeypatch.setattr(api, "_fwd_raw", lambda packed, stream: _lib.SAS_EINVAL)
    t = torch.zeros(1, dtype=torch.int32)
    args = (r, None, t.device, t, t, None, None, t, None, t, t, torch.zeros(16), False)
    with pytest.raises(ValueError, match="^sparse_attn_sharedkv_tree"):
        api._run_cached(*args, torch.zeros(1, 1, dtype=torch.int64))
    with pytest.raises(ValueError, match="^sparse_attn_sharedkv[^_]"):
        api._run_cached(*args)


# ---------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------

class Case:
    """Inputs on the CPU, drawn from `seed`."""

    def __init__(self, kind, dt, H, D, ql, kl, K=0, ratio=4, win=128, bs=64, words=None, reach=9, holes=False, tail=0,
                 trees=None, seed=3):
        g = torch.Generator().manual_seed(seed)
        self.kind, self.ql, self.kl, self.ratio, self.win, self.bs, self.H, self.D = kind, ql, kl, ratio, win, bs, H, D
        self.fp8 = dt == "fp8"
        self.dt = torch.float16 if dt == "fp16" else torch.bfloat16
        self.scale = D ** -0.5
        n = sum(ql)
        self.T = n + tail
        self.trees = trees or [R.random_tree(m, g, reach) for m in ql]
        self.words = words or max(1, -(-max(ql) // 64))
        self.mask = torch.cat([R.mask_of(self.trees, self.words),
                               torch.randint(-2 ** 62, 2 ** 62, (tail, self.words), generator=g)])
        self.q = torch.randn(self.T, H, D, generator=g).to(self.dt)
        self.sinks = torch.randn(H, generator=g)
        self.rows, self.cache, self.table = self._cache(kl, bs, g)
        self.crows = self.ccache = self.ctable = self.idx = None
        if kind != "swa":
            self.crows, self.ccache, self.ctable = self._cache([k // ratio for k in kl], bs, g)
        if kind == "scfa":
            # a few beyond the threshold, -1 here and there
            top = max(1, max(kl) // ratio + 2)
            self.idx = torch.stack([torch.randperm(max(top, K), generator=g)[:K] for _ in range(self.T)])
            self.idx = torch.where(self.idx < top, self.idx, -1).to(torch.int32).view(self.T, 1, K)
        if holes:
            self.table[0, 0] = -1
        self.cu = torch.zeros(len(ql) + 1, dtype=torch.int32)
        self.cu[1:] = torch.tensor(ql).cumsum(0)
        self.used = torch.tensor(kl, dtype=torch.int32)

    def _cache(self, lens, bs, g):
        per = max(1, max(-(-max(x, 1) // bs) for x in lens))
        nb = per * len(lens) + 2
        table = torch.randperm(nb, generator=g)[:per * len(lens)].to(torch.int32).view(len(lens), per)
        rows = torch.randn(nb * bs, self.D, generator=g).to(self.dt)
        if self.fp8:
            cache = paged.quantize_kv_fp8(rows.view(nb, bs, 1, self.D))
            return paged.dequantize_kv_fp8(cache).view(nb * bs, self.D), cache, table
        return rows, rows.view(nb, bs, 1, self.D), table

    def kwargs(self, host_lens=False):
        mv = lambda t: None if t is None else t.cuda()  # noqa: E731
        lens = (lambda t: t) if host_lens else mv
        return dict(ori_kv=mv(self.cache), cmp_kv=mv(self.ccache), cmp_sparse_indices=mv(self.idx),
                    ori_block_table=mv(self.table), cmp_block_table=mv(self.ctable), cu_seqlens_q=lens(self.cu),
                    seqused_kv=lens(self.used), sinks=mv(self.sinks), softmax_scale=self.scale,
                    cmp_ratio=self.ratio if self.kind != "swa" else None, ori_win_left=self.win - 1)

    def ref(self):
        return R.attention(self.q, self.rows, self.crows, self.table, self.ctable,
                           None if self.idx is None else self.idx[:, 0], self.trees, self.ql, self.kl, self.sinks,
                           self.scale, self.win, self.bs, self.bs, self.ratio, self.T)

    def check(self, out, lse):
        ref, ref_lse, mag = self.ref()
        h = torch.finfo(self.dt).eps / 2
        bound = 1.5 * h * (mag + ref.abs()) + (2.0 ** -12 if self.dt is torch.float16 else 2.0 ** -16)
        err = (out.cpu().double() - ref).abs()
        assert bool((err <= bound).all()), f"worst {float((err / bound).max()):.3g} of the bound"
        assert float((lse.cpu().double() - ref_lse).abs().max()) <= 1e-3
        assert bool((out.cpu()[sum(self.ql):] == 0).all()) and bool((lse.cpu()[sum(self.ql):] == 0).all())


def _run(c, **kw):
    from dsv4_amd.api import sparse_attn_sharedkv_tree
    return sparse_attn_sharedkv_tree(c.q.cuda(), tree_mask=c.mask.cuda(), return_softmax_lse=True, **c.kwargs(**kw))


CASES = {
    "one": dict(kind="scfa", dt="bf16", H=16, D=576, ql=[1], kl=[200], K=64),
    "tree8_h16": dict(kind="scfa", dt="bf16", H=16, D=576, ql=[8], kl=[700], K=64),
    "batch_h64": dict(kind="scfa", dt="bf16", H=64, D=576, ql=[12, 0, 5, 30], kl=[400, 9, 5, 900], K=200),
    "fp16_512": dict(kind="scfa", dt="fp16", H=32, D=512, ql=[7, 20], kl=[300, 31], K=130, bs=16),
    "fp8": dict(kind="scfa", dt="fp8", H=32, D=576, ql=[16, 3], kl=[600, 70], K=256, ratio=8),
    "fp8_h16_swa": dict(kind="swa", dt="fp8", H=16, D=576, ql=[9], kl=[300]),
    "fp8_h128": dict(kind="scfa", dt="fp8", H=128, D=576, ql=[5], kl=[500], K=100),
    "swa": dict(kind="swa", dt="bf16", H=64, D=512, ql=[40, 3], kl=[300, 3]),
    "swa_many": dict(kind="swa", dt="bf16", H=64, D=512, ql=[17] * 20, kl=[30 + 20 * i for i in range(20)], bs=16),
    "swa_wide": dict(kind="swa", dt="fp16", H=16, D=576, ql=[10, 6], kl=[900, 100], win=600),
    "cfa": dict(kind="cfa", dt="bf16", H=64, D=576, ql=[9, 14], kl=[800, 90], ratio=8),
    "cfa_many": dict(kind="cfa", dt="fp16", H=64, D=512, ql=[64] * 17, kl=[300 + i for i in range(17)], ratio=16),
    "narrow": dict(kind="scfa", dt="bf16", H=64, D=576, ql=[30], kl=[90], K=70, win=3, reach=1),
    "window_of_one": dict(kind="swa", dt="bf16", H=16, D=512, ql=[6], kl=[40], win=1),
    "two_words": dict(kind="scfa", dt="bf16", H=64, D=576, ql=[100, 64, 65], kl=[300, 64, 400], K=90),
    "deep_chain": dict(kind="swa", dt="bf16", H=16, D=512, ql=[190], kl=[200], reach=1),
    "many_words": dict(kind="swa", dt="bf16", H=16, D=512, ql=[330], kl=[340], words=64, reach=300),
    "missing_rows": dict(kind="scfa", dt="bf16", H=64, D=576, ql=[12, 70], kl=[5, 30], K=70),
    "no_committed": dict(kind="scfa", dt="bf16", H=16, D=576, ql=[12], kl=[12], K=64, ratio=1),
    "hole": dict(kind="swa", dt="bf16", H=64, D=576, ql=[4, 4], kl=[70, 90], holes=True),
    "behind_the_last": dict(kind="scfa", dt="bf16", H=64, D=576, ql=[4, 5], kl=[70, 90], K=64, tail=6),
    # more (token, 64 heads) items than compute units: two workgroups a unit
    "pairs": dict(kind="scfa", dt="bf16", H=64, D=576, ql=[30, 0, 41] + [24] * 9, kl=[300, 9, 41] + [40 + 70 * i for i in range(9)],
                  K=150, tail=5, holes=True),
    "pairs_fp16": dict(kind="scfa", dt="fp16", H=128, D=512, ql=[70, 65], kl=[400, 65], K=90, bs=16),
    "pairs_narrow": dict(kind="swa", dt="bf16", H=64, D=576, ql=[60] * 5, kl=[60, 61, 70, 200, 500], win=1),
    "pairs_missing": dict(kind="scfa", dt="bf16", H=64, D=576, ql=[130, 140], kl=[5, 30], K=70, win=200),
    "pairs_fp8": dict(kind="scfa", dt="fp8", H=64, D=576, ql=[30, 0, 41] + [24] * 9, kl=[300, 9, 41] + [40 + 70 * i for i in range(9)],
                      K=150, ratio=8, tail=5, holes=True),
    "pairs_fp8_swa": dict(kind="swa", dt="fp8", H=128, D=576, ql=[60] * 3, kl=[60, 61, 500], win=3),
    "pairs_fp8_cfa": dict(kind="cfa", dt="fp8", H=128, D=576, ql=[66, 70], kl=[5, 800], ratio=4, win=200),
    "long_topk": dict(kind="scfa", dt="bf16", H=128, D=576, ql=[33], kl=[5000], K=1024),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(CASES))
def test_gpu_tree(name):
    c = Case(**CASES[name])
    out, lse = _run(c)
    c.check(out, lse)
    again, lse2 = _run(c)                       # the kept resolution
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "fp8"])
def test_gpu_rows_without_bits(dt):
    """Masks that leave the drafts out, a tree whose nodes leave themselves out,
    a sequence without committed rows whose token attends nothing: the sink alone."""
    trees = [[[], [0], [0, 2], []], [[], [0, 1]]]
    c = Case(kind="scfa", dt=dt, H=32, D=576, ql=[4, 2], kl=[60, 2], K=64, trees=trees)
    out, lse = _run(c)
    c.check(out, lse)
    assert bool((out[4] == 0).all()) and torch.allclose(lse[4].cpu(), c.sinks, atol=1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "fp8"])
def test_gpu_pairs_rows_without_bits(dt):
    """As above, with more items than compute units: half the trees attend
    nothing, some of them without committed rows; a sink of -inf beside them."""
    trees = [[[]] * 20 if b % 2 else [list(range(i + 1)) for i in range(20)] for b in range(14)]
    c = Case(kind="scfa", dt=dt, H=64, D=576, ql=[20] * 14, kl=[20 + 9 * (b // 2) for b in range(14)], K=64, trees=trees)
    out, lse = _run(c)
    c.check(out, lse)
    assert bool((out[20:40] == 0).all()) and torch.allclose(lse[20].cpu(), c.sinks, atol=1e-6)
    c.sinks[3] = -float("inf")
    out, lse = _run(c)
    assert bool(torch.isfinite(out).all()) and bool((lse[20:40, 3] == -float("inf")).all())


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dt,H,D", [("scfa", "bf16", 64, 576), ("swa", "fp16", 16, 512), ("cfa", "bf16", 32, 512),
                                         ("scfa", "fp8", 64, 576)])
def test_gpu_chain_is_the_linear_operator(kind, dt, H, D):
    """Chains: the same rows in the same order, so the same bits; bits past the
    nodes change nothing."""
    from dsv4_amd.api import sparse_attn_sharedkv
    ql, kl = [1, 3, 6], [400, 80, 4]
    c = Case(kind=kind, dt=dt, H=H, D=D, ql=ql, kl=kl, K=64 if kind == "scfa" else 0,
             trees=[[list(range(i + 1)) for i in range(n)] for n in ql])
    want, want_lse = sparse_attn_sharedkv(c.q.cuda(), return_softmax_lse=True, **c.kwargs())
    out, lse = _run(c)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    c.mask[:, 0] |= 3 << 20
    out, lse = _run(c, host_lens=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.gpu
def test_gpu_layout_bsnd_strided_mask_and_streams():
    from dsv4_amd.api import sparse_attn_sharedkv_tree
    c = Case(kind="scfa", dt="bf16", H=64, D=576, ql=[6, 6, 6], kl=[100, 50, 300], K=64)
    want, want_lse = _run(c)
    kw = c.kwargs()
    kw.pop("cu_seqlens_q")
    idx = kw.pop("cmp_sparse_indices")
    out, lse = sparse_attn_sharedkv_tree(
        c.q.view(3, 6, 64, 576).cuda(), tree_mask=c.mask.view(3, 6, 1).cuda(), layout_q="BSND", return_softmax_lse=True,
        cmp_sparse_indices=idx.view(3, 6, 1, 64), **kw)
    assert torch.equal(out.view_as(want), want) and torch.equal(lse.view_as(want_lse), want_lse)
    wide = torch.full((18, 5), -1, dtype=torch.int64, device="cuda")
    wide[:, 2] = c.mask[:, 0].cuda()
    kw = c.kwargs()
    out = sparse_attn_sharedkv_tree(c.q.cuda(), tree_mask=wide[:, 2:3], **kw)
    assert torch.equal(out, want)
    q, m = c.q.cuda(), c.mask.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = sparse_attn_sharedkv_tree(q, tree_mask=m, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)
    out = sparse_attn_sharedkv_tree(q[:0], tree_mask=m[:0], **{**kw, "cmp_sparse_indices": kw["cmp_sparse_indices"][:0]})
    assert out.shape == (0, 64, 512)
    with pytest.raises(ValueError, match="q's device"):
        sparse_attn_sharedkv_tree(q, tree_mask=c.mask, **kw)


@pytest.mark.gpu
def test_gpu_non_finite_rows_that_are_masked():
    """Rows no token attends may hold anything: other branches' nodes, rows
    before the window, unused blocks, compressed rows past the threshold."""
    c = Case(kind="scfa", dt="bf16", H=64, D=576, ql=[12], kl=[300], K=64, win=16)
    used = set()
    for nodes in c.trees[0][:6]:
        at, pos = R.window(nodes, 288, 12, 16)
        used |= {int(c.table[0, a // 64]) * 64 + a % 64 for a in at}
    keep = 6
    c.ql, c.T = [keep], keep
    # nodes 6 .. 11 stay in the cache as rows past this call's tokens: queries 0 .. 5 of 12 nodes
    c.q, c.mask, c.idx = c.q[:12], c.mask[:12], c.idx[:12]
    bad = torch.ones(c.rows.shape[0], dtype=torch.bool)
    bad[list(used)] = False
    from dsv4_amd.api import sparse_attn_sharedkv_tree
    kw = c.kwargs()
    clean = sparse_attn_sharedkv_tree(c.q.cuda(), tree_mask=c.mask.cuda(), **kw)
    rows = c.rows.clone()
    rows[bad] = float("nan")
    kw["ori_kv"] = rows.view_as(c.cache).cuda()
    cr = c.crows.clone()
    past = [int(c.ctable[0, a // 64]) * 64 + a % 64 for a in range(300 // 4, c.ctable.shape[1] * 64)]
    cr[past] = float("inf")
    kw["cmp_kv"] = cr.view_as(c.ccache).cuda()
    out = sparse_attn_sharedkv_tree(c.q.cuda(), tree_mask=c.mask.cuda(), **kw)
    assert torch.equal(out[:keep], clean[:keep])


@pytest.mark.gpu
def test_gpu_draft_step_append_and_tree_captured():
    """A verification step: the drafts' rows appended at their slots, rotated by
    their depths, and attended as a tree; captured once, replayed on new
    drafts, trees and caches in the same buffers."""
    from dsv4_amd.api import sparse_attn_sharedkv_tree
    from dsv4_amd.cache import append_kv_cache
    from dsv4_amd.rope import rope_table
    c = Case(kind="scfa", dt="bf16", H=64, D=576, ql=[9, 4, 20], kl=[100, 50, 300], K=64)
    g = torch.Generator().manual_seed(8)
    kw = c.kwargs()
    raw_q, raw_kv = torch.randn(33, 64, 576).to(torch.bfloat16).cuda(), torch.randn(33, 576).to(torch.bfloat16).cuda()
    mask, rope = c.mask.cuda(), rope_table(400)

    def depths(trees):
        return torch.tensor([k - m + len(nodes) - 1 for m, k, t in zip(c.ql, c.kl, trees) for nodes in t], dtype=torch.int32)

    pos = depths(c.trees).cuda()

    def step():
        q = append_kv_cache(raw_kv, kw["ori_kv"], kw["ori_block_table"], kw["cu_seqlens_q"], kw["seqused_kv"], table=rope,
                            positions=pos, norm_dim=512, q=raw_q, q_norm_dim=512)
        return q, sparse_attn_sharedkv_tree(q, tree_mask=mask, return_softmax_lse=True, **kw)

    q, (out, lse) = step()
    torch.cuda.synchronize()
    c.q, c.rows = q.cpu(), kw["ori_kv"].cpu().view(-1, 576)
    c.check(out, lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cq, (cout, clse) = step()
    for _ in range(3):
        c.trees = [R.random_tree(m, g) for m in c.ql]
        mask.copy_(R.mask_of(c.trees, 1))
        pos.copy_(depths(c.trees))
        raw_q.copy_(torch.randn(33, 64, 576, generator=g))
        raw_kv.copy_(torch.randn(33, 576, generator=g))
        graph.replay()
        got = cout.clone(), clse.clone()
        torch.cuda.synchronize()
        _, (out, lse) = step()
        assert torch.equal(out, got[0]) and torch.equal(lse, got[1])
        c.q, c.rows = cq.cpu(), kw["ori_kv"].cpu().view(-1, 576)
        c.check(*got)


# windows on either side of 32 (token, 64 heads) items, fp8 rows from half as many items
# as compute units
MORE = {
    "window_31": dict(kind="swa", dt="bf16", H=64, D=576, ql=[31], kl=[500]),
    "window_32": dict(kind="swa", dt="fp16", H=64, D=512, ql=[20, 12], kl=[25, 700], bs=16),
    "window_32_h128": dict(kind="swa", dt="bf16", H=128, D=576, ql=[1] * 16, kl=[1, 2, 31, 32, 33, 64, 127, 128] * 2, tail=3),
    "window_32_fp8": dict(kind="swa", dt="fp8", H=64, D=576, ql=[33], kl=[90], win=64, holes=True),
    "half_fp8": dict(kind="scfa", dt="fp8", H=64, D=576, ql=[64, 66], kl=[300, 5000], K=512),
    "half_fp8_h128": dict(kind="cfa", dt="fp8", H=128, D=576, ql=[33, 34], kl=[2000, 40], ratio=8, win=100),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(MORE))
def test_gpu_tree_around_the_rules(name):
    c = Case(**MORE[name])
    out, lse = _run(c)
    c.check(out, lse)


@pytest.mark.gpu
def test_gpu_pairs_fp8_rows_of_far_apart_scales():
    """A row's groups of 128 channels and the rows among themselves lie up to 2^16
    apart; rows of zeros between them."""
    c = Case(kind="scfa", dt="fp8", H=64, D=576, ql=[40] * 7, kl=[200 + 30 * i for i in range(7)], K=96)
    g = torch.Generator().manual_seed(8)
    for name in ("cache", "ccache"):
        rows = torch.randn(*getattr(c, name).shape[:2], 1, 576, generator=g)
        e = torch.randint(-16, 1, (*rows.shape[:3], 5), generator=g).repeat_interleave(128, -1)[..., :576]
        rows = torch.where(torch.rand(rows.shape[:3] + (1,), generator=g) < 0.1, 0.0, rows * torch.exp2(e.float()))
        cache = paged.quantize_kv_fp8(rows.to(torch.bfloat16))
        setattr(c, name, cache)
        setattr(c, {"cache": "rows", "ccache": "crows"}[name], paged.dequantize_kv_fp8(cache).view(-1, 576))
    out, lse = _run(c)
    c.check(out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["swa", "scfa"])
def test_gpu_empty_call_and_nodes_past_the_words(kind):
    from dsv4_amd.api import sparse_attn_sharedkv_tree
    c = Case(kind=kind, dt="bf16", H=64, D=512, ql=[80], kl=[200], K=64, reach=1)
    kw = c.kwargs()
    none = dict(kw, cu_seqlens_q=torch.zeros_like(kw["cu_seqlens_q"]))
    if kind == "scfa":
        none["cmp_sparse_indices"] = kw["cmp_sparse_indices"][:0]
    out, lse = sparse_attn_sharedkv_tree(c.q.cuda()[:0], tree_mask=c.mask.cuda()[:0], return_softmax_lse=True, **none)
    assert out.shape == (0, 64, 512) and lse.shape == (0, 64)
    # one word: what the first 64 nodes of the chain are for the others
    c.trees = [[[j for j in t if j < 64] for t in c.trees[0]]]
    c.mask = c.mask[:, :1].contiguous()
    c.check(*_run(c))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "fp8"])
@pytest.mark.parametrize("ql", [[3, 2], [140, 135]], ids=["few", "pairs"])
def test_gpu_cache_past_32_bits(dt, ql):
    """The rows of a small cache behind 4 GiB of others give the same bits."""
    from dsv4_amd.api import sparse_attn_sharedkv_tree
    c = Case(kind="scfa", dt=dt, H=64, D=576, ql=ql, kl=[q + 100 for q in ql], K=64)
    want = _run(c)
    kw = c.kwargs()
    for name, table in (("ori_kv", "ori_block_table"), ("cmp_kv", "cmp_block_table")):
        x = kw[name]
        ahead = (1 << 32) // (x[0].numel() * x.element_size()) + 1
        far = torch.zeros(ahead + x.shape[0], *x.shape[1:], dtype=x.dtype, device="cuda")
        far[ahead:] = x
        kw[name], kw[table] = far, torch.where(kw[table] >= 0, kw[table] + ahead, kw[table])
    got = sparse_attn_sharedkv_tree(c.q.cuda(), tree_mask=c.mask.cuda(), return_softmax_lse=True, **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    c.check(*got)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp8"])
@pytest.mark.parametrize("scale", [-0.06, 0.0])
def test_gpu_pairs_scales_of_other_signs(dt, scale):
    c = Case(kind="scfa", dt=dt, H=64, D=576, ql=[45] * 6, kl=[45 + 60 * i for i in range(6)], K=64)
    c.scale = scale
    c.check(*_run(c))


@pytest.mark.gpu
def test_gpu_pairs_on_another_stream_captured():
    """Replays on new inputs give what the eager call gives."""
    from dsv4_amd.api import sparse_attn_sharedkv_tree
    for dt in ("bf16", "fp8"):
        c = Case(kind="scfa", dt=dt, H=64, D=576, ql=[45] * 6, kl=[45 + 60 * i for i in range(6)], K=64)
        q, mask, kw = c.q.cuda(), c.mask.cuda(), c.kwargs()
        eager = sparse_attn_sharedkv_tree(q, tree_mask=mask, **kw)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            assert torch.equal(sparse_attn_sharedkv_tree(q, tree_mask=mask, **kw), eager)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = sparse_attn_sharedkv_tree(q, tree_mask=mask, **kw)
        for _ in range(3):
            q.copy_(torch.randn(q.shape, device="cuda"))
            graph.replay()
            got = captured.clone()
            torch.cuda.synchronize()
            assert torch.equal(got, sparse_attn_sharedkv_tree(q, tree_mask=mask, **kw))


# heads that do not fill a workgroup's four waves of sixteen
PARTS = {
    "h16": dict(kind="scfa", dt="bf16", H=16, D=576, ql=[90, 0, 100, 77], kl=[300, 9, 100, 700], K=100, tail=4, holes=True),
    "h48_fp16": dict(kind="scfa", dt="fp16", H=48, D=512, ql=[150, 130], kl=[400, 131], K=90, bs=16),
    "h96": dict(kind="cfa", dt="bf16", H=96, D=576, ql=[70, 65], kl=[400, 65], ratio=4, win=200),
    "h80_window": dict(kind="swa", dt="bf16", H=80, D=512, ql=[20, 3], kl=[300, 3]),
    "h16_window": dict(kind="swa", dt="fp16", H=16, D=576, ql=[33], kl=[90], win=100),
    "h16_fp8": dict(kind="scfa", dt="fp8", H=16, D=576, ql=[140, 130], kl=[300, 131], K=100, tail=2, holes=True),
    "h48_fp8": dict(kind="cfa", dt="fp8", H=48, D=576, ql=[140, 130], kl=[5, 700], ratio=8, win=60),
    "h112_fp8_window": dict(kind="swa", dt="fp8", H=112, D=576, ql=[60, 5], kl=[60, 300], win=64),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(PARTS))
def test_gpu_tree_heads_short_of_a_workgroup(name):
    c = Case(**PARTS[name])
    guard = _run(c)
    c.check(*guard)
    assert all(torch.equal(a, b) for a, b in zip(guard, _run(c)))


@pytest.mark.gpu
@pytest.mark.parametrize("dt,H", [("bf16", 64), ("fp8", 32)])
def test_gpu_branches_across_a_compression_boundary(dt, H):
    """Nodes on both sides of a multiple of the ratio, two branches: rows listed as
    indices keep each node to the committed compressed rows and those of its own
    branch; the dense form attends the shared row beyond the boundary too, as
    documented."""
    ratio, ql, kl = 8, [14, 9], [59 + 14, 121 + 9]
    trees = []
    for m in ql:   # node 0, then branches of odd and even nodes
        t = [[0]]
        for i in range(1, m):
            t.append(t[max(0, i - 2)] + [i] if i > 2 else [0, i])
        trees.append(t)
    c = Case(kind="cfa", dt=dt, H=H, D=576, ql=ql, kl=kl, ratio=ratio, trees=trees)
    deep = [(k - m + len(t)) // ratio > (k - m) // ratio for m, k, ts in zip(ql, kl, trees) for t in ts]
    assert any(deep) and not all(deep)
    out, lse = _run(c)
    c.check(out, lse)
    # the first branch's nodes alone have rows past the boundary
    top = max(kl) // ratio
    rows = []
    for m, k, ts in zip(ql, kl, trees):
        for t in ts:
            limit = (k - m + len(t)) // ratio if 1 in t else (k - m) // ratio
            rows.append([j if j < limit else -1 for j in range(top)])
    c.kind, c.idx = "scfa", torch.tensor(rows, dtype=torch.int32)[:, None]
    out2, lse2 = _run(c)
    c.check(out2, lse2)
    other = torch.tensor([d and 1 not in t for d, t in zip(deep, [t for ts in trees for t in ts])])
    assert bool(other.any()) and bool((lse2[other] < lse[other]).all())

"""Norms and rotation of queries and KV rows (norm_rope, its backward and
autograd binding) and the cache append: the 64-bit CPU oracle pinned by known
rotations and central differences, argument errors without a device, and the
kernels against the oracle.

Tolerances, with h = finfo(dtype).eps / 2 (half a step) and e = 2^-24 the fp32
half step. A normed channel x r w: the sum of n <= 1024 squares is off by at most
(n / 8 + 3) e relative (a lane's chain, then three adds), halved by the root;
rsqrt, the mean and the three products add 5 e: below 72 e < 2^-17. A rotation adds
3 e of |a| + |b|. So an output is within h |y| + 2^-17 (|a| + |b|) of y, and |a| + |b| <=
2 max|y| over the row. A row's gradient has r g, within 2^-17 r |g|, and r x^ m^ (x^ =
x r, m^ the mean of g x^), whose two sums put it within 2^-16 |x^| r max|g|, |x^| below 6
here: h |dx| + 2^-15 max(|dx|, 2 r max|dy| max|w|) of the row (|u| <= sqrt(2) max|dy|).
A weight's gradient sums N terms in
chains of at most 64 and a tree: 2^-17 (terms) + (64 + 16) e < 2^-16 of the sum of
their absolute values. fp16 results below 2^-14 round by 2^-25 absolutely."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from dsv4_amd import _lib, paged
from oracle import rope_ref as R

NAN = float("nan")


def _half_step(dt):
    return torch.finfo(dt).eps / 2


def _close(got, ref, dt, slack):
    """got within half a step of ref, plus `slack` (a tensor) of fp32 error."""
    ref = ref.double()
    bound = _half_step(dt) * ref.abs() * (1 + 2.0 ** -8) + slack + (2.0 ** -25 if dt is torch.float16 else 1e-38)
    bad = (got.double() - ref).abs() > bound
    assert not bool(bad.any()), (f"{int(bad.sum())} of {bad.numel()} outside, worst "
                                 f"{float(((got.double() - ref).abs() / bound).max()):.3g} of the bound")


def _table(rows, rope_dim, seed=5):
    """Angles of random positions (exactly representable pairs are not needed)."""
    from dsv4_amd.rope import rope_table
    return rope_table(rows, rope_dim, device="cpu") if rope_dim else None


# ---------------------------------------------------------------------------
# oracle
# ---------------------------------------------------------------------------

def test_oracle_known_rotations():
    y = torch.tensor([9.0, 1.0, 2.0, 3.0, 4.0], dtype=torch.float64)
    quarter = torch.tensor([[0.0, 1.0], [-1.0, 0.0]], dtype=torch.float64)   # 90, 180 degrees
    assert R.rotate(y, quarter, False, False).tolist() == [9.0, -2.0, 1.0, -3.0, -4.0]
    assert R.rotate(y, quarter, True, False).tolist() == [9.0, -3.0, -2.0, 1.0, -4.0]
    assert R.rotate(y, quarter, False, True).tolist() == [9.0, 2.0, -1.0, -3.0, -4.0]
    t = _table(50, 8).double()
    x = torch.randn(50, 12, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    for half in (False, True):
        back = R.rotate(R.rotate(x, t, half, False), t, half, True)
        assert torch.allclose(back, x, atol=1e-6)   # the table is fp32: c^2 + s^2 = 1 within 2^-23


def _unit_mean_square(mean_over=None):
    x = torch.randn(7, 24, dtype=torch.float64, generator=torch.Generator().manual_seed(2))
    y = R.norm(x, 16, None, 0.0, mean_over)
    assert torch.allclose((y[:, :16] ** 2).mean(-1), torch.ones(7, dtype=torch.float64), atol=1e-12)
    assert torch.equal(y[:, 16:], x[:, 16:])


def test_oracle_norm_gives_unit_mean_square():
    _unit_mean_square()


def test_oracle_planted_wrong_mean_fails():
    with pytest.raises(AssertionError):
        _unit_mean_square(mean_over=17)


@pytest.mark.parametrize("half,inverse,n", [(False, False, 24), (True, False, 16), (True, True, 8), (False, True, 0)])
def test_oracle_gradients_against_differences(half, inverse, n):
    """Central differences of the forward in 64 bits, step 1e-5: truncation and
    cancellation stay below 1e-8 for values of order one."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3, 24, dtype=torch.float64, generator=g)
    w = 1 + 0.3 * torch.randn(n, dtype=torch.float64, generator=g) if n else None
    dy = torch.randn(3, 24, dtype=torch.float64, generator=g)
    cs = _table(20, 16)[[3, 7, 19]]
    dx, dw, _ = R.norm_rope_grad(dy, x, n, w, cs, half, inverse)

    def loss(x_, w_):
        return float((R.norm_rope(x_, n, w_, cs, half, inverse) * dy).sum())

    for i in range(3):
        for j in range(24):
            d = torch.zeros_like(x)
            d[i, j] = 1e-5
            assert abs((loss(x + d, w) - loss(x - d, w)) / 2e-5 - float(dx[i, j])) < 1e-8
    for j in range(n):
        d = torch.zeros_like(w)
        d[j] = 1e-5
        assert abs((loss(x, w + d) - loss(x, w - d)) / 2e-5 - float(dw[j])) < 1e-8


def test_rope_table_values():
    from dsv4_amd.rope import rope_table
    t = rope_table(70000, 64, device="cpu")
    assert t.shape == (70000, 32, 2) and t.dtype is torch.float32
    a = 69999 / 10000.0 ** (2 * 3 / 64)
    want = torch.tensor([a], dtype=torch.float64)
    assert abs(float(t[69999, 3, 0]) - float(want.cos())) < 1e-7 and abs(float(t[69999, 3, 1]) - float(want.sin())) < 1e-7
    for bad in ((0, 64), (4, 7), (4, 0)):
        with pytest.raises(ValueError, match="rope_table"):
            rope_table(*bad, device="cpu")


# ---------------------------------------------------------------------------
# argument errors (no device)
# ---------------------------------------------------------------------------

FAKE = 1 << 20


def _args(**over):
    a = _lib.SasNormRopeArgs(T=4, H=16, D=512, q_stride_t=8192, q_stride_h=512, kv_stride_t=512, table_rows=100,
                             rope_dim=64, q_norm_dim=512, kv_norm_dim=512, dtype=_lib.SAS_DT_BF16,
                             weight_dtype=_lib.SAS_DT_FP32, eps=1e-6)
    for f in ("q", "kv", "q_weight", "kv_weight", "positions", "table", "q_out", "kv_out"):
        setattr(a, f, FAKE)
    for k, v in over.items():
        setattr(a, k, v)
    return a


BAD = [
    ({"D": 4}, "multiple of 8"), ({"D": 1032}, "multiple of 8"), ({"T": -1}, "negative"), ({"dtype": 2}, "bf16 or fp16"),
    ({"weight_dtype": 1}, "weights"), ({"flags": 8}, "flags"), ({"rope_dim": 4}, "rope_dim"), ({"rope_dim": 520}, "rope_dim"),
    ({"rope_dim": 24, "flags": 1}, "rope_dim"), ({"q_norm_dim": 12}, "norm dims"), ({"kv_norm_dim": 520}, "norm dims"),
    ({"eps": -1.0}, "eps"), ({"eps": NAN}, "eps"), ({"T": 1 << 30}, "2^31"), ({"H": 0}, "go together"),
    ({"q": None}, "go together"), ({"table": None}, "table"), ({"table_rows": 0}, "table"), ({"q_stride_h": 500}, "strides"),
    ({"kv_stride_t": 4}, "strides"), ({"q": FAKE + 2}, "aligned"), ({"kv_out": FAKE + 8}, "aligned"),
    ({"q_weight": FAKE + 4}, "aligned"), ({"q": None, "H": 0, "kv": None}, "null"),
]


@pytest.mark.parametrize("over,needle", BAD, ids=[str(i) for i in range(len(BAD))])
def test_abi_refuses(over, needle):
    L = _lib.lib()
    assert L.sas_norm_rope_v1(C.byref(_args(**over)), None) == _lib.SAS_EINVAL
    assert needle in L.sas_last_error().decode(), L.sas_last_error().decode()
    ba = _lib.SasNormRopeBwdArgs(fwd=_args(**over))
    assert L.sas_norm_rope_bwd_v1(C.byref(ba), None) == _lib.SAS_EINVAL
    assert needle in L.sas_last_error().decode()
    ca = _lib.SasCacheAppendArgs(rope=_args(**over), cu_seqlens_q=FAKE, act_kv=FAKE, block_table=FAKE, cache=FAKE, B=1,
                                 bt_stride=1, block_size=64, num_blocks=1)
    assert L.sas_cache_append_v1(C.byref(ca), None) == _lib.SAS_EINVAL
    assert needle in L.sas_last_error().decode()


def test_abi_refuses_outputs_workspaces_and_caches():
    L = _lib.lib()
    assert L.sas_norm_rope_v1(None, None) == _lib.SAS_EINVAL
    assert L.sas_norm_rope_bwd_v1(None, None) == _lib.SAS_EINVAL
    assert L.sas_cache_append_v1(None, None) == _lib.SAS_EINVAL
    for f in ("q_out", "kv_out", "positions"):
        assert L.sas_norm_rope_v1(C.byref(_args(**{f: None})), None) == _lib.SAS_EINVAL
        assert "null" in L.sas_last_error().decode()
    assert L.sas_norm_rope_v1(C.byref(_args(T=0, q=None, kv=None)), None) == _lib.SAS_OK

    def grad(**over):
        b = _lib.SasNormRopeBwdArgs(fwd=_args(), dq_out=FAKE, dkv_out=FAKE, dq=FAKE, dkv=FAKE, dq_weight=FAKE,
                                    dkv_weight=FAKE, dq_out_stride_t=8192, dq_out_stride_h=512, dkv_out_stride_t=512)
        for k, v in over.items():
            setattr(b, k, v)
        return b

    n = C.c_size_t(0)
    assert L.sas_norm_rope_bwd_plan(C.byref(grad()), C.byref(n)) == _lib.SAS_OK and n.value > 0
    assert L.sas_norm_rope_bwd_v1(C.byref(grad()), None) == _lib.SAS_ENOWS
    assert L.sas_norm_rope_bwd_v1(C.byref(grad(workspace=FAKE, workspace_bytes=n.value - 1)), None) == _lib.SAS_ENOWS
    for f, v, needle in (("dq_out", None, "null"), ("dkv", None, "null"), ("dq_out_stride_h", 4, "strides"),
                         ("dkv_out", FAKE + 2, "aligned")):
        assert L.sas_norm_rope_bwd_v1(C.byref(grad(**{f: v})), None) == _lib.SAS_EINVAL
        assert needle in L.sas_last_error().decode()
    b = grad(fwd=_args(q_weight=None))
    assert L.sas_norm_rope_bwd_plan(C.byref(b), C.byref(n)) == _lib.SAS_EINVAL
    assert "weight" in L.sas_last_error().decode()
    assert L.sas_norm_rope_bwd_plan(C.byref(grad(dq_weight=None, dkv_weight=None)), C.byref(n)) == _lib.SAS_OK
    assert n.value == 0

    def append(**over):
        a = _lib.SasCacheAppendArgs(rope=_args(), cu_seqlens_q=FAKE, act_kv=FAKE, block_table=FAKE, cache=FAKE, B=1,
                                    bt_stride=1, block_size=64, num_blocks=1, cache_dtype=_lib.SAS_DT_BF16)
        for k, v in over.items():
            setattr(a, k, v)
        return a

    for over, needle in (({"B": 0}, "bad sizes"), ({"block_size": 0}, "bad sizes"), ({"cache_dtype": 1}, "cache dtype"),
                         ({"cache_dtype": 2}, "D = 576"), ({"num_blocks": 1 << 31}, "32-bit"), ({"cache": None}, "null"),
                         ({"act_kv": None}, "null"), ({"cache": FAKE + 8}, "aligned"), ({"rope": _args(kv=None)}, "null")):
        assert L.sas_cache_append_v1(C.byref(append(**over)), None) == _lib.SAS_EINVAL, over
        assert needle in L.sas_last_error().decode(), (over, L.sas_last_error().decode())


def test_python_refuses_host_tensors():
    from dsv4_amd.cache import append_kv_cache
    from dsv4_amd.rope import norm_rope, norm_rope_backward
    q = torch.zeros(2, 16, 512, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        norm_rope(q)
    with pytest.raises(ValueError, match="needed"):
        norm_rope(None)
    with pytest.raises(ValueError, match="bf16 or fp16"):
        norm_rope(q.float())
    with pytest.raises(ValueError, match="GPU"):
        norm_rope_backward(q, q)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="kv must be"):
        append_kv_cache(q, q, i, i, i)
    with pytest.raises(ValueError, match="GPU"):
        append_kv_cache(q[:, 0], q, i, i, i)


# ---------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------

# dtype, T, H, D, R, qn, kn, half, inverse, weights, wide
CASES = [
    ("bf16", 1, 16, 512, 64, 512, 512, False, False, "f32", False),
    ("bf16", 33, 64, 512, 64, 512, 512, False, False, None, False),
    ("fp16", 19, 16, 576, 64, 576, 512, True, False, "f32", True),
    ("bf16", 130, 7, 576, 64, 512, 0, False, True, "x", False),
    ("bf16", 257, 3, 128, 64, 128, 64, True, True, "x", True),
    ("fp16", 65, 1, 512, 64, 0, 512, False, False, "f32", True),
    ("fp16", 40, 5, 1024, 128, 1024, 8, True, False, "x", False),
    ("bf16", 40, 9, 640, 32, 600, 640, False, False, "f32", False),
    ("fp16", 9, 2, 24, 16, 16, 24, True, False, "f32", False),
    ("bf16", 12, 4, 8, 8, 8, 0, False, False, "x", False),
    ("bf16", 30, 8, 512, 0, 512, 512, False, False, "f32", False),
    ("fp16", 30, 11, 512, 512, 256, 512, True, True, None, False),
    ("bf16", 21, 16, 576, 96, 576, 512, True, False, "f32", True),
    ("bf16", 700, 16, 512, 64, 512, 512, False, False, "f32", False),
]
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _make(case, seed=11):
    dt, T, H, D, Rd, qn, kn, half, inverse, wt, wide = case
    dt = DT[dt]
    g = torch.Generator().manual_seed(seed)
    rows = 400
    both = torch.randn(T, (H + 1) * D + 16, generator=g).to(dt)
    q, kv = both[:, :H * D].view(T, H, D), both[:, H * D:(H + 1) * D]
    if not wide:
        q, kv = q.clone().contiguous(), kv.contiguous()
    pos = torch.randint(0, rows, (T,), generator=g, dtype=torch.int32)
    if T > 4:
        pos[1], pos[T - 2] = -1, rows      # padding
    table = _table(rows, Rd)
    wdt = {"f32": torch.float32, "x": dt, None: None}[wt]

    def w(n):
        return (1 + 0.2 * torch.randn(n, generator=g)).to(wdt) if wdt is not None and n else None

    return q, kv, pos if Rd else None, table, w(qn), w(kn)


def _refs(case, made):
    dt, T, H, D, Rd, qn, kn, half, inverse, wt, wide = case
    q, kv, pos, table, qw, kw = made
    ok = torch.ones(T, dtype=torch.bool) if pos is None else (pos >= 0) & (pos < table.shape[0])
    cs = None if pos is None else table[pos.long().clamp(0, table.shape[0] - 1)]
    return ok, cs, (None if cs is None else cs[:, None])


def _kw(case, made, dev="cuda"):
    _, _, _, _, _, qn, kn, half, inverse, _, _ = case
    mv = lambda t: None if t is None else t.to(dev)  # noqa: E731
    _, _, pos, table, qw, kw = made
    return dict(positions=mv(pos), table=mv(table), q_norm_dim=qn, kv_norm_dim=kn, q_weight=mv(qw), kv_weight=mv(kw),
                interleaved=not half, inverse=inverse)


def _dev(made, wide):
    """q and kv on the GPU, still slices of one tensor where they were."""
    q, kv = made[0], made[1]
    if not wide:
        return q.cuda(), kv.cuda()
    T, H, D = q.shape
    both = torch.empty(T, (H + 1) * D + 16, dtype=q.dtype, device="cuda")
    dq, dkv = both[:, :H * D].view(T, H, D), both[:, H * D:(H + 1) * D]
    dq.copy_(q)
    dkv.copy_(kv)
    return dq, dkv


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=["-".join(map(str, c)) for c in CASES])
def test_gpu_forward(case):
    from dsv4_amd.rope import norm_rope
    dt, half, inverse = DT[case[0]], case[7], case[8]
    made = _make(case)
    ok, cs, csq = _refs(case, made)
    qo, ko = norm_rope(*_dev(made, case[10]), **_kw(case, made))
    assert qo.is_contiguous() and ko.is_contiguous() and qo.dtype is dt
    for got, x, n, w, c in ((qo, made[0], case[5], made[4], csq), (ko, made[1], case[6], made[5], cs)):
        ref = R.norm_rope(x, n, w, c, half, inverse)
        ref = torch.where(ok.view(-1, *[1] * (ref.dim() - 1)), ref, 0.0)
        _close(got.cpu(), ref, dt, 2.0 ** -16 * ref.abs().amax(-1, keepdim=True))
        assert bool((got.cpu()[~ok] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=["-".join(map(str, c)) for c in CASES])
def test_gpu_backward(case):
    from dsv4_amd.rope import norm_rope_backward
    dt, half, inverse = DT[case[0]], case[7], case[8]
    made = _make(case)
    g = torch.Generator().manual_seed(17)
    q, kv = made[0], made[1]
    dqo, dko = torch.randn(q.shape, generator=g).to(dt), torch.randn(kv.shape, generator=g).to(dt)
    ok, cs, csq = _refs(case, made)
    dq_, dkv_ = _dev(made, case[10])
    got = norm_rope_backward(dqo.cuda(), dq_, dko.cuda(), dkv_, **_kw(case, made))
    again = norm_rope_backward(dqo.cuda(), dq_, dko.cuda(), dkv_, **_kw(case, made))
    for a, b in zip(got, again):
        assert a is b is None or torch.equal(a, b)      # no order that varies
    for dx, dw, x, dy, n, w, c in ((got[0], got[2], q, dqo, case[5], made[4], csq), (got[1], got[3], kv, dko, case[6], made[5], cs)):
        dy = torch.where(ok.view(-1, *[1] * (dy.dim() - 1)), dy.double(), 0.0)
        ref, rw, total = R.norm_rope_grad(dy, x, n, w, c, half, inverse)
        r = 1.0 / torch.sqrt((x[..., :n].double() ** 2).mean(-1, keepdim=True) + 1e-6) if n else 1.0
        big = torch.maximum(ref.abs().amax(-1, keepdim=True),
                            r * dy.abs().amax(-1, keepdim=True) * 2 * (1.0 if w is None else float(w.abs().max())))
        _close(dx.cpu(), ref, dt, 2.0 ** -15 * big)
        assert bool((dx.cpu()[~ok] == 0).all())
        if w is None:
            assert dw is None
        else:
            assert dw.dtype is w.dtype and dw.shape == w.shape
            step = 0.0 if w.dtype is torch.float32 else _half_step(w.dtype)
            assert bool(((dw.cpu().double() - rw).abs() <= step * rw.abs() * 1.01 + 2.0 ** -16 * total + 1e-30).all())


@pytest.mark.gpu
def test_gpu_backward_many_rows_and_shared_inputs():
    """More rows than workgroups at once; queries expanded over heads, a
    gradient expanded over channels' rows: autograd sums what was shared."""
    from dsv4_amd.rope import norm_rope_autograd, rope_table
    T, H, D = 900, 64, 512
    g = torch.Generator(device="cuda").manual_seed(1)
    one = torch.randn(T, 1, D, generator=g, device="cuda").to(torch.bfloat16).requires_grad_()
    kv = torch.randn(T, D, generator=g, device="cuda").to(torch.bfloat16).requires_grad_()
    w = (1 + 0.1 * torch.randn(D, generator=g, device="cuda")).requires_grad_()
    pos = torch.arange(T, device="cuda", dtype=torch.int32)
    table = rope_table(T)
    qo, ko = norm_rope_autograd(one.expand(T, H, D), kv, positions=pos, table=table, q_weight=w, kv_weight=w)
    dy = torch.randn(1, 1, D, generator=g, device="cuda").to(torch.bfloat16)
    d1, dkv, dw = torch.autograd.grad([qo, ko], [one, kv, w], [dy.expand(T, H, D), dy[0].expand(T, D)])
    cs = table.cpu()[:, None]
    # bf16 gradients of 64 equal heads, summed by torch in fp32 and rounded to bf16
    ref, rw, total = R.norm_rope_grad(dy.cpu().expand(T, 1, D), one.detach().cpu(), D, w.detach().cpu(), cs)
    each = ref.to(torch.bfloat16).double()
    # an element may round to either neighbour where fp32 decides: one step of each head's gradient, one of the sum's
    assert bool(((d1.cpu().double() - 64 * each).abs() <= 64 * (2.0 ** -7 * ref.abs() + 2.0 ** -15 * ref.abs().amax(-1, keepdim=True)) +
                 2.0 ** -8 * 64 * ref.abs()).all())
    _, rw2, total2 = R.norm_rope_grad(dy.cpu()[0].expand(T, D), kv.detach().cpu(), D, w.detach().cpu(), cs[:, 0])
    tot = 64 * total + total2
    # chains: 57600 rows over 512 workgroups of 32 rows, 4 a lane; torch adds the two gradients
    assert bool(((dw.cpu().double() - (64 * rw + rw2)).abs() <= 2.0 ** -16 * tot).all())


@pytest.mark.gpu
def test_gpu_forms_of_calls():
    """BSND, kv alone, q alone, unaligned and transposed rows (copied), int64
    positions, empty calls."""
    from dsv4_amd.rope import norm_rope, norm_rope_backward, rope_table
    g = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randn(3, 5, 16, 512, generator=g, device="cuda").to(torch.bfloat16)
    kv = torch.randn(3, 5, 512, generator=g, device="cuda").to(torch.bfloat16)
    pos = torch.randint(0, 90, (3, 5), generator=g, device="cuda")
    table = rope_table(90)
    qo, ko = norm_rope(q, kv, positions=pos, table=table)
    assert qo.shape == q.shape and ko.shape == kv.shape
    flat = dict(positions=pos.view(15).int(), table=table)
    assert torch.equal(norm_rope(q.view(15, 16, 512), **flat), qo.view(15, 16, 512))
    assert torch.equal(norm_rope(None, kv.view(15, 512), **flat), ko.view(15, 512))
    assert torch.equal(norm_rope(q.transpose(0, 1), kv.transpose(0, 1), positions=pos.t(), table=table)[0], qo.transpose(0, 1))
    odd = torch.empty(15 * 16 * 512 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(15, 16, 512)
    odd.copy_(q.view(15, 16, 512))
    assert odd.data_ptr() % 16 and torch.equal(norm_rope(odd, **flat), qo.view(15, 16, 512))
    turned = q.view(15, 16, 512).transpose(1, 2).contiguous().transpose(1, 2)
    assert turned.stride(-1) != 1 and torch.equal(norm_rope(turned, **flat), qo.view(15, 16, 512))
    # heads before tokens, as some projections lie
    heads = q.view(15, 16, 512).transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(norm_rope(heads, **flat), qo.view(15, 16, 512))
    e = norm_rope(q[:0], kv[:0], positions=pos[:0], table=table)
    assert e[0].shape == (0, 5, 16, 512) and e[1].shape == (0, 5, 512)
    w = torch.ones(512, device="cuda")
    dq, dkv, dqw, dkw = norm_rope_backward(q[:0], q[:0], kv[:0], kv[:0], positions=pos[:0], table=table, q_weight=w, kv_weight=w)
    assert dq.shape == (0, 5, 16, 512) and bool((dqw == 0).all()) and bool((dkw == 0).all())
    dq, dkv, dqw, dkw = norm_rope_backward(q, q, positions=pos, table=table, q_norm_dim=0, q_weight=w[:0])
    assert dkv is None and dkw is None and dqw.shape == (0,)
    for bad, match in (({"positions": pos[:2]}, "positions must be"), ({"positions": None}, "positions are needed"),
                       ({"q_weight": w[:8]}, "q_weight must be"), ({"q_weight": w.double()}, "q_weight must be fp32"),
                       ({"table": table.double()}, "table must be"), ({"table": table.cpu()}, "one device"),
                       ({"q_norm_dim": 12}, "norm dims"), ({"eps": -1.0}, "eps")):
        with pytest.raises(ValueError, match=match):
            norm_rope(q, **{"positions": pos, "table": table, **bad})
    with pytest.raises(ValueError, match="kv must be"):
        norm_rope(q, kv[:, :4], positions=pos, table=table)
    with pytest.raises(ValueError, match="dq_out must be"):
        norm_rope_backward(None, q, positions=pos, table=table)


@pytest.mark.gpu
def test_gpu_rotation_undone_and_non_finite_rows():
    """The inverse takes the rotation back within two roundings; infinities and
    NaN stay in their rows."""
    from dsv4_amd.rope import norm_rope, norm_rope_backward, rope_table
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(50, 16, 512, generator=g, device="cuda").to(torch.bfloat16)
    pos = torch.randint(0, 5000, (50,), generator=g, device="cuda").int()
    table = rope_table(5000)
    y = norm_rope(x, positions=pos, table=table, q_norm_dim=0)
    assert torch.equal(y[..., :448], x[..., :448])
    z = norm_rope(y, positions=pos, table=table, q_norm_dim=0, inverse=True)
    # each rounding: 2^-8 of a channel, and a rotation carries the pair's into one channel
    pair = x[..., 448:].float().unflatten(-1, (32, 2)).abs().sum(-1, keepdim=True).expand(-1, -1, -1, 2).flatten(-2)
    assert bool(((z[..., 448:].float() - x[..., 448:].float()).abs() <= 2.0 ** -8 * 2.1 * pair).all())
    clean = norm_rope(x, positions=pos, table=table)
    bad = x.clone()
    bad[7, 3, 5], bad[9, 0, 500] = float("inf"), NAN
    out = norm_rope(bad, positions=pos, table=table)
    hit = torch.zeros(50, 16, dtype=torch.bool, device="cuda")
    hit[7, 3] = hit[9, 0] = True
    assert torch.equal(out[~hit], clean[~hit])
    dq = norm_rope_backward(x, bad, positions=pos, table=table)[0]
    assert torch.equal(dq[~hit], norm_rope_backward(x, x, positions=pos, table=table)[0][~hit])


# ---------------------------------------------------------------------------
# cache append
# ---------------------------------------------------------------------------

def _append_case(dt, fp8, q_lens, kv_lens, D, bs, H, tail=3, seed=21, own_pos=False, holes=True):
    g = torch.Generator().manual_seed(seed)
    B, T = len(q_lens), sum(q_lens) + tail
    per = max(1, max(-(-max(k, 1) // bs) for k in kv_lens))
    nb = B * per + 2
    table = torch.randperm(nb, generator=g)[:B * per].to(torch.int32).reshape(B, per)
    if holes:
        table[0, (kv_lens[0] - 1) // bs] = -1
        table[B - 1, 0] = nb + 4
    cu = torch.zeros(B + 1, dtype=torch.int32)
    cu[1:] = torch.tensor(q_lens).cumsum(0)
    kv = torch.randn(T, D, generator=g)
    if T > 6:
        kv[2, :128] = 0.0
        kv[3] *= 1e-3
        kv[5] *= 300.0
    kv = kv.to(dt)
    q = torch.randn(T, H, D, generator=g).to(dt) if H else None
    w = 1 + 0.2 * torch.randn(512, generator=g)
    pos = torch.randint(-1, 303, (T,), generator=g, dtype=torch.int32) if own_pos else None
    row = 656 if fp8 else D * 2
    cache = torch.randint(0, 255, (nb, bs, 1, row), generator=g, dtype=torch.uint8)
    return q, kv, cache if fp8 else cache.view(dt), table, cu, torch.tensor(kv_lens, dtype=torch.int32), w, pos


APPENDS = [
    # dtype, fp8, query lengths, kv lengths, D, block, heads, norm channels, own positions, rope_dim, half
    ("bf16", False, [1] * 5, [70, 1, 300, 64, 65], 512, 64, 16, 512, False, 64, False),
    ("fp16", False, [4, 0, 9, 1], [9, 33, 200, 1], 576, 16, 3, 512, True, 64, True),
    ("bf16", True, [3, 40, 1, 0, 5], [290, 50, 1, 20, 64], 576, 64, 16, 512, False, 64, False),
    ("bf16", True, [7, 11], [7, 30], 576, 16, 0, 0, True, 64, True),
    ("bf16", True, [6, 2], [60, 30], 576, 64, 5, 512, False, 32, False),       # every row's block missing
    ("bf16", True, [6, 20], [80, 130], 576, 64, 5, 512, False, 32, False),
    ("bf16", False, [5, 3], [3, 40], 512, 64, 9, 512, False, 64, False),       # more new rows than positions
    ("fp16", False, [1] * 70 + [0, 2, 3], [40] * 73, 512, 16, 8, 512, False, 64, False),
    ("bf16", True, [1] * 130, [17] * 130, 576, 16, 2, 512, False, 64, False),
    ("bf16", False, [0] * 63 + [2, 1, 0, 4], [12] * 67, 128, 16, 1, 64, False, 64, False),
    ("bf16", False, [5, 6], [20, 20], 512, 64, 4, 512, False, 0, False),       # no rotation
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", APPENDS, ids=[str(i) for i in range(len(APPENDS))])
def test_gpu_append(case):
    from dsv4_amd.cache import append_kv_cache
    dt, fp8, ql, kl, D, bs, H, n, own_pos, Rd, half = case
    dt = DT[dt]
    q, kv, cache, table, cu, used, w, pos = _append_case(dt, fp8, ql, kl, D, bs, H, own_pos=own_pos)
    w = w[:n] if n else None
    rope = _table(302, Rd)
    d = cache.cuda()
    mv = lambda t: None if t is None else t.cuda()  # noqa: E731
    got_q = append_kv_cache(mv(kv), d, mv(table), mv(cu), mv(used), table=mv(rope), positions=mv(pos), norm_dim=n,
                            weight=mv(w), interleaved=not half, q=mv(q), q_norm_dim=D)
    T, nb = kv.shape[0], cache.shape[0]
    places = R.slots(cu, used, T)
    at = [None if p is None else p[1] if pos is None else int(pos[t]) for t, p in enumerate(places)]
    ok = torch.tensor([a is not None and (not Rd or 0 <= a < 302) for a in at])
    cs = rope[torch.tensor([a if o else 0 for a, o in zip(at, ok.tolist())])] if Rd else None
    flat = R.rows_of([p if o else None for p, o in zip(places, ok.tolist())], table, bs, nb)
    ref = R.norm_rope(kv, n, w, cs, half)
    out = d.cpu().view(torch.uint8).reshape(nb * bs, -1)
    before = cache.view(torch.uint8).reshape(nb * bs, -1)
    touched = [f for f in flat if f is not None]
    assert len(set(touched)) == len(touched)
    rest = torch.ones(nb * bs, dtype=torch.bool)
    rest[touched] = False
    assert torch.equal(out[rest], before[rest])          # every other row as it was
    src = torch.tensor([t for t, f in enumerate(flat) if f is not None], dtype=torch.int64)
    rows, want = out[torch.tensor(touched, dtype=torch.int64)], ref[src]
    big = want.abs().amax(-1, keepdim=True)
    if not fp8:
        _close(rows.view(dt), want, dt, 2.0 ** -16 * big)
    else:
        lat = want[:, :512].unflatten(-1, (4, 128))
        amax = lat.abs().amax(-1)
        scale = rows[:, 512:528].contiguous().view(torch.float32).double()
        assert bool(((scale - torch.where(amax > 0, amax / 448, 1.0)).abs() <= 2.0 ** -16 * big / 448).all())
        got = rows[:, :512].contiguous().view(torch.float8_e4m3fn).double().unflatten(-1, (4, 128)) * scale[..., None]
        # half a step of e4m3: 2^-4 relative, or 2^-10 of the scale below 2^-6
        bound = torch.maximum(lat.abs() * 2.0 ** -4, 2.0 ** -10 * scale[..., None]) * (1 + 2.0 ** -10)
        assert bool(((got - lat).abs() <= bound + 2.0 ** -15 * big[..., None]).all())
        _close(rows[:, 528:].contiguous().view(torch.bfloat16), want[:, 512:], torch.bfloat16, 2.0 ** -16 * big)
    if H:
        ref_q = R.norm_rope(q, D, None, None if cs is None else cs[:, None], half)
        ref_q = torch.where(ok.view(-1, 1, 1), ref_q, 0.0)
        _close(got_q.cpu(), ref_q, dt, 2.0 ** -16 * ref_q.abs().amax(-1, keepdim=True))
    else:
        assert got_q is None


@pytest.mark.gpu
def test_gpu_append_refuses():
    from dsv4_amd.cache import append_kv_cache
    from dsv4_amd.rope import rope_table
    q, kv, cache, table, cu, used, w, _ = [t.cuda() if t is not None else None for t in
                                           _append_case(torch.bfloat16, False, [2, 3], [5, 9], 512, 16, 4)]
    rope = rope_table(20)
    ok = dict(kv=kv, cache=cache, block_table=table, cu_seqlens_q=cu, seqused_kv=used, table=rope, weight=w, norm_dim=512, q=q)
    before = cache.clone()
    for over, match in (({"kv": kv[0]}, "kv must be"), ({"q": q[1:]}, "kv must be"), ({"cache": cache[0]}, "cache must be"),
                        ({"cache": cache.half()}, "cache must hold"), ({"cache": cache[::2]}, "contiguous"),
                        ({"cu_seqlens_q": cu[1:]}, "must agree"), ({"block_table": table[:1]}, "must agree"),
                        ({"seqused_kv": used.cpu()}, "kv's device"), ({"table": rope.cpu()}, "one device"),
                        ({"weight": w[:100]}, "weight must be"), ({"positions": cu}, "positions must be"),
                        ({"cache": torch.zeros(4, 16, 1, 656, dtype=torch.uint8, device="cuda")}, "fp8"),
                        ({"norm_dim": 4, "weight": None}, "norm dims")):
        with pytest.raises(ValueError, match=match):
            append_kv_cache(**{**ok, **over})
    assert torch.equal(cache.view(torch.uint8), before.view(torch.uint8))


@pytest.mark.gpu
def test_gpu_append_then_attention_and_capture():
    """A layer's step as it is used: append with the queries, attention over the
    cache, the output rotated back; eager on a side stream, then captured and
    replayed with new inputs, every replay as the eager call."""
    from dsv4_amd.api import sparse_attn_sharedkv
    from dsv4_amd.cache import append_kv_cache
    from dsv4_amd.rope import norm_rope, rope_table
    ql, kl, D, bs, H = [1, 3, 2, 1], [40, 77, 150, 1], 512, 16, 16
    q, kv, cache, table, cu, used, w, _ = [t.cuda() if t is not None else None for t in _append_case(
        torch.bfloat16, False, ql, kl, D, bs, H, tail=0, holes=False)]
    cache = torch.randn(cache.shape, device="cuda").to(torch.bfloat16)
    rope, sinks = rope_table(200), torch.zeros(H, device="cuda")
    pos = torch.cat([torch.arange(k - m, k) for m, k in zip(ql, kl)]).int().cuda()

    def step():
        qr = append_kv_cache(kv, cache, table, cu, used, table=rope, norm_dim=512, weight=w, q=q)
        out = sparse_attn_sharedkv(qr, ori_kv=cache, ori_block_table=table, cu_seqlens_q=cu, seqused_kv=used, sinks=sinks,
                                   softmax_scale=D ** -0.5)
        return qr, out, norm_rope(out, positions=pos, table=rope, q_norm_dim=0, inverse=True)

    eager = step()
    want_q, want_kv = norm_rope(q, kv, positions=pos, table=rope, kv_weight=w)
    assert torch.equal(eager[0], want_q)
    at = R.rows_of(R.slots(cu.cpu(), used.cpu(), len(pos)), table.cpu(), bs, cache.shape[0])
    assert torch.equal(cache.view(-1, D)[at], want_kv)
    # the attention over what was appended, in 64 bits
    t = 0
    for b, (m, k) in enumerate(zip(ql, kl)):
        rows = cache.view(-1, D)[R.rows_of([(b, i) for i in range(k)], table.cpu(), bs, cache.shape[0])].double().cpu()
        for i in range(m):
            p = k - m + i
            keys = rows[max(0, p - 127):p + 1]
            x = torch.cat([want_q[t].double().cpu() @ keys.t() * D ** -0.5, torch.zeros(H, 1, dtype=torch.float64)], 1)
            ref = torch.softmax(x, 1)[:, :-1] @ keys
            assert torch.allclose(eager[1][t].double().cpu(), ref, atol=2e-2, rtol=2e-2)
            t += 1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a, b in zip(step(), eager):
            assert torch.equal(a, b)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(4):
        q.copy_(torch.randn(q.shape, device="cuda"))
        kv.copy_(torch.randn(kv.shape, device="cuda"))
        graph.replay()
        got = [x.clone() for x in captured]
        after = cache.clone()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b), k
        assert torch.equal(after, cache)


@pytest.mark.gpu
def test_gpu_training_step_through_the_attention():
    """norm_rope_autograd -> attention over the rows it made -> a captured
    backward of the norms: gradients of the raw projections and weights flow
    through both operators."""
    from dsv4_amd.api import sparse_attn_sharedkv_autograd
    from dsv4_amd.rope import norm_rope_autograd, norm_rope_backward, rope_table
    T, H, D, bs = 96, 32, 512, 32
    g = torch.Generator(device="cuda").manual_seed(4)
    q = torch.randn(T, H, D, generator=g, device="cuda").to(torch.bfloat16).requires_grad_()
    kv = torch.randn(T, D, generator=g, device="cuda").to(torch.bfloat16).requires_grad_()
    w = (1 + 0.1 * torch.randn(D, generator=g, device="cuda")).requires_grad_()
    pos = torch.arange(T, device="cuda", dtype=torch.int32)
    rope = rope_table(T)
    kw = dict(ori_block_table=torch.arange(T // bs, device="cuda", dtype=torch.int32)[None],
              cu_seqlens_q=torch.tensor([0, T], device="cuda", dtype=torch.int32),
              seqused_kv=torch.tensor([T], device="cuda", dtype=torch.int32), softmax_scale=D ** -0.5, ori_win_left=31)
    sinks = torch.zeros(H, device="cuda")
    qr, kr = norm_rope_autograd(q, kv, positions=pos, table=rope, kv_weight=w)
    qr.retain_grad()
    kr.retain_grad()
    out = sparse_attn_sharedkv_autograd(qr, ori_kv=kr.view(T // bs, bs, 1, D), sinks=sinks, **kw)
    dout = torch.randn(out.shape, generator=g, device="cuda").to(torch.bfloat16)
    out.backward(dout)
    want = norm_rope_backward(qr.grad, q.detach(), kr.grad, kv.detach(), positions=pos, table=rope, kv_weight=w.detach())
    assert torch.equal(q.grad, want[0]) and torch.equal(kv.grad, want[1]) and torch.equal(w.grad, want[3])
    assert all(bool(torch.isfinite(t).all()) and float(t.abs().max()) > 0 for t in (q.grad, kv.grad, w.grad))
    # the whole step against 64-bit autograd on the CPU
    q64, kv64, w64 = (t.detach().cpu().double().requires_grad_() for t in (q, kv, w))
    cs = torch.view_as_complex(rope.cpu().double())

    def turn(x, c):
        z = torch.view_as_complex(x[..., 448:].unflatten(-1, (32, 2)).contiguous()) * c
        return torch.cat([x[..., :448], torch.view_as_real(z).flatten(-2)], -1)

    qn = q64 / torch.sqrt((q64 ** 2).mean(-1, keepdim=True) + 1e-6)
    kn = kv64 / torch.sqrt((kv64 ** 2).mean(-1, keepdim=True) + 1e-6) * w64
    qn, kn = turn(qn, cs[:, None]), turn(kn, cs)
    x = torch.einsum("thd,sd->hts", qn, kn) * D ** -0.5
    i = torch.arange(T)
    x = x.masked_fill(~((i[None] <= i[:, None]) & (i[None] > i[:, None] - 32)), -float("inf"))
    x = torch.cat([x, torch.zeros(H, T, 1, dtype=torch.float64)], 2)
    o = torch.einsum("hts,sd->thd", torch.softmax(x, 2)[..., :T], kn)
    ref = torch.autograd.grad(o, [q64, kv64, w64], dout.cpu().double())
    for name, a, b in (("q", q.grad, ref[0]), ("kv", kv.grad, ref[1]), ("w", w.grad, ref[2])):
        # rotated rows, P, dS, the attention's gradients: some six roundings of 2^-8 each
        rel = float((a.cpu().double() - b).norm() / b.norm())
        assert rel <= 6 * 2.0 ** -8, (name, rel)
    # captured: the kernels' backward, replayed on new gradients
    gq, gk = qr.grad.clone(), kr.grad.clone()
    args = dict(positions=pos, table=rope, kv_weight=w.detach())
    graph = torch.cuda.CUDAGraph()
    qd, kd = q.detach(), kv.detach()
    norm_rope_backward(gq, qd, gk, kd, **args)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = norm_rope_backward(gq, qd, gk, kd, **args)
    for _ in range(3):
        gq.copy_(torch.randn(gq.shape, device="cuda"))
        gk.copy_(torch.randn(gk.shape, device="cuda"))
        graph.replay()
        got = [None if t is None else t.clone() for t in captured]
        torch.cuda.synchronize()
        for a, b in zip(got, norm_rope_backward(gq, qd, gk, kd, **args)):
            assert a is b is None or torch.equal(a, b)


def test_abi_refuses_more_rows_than_a_launch_has_threads_for():
    L = _lib.lib()
    small = dict(H=0, q=None, q_out=None, D=8, kv_stride_t=8, rope_dim=0, kv_norm_dim=8, q_norm_dim=0)
    for over in (dict(small, T=1 << 28), dict(T=(1 << 24) - 1, H=16, kv=None)):
        if "kv" in over:   # the queries alone reach it from 2^28 - 31 rows on
            over["T"] += 1
        assert L.sas_norm_rope_v1(C.byref(_args(**over)), None) == _lib.SAS_EINVAL
        assert "2^28" in L.sas_last_error().decode()
        ca = _lib.SasCacheAppendArgs(rope=_args(**over), cu_seqlens_q=FAKE, act_kv=FAKE, block_table=FAKE, cache=FAKE, B=1,
                                     bt_stride=1, block_size=64, num_blocks=1, cache_dtype=_lib.SAS_DT_BF16)
        assert L.sas_cache_append_v1(C.byref(ca), None) == _lib.SAS_EINVAL
        assert "2^28" in L.sas_last_error().decode()
    n = C.c_size_t(0)
    ba = _lib.SasNormRopeBwdArgs(fwd=_args(T=(1 << 28) // 17 - 16), dq_weight=FAKE)
    assert L.sas_norm_rope_bwd_plan(C.byref(ba), C.byref(n)) == _lib.SAS_OK and n.value > 0


@pytest.mark.gpu
def test_gpu_positions_without_a_table_are_not_read():
    """The same signature twice: the second call takes the kept resolution."""
    from dsv4_amd.cache import append_kv_cache
    from dsv4_amd.rope import norm_rope, norm_rope_backward
    q = torch.randn(40, 16, 512, device="cuda").to(torch.bfloat16)
    kv = q[:, 0].contiguous()
    want = norm_rope(q, kv)
    for pos in (torch.zeros(3, dtype=torch.int64, device="cuda"), torch.zeros(40, dtype=torch.int32)):
        for _ in range(2):
            assert all(torch.equal(a, b) for a, b in zip(norm_rope(q, kv, positions=pos), want))
        grads = [norm_rope_backward(q, q, positions=pos)[0] for _ in range(2)]
        assert torch.equal(*grads) and torch.equal(grads[0], norm_rope_backward(q, q)[0])
        for _ in range(2):
            cache = torch.zeros(3, 16, 1, 512, device="cuda", dtype=torch.bfloat16)
            args = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([[0, 1, 2]], [0, 40], [40])]
            assert torch.equal(append_kv_cache(kv, cache, *args, positions=pos, q=q), want[0])
            assert torch.equal(cache.view(48, 512)[:40], want[1])


@pytest.mark.gpu
def test_gpu_scalars_in_tensors_are_read_anew():
    from dsv4_amd.rope import norm_rope
    q = torch.randn(4, 16, 128, device="cuda").to(torch.bfloat16)
    eps = torch.tensor(1e-6)
    n = torch.tensor(128)
    norm_rope(q, eps=eps, q_norm_dim=n)
    eps.fill_(1.0)
    n.fill_(64)
    assert torch.equal(norm_rope(q, eps=eps, q_norm_dim=n), norm_rope(q, eps=1.0, q_norm_dim=64))


@pytest.mark.gpu
def test_gpu_positions_past_32_bits_are_padding():
    from dsv4_amd.cache import append_kv_cache
    from dsv4_amd.rope import norm_rope, norm_rope_backward, rope_table
    q = torch.randn(6, 16, 512, device="cuda").to(torch.bfloat16)
    kv = q[:, 0].contiguous()
    pos = torch.tensor([3, -1, 2 ** 32 + 3, -2 ** 63, 2 ** 63 - 1, -2 ** 32 + 3], device="cuda")
    table = rope_table(8)
    a = norm_rope(q, positions=pos, table=table)
    assert torch.equal(a[0], norm_rope(q[:1], positions=pos[:1].int(), table=table)[0]) and bool((a[1:] == 0).all())
    d = norm_rope_backward(q, q, positions=pos, table=table)[0]
    assert bool((d[0] != 0).any()) and bool((d[1:] == 0).all())
    cache = torch.zeros(1, 16, 1, 512, device="cuda", dtype=torch.bfloat16)
    args = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([[0]], [0, 6], [6])]
    assert torch.equal(append_kv_cache(kv, cache, *args, table=table, positions=pos, q=q), a)
    assert bool((cache[0, 0] != 0).any()) and bool((cache[0, 1:] == 0).all())
    for bad in (pos.float(), pos > 0):
        with pytest.raises(ValueError, match="integers"):
            norm_rope(q, positions=bad, table=table)


@pytest.mark.gpu
def test_gpu_offsets_past_32_bits():
    """Rows, gradients, table and cache of more than 4 GiB: the last tokens are what
    a call of their own gives."""
    from dsv4_amd.cache import append_kv_cache
    from dsv4_amd.rope import norm_rope, norm_rope_backward, rope_table
    g = torch.Generator(device="cuda").manual_seed(5)
    T, H, D, k = 60000, 64, 576, 50
    table = rope_table(1 << 16)
    q = torch.empty(T, H, D, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    assert q.numel() * 2 > 1 << 32
    pos = torch.arange(T, device="cuda", dtype=torch.int32)
    last = dict(positions=pos[-k:], table=table)
    out = norm_rope(q, positions=pos, table=table)
    assert torch.equal(out[-k:], norm_rope(q[-k:], **last))
    d = norm_rope_backward(out, q, positions=pos, table=table)[0]
    assert torch.equal(d[-k:], norm_rope_backward(out[-k:], q[-k:], **last)[0])
    del out, d
    # a table of 2^27 rows of 8 rotated channels
    n = 1 << 27
    wide = torch.zeros(n, 4, 2, device="cuda")
    wide[-k:] = rope_table(k, 8)
    far = dict(positions=torch.arange(n - k, n, device="cuda", dtype=torch.int32), table=wide)
    near = dict(positions=torch.arange(k, device="cuda", dtype=torch.int32), table=rope_table(k, 8))
    assert torch.equal(norm_rope(q[:k], **far), norm_rope(q[:k], **near))
    del wide, far
    kv = q[:k, 0].contiguous()
    del q
    for dt, row in ((torch.bfloat16, D), (torch.uint8, 656)):
        blocks = (1 << 32) // (64 * row * dt.itemsize) + 2
        cache = torch.zeros(blocks, 64, 1, row, device="cuda", dtype=dt)
        small = torch.zeros(1, 64, 1, row, device="cuda", dtype=dt)
        cu, used = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, k], [k]))
        for c, b in ((cache, blocks - 1), (small, 0)):
            append_kv_cache(kv, c, torch.tensor([[b]], dtype=torch.int32, device="cuda"), cu, used, table=table)
        assert bool((small != 0).any()) and torch.equal(cache[-1], small[0])
        del cache


# ---------------------------------------------------------------------------
# fp8 appends of rows out of the ordinary
# ---------------------------------------------------------------------------

def _append_fp8(kv, n, rope_dim=0, **kw):
    """The 656-byte rows that an append of kv [T, 576] (one sequence) leaves, on the CPU."""
    from dsv4_amd.cache import append_kv_cache
    T = kv.shape[0]
    cache = torch.zeros(-(-T // 16), 16, 1, 656, dtype=torch.uint8, device="cuda")
    table = torch.arange(cache.shape[0], dtype=torch.int32, device="cuda")[None]
    cu, used = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, T], [T]))
    rope = _table(T, rope_dim)
    append_kv_cache(kv.cuda(), cache, table, cu, used, norm_dim=n, table=None if rope is None else rope.cuda(), **kw)
    return cache.view(-1, 656)[:T].cpu()


def _check_fp8(rows, y, slack):
    """rows against y [T, 576] in 64 bits, by 128-channel groups: the scale amax / 448 (1
    where amax is 0 or NaN), each byte within half a step of its value, a NaN where the
    value over the scale is one. `slack` [T, 1]: the fp32 error of y."""
    lat = y[:, :512].unflatten(-1, (4, 128))
    amax = lat.abs().amax(-1)                       # (torch's keeps a NaN)
    scale = rows[:, 512:528].contiguous().view(torch.float32).double()
    want = torch.where(amax > 0, amax / 448, 1.0)
    inf = want.isinf()
    assert torch.equal(scale.isinf(), inf)
    # (half a step of the smallest floats below 2^-126)
    assert bool(((scale - want).abs() <= 2.0 ** -16 * want + slack / 448 + 2.0 ** -150)[~inf].all())
    # what the byte stands for: the value over the scale, clamped (scale 1 beside a NaN)
    code = rows[:, :512].contiguous().view(torch.float8_e4m3fn).double().unflatten(-1, (4, 128))
    val = (lat / want[..., None]).clamp(-448, 448)
    assert torch.equal(code.isnan(), val.isnan())
    bound = torch.maximum(val.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10, dtype=torch.float64)) * (1 + 2.0 ** -10)
    bound = bound + slack[..., None] / scale[..., None]
    assert bool(((code - val).abs() <= bound)[~val.isnan()].all())


@pytest.mark.gpu
@pytest.mark.parametrize("rope_dim", [0, 32], ids=["plain", "rotated32"])
@pytest.mark.parametrize("n", [0, 256, 512, 576])
def test_gpu_append_fp8_keeps_nan_and_infinities(n, rope_dim):
    """A channel that is NaN or infinite: the row is what the formulas and the codec
    make of it, no finite value in its place; the rows beside it are as without it."""
    g = torch.Generator().manual_seed(31)
    clean = torch.randn(40, 576, generator=g).to(torch.bfloat16)
    kv = clean.clone()
    bad = {3: (5, NAN), 4: (300, float("inf")), 9: (511, -float("inf")), 10: (255, NAN), 11: (575, NAN), 17: (560, float("inf"))}
    for r, (c, v) in bad.items():
        kv[r, c] = v
    kv[20, 130], kv[20, 140], kv[20, 400] = float("inf"), NAN, -NAN
    kv[21, 0:512:3] = float("inf")
    rows, want = _append_fp8(kv, n, rope_dim), _append_fp8(clean, n, rope_dim)
    hit = torch.zeros(40, dtype=torch.bool)
    hit[[*bad, 20, 21]] = True
    assert torch.equal(rows[~hit], want[~hit])
    y = R.norm_rope(kv, n, None, _table(40, rope_dim) if rope_dim else None)
    big = y.abs().nan_to_num(0.0, 0.0, 0.0).amax(-1, keepdim=True)
    _check_fp8(rows, y, 2.0 ** -16 * big)
    tail = rows[:, 528:].contiguous().view(torch.bfloat16).double()
    assert torch.equal(tail.isnan(), y[:, 512:].isnan()) and torch.equal(tail.isinf(), y[:, 512:].isinf())


@pytest.mark.gpu
def test_gpu_fp8_rows_of_nan_reach_the_attention():
    """A token that attends an appended NaN row gives NaN, as over a bf16 cache; the
    tokens before it, and the other sequence's, what they gave without it."""
    from dsv4_amd.api import sparse_attn_sharedkv, sparse_attn_sharedkv_tree
    from dsv4_amd.cache import append_kv_cache
    g = torch.Generator().manual_seed(32)
    q = torch.randn(16, 16, 576, generator=g).to(torch.bfloat16).cuda()
    clean = torch.randn(16, 576, generator=g).to(torch.bfloat16)
    kv = clean.clone()
    kv[5, 17] = NAN
    table = torch.tensor([[0], [1]], dtype=torch.int32, device="cuda")
    cu, used = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 9, 16], [9, 7]))
    mask = torch.tensor([(2 << i) - 1 for i in (*range(9), *range(7))], dtype=torch.int64, device="cuda")[:, None]
    outs = []
    for rows, row in ((clean, 656), (kv, 656), (kv, 576)):
        cache = torch.zeros(2, 16, 1, row, dtype=torch.uint8 if row == 656 else torch.bfloat16, device="cuda")
        append_kv_cache(rows.cuda(), cache, table, cu, used, norm_dim=512)
        kw = dict(ori_kv=cache, ori_block_table=table, cu_seqlens_q=cu, seqused_kv=used, sinks=torch.zeros(16, device="cuda"),
                  softmax_scale=0.04)
        outs.append((sparse_attn_sharedkv(q, **kw), sparse_attn_sharedkv_tree(q, tree_mask=mask, **kw)))
    sees = torch.zeros(16, dtype=torch.bool)
    sees[5:9] = True
    for without, fp8, bf16 in zip(*outs):
        assert bool(fp8[sees].isnan().all()) and bool(bf16[sees].isnan().all())
        assert torch.equal(fp8[~sees], without[~sees])


@pytest.mark.gpu
@pytest.mark.parametrize("rope_dim", [0, 32], ids=["plain", "rotated32"])
@pytest.mark.parametrize("n,eps", [(0, 0.0), (512, 1e-6), (512, 1e-12)])
def test_gpu_append_fp8_groups_of_tiny_channels(n, eps, rope_dim):
    """Groups whose channels lie below 1e-34 down to the smallest bf16 values, zeros among
    them: 448 over their maximum, times the norm's factor, is past the largest float."""
    g = torch.Generator().manual_seed(33)
    kv = torch.randn(24, 576, generator=g)
    zero = torch.rand(24, 512, generator=g) < 0.3
    kv[:, :512] = torch.where(zero, 0.0, kv[:, :512] * 10.0 ** -torch.linspace(33, 40.4, 24)[:, None])
    kv[::4, 128:256] = 0.0
    kv[5, 256:384] = 0.0
    kv[5, 300] = -1e-40                              # one channel, the others zeros
    kv = kv.to(torch.bfloat16)
    rows = _append_fp8(kv, n, rope_dim, eps=eps)
    y = R.norm_rope(kv, n, None, _table(24, rope_dim) if rope_dim else None, eps=eps)
    # by groups: each is of its own magnitude; fp32 values below 2^-126 have steps of 2^-149
    big = y[:, :512].unflatten(-1, (4, 128)).abs().amax(-1)
    _check_fp8(rows, y, 2.0 ** -16 * big + 2.0 ** -149 * (n > 0))
    zeros = rows[:, :512][kv[:, :512] == 0]
    assert bool(((zeros == 0) | (zeros == 0x80)).all())


# ---------------------------------------------------------------------------
# calls past the caches: rows read (and written) non-temporally, by builds and
# branches of their own
# ---------------------------------------------------------------------------

def _randn(shape, dt, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.empty(shape, device="cuda", dtype=dt).normal_(generator=g)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,fp8,D,rope_dim,half", [
    ("bf16", False, 512, 64, False), ("fp16", False, 576, 64, True), ("bf16", True, 576, 64, False),
    ("bf16", True, 576, 32, True), ("fp16", False, 640, 32, False)])
def test_gpu_append_past_the_caches(dt, fp8, D, rope_dim, half):
    """2501 tokens of 64 heads, more than 128 MB of rows: the same bits as the same
    tokens in steps of 400."""
    from dsv4_amd.cache import append_kv_cache
    from dsv4_amd.rope import rope_table
    T, H, bs, step = 2501, 64, 64, 400
    assert T * (H + 1) * D * 4 >= 256e6 > step * (H + 1) * D * 4
    q, kv = _randn((T, H, D), DT[dt], 41), _randn((T, D), DT[dt], 42)
    w = 1 + 0.2 * torch.randn(D, device="cuda")
    blocks = -(-T // bs)
    table = torch.randperm(blocks + 2, device="cuda")[:blocks].to(torch.int32)[None]
    kw = dict(table=rope_table(T, rope_dim), norm_dim=512, weight=w[:512], interleaved=not half, q_norm_dim=D, q_weight=w)
    row = dict(device="cuda", dtype=torch.uint8 if fp8 else DT[dt])

    def append(cache, a, b):
        cu, used = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, b - a], [b]))
        return append_kv_cache(kv[a:b], cache, table, cu, used, q=q[a:b], **kw)

    one = torch.zeros(blocks + 2, bs, 1, 656 if fp8 else D, **row)
    many = torch.zeros_like(one)
    got = append(one, 0, T)
    want = torch.cat([append(many, a, min(a + step, T)) for a in range(0, T, step)])
    assert torch.equal(got, want) and torch.equal(one, many) and bool((one != 0).any())


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D,rope_dim,half,T", [
    ("fp16", 576, 64, True, 2501), ("fp16", 512, 64, False, 8001), ("bf16", 576, 64, True, 7001), ("bf16", 640, 32, False, 2501),
    ("fp16", 128, 64, True, 16001)])
def test_gpu_forward_past_the_caches(dt, D, rope_dim, half, T):
    """The same bits as the tokens in calls that stay within them; 512 MB and more are
    written past the caches too."""
    from dsv4_amd.rope import norm_rope, rope_table
    H, step = 64, 800
    assert T * (H + 1) * D * 4 >= 256e6 > step * (H + 1) * D * 4
    q, kv = _randn((T, H, D), DT[dt], 43), _randn((T, D), DT[dt], 44)
    w = 1 + 0.2 * torch.randn(D, device="cuda")
    pos, table = torch.randint(-1, 5001, (T,), device="cuda", dtype=torch.int32), rope_table(5000, rope_dim)
    kw = dict(table=table, q_norm_dim=512 if D > 512 else D, kv_norm_dim=D, kv_weight=w, interleaved=not half)
    got = norm_rope(q, kv, positions=pos, **kw)
    for a in range(0, T, step):
        part = norm_rope(q[a:a + step], kv[a:a + step], positions=pos[a:a + step], **kw)
        assert all(torch.equal(x[a:a + step], y) for x, y in zip(got, part))


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D,rope_dim,half", [("bf16", 512, 64, False), ("fp16", 576, 64, True), ("bf16", 640, 32, True)])
def test_gpu_backward_past_the_caches(dt, D, rope_dim, half):
    """Rows' gradients as in calls of 200 tokens; weights' against 64 bits: chains of 8 rows
    a lane, 6 adds over the workgroup's, 12 and 64 over the workgroups: 90 e < 2^-17, and
    2^-17 of each term."""
    from dsv4_amd.rope import norm_rope_backward, rope_table
    T, H, step = 1501, 64, 200
    assert T * (H + 1) * D * 6 >= 256e6 > step * (H + 1) * D * 6
    q, kv = _randn((T, H, D), DT[dt], 45), _randn((T, D), DT[dt], 46)
    gq, gk = _randn((T, H, D), DT[dt], 47), _randn((T, D), DT[dt], 48)
    w = 1 + 0.2 * torch.randn(D, device="cuda")
    pos, table = torch.randint(0, 5000, (T,), device="cuda", dtype=torch.int32), rope_table(5000, rope_dim)
    kw = dict(table=table, q_norm_dim=512, q_weight=w[:512], kv_weight=w, interleaved=not half)
    dq, dkv, dqw, dkw = norm_rope_backward(gq, q, gk, kv, positions=pos, **kw)
    for a in range(0, T, step):
        s = slice(a, a + step)
        part = norm_rope_backward(gq[s], q[s], gk[s], kv[s], positions=pos[s], **kw)
        assert torch.equal(dq[s], part[0]) and torch.equal(dkv[s], part[1])
    cs = table[pos.long()]
    for dw, dy, x, n, c in ((dqw, gq, q, 512, cs[:, None]), (dkw, gk, kv, D, cs)):
        _, want, total = R.norm_rope_grad(dy, x, n, w[:n], c, half)
        assert bool(((dw.double() - want).abs() <= 2.0 ** -16 * total).all())


def test_abi_names_the_most_rows_of_a_call():
    L = _lib.lib()
    n = C.c_size_t(0)
    for T, ok in (((1 << 28) - 32, True), ((1 << 28) - 31, False), (1 << 28, False), (1 << 31, False), (1 << 40, False)):
        a = _args(T=T, H=0, q=None, q_out=None, D=8, kv_stride_t=8, rope_dim=0, kv_norm_dim=8, q_norm_dim=0)
        rc = L.sas_norm_rope_bwd_plan(C.byref(_lib.SasNormRopeBwdArgs(fwd=a)), C.byref(n))   # (launches nothing)
        assert rc == (_lib.SAS_OK if ok else _lib.SAS_EINVAL)
        if not ok:
            assert "at most 2^28 - 32" in L.sas_last_error().decode()


@pytest.mark.gpu
@pytest.mark.parametrize("H", [16, 32, 48, 64, 128])
@pytest.mark.parametrize("T", [9, 300])
def test_gpu_fp8_rows_of_nan_reach_every_kernel(T, H):
    """As above over the kernels that head and token counts choose, compressed rows among
    the keys: one NaN row of each cache; tokens that attend neither as without them."""
    from dsv4_amd.api import sparse_attn_sharedkv, sparse_attn_sharedkv_tree
    from dsv4_amd.cache import append_kv_cache
    g = torch.Generator().manual_seed(34)
    q = torch.randn(T, H, 576, generator=g).to(torch.bfloat16).cuda()
    blocks = -(-T // 64) + 1
    table = torch.arange(blocks, dtype=torch.int32, device="cuda")[None]
    cu, used = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, T], [T]))
    idx = torch.full((T, 1, 40), -1, dtype=torch.int32)
    for t in range(T):
        n = min((t + 1) // 4, 40)
        idx[t, 0, :n] = torch.randperm((t + 1) // 4, generator=g)[:n]
    words = -(-T // 64)
    mask = [[(1 << min(64, t + 1 - 64 * w)) - 1 if t >= 64 * w else 0 for w in range(words)] for t in range(T)]
    mask = torch.tensor([[x - (1 << 64) if x >> 63 else x for x in m] for m in mask], dtype=torch.int64).cuda()
    clean, cmp_clean = (torch.randn(n, 576, generator=g).to(torch.bfloat16) for n in (T, max(T // 4, 1)))
    kv, cmp = clean.clone(), cmp_clean.clone()
    kv[5, 17], cmp[1, 400] = NAN, NAN

    def caches(rows, cmp_rows):
        out = []
        for r in (rows, cmp_rows):
            c = torch.zeros(blocks, 64, 1, 656, dtype=torch.uint8, device="cuda")
            n = r.shape[0]
            append_kv_cache(r.cuda(), c, table, *(torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, n], [n])), norm_dim=512)
            out.append(c)
        return dict(ori_kv=out[0], cmp_kv=out[1])

    kw = dict(ori_block_table=table, cmp_block_table=table, cmp_sparse_indices=idx.cuda(), cmp_ratio=4, cu_seqlens_q=cu,
              seqused_kv=used, sinks=torch.zeros(H, device="cuda"), softmax_scale=0.04, ori_win_left=31)
    t = torch.arange(T)
    sees = ((t >= 5) & (t - 31 <= 5)) | (idx[:, 0] == 1).any(1)
    assert bool(sees.any()) and not bool(sees.all())
    for call in (lambda c: sparse_attn_sharedkv(q, **kw, **c), lambda c: sparse_attn_sharedkv_tree(q, tree_mask=mask, **kw, **c)):
        without, out = call(caches(clean, cmp_clean)), call(caches(kv, cmp))
        assert bool(out[sees].isnan().all()) and torch.equal(out[~sees], without[~sees])

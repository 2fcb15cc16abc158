"""Performance cases of the operators around the attention: what a serving or
training program has them do, in their plain form or through the framework's
entry points.

A case is a dict of plain values. ``op`` is the call:

``rope``    norms of queries and KV rows for each head, rotated by their
            positions, in one pass (``norm_rope``);
``grad``    its backward (``norm_rope_backward``): the gradients of queries,
            KV rows and norm weights;
``append``  the new KV rows of a step normed, rotated and written into the
            paged cache, with the step's queries where ``H`` is set
            (``append_kv_cache``);
``tree``    attention of a tree of draft tokens over the caches
            (``sparse_attn_sharedkv_tree``).

The other fields are the shape: ``B`` sequences of ``q_lo .. q_hi`` new tokens,
the last ones of ``kv_lo .. kv_hi`` positions, drawn from ``lens`` (as the
trees are, so that both are part of the case); ``H`` heads of ``D`` channels,
of which the first ``qn`` (queries) and ``kn`` (KV rows) are normed and the last
``R`` rotated, in adjacent pairs or (``half``) channel i with i + R / 2; ``wide``
queries are a slice of a wider projection. Caches have blocks of ``bs`` rows
of type ``dt``; window ``win``, top-k ``K``, compressed ratio ``ratio``.

Activations and gradients are N(0, 1), norm weights 1 + N(0, 0.1), cache blocks a
random permutation, top-k positions distinct and uniform below a token's
causal threshold, -1 padded. ``table`` holds the (cos, sin) pairs of every
position in 32 bits, made once, as a program keeps it.
"""

import functools
import math
import random

import torch

own = False

DV = 512
DEV = "cuda"
EPS = 1e-6
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp8": torch.bfloat16}


def _rope(name, op="rope", B=1, q=(1, 1), kv=(1024, 8192), H=64, D=512, qn=512, kn=512, qw=False, R=64, half=False,
          inverse=False, wide=False, dt="bf16", lens=0):
    return {"name": name, "op": op, "B": B, "q_lo": q[0], "q_hi": q[1], "kv_lo": kv[0], "kv_hi": kv[1], "H": H, "D": D,
            "qn": qn, "kn": kn, "qw": qw, "R": R, "half": half, "inverse": inverse, "wide": wide, "dt": dt, "lens": lens}


def _append(name, B, q, kv, H=0, D=512, qn=512, kn=512, bs=64, half=False, dt="bf16", lens=0):
    return {"name": name, "op": "append", "B": B, "q_lo": q[0], "q_hi": q[1], "kv_lo": kv[0], "kv_hi": kv[1], "H": H,
            "D": D, "qn": qn, "kn": kn, "qw": False, "R": 64, "half": half, "inverse": False, "wide": False, "bs": bs,
            "dt": dt, "lens": lens}


def _tree(name, kind="scfa", B=1, H=64, D=576, K=512, ratio=4, win=128, bs=64, dt="bf16", q=(8, 8), kv=(2048, 2048),
          lens=0):
    return {"name": name, "op": "tree", "kind": kind, "B": B, "H": H, "D": D, "K": K if kind == "scfa" else 0,
            "ratio": ratio, "win": win, "bs": bs, "dt": dt, "q_lo": q[0], "q_hi": q[1], "kv_lo": kv[0], "kv_hi": kv[1],
            "lens": lens}


def listed():
    return [
        # a decode step of 32 sequences: every head of the queries and the KV row normed
        _rope("rope_step", B=32, q=(1, 1), kv=(1024, 32768), lens=11),
        # a prompt of 8192 tokens
        _rope("rope_8k", q=(8192, 8192), kv=(8192, 8192), lens=12),
        # packed prompts of odd lengths, few heads, latent rows, half-split pairs, queries sliced from a projection
        _rope("rope_packed", B=5, q=(300, 1900), kv=(2000, 9000), H=16, D=576, qn=576, kn=512, qw=True, half=True,
              wide=True, dt="fp16", lens=13),
        # the layer's backward on a sequence of 4096 tokens, latent rows with weights
        _rope("grad_4k", op="grad", q=(4096, 4096), kv=(4096, 4096), D=576, qn=512, kn=512, qw=True, lens=14),
        # the backward of short packed sequences, few heads
        _rope("grad_packed", op="grad", B=6, q=(40, 250), kv=(300, 4000), H=16, qw=True, dt="fp16", lens=15),
        # a decode step's rows and queries: one launch's latency
        _append("append_step", B=32, q=(1, 1), kv=(1024, 32768), H=64, lens=16),
        # prompt chunks of eight sequences quantised into fp8 rows
        _append("append_fp8_32k", B=8, q=(4096, 4096), kv=(4096, 16384), D=576, dt="fp8", lens=17),
        # draft tokens of sixteen sequences with their queries, 128 heads
        _append("append_drafts", B=16, q=(3, 60), kv=(1024, 65536), H=128, D=576, qn=0, dt="fp16", lens=18),
        # one user's tree of eight draft tokens, few heads: a call's latency
        _tree("tree_1x8", H=16, K=64, lens=19),
        # a serving batch's trees over mixed contexts
        _tree("tree_16x32", B=16, q=(20, 40), kv=(8192, 32768), lens=20),
        # large trees over long fp8 contexts, compressed 128 to 1, 128 heads
        _tree("tree_fp8_128k", B=4, H=128, K=1024, ratio=128, dt="fp8", q=(64, 64), kv=(131072, 131072), lens=21),
        # a window-only layer's trees
        _tree("tree_window", kind="swa", B=24, D=512, bs=128, dt="fp16", q=(12, 17), kv=(60, 8192), lens=22),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng: random.Random):
    limit = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        del c["name"]
        if _cost(c) <= limit:
            return c


def _draw(rng):
    lens = rng.randrange(1 << 20)
    what = rng.choices(["rope", "grad", "append", "tree"], [3, 2, 3, 4])[0]
    D = rng.choice([512, 512, 576])
    H = rng.choice([16, 32, 64, 64, 64, 128])
    half = rng.random() < 0.25
    dt = rng.choice(["bf16", "bf16", "fp16"])
    if what == "tree":
        kind = rng.choices(["scfa", "swa", "cfa"], [6, 2, 2])[0]
        if rng.random() < 0.35:
            dt, D = "fp8", 576
        hi = _log(rng, 2, 100)
        kv = _log(rng, max(hi, 200), 65536)
        return _tree("", kind=kind, B=_log(rng, 1, 32), H=H, D=D, K=rng.choice([64, 512, 512, 1024, rng.randrange(40, 1100)]),
                     ratio=rng.choice([4, 4, 8, 128]) if kind == "scfa" else 128,
                     win=rng.choice([128, 128, 128, 64, rng.randrange(1, 257)]), bs=rng.choice([64, 64, 128, 16]), dt=dt,
                     q=(max(1, hi // rng.choice([1, 2, 5])), hi), kv=(max(hi, kv // rng.choice([1, 4, 30])), kv), lens=lens)
    qn = rng.choice([D, D, 512, 0])
    hi = _log(rng, 1, 8192)
    B = rng.randrange(1, max(2, min(32, 16384 // hi) + 1))
    q = (max(1, hi // rng.choice([1, 2, 5])), hi)
    kv = (hi, hi + _log(rng, 64, 32768))
    if what == "append":
        fp8 = rng.random() < 0.4
        return _append("", B=B, q=q, kv=kv, H=rng.choice([0, H]), D=576 if fp8 else D, qn=min(qn, 576 if fp8 else D),
                       kn=rng.choice([512, 512, 0]), bs=rng.choice([64, 64, 128, 16]), half=half, dt="fp8" if fp8 else dt,
                       lens=lens)
    return _rope("", op=what, B=B, q=q, kv=kv, H=H, D=D, qn=qn, kn=rng.choice([512, 512, D]), qw=rng.random() < 0.4,
                 half=half, inverse=rng.random() < 0.2, wide=rng.random() < 0.3, dt=dt, lens=lens)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _lengths(c):
    r = random.Random(c["lens"])
    kv = [r.randint(c["kv_lo"], c["kv_hi"]) for _ in range(c["B"])]
    return [min(r.randint(c["q_lo"], c["q_hi"]), n) for n in kv], kv


def _trees(c):
    """Per sequence, each node's set of attended draft slots (its ancestors and
    itself) as an integer of bits."""
    r = random.Random(c["lens"] + 1)
    trees = []
    for n in _lengths(c)[0]:
        bits = [1]
        for s in range(1, n):
            bits.append(bits[r.randrange(max(0, s - 9), s)] | 1 << s)
        trees.append(bits)
    return trees


def _normal(shape, dtype, gen):
    out = torch.empty(shape, dtype=dtype, device=DEV)
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 27):
        part = flat[i:i + (1 << 27)]
        part.copy_(torch.randn(part.numel(), generator=gen, device=DEV))
    return out


def _fp8_rows(blocks, bs, gen):
    """Cache rows of 656 bytes: 512 e4m3 latent values, four scales, 64 bf16
    rope channels, from N(0, 1) channels (amax / 448 a 128-channel group)."""
    rows = torch.empty((blocks * bs, 656), dtype=torch.uint8, device=DEV)
    for i in range(0, rows.shape[0], 1 << 17):
        part = rows[i:i + (1 << 17)]
        n = part.shape[0]
        x = torch.randn((n, 576), generator=gen, device=DEV)
        lat = x[:, :512].reshape(n, 4, 128)
        scale = lat.abs().amax(-1) / 448.0
        part[:, :512] = (lat / scale[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).reshape(n, 512)
        part[:, 512:528] = scale.contiguous().view(torch.uint8)
        part[:, 528:] = x[:, 512:].to(torch.bfloat16).contiguous().view(torch.uint8)
    return rows.view(blocks, bs, 1, 656)


def _block_table(lens, bs, gen):
    """Shuffled block table of the sequences, -1 = unused, and the pool's blocks."""
    n = [max(1, -(-x // bs)) for x in lens]
    pool = sum(n) + 3
    perm = torch.randperm(pool, generator=gen, device=DEV).to(torch.int32)
    table = torch.full((len(n), max(n)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, m in enumerate(n):
        table[b, :m] = perm[at:at + m]
        at += m
    return table, pool


def _top_k(bounds, K, gen):
    """Per token: distinct positions, uniform below its threshold, -1 padded."""
    n = max(1, max(bounds))
    idx = torch.full((len(bounds), 1, K), -1, dtype=torch.int32, device=DEV)
    thr = torch.tensor(bounds, device=DEV)
    step = max(1, (1 << 25) // n)
    for i in range(0, len(bounds), step):
        t = thr[i:i + step, None]
        score = torch.rand((t.shape[0], n), generator=gen, device=DEV)
        score.masked_fill_(torch.arange(n, device=DEV)[None, :] >= t, -1.0)
        best, at = score.topk(min(K, n), dim=1)
        idx[i:i + step, 0, :at.shape[1]] = torch.where(best >= 0, at, -1).to(torch.int32)
    return idx


def _cu(lens):
    cu = [0]
    for m in lens:
        cu.append(cu[-1] + m)
    return cu


def _angles(rows, R):
    """(cos, sin) of position p and pair i at [p, i]: angle p / 10000^(2 i / R), in 64 bits."""
    f = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device=DEV) / R)
    a = torch.arange(rows, dtype=torch.float64, device=DEV)[:, None] * f
    return torch.stack([a.cos(), a.sin()], -1).to(torch.float32)


def _prologue(c, gen):
    """Inputs of rope, grad and append."""
    q_lens, kv_lens = _lengths(c)
    T, H, D, dt = sum(q_lens), c["H"], c["D"], _DT[c["dt"]]
    i32 = dict(dtype=torch.int32, device=DEV)
    pos = torch.cat([torch.arange(k - m, k, **i32) for m, k in zip(q_lens, kv_lens)])
    s = {"pos": pos, "table": _angles(c["kv_hi"], c["R"]), "q": None, "half": c["half"], "inverse": c["inverse"],
         "qn": c["qn"], "kn": c["kn"], "qw": None, "kw": None, "bs": c.get("bs"), "fp8": c["dt"] == "fp8"}
    if c["wide"]:   # one projection's output: the queries, then the KV row
        both = _normal((T, (H + 1) * D), dt, gen)
        s["q"], s["kv"] = both[:, :H * D].view(T, H, D), both[:, H * D:]
    else:
        s["kv"] = _normal((T, D), dt, gen)
        if H:
            s["q"] = _normal((T, H, D), dt, gen)
    if c["kn"]:
        s["kw"] = 1 + 0.1 * torch.randn(c["kn"], generator=gen, device=DEV)
    if c["qw"] and c["qn"]:
        s["qw"] = 1 + 0.1 * torch.randn(c["qn"], generator=gen, device=DEV)
    if c["op"] == "grad":
        s["dq_out"], s["dkv_out"] = _normal((T, H, D), dt, gen), _normal((T, D), dt, gen)
    if c["op"] == "append":
        s["bt"], pool = _block_table(kv_lens, c["bs"], gen)
        s["cu"], s["used"] = torch.tensor(_cu(q_lens), **i32), torch.tensor(kv_lens, **i32)
        fp8 = c["dt"] == "fp8"
        s["cache"] = torch.zeros((pool, c["bs"], 1, 656 if fp8 else D), dtype=torch.uint8 if fp8 else dt, device=DEV)
    return s


def _tree_inputs(c, gen):
    q_lens, kv_lens = _lengths(c)
    T, H, D, bs, dt = sum(q_lens), c["H"], c["D"], c["bs"], _DT[c["dt"]]
    rows = (lambda n: _fp8_rows(n, bs, gen)) if c["dt"] == "fp8" else (lambda n: _normal((n, bs, 1, D), dt, gen))
    words = -(-max(q_lens) // 64)
    flat = [(b >> 64 * w) & ((1 << 64) - 1) for t in _trees(c) for b in t for w in range(words)]
    mask = torch.tensor([x - (1 << 64) if x >> 63 else x for x in flat], dtype=torch.int64, device=DEV).view(T, words)
    # the dense compressed scenario reads its slot count from the lengths: host tensors
    i32 = dict(dtype=torch.int32, device="cpu" if c["kind"] == "cfa" else DEV)
    bt, pool = _block_table(kv_lens, bs, gen)
    kw = {"ori_kv": rows(pool), "ori_block_table": bt, "cu_seqlens_q": torch.tensor(_cu(q_lens), **i32),
          "seqused_kv": torch.tensor(kv_lens, **i32), "sinks": torch.randn(H, generator=gen, device=DEV),
          "softmax_scale": 1.0 / math.sqrt(D), "ori_win_left": c["win"] - 1}
    if c["kind"] != "swa":
        cmp_lens = [k // c["ratio"] for k in kv_lens]
        kw["cmp_block_table"], pool = _block_table(cmp_lens, bs, gen)
        kw["cmp_kv"] = rows(pool)
        kw["cmp_ratio"] = c["ratio"]
    if c["kind"] == "scfa":
        bounds = [(k - m + bin(b).count("1")) // c["ratio"] for m, k, t in zip(q_lens, kv_lens, _trees(c)) for b in t]
        kw["cmp_sparse_indices"] = _top_k(bounds, c["K"], gen)
    return {"q": _normal((T, H, D), dt, gen), "mask": mask, "kw": kw,
            "J": max(k // c["ratio"] for k in kv_lens) if c["kind"] == "cfa" else c["K"]}


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = _tree_inputs(case, gen) if case["op"] == "tree" else _prologue(case, gen)
    s["op"] = case["op"]
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _rotate(y, cs, half, inverse):
    """The last R channels of ``y`` rotated by the angles ``cs [..., R / 2, 2]``."""
    R = 2 * cs.shape[-2]
    cos, sin = cs[..., 0], -cs[..., 1] if inverse else cs[..., 1]
    head, tail = y[..., :y.shape[-1] - R], y[..., y.shape[-1] - R:]
    if half:
        a, b = tail[..., :R // 2], tail[..., R // 2:]
        return torch.cat([head, a * cos - b * sin, a * sin + b * cos], -1)
    a, b = tail[..., 0::2], tail[..., 1::2]
    return torch.cat([head, torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)], -1)


def _normed(x, n, w):
    """x in 32 bits with its first n channels normed and weighted."""
    x = x.float()
    if n == 0:
        return x
    h = x[..., :n]
    h = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
    return torch.cat([h if w is None else h * w, x[..., n:]], -1)


def _normed_grad(x, u, n, w):
    """Gradients of x and w for a gradient u of _normed(x, n, w)."""
    if n == 0:
        return u, None
    x = x[..., :n].float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    xh, un = x * r, u[..., :n]
    g = un if w is None else un * w
    dx = r * (g - xh * (g * xh).mean(-1, keepdim=True))
    dw = None if w is None else (un * xh).reshape(-1, n).sum(0)
    return torch.cat([dx, u[..., n:]], -1), dw


def _plain_rope(s):
    cs = s["table"][s["pos"]]
    dt = s["kv"].dtype
    kv = _rotate(_normed(s["kv"], s["kn"], s["kw"]), cs, s["half"], s["inverse"])
    q = None if s["q"] is None else _rotate(_normed(s["q"], s["qn"], s["qw"]), cs[:, None], s["half"], s["inverse"]).to(dt)
    return q, kv


def _plain_grad(s):
    cs = s["table"][s["pos"]]
    dt = s["q"].dtype
    dq, dqw = _normed_grad(s["q"], _rotate(s["dq_out"].float(), cs[:, None], s["half"], not s["inverse"]), s["qn"], s["qw"])
    dkv, dkw = _normed_grad(s["kv"], _rotate(s["dkv_out"].float(), cs, s["half"], not s["inverse"]), s["kn"], s["kw"])
    return {"dq": dq.to(dt), "dkv": dkv.to(dt), "dq_weight": dqw, "dkv_weight": dkw}


def _sequences(cu, T):
    """Each token's sequence, and its place in it."""
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(cu, t, right=True) - 1
    return b, t - cu[b]


def _plain_append(s):
    q, kv = _plain_rope(s)
    b, i = _sequences(s["cu"].long(), kv.shape[0])
    at = s["used"].long()[b] - (s["cu"][1:] - s["cu"][:-1]).long()[b] + i
    flat = s["bt"].long()[b, at // s["bs"]] * s["bs"] + at % s["bs"]
    rows = s["cache"].view(-1, s["cache"].shape[-1])
    if s["fp8"]:
        lat = kv[:, :512].reshape(-1, 4, 128)
        amax = lat.abs().amax(-1)
        scale = torch.where(amax > 0, amax / 448.0, 1.0)
        code = (lat / scale[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).reshape(-1, 512)
        kv = torch.cat([code, scale.view(torch.uint8), kv[:, 512:].to(torch.bfloat16).view(torch.uint8)], 1)
    rows[flat] = kv.to(rows.dtype)
    return q


def _rows(cache, flat, f):
    """Cache rows at flat indices, in the type f: fp8 rows as the values they hold."""
    r = cache.view(-1, cache.shape[-1])[flat]
    if cache.dtype is not torch.uint8:
        return r.to(f)
    lat = r[..., :512].view(torch.float8_e4m3fn).to(f).unflatten(-1, (4, 128))
    scale = r[..., 512:528].contiguous().view(torch.float32).to(f)
    return torch.cat([(lat * scale[..., None]).flatten(-2), r[..., 528:].contiguous().view(torch.bfloat16).to(f)], -1)


def _plain_tree(s):
    q, kw = s["q"], s["kw"]
    T, H, D = q.shape
    win, bs = kw["ori_win_left"] + 1, kw["ori_kv"].shape[1]
    cu, used = kw["cu_seqlens_q"].to(DEV).long(), kw["seqused_kv"].to(DEV).long()
    b, _ = _sequences(cu, T)
    aq = (cu[1:] - cu[:-1])[b][:, None]
    n = used[b][:, None] - aq                                          # committed rows
    j = torch.arange(64 * s["mask"].shape[1], device=DEV)
    bits = ((s["mask"][:, j // 64] >> (j % 64)) & 1).bool() & (j < aq) & (n + j >= 0)
    count = bits.sum(1, keepdim=True)
    near = bits.flip(1).long().cumsum(1).flip(1) <= win                # the last `win` of them
    i = torch.arange(win, device=DEV)
    at = torch.cat([n - 1 - i, n + j], 1)
    ok = torch.cat([(i < win - count) & (n - 1 - i >= 0), bits & near], 1)
    at = at.masked_fill(~ok, 0)
    page = kw["ori_block_table"].long()[b[:, None], at // bs] * bs + at % bs
    keys = [_rows(kw["ori_kv"], page.masked_fill(~ok, 0), torch.float32)]
    valid = [ok]
    if "cmp_kv" in kw:
        at = kw["cmp_sparse_indices"].view(T, -1).long() if "cmp_sparse_indices" in kw else torch.arange(
            s["J"], device=DEV).expand(T, -1)
        ok = (at >= 0) & (at < (n.clamp(min=0) + count) // kw["cmp_ratio"])
        at = at.masked_fill(~ok, 0)
        cbs = kw["cmp_kv"].shape[1]
        page = kw["cmp_block_table"].long()[b[:, None], at // cbs] * cbs + at % cbs
        keys.append(_rows(kw["cmp_kv"], page.masked_fill(~ok, 0), torch.float32))
        valid.append(ok)
    k, ok = torch.cat(keys, 1), torch.cat(valid, 1)
    x = torch.matmul(q.float(), k.transpose(1, 2).contiguous()) * kw["softmax_scale"]
    x = x.masked_fill(~ok[:, None], -math.inf)
    sink = kw["sinks"][None, :, None]
    m = torch.maximum(x.amax(2, keepdim=True), sink)
    p = torch.exp(x - m)
    l = p.sum(2, keepdim=True) + torch.exp(sink - m)
    out = torch.matmul(p, k[..., :DV].contiguous()) / l
    return {"out": out.to(q.dtype), "lse": (m + torch.log(l))[..., 0]}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _cache_values(cache):
    """The cache as values: of fp8 rows the latent values, their scales and the rope channels."""
    if cache.dtype is not torch.uint8:
        return {"cache": cache}
    return {"latent": cache[..., :512].view(torch.float8_e4m3fn), "scale": cache[..., 512:528].view(torch.float32),
            "rope": cache[..., 528:].view(torch.bfloat16)}


def _own_kwargs(s):
    return dict(positions=s["pos"], table=s["table"], q_norm_dim=s["qn"], kv_norm_dim=s["kn"], q_weight=s["qw"],
                kv_weight=s["kw"], eps=EPS, interleaved=not s["half"], inverse=s["inverse"])


@functools.cache
def _entries():
    """The framework's entry points."""
    from dsv4_amd.api import sparse_attn_sharedkv_tree
    from dsv4_amd.cache import append_kv_cache
    from dsv4_amd.rope import norm_rope, norm_rope_backward
    return norm_rope, norm_rope_backward, append_kv_cache, sparse_attn_sharedkv_tree


def _run_own(s):
    norm_rope, norm_rope_backward, append_kv_cache, sparse_attn_sharedkv_tree = _entries()
    op = s["op"]
    if op == "tree":
        out, lse = sparse_attn_sharedkv_tree(s["q"], tree_mask=s["mask"], return_softmax_lse=True, **s["kw"])
        return {"out": out, "lse": lse}
    if op == "append":
        q = append_kv_cache(s["kv"], s["cache"], s["bt"], s["cu"], s["used"], table=s["table"], norm_dim=s["kn"],
                            weight=s["kw"], eps=EPS, interleaved=not s["half"], q=s["q"], q_norm_dim=s["qn"])
        return {"q": q, **_cache_values(s["cache"])}
    if op == "rope":
        q, kv = norm_rope(s["q"], s["kv"], **_own_kwargs(s))
        return {"q": q, "kv": kv}
    dq, dkv, dqw, dkw = norm_rope_backward(s["dq_out"], s["q"], s["dkv_out"], s["kv"], **_own_kwargs(s))
    return {"dq": dq, "dkv": dkv, "dq_weight": dqw, "dkv_weight": dkw}


def run(s):
    if own:
        return _run_own(s)
    op = s["op"]
    if op == "tree":
        return _plain_tree(s)
    if op == "append":
        return {"q": _plain_append(s), **_cache_values(s["cache"])}
    if op == "rope":
        q, kv = _plain_rope(s)
        return {"q": q, "kv": kv.to(s["kv"].dtype)}
    return _plain_grad(s)


# ---------------------------------------------------------------------------
# work, 64-bit results
# ---------------------------------------------------------------------------

def work(case):
    c = case
    q_lens, kv_lens = _lengths(c)
    T, H, D = sum(q_lens), c["H"], c["D"]
    row = 656 if c["dt"] == "fp8" else 2 * D
    if c["op"] != "tree":
        rows = T * (H + 1)
        small = T * (4 + 4 * c["R"]) + 4 * c["kn"] + 4 * c["qn"] * c["qw"]
        if c["op"] == "grad":
            return {"bytes": rows * 6 * D + small + 4 * c["kn"] + 4 * c["qn"] * c["qw"], "flops": rows * (14 * D + 3 * c["R"])}
        out = T * (2 * H * D + (row if c["op"] == "append" else 2 * D))
        return {"bytes": rows * 2 * D + out + small, "flops": rows * (5 * D + 3 * c["R"])}
    pairs = rows = 0
    for ql, kl, tree in zip(q_lens, kv_lens, _trees(c)):
        n, cmp_pairs, reach = kl - ql, 0, 0
        for bits in tree:
            count = bin(bits).count("1")
            pairs += min(n + count, c["win"])
            thr = 0 if c["kind"] == "swa" else (n + count) // c["ratio"]
            thr = min(thr, c["K"]) if c["kind"] == "scfa" else thr
            cmp_pairs += thr
            reach = max(reach, thr)
        pairs += cmp_pairs
        rows += ql + min(n, c["win"] - 1) + (reach if c["kind"] == "cfa" else min(cmp_pairs, kl // c["ratio"]))
    return {"bytes": T * (H * (2 * D + 2 * DV + 4) + 4 * c["K"] + 8 * -(-max(q_lens) // 64)) + rows * row,
            "flops": pairs * H * 2 * (D + DV)}


def _turn64(y, cs, half, inverse):
    """``y`` in 64 bits, its last channels rotated as complex numbers by the table's."""
    R = 2 * cs.shape[-2]
    z = torch.view_as_complex(cs.double())
    z = z.conj() if inverse else z
    t = y[..., y.shape[-1] - R:]
    t = torch.stack([t[..., :R // 2], t[..., R // 2:]], -1) if half else t.unflatten(-1, (R // 2, 2))
    t = torch.view_as_real(torch.view_as_complex(t.contiguous()) * z)
    t = torch.cat([t[..., 0], t[..., 1]], -1) if half else t.flatten(-2)
    return torch.cat([y[..., :y.shape[-1] - R], t], -1)


def _heads64(x, n, w, cs, half, inverse):
    if n:
        rms = (x[..., :n].square().sum(-1, keepdim=True) / n + EPS).sqrt()
        first = x[..., :n] / rms
        x = torch.cat([first if w is None else first * w, x[..., n:]], -1)
    return _turn64(x, cs, half, inverse)


def _exact_prologue(c, s):
    cs = s["table"][s["pos"].long()]
    leaf = {"q": s["q"], "kv": s["kv"], "q_weight": s["qw"], "kv_weight": s["kw"]}
    leaf = {k: v.double().requires_grad_(c["op"] == "grad") for k, v in leaf.items() if v is not None}
    kv = _heads64(leaf["kv"], c["kn"], leaf.get("kv_weight"), cs, c["half"], c["inverse"])
    q = _heads64(leaf["q"], c["qn"], leaf.get("q_weight"), cs[:, None], c["half"], c["inverse"]) if "q" in leaf else None
    if c["op"] == "rope":
        return {"q": q, "kv": kv}
    if c["op"] == "grad":
        got = dict(zip(leaf, torch.autograd.grad([q, kv], list(leaf.values()), [s["dq_out"].double(), s["dkv_out"].double()])))
        return {"d" + k: got.get(k) for k in ("q", "kv", "q_weight", "kv_weight")}
    q_lens, kv_lens = _lengths(c)
    cache = torch.zeros((*s["cache"].shape[:2], c["D"]), dtype=torch.float64, device=DEV)
    t = 0
    for b, (m, k) in enumerate(zip(q_lens, kv_lens)):
        at = torch.arange(k - m, k, device=DEV)
        cache[s["bt"][b].long()[at // c["bs"]], at % c["bs"]] = kv[t:t + m]
        t += m
    if c["dt"] != "fp8":
        return {"q": q, "cache": cache.unsqueeze(2)}
    lat = cache[..., :512].unflatten(-1, (4, 128))
    scale = lat.abs().amax(-1) / 448
    written = torch.zeros(cache.shape[:2], dtype=torch.bool, device=DEV)
    t = 0
    for b, (m, k) in enumerate(zip(q_lens, kv_lens)):
        at = torch.arange(k - m, k, device=DEV)
        written[s["bt"][b].long()[at // c["bs"]], at % c["bs"]] = True
    scale = torch.where(scale > 0, scale, written[..., None].double())
    lat = (lat / torch.where(scale > 0, scale, 1.0)[..., None]).flatten(-2)
    return {"q": q, "latent": lat.unsqueeze(2), "scale": scale.unsqueeze(2), "rope": cache[..., 512:].unsqueeze(2)}


def _exact_tree(c, s):
    q, kw = s["q"], s["kw"]
    out = torch.empty((*q.shape[:2], DV), dtype=torch.float64, device=DEV)
    lse = torch.empty(q.shape[:2], dtype=torch.float64, device=DEV)
    q_lens, kv_lens = _lengths(c)
    t = 0
    for b, (m, k, tree) in enumerate(zip(q_lens, kv_lens, _trees(c))):
        n, table = k - m, kw["ori_block_table"][b].long()
        line = list(range(max(0, n - c["win"]), n))                    # the last committed positions
        for bits in tree:
            path = (line + [n + j for j in range(m) if bits >> j & 1])[-c["win"]:]
            at = torch.tensor(path, device=DEV)
            keys = [_rows(kw["ori_kv"], table[at // c["bs"]] * c["bs"] + at % c["bs"], torch.float64)]
            if c["kind"] != "swa":
                thr = (n + bin(bits).count("1")) // c["ratio"]
                at = kw["cmp_sparse_indices"][t, 0].long() if c["kind"] == "scfa" else torch.arange(s["J"], device=DEV)
                at = at[(at >= 0) & (at < thr)]
                page = kw["cmp_block_table"][b].long()[at // c["bs"]] * c["bs"] + at % c["bs"]
                keys.append(_rows(kw["cmp_kv"], page, torch.float64))
            kk = torch.cat(keys)
            x = torch.cat([torch.matmul(q[t].double(), kk.t().contiguous()) * kw["softmax_scale"],
                           kw["sinks"].double()[:, None]], 1)
            lse[t] = torch.logsumexp(x, 1)
            out[t] = torch.matmul(torch.exp(x[:, :-1] - lse[t][:, None]), kk[:, :DV].contiguous())
            t += 1
    return {"out": out, "lse": lse}


def exact(case, seed):
    if case["op"] == "tree" and sum(_lengths(case)[0]) > 4000:
        return None   # token by token: beyond some 20 seconds
    s = prepare(case, seed)
    return _exact_tree(case, s) if case["op"] == "tree" else _exact_prologue(case, s)

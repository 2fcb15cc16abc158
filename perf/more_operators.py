"""Performance cases of caches that stay bounded while a sequence grows without end:
attention whose first rows stay visible beside the window, its gradients, the weight
that attention gives each cache row, and the eviction of the rows that got least.

A case is a dict of plain values. ``op`` is the call:

``first``    attention over the window, the ``F`` first rows and the compressed rows
             (``sparse_attn_sharedkv_first``);
``grad``     its backward (``sparse_attn_sharedkv_first_backward``): the gradients of
             queries, cache rows (in the caches' type, as a step takes them) and sinks;
``weights``  the attention weight of each cache row, the mean over the heads, added up
             over a call's tokens (``add_row_weights``);
``evict``    all but ``budget`` rows of each sequence leave its cache, those with the
             least weight (``evict_kv_cache``).

The other fields are the shape: ``B`` sequences of ``q_lo .. q_hi`` new tokens, the last
ones of ``kv_lo .. kv_hi`` rows, drawn from ``lens``; ``H`` heads of ``D`` channels;
``kind``: the window alone (``swa``), with all compressed rows (``cfa``) or with a
top-k ``K`` of them (``scfa``), ``ratio`` positions to one; window ``win`` (0: every
row). Caches have blocks of ``bs`` rows of type ``dt``; a block that holds no row of the
window or of the first ones is not there. ``first`` and ``recent`` rows are kept from
eviction.

Activations and gradients are N(0, 1), cache blocks a random permutation, top-k
positions distinct and uniform below a token's causal threshold, -1 padded; the
weights that an eviction meets are sums of the kind that attention leaves: a few rows
hold most, many hold nothing.
"""

import functools
import math
import random

import torch

own = False

DV = 512
DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp8": torch.bfloat16}


def _attn(name, op, kind="swa", B=1, H=64, D=576, K=512, ratio=4, win=128, F=4, bs=64, dt="bf16", q=(1, 1),
          kv=(2048, 2048), lens=0):
    return {"name": name, "op": op, "kind": kind, "B": B, "H": H, "D": D, "K": K if kind == "scfa" else 0,
            "ratio": ratio, "win": win, "F": F, "bs": bs, "dt": dt, "q_lo": q[0], "q_hi": q[1], "kv_lo": kv[0],
            "kv_hi": kv[1], "lens": lens}


def _evict(name, B, kv, budget, first=4, recent=128, D=576, bs=64, dt="bf16", lens=0):
    return {"name": name, "op": "evict", "B": B, "D": D, "bs": bs, "dt": dt, "kv_lo": kv[0], "kv_hi": kv[1],
            "budget": budget, "first": first, "recent": recent, "lens": lens}


def listed():
    return [
        # one user's next token in a window-only layer, few heads: a call's latency
        _attn("first_1", "first", H=16, D=512, bs=128, kv=(5000, 5000), lens=31),
        # a decode step of 32 sequences over mixed contexts
        _attn("first_step", "first", kind="scfa", B=32, kv=(1024, 32768), lens=32),
        # a prompt of 8192 tokens in a window-only layer
        _attn("first_8k", "first", D=512, q=(8192, 8192), kv=(8192, 8192), lens=33),
        # prompt chunks of eight long sequences, 128 heads, fp8 rows compressed 128 to 1
        _attn("first_fp8", "first", kind="scfa", B=8, H=128, K=1024, ratio=128, F=8, dt="fp8", q=(60, 200),
              kv=(131072, 131072), lens=34),
        # the layer's backward on a sequence of 4096 tokens
        _attn("grad_4k", "grad", q=(4096, 4096), kv=(4096, 4096), lens=35),
        # the backward of short packed sequences with compressed rows
        _attn("grad_packed", "grad", kind="scfa", B=6, H=32, D=512, K=64, F=16, dt="fp16", q=(70, 250), kv=(300, 4000),
              lens=36),
        # the weights of a decode step of 32 sequences over bounded caches
        _attn("weights_step", "weights", B=32, win=0, F=0, kv=(1900, 2112), lens=37),
        # the last 64 tokens of two long prompts over all their rows, before the first eviction
        _attn("weights_prompt", "weights", B=2, D=512, win=0, F=0, q=(64, 64), kv=(20000, 32768), lens=38),
        # drafted tokens of sixteen sequences: window, first and compressed rows, fp8
        _attn("weights_topk", "weights", kind="scfa", B=16, dt="fp8", q=(1, 4), kv=(8192, 65536), lens=39),
        # one short sequence gives up a few rows: a call's latency
        _evict("evict_1", 1, (300, 300), 256, recent=64, D=512, bs=128, dt="fp16", lens=40),
        # 32 sequences give up their last block's worth of rows between two decode steps
        _evict("evict_step", 32, (2049, 2112), 2048, lens=41),
        # four long fp8 prompts cut down after the prefill
        _evict("evict_prompt", 4, (20000, 32768), 4096, recent=512, dt="fp8", lens=42),
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
    op = rng.choices(["first", "grad", "weights", "evict"], [3, 2, 3, 2])[0]
    D = rng.choice([512, 512, 576])
    H = rng.choice([16, 32, 64, 64, 64, 128])
    bs = rng.choice([64, 64, 128, 16])
    dt = rng.choice(["bf16", "bf16", "fp16"])
    if op != "grad" and rng.random() < 0.3:
        dt, D = "fp8", 576
    if op == "evict":
        hi = _log(rng, 64, 40000)
        lo = max(2, hi // rng.choice([1, 1, 2, 5]))
        budget = max(1, min(lo - rng.choice([1, 1, 17, 64, 300]), hi // rng.choice([1, 1, 2, 8])))
        first = min(budget // 2, rng.choice([0, 1, 4, 4, 16]))
        return _evict("", _log(rng, 1, max(1, min(32, 200000 // hi))), (lo, hi), budget, first,
                      min(budget - first, rng.choice([0, 1, 64, 128, 512])), D, bs, dt, lens)
    kind = rng.choices(["scfa", "swa", "cfa"], [4, 5, 2])[0]
    F = rng.choice([1, 4, 4, 4, 8, 16, 64])
    win = rng.choice([128, 128, 128, 64, rng.randrange(1, 257)])
    if op == "weights" and kind == "swa" and rng.random() < 0.7:   # every row: a bounded cache, or a prompt's end
        win = F = 0
    most = 8192 if op == "first" and kind == "swa" else 4096 if kind == "swa" and win else 64 if not win else 1500
    hi = _log(rng, 64 if op == "grad" and rng.random() < 0.7 else 1, most)
    B = rng.randrange(1, max(2, min(32, most // hi) + 1))
    kv = hi + _log(rng, 64, 32768 if op != "grad" else 4096)
    if not win:
        B = max(1, min(B, 60000 // kv))
    return _attn("", op, kind=kind, B=B, H=H, D=D, K=rng.choice([64, 512, 512, rng.randrange(40, 1100)]),
                 ratio=rng.choice([4, 4, 8, 128]) if kind == "scfa" else 128, win=win, F=F, bs=bs, dt=dt,
                 q=(max(1, hi // rng.choice([1, 2, 5])), hi), kv=(max(hi, kv // rng.choice([1, 2, 10])), kv), lens=lens)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _lengths(c):
    r = random.Random(c["lens"])
    kv = [r.randint(c["kv_lo"], c["kv_hi"]) for _ in range(c["B"])]
    return [min(r.randint(c["q_lo"], c["q_hi"]), n) for n in kv] if "q_lo" in c else None, kv


def _normal(shape, dtype, gen):
    out = torch.empty(shape, dtype=dtype, device=DEV)
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 27):
        part = flat[i:i + (1 << 27)]
        part.copy_(torch.randn(part.numel(), generator=gen, device=DEV))
    return out


def _fp8_rows(blocks, bs, gen):
    """Cache rows of 656 bytes: 512 e4m3 latent values, four scales, 64 bf16 rope
    channels, from N(0, 1) channels (amax / 448 a 128-channel group)."""
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


def _cache(c, blocks, gen):
    if c["dt"] == "fp8":
        return _fp8_rows(blocks, c["bs"], gen)
    return _normal((blocks, c["bs"], 1, c["D"]), _DT[c["dt"]], gen)


def _block_table(lens, bs, gen, first=0, lows=None):
    """Shuffled block table of the sequences and the pool's blocks: those that hold
    rows below ``first`` or from ``lows`` on; -1 = not there."""
    n = max(1, -(-max(lens) // bs))
    blk = torch.arange(n, device=DEV)[None]
    there = blk * bs < torch.tensor(lens, device=DEV)[:, None]
    if lows is not None:
        there &= (blk * bs < first) | (blk >= torch.tensor(lows, device=DEV)[:, None] // bs)
    at = there.view(-1).cumsum(0).view_as(there) - 1
    pool = int(there.sum()) + 3
    perm = torch.randperm(pool, generator=gen, device=DEV)
    return torch.where(there, perm[at.clamp(min=0)], -1).to(torch.int32), pool


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


def _attn_inputs(c, gen):
    q_lens, kv_lens = _lengths(c)
    T, H, D, bs, dt = sum(q_lens), c["H"], c["D"], c["bs"], _DT[c["dt"]]
    # the dense compressed scenario reads its slot count from the lengths: host tensors
    i32 = dict(dtype=torch.int32, device="cpu" if c["kind"] == "cfa" else DEV)
    win = c["win"] or max(kv_lens)
    bt, pool = _block_table(kv_lens, bs, gen, c["F"], [max(0, k - m - win + 1) for m, k in zip(q_lens, kv_lens)])
    kw = {"ori_kv": _cache(c, pool, gen), "ori_block_table": bt, "cu_seqlens_q": torch.tensor(_cu(q_lens), **i32),
          "seqused_kv": torch.tensor(kv_lens, **i32), "softmax_scale": 1.0 / math.sqrt(D), "ori_win_left": win - 1,
          "ori_first": c["F"]}
    if c["kind"] != "swa":
        cmp_lens = [k // c["ratio"] for k in kv_lens]
        kw["cmp_block_table"], pool = _block_table(cmp_lens, bs, gen)
        kw["cmp_kv"] = _cache(c, pool, gen)
        kw["cmp_ratio"] = c["ratio"]
    if c["kind"] == "scfa":
        kw["cmp_sparse_indices"] = _top_k([(k - m + i + 1) // c["ratio"] for m, k in zip(q_lens, kv_lens) for i in range(m)],
                                          c["K"], gen)
    s = {"q": _normal((T, H, D), dt, gen), "sinks": torch.randn(H, generator=gen, device=DEV), "kw": kw, "full": not c["win"],
         "J": max(k // c["ratio"] for k in kv_lens) if c["kind"] == "cfa" else c["K"], "m": max(q_lens), "n": max(kv_lens)}
    if c["op"] == "first":
        return s
    if c["op"] == "grad":
        s["out"], s["lse"] = _plain_first(s).values()
        s["dout"] = _normal((T, H, DV), dt, gen)
        return s
    s["lse"] = _dense_lse(s) if s["full"] else _plain_first(s)["lse"]
    f64 = dict(dtype=torch.float64, device=DEV)
    s["ori_weights"] = torch.zeros((c["B"], bt.shape[1] * bs), **f64)
    if c["kind"] != "swa":
        s["cmp_weights"] = torch.zeros((c["B"], kw["cmp_block_table"].shape[1] * bs), **f64)
    return s


def _evict_inputs(c, gen):
    _, kv_lens = _lengths(c)
    bt, pool = _block_table(kv_lens, c["bs"], gen)
    n = torch.tensor(kv_lens, device=DEV)
    R = bt.shape[1] * c["bs"]
    u = torch.rand((c["B"], R), generator=gen, device=DEV, dtype=torch.float64)
    w = torch.floor(torch.exp(-9 * u) * torch.rand((c["B"], R), generator=gen, device=DEV) * 2.0 ** 36) * 2.0 ** -36
    w.masked_fill_((u > 0.75) | (torch.arange(R, device=DEV) >= n[:, None]), 0.0)
    return {"cache": _cache(c, pool, gen), "bt": bt, "used": n.to(torch.int32), "met": w, "weights": w.clone(),
            "budget": c["budget"], "first": c["first"], "recent": c["recent"]}


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = _evict_inputs(case, gen) if case["op"] == "evict" else _attn_inputs(case, gen)
    s["op"] = case["op"]
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _sequences(cu, T):
    """Each token's sequence, and its place in it."""
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(cu, t, right=True) - 1
    return b, t - cu[b]


def _rows(cache, flat, f):
    """Cache rows at flat indices, in the type f: fp8 rows as the values they hold."""
    r = cache.view(-1, cache.shape[-1])[flat]
    if cache.dtype is not torch.uint8:
        return r.to(f)
    lat = r[..., :512].view(torch.float8_e4m3fn).to(f).unflatten(-1, (4, 128))
    scale = r[..., 512:528].contiguous().view(torch.float32).to(f)
    return torch.cat([(lat * scale[..., None]).flatten(-2), r[..., 528:].contiguous().view(torch.bfloat16).to(f)], -1)


def _pages(table, b, at, ok, bs):
    """Flat cache rows of positions ``at`` of sequences ``b``; masked ones: any row."""
    at = at.masked_fill(~ok, 0)
    page = table.long()[b[:, None], at // bs]
    ok = ok & (page >= 0)
    return (page * bs + at % bs).masked_fill(~ok, 0), ok


def _slots(s):
    """Each token's keys: per cache the sequence of each token, the positions, their
    flat rows and which of them count."""
    kw, T = s["kw"], s["q"].shape[0]
    cu, used = kw["cu_seqlens_q"].to(DEV).long(), kw["seqused_kv"].to(DEV).long()
    b, i = _sequences(cu, T)
    pos = (used - (cu[1:] - cu[:-1]))[b] + i
    low = (pos - kw["ori_win_left"]).clamp(min=0)[:, None]
    f = torch.arange(kw["ori_first"], device=DEV).expand(T, -1)
    w = low + torch.arange(kw["ori_win_left"] + 1, device=DEV)
    at, ok = torch.cat([f, w], 1), torch.cat([f < low, w <= pos[:, None]], 1)
    got = [(b, at, *_pages(kw["ori_block_table"], b, at, ok, kw["ori_kv"].shape[1]))]
    if "cmp_kv" in kw:
        at = kw["cmp_sparse_indices"].view(T, -1).long() if "cmp_sparse_indices" in kw else torch.arange(
            s["J"], device=DEV).expand(T, -1)
        ok = (at >= 0) & (at < ((pos + 1) // kw["cmp_ratio"])[:, None])
        got.append((b, at, *_pages(kw["cmp_block_table"], b, at, ok, kw["cmp_kv"].shape[1])))
    return got


def _keys(s, slots):
    kw = s["kw"]
    k = torch.cat([_rows(cache, x[2], torch.float32) for cache, x in zip((kw["ori_kv"], kw.get("cmp_kv")), slots)], 1)
    return k, torch.cat([x[3] for x in slots], 1)


def _scores(s, k, ok):
    x = torch.matmul(s["q"].float(), k.transpose(1, 2).contiguous()) * s["kw"]["softmax_scale"]
    return x.masked_fill(~ok[:, None], -math.inf)


def _plain_first(s):
    k, ok = _keys(s, _slots(s))
    x = _scores(s, k, ok)
    sink = s["sinks"][None, :, None]
    m = torch.maximum(x.amax(2, keepdim=True), sink)
    p = torch.exp(x - m)
    l = p.sum(2, keepdim=True) + torch.exp(sink - m)
    out = torch.matmul(p, k[..., :DV].contiguous()) / l
    return {"out": out.to(s["q"].dtype), "lse": (m + torch.log(l))[..., 0]}


def _plain_grad(s):
    kw, T = s["kw"], s["q"].shape[0]
    slots = _slots(s)
    k, ok = _keys(s, slots)
    p = torch.exp(_scores(s, k, ok) - s["lse"][..., None])
    dout = s["dout"].float()
    delta = (dout * s["out"].float()).sum(-1)
    ds = p * (torch.matmul(dout, k[..., :DV].transpose(1, 2).contiguous()) - delta[..., None]) * kw["softmax_scale"]
    rows = torch.matmul(ds.transpose(1, 2).contiguous(), s["q"].float())
    rows[..., :DV] += torch.matmul(p.transpose(1, 2).contiguous(), dout)
    n = slots[0][1].shape[1]
    got = {"dq": torch.matmul(ds, k).to(s["q"].dtype), "d_sinks": -(torch.exp(s["sinks"] - s["lse"]) * delta).sum(0),
           "d_ori_kv": _row_sums(kw["ori_kv"], slots[0], rows[:, :n])}
    if "cmp_kv" in kw:
        got["d_cmp_kv"] = _row_sums(kw["cmp_kv"], slots[1], rows[:, n:])
    return got


def _row_sums(cache, slot, rows):
    """Gradients of cache rows summed over the tokens' slots, in the cache's type."""
    d = torch.zeros(cache.shape, dtype=torch.float32, device=DEV)
    d.view(-1, d.shape[-1]).index_add_(0, slot[2].reshape(-1), rows.reshape(-1, rows.shape[-1]))
    return d.to(cache.dtype)


def _padded(s):
    """The sequences' tokens side by side [B, m] (-1: none) and their positions."""
    kw = s["kw"]
    cu, used = kw["cu_seqlens_q"].to(DEV).long(), kw["seqused_kv"].to(DEV).long()
    i = torch.arange(s["m"], device=DEV)
    there = i < (cu[1:] - cu[:-1])[:, None]
    return torch.where(there, cu[:-1, None] + i, -1), (used - (cu[1:] - cu[:-1]))[:, None] + i


def _dense_scores(s):
    """Scores of every token and row of each sequence, [B, m, H, n]; -inf where none."""
    kw = s["kw"]
    t, pos = _padded(s)
    B, n, H = t.shape[0], s["n"], s["q"].shape[1]
    at = torch.arange(n, device=DEV).expand(B, -1)
    flat, ok = _pages(kw["ori_block_table"], torch.arange(B, device=DEV), at, at < kw["seqused_kv"].to(DEV)[:, None],
                      kw["ori_kv"].shape[1])
    k = _rows(kw["ori_kv"], flat, torch.float32)
    x = torch.matmul(s["q"][t.clamp(min=0)].float().flatten(1, 2), k.transpose(1, 2).contiguous()) * kw["softmax_scale"]
    x = x.view(B, -1, H, n)
    return x.masked_fill_(~(ok[:, None] & (at[:, None] <= pos[..., None]) & (t >= 0)[..., None])[:, :, None], -math.inf), t


def _dense_lse(s):
    x, t = _dense_scores(s)
    sink = s["sinks"][:, None]
    m = torch.maximum(x.amax(3, keepdim=True), sink)
    lse = (m + torch.log(torch.exp(x - m).sum(3, keepdim=True) + torch.exp(sink - m)))[..., 0]
    return lse[t >= 0]


def _plain_weights(s):
    if s["full"]:
        x, t = _dense_scores(s)
        p = x.sub_(s["lse"][t.clamp(min=0)][..., None]).exp_()
        s["ori_weights"][:, :s["n"]] += p.sum((1, 2)) / p.shape[2]
        return
    slots = _slots(s)
    p = torch.exp(_scores(s, *_keys(s, slots)) - s["lse"][..., None]).mean(1).double()
    n = slots[0][1].shape[1]
    _add(s["ori_weights"], slots[0], p[:, :n])
    if "cmp_weights" in s:
        _add(s["cmp_weights"], slots[1], p[:, n:])


def _add(weights, slot, p):
    b, at, _, ok = slot
    place = (b[:, None] * weights.shape[1] + at).masked_fill(~ok, 0)
    weights.view(-1).index_add_(0, place.view(-1), p.masked_fill(~ok, 0.0).reshape(-1))


def _plain_evict(s):
    w, bt, bs, used = s["weights"], s["bt"].long(), s["cache"].shape[1], s["used"].long()[:, None]
    B, R = w.shape
    at = torch.arange(R, device=DEV).expand(B, -1)
    key = w.masked_fill((at < s["first"]) | (at >= used - s["recent"]), math.inf).masked_fill(at >= used, -math.inf)
    order = key.sort(dim=1, descending=True, stable=True)[1]
    place = torch.empty_like(order).scatter_(1, order, at)
    stays = (place < s["budget"]) & (at < used)
    used2 = used.clamp(max=s["budget"])
    kept = torch.where(stays, at, R).sort(dim=1)[0]
    kept = torch.nn.functional.pad(kept, (0, max(0, s["budget"] - R)), value=R)[:, :s["budget"]]
    new = torch.arange(kept.shape[1], device=DEV).expand(B, -1)
    ok = kept < R
    b = torch.arange(B, device=DEV)
    src = _pages(bt, b, kept, ok, bs)[0][ok]
    dst = _pages(bt, b, new, ok, bs)[0][ok]
    rows = s["cache"].view(-1, s["cache"].shape[-1])
    rows[dst] = rows[src]
    moved = torch.zeros_like(w)
    m = min(kept.shape[1], R)
    moved[:, :m] = w.gather(1, kept[:, :m].clamp(max=R - 1)).masked_fill(~ok[:, :m], 0.0)
    w.copy_(torch.where(at < used, moved, w))
    return used2[:, 0].to(torch.int32), torch.where(ok, kept, -1).to(torch.int32)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _cache_values(cache):
    """The cache as values: of fp8 rows the latent values, their scales and the rope channels."""
    if cache.dtype is not torch.uint8:
        return {"cache": cache}
    return {"latent": cache[..., :512].view(torch.float8_e4m3fn), "scale": cache[..., 512:528].view(torch.float32),
            "rope": cache[..., 528:].view(torch.bfloat16)}


@functools.cache
def _entries():
    """The framework's entry points."""
    from dsv4_amd.api import add_row_weights, sparse_attn_sharedkv_first, sparse_attn_sharedkv_first_backward
    from dsv4_amd.cache import evict_kv_cache
    return sparse_attn_sharedkv_first, sparse_attn_sharedkv_first_backward, add_row_weights, evict_kv_cache


def _run_own(s):
    first, first_backward, add_row_weights, evict_kv_cache = _entries()
    op = s["op"]
    if op == "first":
        out, lse = first(s["q"], sinks=s["sinks"], return_softmax_lse=True, **s["kw"])
        return {"out": out, "lse": lse}
    if op == "grad":
        dq, d_ori, d_cmp, d_sinks = first_backward(s["dout"], s["q"], s["out"], s["lse"], sinks=s["sinks"], **s["kw"])
        got = {"dq": dq, "d_sinks": d_sinks, "d_ori_kv": d_ori.to(s["q"].dtype)}
        return got if d_cmp is None else {**got, "d_cmp_kv": d_cmp.to(s["q"].dtype)}
    if op == "weights":
        add_row_weights(s["q"], s["lse"], ori_weights=s["ori_weights"], cmp_weights=s.get("cmp_weights"), **s["kw"])
        return _weights(s)
    used, kept = evict_kv_cache(s["cache"], s["weights"], s["bt"], s["used"], budget=s["budget"], keep_first=s["first"],
                                keep_recent=s["recent"])
    return {"used": used, "kept": kept, "weights": s["weights"], **_cache_values(s["cache"])}


def _weights(s):
    return {k: s[k].float() for k in ("ori_weights", "cmp_weights") if k in s}


def run(s):
    op = s["op"]
    if op == "evict":   # the weights that this eviction meets: the last one took them apart
        s["weights"].copy_(s["met"])
    if own:
        return _run_own(s)
    if op == "first":
        return _plain_first(s)
    if op == "grad":
        return _plain_grad(s)
    if op == "weights":
        _plain_weights(s)
        return _weights(s)
    used, kept = _plain_evict(s)
    return {"used": used, "kept": kept, "weights": s["weights"], **_cache_values(s["cache"])}


# ---------------------------------------------------------------------------
# work, 64-bit results
# ---------------------------------------------------------------------------

def work(case):
    c = case
    q_lens, kv_lens = _lengths(c)
    D = c["D"]
    row = 656 if c["dt"] == "fp8" else 2 * D
    if c["op"] == "evict":
        # of each sequence: every weight read; the rows behind the first one that leaves, and their weights, moved
        moved = 0
        for n in kv_lens:
            gone = max(0, n - c["budget"])
            free = max(0, n - c["first"] - c["recent"])
            moved += max(0, c["budget"] - c["first"] - free // (gone + 1)) if gone else 0
        return {"bytes": moved * (2 * row + 8) + sum(kv_lens) * 8 + 4 * c["B"] * c["budget"], "flops": 0}
    T, H, win = sum(q_lens), c["H"], c["win"] or max(kv_lens)
    ori = cmp_ = ori_rows = cmp_rows = 0
    for m, n in zip(q_lens, kv_lens):
        pos = range(n - m, n)
        ori += sum(min(p + 1, win) + min(c["F"], max(0, p + 1 - win)) for p in pos)
        ori_rows += min(n, m - 1 + win) + min(c["F"], max(0, n - m + 1 - win))
        if c["kind"] != "swa":
            pairs = sum(min((p + 1) // c["ratio"], c["K"] or n) for p in pos)
            cmp_ += pairs
            cmp_rows += n // c["ratio"] if c["kind"] == "cfa" else min(pairs, n // c["ratio"])
    pairs, rows = ori + cmp_, ori_rows + cmp_rows
    index = T * 4 * c["K"]
    if c["op"] == "first":
        return {"bytes": T * H * (2 * D + 2 * DV + 4) + rows * row + index, "flops": pairs * H * 2 * (D + DV)}
    if c["op"] == "grad":   # q, out, dout and rows read, dq and the rows' gradients written; five products
        return {"bytes": T * H * (4 * D + 4 * DV + 4) + rows * 2 * row + index, "flops": pairs * H * 2 * (3 * D + 2 * DV)}
    return {"bytes": T * H * (2 * D + 4) + rows * (row + 16) + index, "flops": pairs * H * 2 * D}


def _exact_tokens(c, s):
    """For runs of tokens: (sequence, tokens, positions of the raw rows in 64 bits and
    which of them each token attends, of the compressed rows likewise)."""
    kw = s["kw"]
    q_lens, kv_lens = _lengths(c)
    t = 0
    for b, (m, n) in enumerate(zip(q_lens, kv_lens)):
        step = 1 if c["kind"] == "scfa" else 512 if c["win"] else max(1, min(512, (1 << 26) // (c["H"] * n)))
        for i in range(0, m, step):
            k = min(m, i + step)
            pos = torch.arange(n - m + i, n - m + k, device=DEV)
            low = max(0, n - m + i - (c["win"] or n) + 1)
            at = torch.cat([torch.arange(min(c["F"], low), device=DEV), torch.arange(low, n - m + k, device=DEV)])
            near = at > (pos - (c["win"] or n))[:, None]
            see = (at <= pos[:, None]) & (near | (at < c["F"]))
            caches = [(kw["ori_kv"], kw["ori_block_table"][b].long(), at, see)]
            if c["kind"] != "swa":
                thr = (pos + 1) // c["ratio"]
                at = torch.arange(int(thr[-1]), device=DEV)
                see = at < thr[:, None]
                if c["kind"] == "scfa":
                    at = kw["cmp_sparse_indices"][t + i, 0].long()
                    at = at[(at >= 0) & (at < thr[0])]
                    see = torch.ones((1, at.numel()), dtype=torch.bool, device=DEV)
                caches.append((kw["cmp_kv"], kw["cmp_block_table"][b].long(), at, see))
            flat = [table[at // c["bs"]] * c["bs"] + at % c["bs"] for _, table, at, _ in caches]
            keys = torch.cat([_rows(x[0], f, torch.float64) for x, f in zip(caches, flat)])
            yield b, slice(t + i, t + k), keys, torch.cat([x[3] for x in caches], 1), [x[2] for x in caches], flat
        t += m


def _exact_attn(c, s):
    q, kw, H = s["q"], s["kw"], c["H"]
    f64 = dict(dtype=torch.float64, device=DEV)
    got = {}
    if c["op"] == "first":
        got = {"out": torch.empty((*q.shape[:2], DV), **f64), "lse": torch.empty(q.shape[:2], **f64)}
    elif c["op"] == "grad":
        got = {"dq": torch.empty(q.shape, **f64), "d_sinks": torch.zeros(H, **f64)}
        got.update({"d_" + k: torch.zeros(kw[k].shape, **f64) for k in ("ori_kv", "cmp_kv") if k in kw})
    else:
        got = {k: torch.zeros_like(s[k]) for k in ("ori_weights", "cmp_weights") if k in s}
    for b, t, k, see, ats, flats in _exact_tokens(c, s):
        qd = q[t].double()
        x = torch.matmul(qd.flatten(0, 1), k.t().contiguous()).view(*qd.shape[:2], -1) * kw["softmax_scale"]
        x.masked_fill_(~see[:, None], -math.inf)
        n = ats[0].numel()
        if c["op"] == "first":
            sink = s["sinks"].double()[None, :, None].expand(x.shape[0], -1, 1)
            lse = torch.logsumexp(torch.cat([x, sink], 2), 2)
            got["lse"][t] = lse
            got["out"][t] = torch.matmul(torch.exp(x - lse[..., None]).flatten(0, 1), k[:, :DV].contiguous()).view(
                *qd.shape[:2], DV)
            continue
        p = torch.exp(x - s["lse"][t].double()[..., None])
        if c["op"] == "weights":
            w = p.sum((0, 1)) / H
            got["ori_weights"][b].index_add_(0, ats[0], w[:n])
            if len(ats) > 1:
                got["cmp_weights"][b].index_add_(0, ats[1], w[n:])
            continue
        do = s["dout"][t].double()
        delta = (do * s["out"][t].double()).sum(-1)
        ds = p * (torch.matmul(do.flatten(0, 1), k[:, :DV].t().contiguous()).view_as(p) - delta[..., None]) * kw["softmax_scale"]
        got["dq"][t] = torch.matmul(ds.flatten(0, 1), k).view_as(qd)
        got["d_sinks"] -= (torch.exp(s["sinks"].double() - s["lse"][t].double()) * delta).sum(0)
        d = torch.matmul(ds.flatten(0, 1).t().contiguous(), qd.flatten(0, 1))
        d[:, :DV] += torch.matmul(p.flatten(0, 1).t().contiguous(), do.flatten(0, 1))
        got["d_ori_kv"].view(-1, c["D"]).index_add_(0, flats[0], d[:n])
        if len(flats) > 1:
            got["d_cmp_kv"].view(-1, c["D"]).index_add_(0, flats[1], d[n:])
    return got


def _exact_evict(c, s):
    """Row by row on the host: which stay, then the caches as they have to look."""
    cache, weights = s["cache"].clone(), s["weights"].clone()
    used, kept = [], []
    for b, n in enumerate(_lengths(c)[1]):
        w = s["weights"][b].tolist()
        free = range(c["first"], max(c["first"], n - c["recent"]))
        gone = set(sorted(free, key=lambda j: (w[j], -j))[:max(0, n - c["budget"])])
        stay = [j for j in range(n) if j not in gone]
        used.append(len(stay))
        kept.append(stay + [-1] * (c["budget"] - len(stay)))
        old, new = torch.tensor(stay, device=DEV), torch.arange(len(stay), device=DEV)
        table = s["bt"][b].long()
        cache[table[new // c["bs"]], new % c["bs"]] = s["cache"][table[old // c["bs"]], old % c["bs"]]
        weights[b, :n] = 0
        weights[b, :len(stay)] = s["weights"][b, old]
    return {"used": torch.tensor(used, dtype=torch.int32, device=DEV),
            "kept": torch.tensor(kept, dtype=torch.int32, device=DEV), "weights": weights, **_cache_values(cache)}


def exact(case, seed):
    if case["op"] != "evict" and case["kind"] == "scfa" and sum(_lengths(case)[0]) > 6000:
        return None   # token by token: beyond some 20 seconds
    s = prepare(case, seed)
    return _exact_evict(case, s) if case["op"] == "evict" else _exact_attn(case, s)

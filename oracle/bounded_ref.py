"""ORACLE (test infrastructure only; never imported by the product path).

CPU restatement in 64 bits of what keeps caches bounded: the attention with first rows
that stay visible and its gradients, the weight of cache rows, evictions; token by
token, row by row, with plain lists of positions. The reference's window drops the first
rows (sparse_attn_sharedkv_tilelang/golden.py:125-131, whose causal position, window and
compressed threshold this follows otherwise) and has none of the others.

Pins (tests/test_bounded.py): known key sets; no first rows gives the linear oracle's
result; central differences and the closed-form sink gradient; weights of a token sum to
its share that is not the sink's; known evictions; planted mistakes fail them.
"""

from __future__ import annotations

import torch


def positions(sg, first, win, twice=False):
    """Raw rows of a token at position ``sg``. ``twice`` plants a mistake: first rows
    that the window holds count again."""
    if sg < 0:
        return []
    low = max(0, sg - win + 1)
    return list(range(first if twice else min(first, low))) + list(range(low, sg + 1))


class Keys:
    """The keys of each token: per cache (positions, flat rows)."""

    def __init__(self, table, ctable, indices, q_lens, kv_lens, first, win, bs, cbs, ratio, T):
        self.seq, self.raw, self.cmp = [-1] * T, [([], [])] * T, [([], [])] * T
        pick = lambda tab, at, size: tuple(map(list, zip(*[  # noqa: E731
            (a, tab[a // size] * size + a % size) for a in at if a // size < len(tab) and tab[a // size] >= 0]))) or ([], [])
        t = 0
        for b, (m, n) in enumerate(zip(q_lens, kv_lens)):
            for i in range(m):
                sg = n - m + i
                self.seq[t] = b
                self.raw[t] = pick(table[b].tolist(), positions(sg, first, win), bs)
                if ctable is not None:
                    thr = max(0, (sg + 1) // ratio)
                    at = range(thr) if indices is None else [j for j in indices[t].tolist() if 0 <= j < thr]
                    self.cmp[t] = pick(ctable[b].tolist(), at, cbs)
                t += 1


def _k(keys, t, rows, crows):
    parts = [rows[keys.raw[t][1]].double()]
    if crows is not None:
        parts.append(crows[keys.cmp[t][1]].double())
    return torch.cat(parts)


def attention(keys, q, rows, crows, sinks, scale):
    """(out, lse, sum p |v|); tokens of no sequence give zeros."""
    T, H, _ = q.shape
    out, lse = torch.zeros(T, H, 512, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for t in range(T):
        if keys.seq[t] < 0:
            continue
        k = _k(keys, t, rows, crows)
        x = torch.cat([q[t].double() @ k.t() * scale, sinks.double()[:, None]], 1)
        lse[t] = torch.logsumexp(x, 1)
        p = torch.exp(x[:, :-1] - lse[t][:, None])
        out[t], mag[t] = p @ k[:, :512], p @ k[:, :512].abs()
    return out, lse, mag


def gradients(keys, dout, q, out, lse, rows, crows, sinks, scale, half, sign=1.0):
    """({name: gradient}, {name: bound}) from a forward's own ``out`` and ``lse``. The
    bounds are those of P and dS rounded to the query's type (half a step: ``half``) before
    the products; see tests/test_bounded.py. ``sign`` plants a mistake in dS."""
    T, H, D = q.shape
    z = lambda *s: torch.zeros(*s, dtype=torch.float64)  # noqa: E731
    g = {"dq": z(T, H, D), "rows": z(*rows.shape), "crows": None if crows is None else z(*crows.shape), "sinks": z(H)}
    e = {k: None if v is None else torch.zeros_like(v) for k, v in g.items()}
    tiny = 2.0 ** -25 if half == 2.0 ** -11 else 0.0   # half a step of fp16's smallest numbers
    for t in range(T):
        if keys.seq[t] < 0:
            continue
        k, qt, do = _k(keys, t, rows, crows), q[t].double(), dout[t].double()
        p = torch.exp(qt @ k.t() * scale - lse[t].double()[:, None])
        delta = (do * out[t].double()).sum(1, keepdim=True)
        terms = (do * out[t].double()).abs().sum(1, keepdim=True)
        dp = do @ k[:, :512].t()
        ds = sign * p * (dp - delta) * scale
        off = 1.5 * half * p * ((dp - delta).abs() + (do.abs() @ k[:, :512].abs().t() + terms) / 16) * scale + tiny
        g["dq"][t] = ds @ k
        e["dq"][t] = off @ k.abs() + half * g["dq"][t].abs()
        share = torch.exp(sinks.double() - lse[t].double())
        g["sinks"] -= share * delta[:, 0]
        e["sinks"] += 2.0 ** -13 * share * terms[:, 0]
        d, de = ds.t() @ qt, off.t() @ qt.abs()
        d[:, :512] += p.t() @ do
        de[:, :512] += (1.5 * half * p + tiny).t() @ do.abs()
        n = len(keys.raw[t][1])
        for at, name, sl in ((keys.raw[t][1], "rows", slice(0, n)), (keys.cmp[t][1], "crows", slice(n, None))):
            if at:
                i = torch.tensor(at)
                g[name].index_add_(0, i, d[sl])
                e[name].index_add_(0, i, de[sl])
    return g, e


def weights(keys, q, lse, rows, crows, scale, B, R, RC):
    """(raw [B, R], compressed [B, RC]) weights of a call; positions past R are dropped."""
    w, wc = torch.zeros(B, R, dtype=torch.float64), torch.zeros(B, RC, dtype=torch.float64)
    for t in range(q.shape[0]):
        if keys.seq[t] < 0:
            continue
        p = torch.exp(q[t].double() @ _k(keys, t, rows, crows).t() * scale - lse[t].double()[:, None]).mean(0)
        n = len(keys.raw[t][0])
        for to, at, part in ((w, keys.raw[t][0], p[:n]), (wc, keys.cmp[t][0], p[n:])):
            for j, x in zip(at, part.tolist()):
                if j < to.shape[1]:
                    to[keys.seq[t], j] += x
    return w, wc


def evict(cache, w, table, used, budget, first, recent, high=False):
    """(cache, weights, lengths, kept) after an eviction of ``cache [num_blocks, bs, ..]``.
    ``high`` plants a mistake: of equal weights the highest positions stay."""
    cache, old, w, was = cache.clone(), cache, w.clone(), w
    bs, out, lists = cache.shape[1], [], []
    for b, n in enumerate(max(0, int(x)) for x in used):
        tab = table[b].tolist()
        place = lambda j: (tab[j // bs], j % bs) if j // bs < len(tab) and 0 <= tab[j // bs] < cache.shape[0] else None  # noqa: E731
        stay = list(range(n))
        if n > budget:
            val = lambda j: was[b, j].item() if j < was.shape[1] else 0.0  # noqa: E731
            key = lambda j: (val(j) == val(j), val(j) if val(j) == val(j) else 0.0, j if high else -j)  # noqa: E731
            cand = sorted(range(first, n - recent), key=key, reverse=True)
            stay = sorted(list(range(first)) + cand[:budget - first - recent] + list(range(n - recent, n)))
            for i, j in enumerate(stay):
                if i != j and place(i) and place(j):
                    cache[place(i)] = old[place(j)]
            for i in range(min(n, was.shape[1])):
                w[b, i] = val(stay[i]) if i < budget else 0.0
        out.append(len(stay))
        lists.append(stay + [-1] * (budget - len(stay)))
    return cache, w, torch.tensor(out, dtype=torch.int32), torch.tensor(lists, dtype=torch.int32).view(len(out), budget)

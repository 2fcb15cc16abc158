"""ORACLE (test infrastructure only; never imported by the product path).

CPU restatement in 64 bits of the attention for trees of drafted tokens
(``sas_fwd_tree_v1``), token by token with plain lists of cache positions. The
reference takes chains only (sparse_attn_sharedkv_tilelang/golden.py:69-204, whose
window, causal threshold and sink this follows for a node's own position).

Pins (tests/test_tree.py): a chain's mask gives the linear oracle's result; known
windows of a small tree; a planted mistake (a node that does not attend itself)
fails them.
"""

from __future__ import annotations

import torch


def mask_of(trees, words):
    """int64 ``[T, words]`` of per-token sets of attended nodes."""
    out = torch.zeros(sum(len(t) for t in trees), words, dtype=torch.int64)
    r = 0
    for t in trees:
        for nodes in t:
            for j in nodes:
                out[r, j // 64] |= (1 << (j % 64)) - (1 << 64 if j % 64 == 63 else 0)
            r += 1
    return out


def random_tree(n, gen, reach=9):
    """Per node of a random tree the set of its ancestors and itself."""
    nodes = [[0]] if n else []
    for s in range(1, n):
        parent = int(torch.randint(max(0, s - reach), s, (1,), generator=gen))
        nodes.append(nodes[parent] + [s])
    return nodes


def window(nodes, n, aq, win, attend_self=True):
    """(positions of the window's cache rows, the token's position) of a token that
    attends ``nodes`` among ``aq`` nodes behind ``n`` rows (n < 0: nodes before position 0
    are missing). ``attend_self`` exists so a test can plant a mistake."""
    nodes = sorted(j for j in nodes if j < aq and n + j >= 0)
    if not attend_self:
        nodes = nodes[:-1]
    line = list(range(max(n, 0))) + [n + j for j in nodes]
    return line[-win:], len(line) - 1


def attention(q, rows, cmp_rows, table, cmp_table, indices, trees, q_lens, kv_lens, sinks, scale, win, bs, cbs, ratio, T):
    """(out, lse, sum p |v|) for tokens packed as ``q [T, H, D]``; ``rows`` / ``cmp_rows``
    are the caches' values ``[num_blocks * bs, D]`` (cmp_rows None: window only; indices
    None: dense compressed rows)."""
    H = q.shape[1]
    out, lse = torch.zeros(T, H, 512, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    mag = torch.zeros_like(out)
    t = 0
    for b, (aq, kv) in enumerate(zip(q_lens, kv_lens)):
        for nodes in trees[b]:
            at, pos = window(nodes, kv - aq, aq, win)
            pick = lambda tab, at_, size: [tab[a // size] * size + a % size for a in at_  # noqa: E731
                                           if a // size < len(tab) and tab[a // size] >= 0]
            keys = [rows[pick(table[b].tolist(), at, bs)]]
            if cmp_rows is not None:
                thr = (pos + 1) // ratio
                sel = range(thr) if indices is None else [i for i in indices[t].tolist() if 0 <= i < thr]
                keys.append(cmp_rows[pick(cmp_table[b].tolist(), sel, cbs)])
            k = torch.cat(keys).double()
            x = torch.cat([q[t].double() @ k.t() * scale, sinks.double()[:, None]], 1)
            lse[t] = torch.logsumexp(x, 1)
            p = torch.exp(x[:, :-1] - lse[t][:, None])
            out[t], mag[t] = p @ k[:, :512], p @ k[:, :512].abs()
            t += 1
    return out, lse, mag

"""CPU restatement of the paged latent cache's operators (float64, one sequence, token and slot at a
time).  The reference keeps contiguous caches (``oracle/v4_fast.py:93-96,150-159`` of it); the attention is
``ref_torch/sparse_attn.py:23-34`` over the rows a token sees."""
import torch

F64 = torch.float64


def rows(pages, scales, table_row, n):
    """The first n rows [n, D] of a sequence (float64) and which of them lie in valid pages; fp8 pages are
    decoded."""
    P, D = pages.shape[1:]
    out, ok = torch.zeros(n, D, dtype=F64), torch.zeros(n, dtype=torch.bool)
    for j in range(n):
        col = j // P
        page = int(table_row[col]) if col < table_row.shape[0] else -1
        if 0 <= page < pages.shape[0]:
            ok[j] = True
            r = pages[page, j % P].to(F64)
            if scales is not None:
                r = r * scales[page, j % P].to(F64).repeat_interleave(64)
            out[j] = r
    return out, ok


def paged_attn(q, pages, table, lens, cu, scale, sink=None, window=0, first=0, dv=512, scales=None):
    """(out, spread) [T, H, dv] float64: the result and sum p |v| / denominator, by which roundings of the
    probabilities are bounded."""
    T, H, D = q.shape
    out, spread = torch.zeros(T, H, dv, dtype=F64), torch.zeros(T, H, dv, dtype=F64)
    for b in range(table.shape[0]):
        n = int(cu[b + 1]) - int(cu[b])
        if n <= 0:
            continue
        kv, ok = rows(pages, scales, table[b], max(int(lens[b]), 0))
        for i in range(n):
            t, p = int(cu[b]) + i, int(lens[b]) - n + i
            seen = [j for j in range(p + 1) if ok[j] and (window == 0 or j > p - window or j < first)]
            if not seen:
                continue
            v = kv[seen]
            s = q[t].to(F64) @ v.T * scale
            m = s.amax(dim=1, keepdim=True)
            if sink is not None:
                m = torch.maximum(m, sink.to(F64)[:, None])
            e = torch.exp(s - m)
            den = e.sum(1, keepdim=True)
            if sink is not None:
                den = den + torch.exp(sink.to(F64)[:, None] - m)
            out[t], spread[t] = e @ v[:, :dv] / den, e @ v[:, :dv].abs() / den
    return out, spread


def positions(lens, cu):
    """(sequence, position) of every token below cu[-1]."""
    got = []
    for b in range(len(lens)):
        n = int(cu[b + 1]) - int(cu[b])
        got += [(b, int(lens[b]) - n + i) for i in range(n)]
    return got


def norm_rope(x, w, norm, norm_dims, cos, sin, eps):
    """[heads, D] float64: RMS norm of the first norm_dims channels, rotation of the last 2 len(cos) as pairs."""
    x = x.to(F64).clone()
    if norm:
        h = x[:, :norm_dims]
        x[:, :norm_dims] = h / torch.sqrt(h.square().mean(1, keepdim=True) + eps) * (1.0 if w is None else w.to(F64))
    rd = 2 * cos.shape[0]
    if rd:
        at = x.shape[1] - rd
        a, b, c, s = x[:, at::2].clone(), x[:, at + 1::2].clone(), cos.to(F64), sin.to(F64)
        x[:, at::2], x[:, at + 1::2] = a * c - b * s, a * s + b * c
    return x


def fp8_scale(y):
    """Power-of-two scales of the 64-channel blocks of y [..., D] (float64)."""
    amax = y.unflatten(-1, (-1, 64)).abs().amax(-1).clamp(min=1e-4)
    return torch.exp2(torch.ceil(torch.log2(amax / 448.0)))


def update_pages(pages, table, lens, refs, parent, grow):
    """New (table, lens, refs, granted) and the page copies [(source, destination, rows)] as lists."""
    S, M = len(table), len(table[0])
    P, n_pages = pages
    free = [i for i in range(n_pages) if refs[i] == 0]
    new_t, new_l, granted, copies = [list(r) for r in table], list(lens), [0] * S, []
    asked = 0
    for s in range(S):
        p, g = parent[s], grow[s]
        if not -1 <= p < S:
            continue
        have = lens[p] if p >= 0 else 0
        if have < 0 or not 0 <= have + g < 1 << 31 or -(-(have + g) // P) > M:
            continue
        pages_now = -(-(have + g) // P)
        rows_kept = min(have, have + g)     # a negative growth gives rows back
        kept = rows_kept // P
        tail = table[p][kept] if p >= 0 and rows_kept % P else -1
        if p == s and rows_kept % P and (g == 0 or not 0 <= tail < n_pages or refs[tail] <= 1):
            kept, tail = kept + 1, -1   # keeps its own partly filled page, which no other slot holds
        at = asked
        asked += pages_now - kept
        if asked > len(free):
            continue
        granted[s], new_l[s] = 1, have + g
        fresh = free[at:asked]
        new_t[s] = (list(table[p][:kept]) if p >= 0 else []) + fresh
        new_t[s] += [-1] * (M - len(new_t[s]))
        if 0 <= tail < n_pages:
            copies.append((tail, fresh[0], rows_kept % P))
    new_r = list(refs)
    for s in range(S):
        if granted[s]:
            for row, n, by in ((table[s], lens[s], -1), (new_t[s], new_l[s], 1)):
                for page in row[:-(-n // P)]:
                    if 0 <= page < n_pages:
                        new_r[page] += by
    return new_t, new_l, new_r, granted, copies


def compact_pages(table, refs):
    """New (table, refs, live) and the moves [(source, destination)]."""
    n = len(refs)
    live = sum(r > 0 for r in refs)
    moves = list(zip([i for i in range(live, n) if refs[i] > 0], [i for i in range(live) if refs[i] <= 0]))
    to = dict(moves)
    new_r = list(refs)
    for a, b in moves:
        new_r[b], new_r[a] = refs[a], 0
    new_t = [[to.get(p, p) if 0 <= p < n and refs[p] > 0 else -1 for p in row] for row in table]
    return new_t, new_r, live, moves

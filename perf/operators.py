"""Timed and checked cases of the paged latent cache: what a server of many sequences does with it.

The kinds:

* ``attn``     ``paged.paged_attn``: attention of the newest tokens of a ragged batch over the pages
               (decode: one token a sequence; a prompt's chunk; a window with a few first tokens).
* ``append``   ``paged.paged_append``: per-head query norm, row norm, RoPE and the write of the new rows
               into their pages, from the projections' results.
* ``update``   ``paged.update_pages``: slots forked, freed and grown between two steps.
* ``compact``  ``paged.compact_pages``: the live pages moved together at the pool's start.

``run`` computes them in plain torch where ``own`` is false, through the framework where it is true;
``exact`` restates the floating ones in float64.
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
DV = 512
ROPE = 64
EPS = 1e-6


def _paged():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "deepseek-v4-flash-mlx_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from smla import paged
    return paged


def listed():
    return [
        # one sequence's next token at 4 K context: the smallest call, where latency counts
        {"name": "attn_token", "kind": "attn", "B": 1, "n_lo": 1, "n_hi": 1, "l_lo": 4097, "l_hi": 4097, "H": 64, "D": 576,
         "P": 64, "kv": "bf16", "window": 0, "first": 0, "sink": False, "mix": 1},
        # a decode step of 32 sequences of unlike lengths, the layer's 64 heads
        {"name": "attn_decode", "kind": "attn", "B": 32, "n_lo": 1, "n_hi": 1, "l_lo": 2000, "l_hi": 32768, "H": 64, "D": 576,
         "P": 64, "kv": "bf16", "window": 0, "first": 0, "sink": False, "mix": 2},
        # four draft tokens each of 64 sequences over fp8 pages, 16 heads (a quarter of the layer's), sinks
        {"name": "attn_draft_fp8", "kind": "attn", "B": 64, "n_lo": 2, "n_hi": 4, "l_lo": 1000, "l_hi": 16384, "H": 16, "D": 512,
         "P": 32, "kv": "fp8", "window": 0, "first": 0, "sink": True, "mix": 3},
        # a prompt of 4096 tokens in the layer's 128-row window with 4 first tokens kept
        {"name": "attn_window", "kind": "attn", "B": 1, "n_lo": 4096, "n_hi": 4096, "l_lo": 4096, "l_hi": 4096, "H": 64, "D": 512,
         "P": 64, "kv": "bf16", "window": 128, "first": 4, "sink": True, "mix": 4},
        # a 2048-token chunk at the end of a 32 K prompt: the largest
        {"name": "attn_chunk", "kind": "attn", "B": 1, "n_lo": 2048, "n_hi": 2048, "l_lo": 32768, "l_hi": 32768, "H": 64, "D": 576,
         "P": 64, "kv": "bf16", "window": 0, "first": 0, "sink": False, "mix": 5},
        # the new rows of a decode step of 8 sequences: latency again
        {"name": "append_step", "kind": "append", "B": 8, "n_lo": 1, "n_hi": 1, "ctx": 5000, "H": 64, "D": 512, "P": 64,
         "x": "f32", "kv": "sim", "q_norm": True, "mix": 6},
        # a 4096-token prompt's queries and rows from fp32 projections
        {"name": "append_prompt", "kind": "append", "B": 1, "n_lo": 4096, "n_hi": 4096, "ctx": 0, "H": 64, "D": 512, "P": 64,
         "x": "f32", "kv": "bf16", "q_norm": True, "mix": 7},
        # chunks of 5 sequences, bf16 projections, e4m3 pages of 576-wide rows
        {"name": "append_fp8", "kind": "append", "B": 5, "n_lo": 100, "n_hi": 333, "ctx": 8000, "H": 16, "D": 576, "P": 32,
         "x": "bf16", "kv": "fp8", "q_norm": False, "mix": 8},
        # every sequence of a step grows by a token
        {"name": "update_step", "kind": "update", "S": 32, "M": 128, "P": 64, "D": 576, "layers": 1, "pages": 1500, "kv": "bf16",
         "how": "grow", "grow": 1, "mix": 9},
        # beams reordered and forked, some slots freed, others started; eight layers share the table
        {"name": "update_fork", "kind": "update", "S": 160, "M": 64, "P": 64, "D": 576, "layers": 8, "pages": 2048, "kv": "bf16",
         "how": "fork", "grow": 40, "mix": 10},
        # a small pool with its live pages scattered, and a large one
        {"name": "compact_small", "kind": "compact", "S": 8, "M": 40, "P": 64, "D": 512, "layers": 1, "pages": 300, "kv": "bf16",
         "mix": 11},
        {"name": "compact_large", "kind": "compact", "S": 64, "M": 128, "P": 64, "D": 576, "layers": 1, "pages": 8192, "kv": "bf16",
         "mix": 12},
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "append", "append", "update", "compact"])
    c = {"kind": kind, "P": rng.choice([16, 32, 64, 128]), "D": rng.choice([512, 576]), "mix": rng.randint(100, 1 << 30)}
    if kind == "attn":
        how = rng.choice(["token", "draft", "chunk", "window"])
        c["H"] = rng.choice([8, 16, 32, 64, 64, 128, rng.randint(1, 80)])
        c["n_hi"] = {"token": 1, "draft": rng.randint(2, 8)}.get(how) or _logint(rng, 16, 2048)
        c["n_lo"] = 1 if rng.random() < 0.3 else max(1, c["n_hi"] * 2 // 3)
        c["l_hi"] = c["n_hi"] + _logint(rng, 64, 32000 if how != "window" else 6000)
        c["l_lo"] = max(c["n_hi"], c["l_hi"] // rng.choice([1, 2, 8]))
        most = (1 << 31) // (c["H"] * c["n_hi"] * c["l_hi"])  # half of the largest listed case's scores
        if most < 1:
            c["l_hi"] = max(c["n_hi"], (1 << 31) // (c["H"] * c["n_hi"]))
            c["l_lo"] = min(c["l_lo"], c["l_hi"])
        c["B"] = max(1, min(_logint(rng, 1, 64), most, (1 << 20) // c["l_hi"]))
        c["window"], c["first"] = (_logint(rng, 32, 4096), rng.choice([0, 1, 4, 37])) if how == "window" else (0, 0)
        c["sink"] = rng.random() < 0.5
        c["kv"] = rng.choice(["bf16", "bf16", "fp8"])
    elif kind == "append":
        c["H"] = rng.choice([8, 16, 32, 64, rng.randint(1, 80)])
        c["B"] = _logint(rng, 1, 64)
        c["n_hi"] = _logint(rng, 1, max(1, min(4096, 262144 // (c["H"] * c["B"]))))
        c["n_lo"] = max(1, c["n_hi"] // 2)
        c["ctx"] = rng.choice([0, rng.randint(1, 4000)])
        c["x"] = rng.choice(["f32", "bf16"])
        c["kv"] = rng.choice(["bf16", "fp8", "sim"])
        c["q_norm"] = rng.random() < 0.6
    else:
        c["S"] = _logint(rng, 1, 160)
        c["M"] = _logint(rng, 4, 128)
        c["pages"] = max(8, min(8192, int(c["S"] * c["M"] * rng.uniform(0.7, 1.3))))
        c["layers"] = rng.randint(1, 3) if c["pages"] * c["P"] <= 65536 else 1
        c["kv"] = rng.choice(["bf16", "bf16", "fp8"])
        if kind == "update":
            c["how"], c["grow"] = rng.choice(["grow", "fork"]), _logint(rng, 1, 200)
    return c


# ---------------------------------------------------------------------------------------------
# what a case says apart from the values: lengths, parents, holes

def _lengths(c):
    r = random.Random(c["mix"])
    if c["kind"] == "append":
        n = [r.randint(c["n_lo"], c["n_hi"]) for _ in range(c["B"])]
        return n, [k + (r.randint(0, c["ctx"]) if c["ctx"] else 0) for k in n]
    n = [r.randint(c["n_lo"], c["n_hi"]) for _ in range(c["B"])]
    return n, [r.randint(c["l_lo"], c["l_hi"]) for _ in range(c["B"])]


def _slots(c):
    """Rows of each slot, the rows that an odd slot shares with the one before it, parents, growth."""
    r = random.Random(c["mix"])
    S, M, P = c["S"], c["M"], c["P"]
    room = c["pages"] * 3 // 4  # a quarter of the pool stays free
    lens, shared = [], []
    for s in range(S):
        n = 0 if r.random() < 0.1 and S > 1 else r.randint(1, max(1, (M * P * 3) // 4))
        n = min(n, max(0, room) * P)
        room -= -(-n // P)
        lens.append(n)
        shared.append(min(n // P, lens[s - 1] // P) // 2 if s % 2 else 0)
    parent, grow = list(range(S)), [c.get("grow", 0)] * S
    if c.get("how") == "fork":
        grow = [r.randint(0, c["grow"]) for _ in range(S)]
        for s in range(S):
            u = r.random()
            if u < 0.5:
                parent[s] = r.randint(max(0, s - s % 8), min(S - 1, s - s % 8 + 7))
            elif u < 0.6:
                parent[s] = -1
    return lens, shared, parent, grow


class _Draw:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(int(seed))

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        x = torch.randn(*shape, generator=self.g, device=DEV, dtype=dtype)
        return x if std == 1.0 else x.mul_(std)

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device=DEV).to(torch.int32)


def _pool(r, shape, kv):
    """Pages of rows: bf16, or e4m3 codes with a power-of-two scale per 64 channels."""
    if kv != "fp8":
        return r.normal(*shape, dtype=torch.bfloat16), None
    codes = r.normal(*shape, std=60.0, dtype=torch.bfloat16).clamp_(-448, 448).to(torch.float8_e4m3fn)
    e = torch.randint(-7, -5, (*shape[:-1], shape[-1] // 64), generator=r.g, device=DEV)
    return codes, torch.exp2(e.float())


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    c, r = case, _Draw(seed)
    st = {"case": dict(c)}
    P, D = c["P"], c["D"]
    if c["kind"] in ("attn", "append"):
        n, lens = _lengths(c)
        cols = [-(-x // P) for x in lens]
        M, total = max(cols), sum(cols)
        st["pages"], st["scales"] = _pool(r, (total + 5, P, D), c["kv"])
        perm = r.perm(total + 5)
        table = torch.full((len(n), M), -1, dtype=torch.int32, device=DEV)
        at = 0
        for b, k in enumerate(cols):
            table[b, :k] = perm[at:at + k]
            at += k
        cu = [0]
        for k in n:
            cu.append(cu[-1] + k)
        st.update(table=table, lens=_i32(lens), cu=_i32(cu), n_max=max(n), l_max=max(lens))
        T, H = cu[-1], c["H"]
        if c["kind"] == "attn":
            st["q"] = r.normal(T, H, D, dtype=torch.bfloat16)
            st["sink"] = r.normal(H) if c["sink"] else None
        else:
            dt = torch.float32 if c["x"] == "f32" else torch.bfloat16
            st["q"] = r.normal(T, H, D, dtype=dt)
            st["kv_in"] = r.normal(T, D + 1024, dtype=dt)[:, 1024:]  # a slice of a wider projection
            st["norm_w"] = 1.0 + 0.1 * r.normal(DV)
            f = 10000.0 ** (-torch.arange(0, ROPE, 2, device=DEV, dtype=torch.float64) / ROPE)
            a = torch.arange(max(lens), device=DEV, dtype=torch.float64)[:, None] * f
            st["cos"], st["sin"] = a.cos().float(), a.sin().float()
        return st
    lens, shared, parent, grow = _slots(c)
    S, M, n_pages = c["S"], c["M"], c["pages"]
    cols = [-(-x // P) for x in lens]
    perm = r.perm(n_pages)
    table = torch.full((S, M), -1, dtype=torch.int32, device=DEV)
    at = 0
    for s, k in enumerate(cols):
        table[s, :k] = perm[at:at + k]
        at += k
        if shared[s]:
            table[s, :shared[s]] = table[s - 1, :shared[s]]
    live = table[table >= 0].long()
    refs = torch.zeros(n_pages, dtype=torch.int32, device=DEV).index_add_(0, live, torch.ones_like(live, dtype=torch.int32))
    if c["kind"] == "compact":
        refs[perm[-(n_pages // 10):].long()] += 1  # pages that something beside the table holds
    st["pages"], st["scales"] = _pool(r, (c["layers"], n_pages, P, D), c["kv"])
    st.update(table=table, lens=_i32(lens), refs=refs, parent=_i32(parent), grow=_i32(grow))
    return st


# ---------------------------------------------------------------------------------------------
# the plain forms

def _rows_plain(pages, scales, table):
    """[B, columns * P, D] fp32 rows of a table (-1 read as page 0: masked later)."""
    at = table.clamp(min=0).long()
    x = pages[at].float()
    if scales is not None:
        x = (x.unflatten(-1, (-1, 64)) * scales[at].unsqueeze(-1)).flatten(-2)
    return x.flatten(1, 2)


def _attn_plain(st):
    c = st["case"]
    q, lens, cu = st["q"], st["lens"], st["cu"]
    T, H, D = q.shape
    P, B, n_max = c["P"], c["B"], st["n_max"]
    kv = _rows_plain(st["pages"], st["scales"], st["table"])
    L = kv.shape[1]
    n = cu[1:] - cu[:-1]
    i = torch.arange(n_max, device=DEV)
    tok = (cu[:-1, None] + i).clamp(max=T - 1).long()  # [B, n_max]
    s = torch.matmul(q[tok].float().view(B, n_max * H, D), kv.transpose(1, 2)).mul_(D ** -0.5).view(B, n_max, H, L)
    pos = (lens - n)[:, None] + i  # [B, n_max]
    j = torch.arange(L, device=DEV)
    seen = j <= pos[..., None]
    if c["window"]:
        seen &= (j > pos[..., None] - c["window"]) | (j < c["first"])
    seen &= (st["table"] >= 0).repeat_interleave(P, dim=1)[:, None]
    s.masked_fill_(~seen[:, :, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    if st["sink"] is not None:
        m = torch.maximum(m, st["sink"][:, None])
    m = torch.where(m == -math.inf, 0.0, m)
    p = s.sub_(m).exp_()
    den = p.sum(-1, keepdim=True)
    if st["sink"] is not None:
        den = den + torch.exp(st["sink"][:, None] - m)
    o = torch.matmul(p.view(B, n_max * H, L), kv[..., :DV]).view(B, n_max, H, DV)
    o = torch.where(den > 0, o / den, 0.0).to(torch.bfloat16)
    out = torch.zeros(T, H, DV, dtype=torch.bfloat16, device=DEV)
    mine = i < n[:, None]
    out[tok[mine]] = o[mine]
    return out


def _norm_rope_plain(x, w, norm, cos, sin):
    """x [T, heads, D] fp32: RMS norm of the first 512 channels, rotation of the last 64 as pairs."""
    if norm:
        head = x[..., :DV]
        y = head * torch.rsqrt(head.square().mean(-1, keepdim=True) + EPS)
        x = torch.cat([y if w is None else y * w, x[..., DV:]], dim=-1)
    a, b = x[..., -ROPE::2], x[..., 1 - ROPE::2]
    turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    return torch.cat([x[..., :-ROPE], turned], dim=-1)


def _fp8_plain(x):
    """e4m3 codes and power-of-two scales per 64 channels."""
    y = x.unflatten(-1, (-1, 64))
    amax = y.abs().amax(-1, keepdim=True).clamp(min=1e-4)
    m, e = torch.frexp(amax / 448.0)
    s = torch.ldexp(torch.ones_like(amax), torch.where(m == 0.5, e - 1, e))
    return (y / s).clamp(-448, 448).to(torch.float8_e4m3fn).flatten(-2), s.squeeze(-1)


def _append_plain(st):
    c = st["case"]
    cu, lens = st["cu"], st["lens"]
    t = torch.arange(st["q"].shape[0], device=DEV, dtype=torch.int32)
    b = torch.searchsorted(cu[1:], t, right=True)
    pos = (lens - (cu[1:] - cu[:-1]))[b] + t - cu[:-1][b]
    cos, sin = st["cos"][pos.long()][:, None], st["sin"][pos.long()][:, None]
    q = _norm_rope_plain(st["q"].float(), None, c["q_norm"], cos, sin).to(torch.bfloat16)
    kv = _norm_rope_plain(st["kv_in"].float()[:, None], st["norm_w"], True, cos, sin)[:, 0]
    page, row = st["table"][b, (pos // c["P"]).long()].long(), (pos % c["P"]).long()
    if c["kv"] == "fp8":
        codes, s = _fp8_plain(kv)
        st["pages"].view(torch.uint8)[page, row] = codes.view(torch.uint8)
        st["scales"][page, row] = s
        return {"q": q, "pages": st["pages"], "scales": st["scales"]}
    if c["kv"] == "sim":
        codes, s = _fp8_plain(kv[:, :-ROPE])
        flat = (codes.float().unflatten(-1, (-1, 64)) * s.unsqueeze(-1)).flatten(-2)
        kv = torch.cat([flat, kv[:, -ROPE:]], dim=-1)
    st["pages"][page, row] = kv.to(torch.bfloat16)
    return {"q": q, "pages": st["pages"]}


def _update_plain(st):
    c = st["case"]
    table, lens, refs, parent, grow = (st[k] for k in ("table", "lens", "refs", "parent", "grow"))
    P, (S, M), n_pages = c["P"], table.shape, refs.shape[0]
    slot, col = torch.arange(S, device=DEV, dtype=torch.int32), torch.arange(M, device=DEV, dtype=torch.int32)
    p = parent.clamp(0, S - 1).long()
    have = torch.where(parent >= 0, lens[p], 0)
    new = have + grow
    up = lambda n: torch.div(n + P - 1, P, rounding_mode="floor")  # noqa: E731
    keep = parent == slot
    full = torch.where(keep, up(have), torch.div(have, P, rounding_mode="floor"))
    ok = (parent >= -1) & (parent < S) & (grow >= 0) & (up(new) <= M)
    need = torch.where(ok, up(new) - full, 0)
    last = need.cumsum(0).to(torch.int32)
    order = torch.argsort((refs != 0).to(torch.int32), stable=True).to(torch.int32)  # free pages first, ascending
    ok &= last <= (refs == 0).sum()
    fresh = order[((last - need)[:, None] + col - full[:, None]).clamp(0, n_pages - 1).long()]
    now = torch.where(col < full[:, None], table[p], torch.where(col < up(new)[:, None], fresh, -1))
    now = torch.where(ok[:, None], now, table)
    lens2 = torch.where(ok, new, lens)
    was = torch.where(ok[:, None] & (col < up(lens)[:, None]), table, -1)
    takes = torch.where(ok[:, None] & (col < up(new)[:, None]), now, -1)
    refs2 = refs.clone()
    for ids, by in ((was, -1), (takes, 1)):
        at = ids.flatten()
        refs2.index_add_(0, at.clamp(min=0).long(), torch.where(at >= 0, by, 0).to(torch.int32))
    part = torch.where(ok & ~keep & (parent >= 0), have % P, 0)
    some = (part > 0).nonzero()[:, 0]
    src = table[p[some], full[some].long()].long()
    dst = now[some, full[some].long()].long()
    rows = torch.arange(P, device=DEV) < part[some, None]
    for pool in (st["pages"], st["scales"]):
        if pool is not None:
            raw = pool.view(torch.uint8) if pool.dtype == torch.float8_e4m3fn else pool
            raw[:, dst] = torch.where(rows[..., None], raw[:, src], raw[:, dst])
    return {"table": now, "lens": lens2, "refs": refs2, "granted": ok.to(torch.int32), "pages": st["pages"],
            "scales": st["scales"]}


def _compact_plain(st):
    table, refs = st["table"], st["refs"]
    n_pages = refs.shape[0]
    live = refs > 0
    n_live = live.sum()
    page = torch.arange(n_pages, device=DEV)
    src, dst = page[live & (page >= n_live)], page[~live & (page < n_live)]
    to = torch.where(live, page, -1)
    to[src] = dst
    inside = (table >= 0) & (table < n_pages)
    table2 = torch.where(inside, to[table.clamp(0, n_pages - 1).long()], -1).to(torch.int32)
    refs2 = refs.clone()
    refs2[dst] = refs[src]
    refs2[src] = 0
    for pool in (st["pages"], st["scales"]):
        if pool is not None:
            raw = pool.view(torch.uint8) if pool.dtype == torch.float8_e4m3fn else pool
            raw[:, dst] = raw[:, src]
    return {"table": table2, "refs": refs2, "live": n_live.to(torch.int32).view(1), "pages": st["pages"],
            "scales": st["scales"]}


def run(state):
    st, c = state, state["case"]
    if not own:
        return {"attn": _attn_plain, "append": _append_plain, "update": _update_plain, "compact": _compact_plain}[c["kind"]](st)
    paged = _paged()
    if c["kind"] == "attn":
        return paged.paged_attn(st["q"], st["pages"], st["table"], st["lens"], st["cu"], c["D"] ** -0.5, attn_sink=st["sink"],
                                window=c["window"], first=c["first"], dv=DV, page_scales=st["scales"])
    if c["kind"] == "append":
        q = paged.paged_append(st["q"], st["kv_in"], st["pages"], st["table"], st["lens"], st["cu"], st["cos"], st["sin"],
                               kv_norm=st["norm_w"], q_norm=c["q_norm"], norm_dims=DV, page_scales=st["scales"],
                               fp8_sim=c["kv"] == "sim", eps=EPS)
        out = {"q": q, "pages": st["pages"]}
        if c["kv"] == "fp8":
            out["scales"] = st["scales"]
        return out
    if c["kind"] == "update":
        table, lens, refs, granted = paged.update_pages(st["pages"], st["table"], st["lens"], st["refs"], st["parent"],
                                                        st["grow"], page_scales=st["scales"])
        return {"table": table, "lens": lens, "refs": refs, "granted": granted, "pages": st["pages"], "scales": st["scales"]}
    table, refs, live = paged.compact_pages(st["pages"], st["table"], st["refs"], page_scales=st["scales"])
    return {"table": table, "refs": refs, "live": live, "pages": st["pages"], "scales": st["scales"]}


# ---------------------------------------------------------------------------------------------

def work(case):
    c = case
    P, D = c["P"], c["D"]
    row = D + D // 64 * 4 if c["kv"] == "fp8" else 2 * D
    if c["kind"] in ("attn", "append"):
        n, lens = _lengths(c)
        T, H = sum(n), c["H"]
        table = 4 * sum(-(-x // P) for x in lens)
        if c["kind"] == "append":
            size = 4 if c["x"] == "f32" else 2
            return {"bytes": T * (H * D * (size + 2) + D * size + row + 2 * 4 * ROPE // 2) + 4 * T, "flops": 8 * T * (H + 1) * D}
        pairs = rows = 0
        for k, length in zip(n, lens):
            w, f = c["window"] or length, c["first"] if c["window"] else 0
            for p in range(length - k, length):
                lo = max(0, p - w + 1)
                pairs += p + 1 - lo + min(f, lo)
            lo = max(0, length - k - w + 1)
            rows += length - lo + min(f, lo)
        return {"bytes": 2 * T * H * (D + DV) + rows * row + table, "flops": 2 * pairs * H * (D + DV)}
    lens, shared, parent, grow = _slots(c)
    state = 4 * (2 * c["S"] * c["M"] + 4 * c["S"] + 2 * c["pages"])
    if c["kind"] == "update":
        tails = sum(lens[p] % P for s, p in enumerate(parent) if p not in (s, -1))
        return {"bytes": state + 2 * c["layers"] * row * tails, "flops": 0}
    live = sum(-(-x // P) - k for x, k in zip(lens, shared)) + c["pages"] // 10
    moved = live * (c["pages"] - live) // c["pages"]  # live pages behind the first `live` ids, of a random order
    return {"bytes": state + 2 * c["layers"] * row * P * moved, "flops": 0}


def _attn_exact(st):
    c = st["case"]
    P, D, H, dd = c["P"], c["D"], c["H"], torch.float64
    out = torch.zeros(st["q"].shape[0], H, DV, dtype=dd, device=DEV)
    cu, lens = st["cu"].tolist(), st["lens"].tolist()
    for b, length in enumerate(lens):
        ids = st["table"][b, :-(-length // P)].long()
        kv = st["pages"][ids].to(dd)
        if st["scales"] is not None:
            kv = kv * st["scales"][ids].to(dd).repeat_interleave(64, dim=-1)
        kv = kv.reshape(-1, D)[:length]
        first_pos = length - (cu[b + 1] - cu[b])
        step = max(1, (1 << 28) // (H * length))
        for t0 in range(cu[b], cu[b + 1], step):
            t1 = min(cu[b + 1], t0 + step)
            x = torch.einsum("thd,jd->thj", st["q"][t0:t1].to(dd), kv) / math.sqrt(D)
            p = first_pos + torch.arange(t0 - cu[b], t1 - cu[b], device=DEV)[:, None]
            j = torch.arange(length, device=DEV)[None]
            hide = j > p
            if c["window"]:
                hide |= (j <= p - c["window"]) & (j >= c["first"])
            x = x.masked_fill(hide[:, None], -math.inf)
            if st["sink"] is not None:
                x = torch.cat([x, st["sink"].to(dd)[None, :, None].expand(t1 - t0, H, 1)], dim=-1)
            out[t0:t1] = torch.einsum("thj,jd->thd", torch.softmax(x, dim=-1)[..., :length], kv[:, :DV])
    return out


def _append_exact(st):
    c, dd = st["case"], torch.float64
    cu, lens = st["cu"].tolist(), st["lens"].tolist()
    pos = torch.cat([torch.arange(n - (cu[b + 1] - cu[b]), n, device=DEV) for b, n in enumerate(lens)])
    seq = torch.cat([torch.full((cu[b + 1] - cu[b],), b, device=DEV) for b in range(len(lens))])
    turn = torch.complex(st["cos"][pos].to(dd), st["sin"][pos].to(dd))

    def through(x, w, norm):
        x = x.to(dd).clone()
        if norm:
            h = x[..., :DV]
            x[..., :DV] = h / torch.sqrt((h * h).sum(-1, keepdim=True) / DV + EPS) * (1.0 if w is None else w.to(dd))
        z = torch.view_as_complex(x[..., -ROPE:].unflatten(-1, (-1, 2)).contiguous())
        x[..., -ROPE:] = torch.view_as_real(z * turn.view(-1, *([1] * (z.dim() - 2)), ROPE // 2)).flatten(-2)
        return x

    out = {"q": through(st["q"], None, c["q_norm"]), "pages": None}
    if c["kv"] == "bf16":
        out["pages"] = st["pages"].to(dd)
        out["pages"][st["table"][seq, pos // c["P"]].long(), pos % c["P"]] = through(st["kv_in"], st["norm_w"], True)
    if c["kv"] == "fp8":
        out["scales"] = None
    return out


def exact(case, seed):
    if case["kind"] not in ("attn", "append"):
        return None
    st = prepare(case, seed)
    return _attn_exact(st) if case["kind"] == "attn" else _append_exact(st)

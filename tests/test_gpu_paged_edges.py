"""GPU tier: the paged latent cache (``smla.paged``) where its inputs leave the ordinary: lengths past the table, rows and
projections that are not finite, refused slots, rows given back.  Tolerances as in ``test_gpu_paged``."""
import random

import pytest
import torch

from conftest import announce
from oracle import paged as op
from test_gpu_paged import BF16, _apply, _cache, _check_attn, _cu, _i32, _tables, _to

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("window,first", [(1, 4), (20, 4), (20, 0), (3, 1), (40, 70), (5, 64), (5, 65), (30, 1 << 29), (1 << 29, 3)])
def test_attn_window_past_the_table(dev, window, first, kv):
    """Rows past the table's columns are not there; the first rows are, also where the whole window lies past the table."""
    from smla import paged
    announce(f"paged_attn lengths past a table of 64 rows, window={window} first={first} {kv}")
    pages, scales, table = _cache(201, [64] * 5, 16, 512, kv)
    lens, cu = [64, 66, 83, 100, 84], _cu([3, 2, 3, 1, 20])
    q = torch.randn(cu[-1], 16, 512, generator=torch.Generator().manual_seed(window % 97 + first % 89)).to(torch.bfloat16)
    dq, dp, ds, dt = _to(dev, q, pages, scales, table)
    out = paged.paged_attn(dq, dp, dt, _i32(lens, dev), _i32(cu, dev), 512 ** -0.5, None, window, first, page_scales=ds)
    torch.cuda.synchronize()
    _check_attn(out, q, pages, scales, table, lens, cu, None, window, first)


@pytest.mark.parametrize("window,first,length", [(150, 1550, 1700), (10, 1 << 29, 5000), (10, 1500, 5000), (700, 900, 2000)])
def test_attn_window_past_the_table_split(dev, window, first, length):
    """The same with rows enough that tiles are split over workgroups."""
    from smla import paged
    announce(f"paged_attn a token at {length} over a table of 1600 rows, window={window} first={first}")
    pages, _, table = _cache(202, [1600], 16, 576)
    q = torch.randn(2, 64, 576, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16)
    dq, dp, dt = _to(dev, q, pages, table)
    out = paged.paged_attn(dq, dp, dt, _i32([length], dev), _i32([0, 2], dev), 576 ** -0.5, None, window, first)
    torch.cuda.synchronize()
    _check_attn(out, q, pages, None, table, [length], [0, 2], None, window, first)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("capture", [False, True])
def test_refused_slots_leave_every_row(dev, kv, capture):
    """update -> append -> attn over a pool that runs out while slots share a full last page: the tokens of a refused slot
    write nothing and give 0, every older row keeps its bits, the granted slots go on, and a refused one does so
    once there are pages again."""
    from smla import paged
    announce(f"a step with refused slots, {kv}, {'captured' if capture else 'eager'}")
    S, M, P, n_pages, H, D, T = 4, 6, 8, 8, 16, 512, 52
    g = torch.Generator().manual_seed(31)
    cos, sin = _to(dev, *_tables(dev, M * P, 64))
    pages = torch.full((n_pages, P, D), float("nan"), dtype=torch.bfloat16, device=dev)
    scales = None
    if kv == "fp8":
        pages = torch.full((n_pages, P, D), 0x7f, dtype=torch.uint8, device=dev)
        scales = torch.full((n_pages, P, D // 64), float("nan"), device=dev)
    zeros = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
    table, lens, refs = torch.full((S, M), -1, dtype=torch.int32, device=dev), zeros(S), zeros(n_pages)
    parent, grow, cu = zeros(S), zeros(S), zeros(S + 1)
    q, x = torch.zeros(T, H, D, device=dev), torch.zeros(T, D, device=dev)
    mine, mine_q = [torch.zeros(T, H, D, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    res = {}

    def step():
        t, n, f, ok = paged.update_pages(pages, table, lens, refs, parent, grow, page_scales=scales)
        kw = dict(page_scales=scales, granted=ok)
        qs = paged.paged_append(q, x, pages, t, n, cu, cos, sin, kv_norm=True, q_norm=True, **kw)
        o = paged.paged_attn(qs, pages, t, n, cu, D ** -0.5, **kw)
        paged.paged_append(q, x, pages, t, n, cu, cos, sin, kv_norm=True, q_norm=True, q_out=mine_q, **kw)
        paged.paged_attn(qs, pages, t, n, cu, D ** -0.5, out=mine, **kw)
        table.copy_(t), lens.copy_(n), refs.copy_(f)
        res.update(q=qs, o=o, ok=ok)

    graph = None
    if capture:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
    dense = [[] for _ in range(S)]
    # (parents, growth, what is granted): slots 0 and 1 share the two whole pages of a prompt of 16, slots 2 and 3 take
    # five of the other six; the last goes to slot 0, then there are none until slot 0 is emptied
    plan = [([-1, -1, -1, -1], [16, 0, 17, 16], [1, 1, 1, 1]), ([0, 0, 2, 3], [0, 0, 0, 0], [1, 1, 1, 1]),
            ([0, 1, 2, 3], [1, 1, 1, 1], [1, 0, 0, 0]), ([0, 1, 2, 3], [7, 0, 2, 0], [1, 1, 1, 1]),
            ([0, 1, 2, 3], [0, 3, 1, 1], [1, 0, 0, 0]), ([0, 0, 2, 3], [0, 3, 0, 0], [1, 0, 0, 0]),
            ([-1, 1, 2, 3], [0, 1, 0, 0], [1, 0, 0, 0]), ([0, 1, 2, 3], [0, 3, 1, 1], [1, 1, 1, 0])]
    for k, (ps, gs, want_ok) in enumerate(plan):
        c = _cu(gs)
        for dst, v in ((parent, ps), (grow, gs), (cu, c)):
            dst.copy_(_i32(v, dev))
        q.copy_(torch.randn(T, H, D, generator=g))
        x.copy_(torch.randn(T, D, generator=g))
        mine.fill_(7.0), mine_q.fill_(7.0)
        t_want, l_want, r_want, ok_want, copies = op.update_pages((P, n_pages), table.tolist(), lens.tolist(), refs.tolist(), ps, gs)
        assert ok_want == want_ok
        before = pages.clone().view(torch.uint8).cpu()
        step() if graph is None else graph.replay()
        torch.cuda.synchronize()
        assert (res["ok"].tolist(), table.tolist(), lens.tolist(), refs.tolist()) == (ok_want, t_want, l_want, r_want)
        dense = [(list(dense[p]) if p >= 0 else []) if ok else dense[s] for s, (p, ok) in enumerate(zip(ps, ok_want))]
        host, hs = pages.cpu(), None if scales is None else scales.cpu()
        hp = host if scales is None else host.view(torch.float8_e4m3fn)
        new = set()
        for s in range(S):
            rows = [hp[t_want[s][j // P], j % P].double() * (1.0 if hs is None else hs[t_want[s][j // P], j % P].double().repeat_interleave(64))
                    for j in range(l_want[s])]
            for j, old in enumerate(dense[s]):
                assert torch.equal(rows[j], old), (k, s, j)
            new |= {(t_want[s][j // P], j % P) for j in range(len(dense[s]), l_want[s])}
            dense[s] = rows
        new |= {(b, j) for _, b, n in copies for j in range(n)}
        changed = (host.view(torch.uint8) != before).flatten(2).any(-1).nonzero().tolist()
        assert {tuple(i) for i in changed} <= new, k
        seen = [n if ok else -1 for n, ok in zip(l_want, ok_want)]     # a refused slot's tokens see nothing
        if c[-1]:
            _check_attn(res["o"], res["q"].cpu(), hp, hs, torch.tensor(t_want), seen, c, None, 0, 0)
        for s in range(S):
            of = slice(c[s], c[s + 1])
            if ok_want[s]:
                assert torch.equal(mine[of], res["o"][of]) and torch.equal(mine_q[of], res["q"][of])
                assert c[s] == c[s + 1] or (res["q"][of] != 0).any(-1).all()
            else:
                assert (mine[of] == 7).all() and (mine_q[of] == 7).all() and not res["o"][of].any() and not res["q"][of].any()
        assert not res["o"][c[-1]:].any() and (mine[c[-1]:] == 7).all()


def test_refused_slots_among_many(dev):
    """Sequences past a wave's lanes, every third refused, tiles split and whole: as with their tokens taken out."""
    from smla import paged
    announce("paged_attn and paged_append of 150 sequences, every third refused")
    r = random.Random(2)
    n = [r.choice([0, 1, 1, 3]) for _ in range(150)]
    lens = [k + r.randint(0, 60) for k in n]
    lens[70], n[70] = 3000, 2
    lens[69], n[69] = 900, 1
    granted = [int(b % 3 != 0) for b in range(150)]
    pages, _, table = _cache(209, lens, 16, 512)
    cu = _cu(n)
    q = torch.randn(cu[-1] + 3, 16, 512, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    dq, dp, dt = _to(dev, q, pages, table)
    ok = _i32(granted, dev)
    out = paged.paged_attn(dq, dp, dt, _i32(lens, dev), _i32(cu, dev), 512 ** -0.5, granted=ok)
    all_ = paged.paged_attn(dq, dp, dt, _i32(lens, dev), _i32(cu, dev), 512 ** -0.5, granted=torch.ones_like(ok))
    assert torch.equal(all_, paged.paged_attn(dq, dp, dt, _i32(lens, dev), _i32(cu, dev), 512 ** -0.5))
    seen = [k if ok else -1 for k, ok in zip(lens, granted)]
    _check_attn(out, q, pages, None, table, seen, cu, None, 0, 0)
    assert not out[cu[-1]:].any()
    before, cos, sin = dp.clone(), *_to(dev, *_tables(dev, 3000, 64))
    mine = torch.full_like(dq, 7.0)
    paged.paged_append(dq, dq[:, 0], dp, dt, _i32(lens, dev), _i32(cu, dev), cos, sin, q_out=mine, granted=ok)
    wrote = (dp != before).any(-1).cpu()
    for b, ok in enumerate(granted):
        for i in range(n[b]):
            j = lens[b] - n[b] + i
            assert bool(wrote[table[b, j // 16], j % 16]) == bool(ok) and bool((mine[cu[b] + i] == 7).all()) != bool(ok)
            wrote[table[b, j // 16], j % 16] = False
    assert not wrote.any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("xdt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kv,kv_norm", [("bf16", True), ("bf16", None), ("sim", True), ("sim", None), ("fp8", True), ("fp8", None)])
def test_append_keeps_what_is_not_finite(dev, bad, xdt, kv, kv_norm):
    """A channel that is not finite shows in the stored row, whatever the pages hold: as it is in bf16, as NaN over its
    64-channel block where that is scaled by its largest magnitude; other blocks, rows and queries are as without it."""
    from smla import paged
    announce(f"paged_append of {bad} {xdt} {kv} norm={kv_norm}")
    D, P, H, rd, lens = 576, 8, 3, 64, [9]
    pages, scales, table = _cache(204, lens, P, D, "fp8" if kv == "fp8" else "bf16")
    g = torch.Generator().manual_seed(4)
    q, x = torch.randn(4, H, D, generator=g).to(xdt), torch.randn(4, D, generator=g).to(xdt)
    x[1, 70], x[3, 5], x[3, 575] = bad, bad, bad
    q[2, 1, 130] = bad
    cos, sin = _tables(dev, 9, rd)
    cu, nd = [0, 4], 512
    args = _to(dev, q, x, pages, table)
    dc, dsn, ds = _to(dev, cos, sin, scales)
    out = paged.paged_append(*args[:3], args[3], _i32(lens, dev), _i32(cu, dev), dc, dsn, kv_norm=kv_norm, q_norm=True, norm_dims=nd,
                             page_scales=ds, fp8_sim=kv == "sim").double().cpu()
    got = args[2].cpu() if kv != "fp8" else args[2].cpu().view(torch.float8_e4m3fn)
    for t, p in enumerate(range(5, 9)):
        y = op.norm_rope(q[t], None, True, nd, cos[p], sin[p], 1e-6)
        assert torch.equal(out[t].isnan(), y.isnan())
        ok = ~y.isnan()
        assert ((out[t] - y).abs() <= BF16 * y.abs() + 2.0 ** -16)[ok].all()
        y = op.norm_rope(x[t, None], None, bool(kv_norm), nd, cos[p], sin[p], 1e-6)[0]
        page = int(table[0, p // P])
        val = got[page, p % P].double()
        coded = {"bf16": 0, "sim": D - rd, "fp8": D}[kv]
        if kv == "fp8":
            val = val * ds.cpu()[page, p % P].double().repeat_interleave(64)
        want = y.clone()
        blocks = want[:coded].unflatten(0, (-1, 64))
        blocks[~blocks.isfinite().all(-1)] = float("nan")
        assert torch.equal(val.isnan(), want.isnan()), t
        inf = want.isinf()
        assert torch.equal(val[inf], want[inf])
        ok = want.isfinite()
        rel = torch.full((D,), BF16, dtype=torch.float64)
        rel[:coded] = 2.0 ** -4
        # (blocks of ordinary values: the largest is at most 2^3, so a subnormal half step is under 2^-10 * 2^-5)
        assert ((val - want).abs() <= rel * want.abs() + 2.0 ** -14)[ok].all(), t


def _held(table, lens, refs, P):
    """The state is sound: every entry of a slot's rows names a page, no other entry does, refs counts them."""
    count = [0] * len(refs)
    for row, n in zip(table, lens):
        used = -(-n // P)
        assert all(p >= 0 for p in row[:used]) and all(p == -1 for p in row[used:])
        for p in row[:used]:
            count[p] += 1
    assert count == refs


@pytest.mark.parametrize("S,M,P,n_pages,D,kv", [(5, 8, 4, 30, 64, "bf16"), (64, 12, 16, 400, 64, "fp8"), (1030, 5, 4, 5000, 64, "bf16"),
                                                (9, 4000, 2, 20000, 64, "bf16")])
def test_rows_given_back(dev, S, M, P, n_pages, D, kv):
    """Growth of either sign over forked slots: pages past the shorter lengths are free again, whichever path the pool takes."""
    from smla import paged
    r = random.Random(S)
    table, lens, refs = [[-1] * M for _ in range(S)], [0] * S, [0] * n_pages
    g = torch.Generator().manual_seed(S)
    pool = torch.randint(0, 256, (n_pages, P, D * (1 if kv == "fp8" else 2)), generator=g, dtype=torch.uint8)
    pool = pool if kv == "fp8" else pool.view(torch.bfloat16)
    sc = torch.randn(n_pages, P, D // 64, generator=g) if kv == "fp8" else None
    dp, ds = _to(dev, pool, sc)
    for k in range(8):
        announce(f"update_pages with rows given back, S={S} M={M} P={P} n_pages={n_pages} {kv} step {k}")
        parent = [r.choice([s, s, s, r.randrange(S), -1]) for s in range(S)]
        have = [lens[p] if p >= 0 else 0 for p in parent]
        most = max(1, min(M * P, n_pages * P // S) // 2)
        grow = [r.choice([0, 1, r.randint(0, most), -1, -r.randint(0, h), -h, -h - 1 if r.random() < 0.1 else 0, -r.randint(0, 2 * P)])
                for h in have]
        t2, l2, r2, ok, copies = op.update_pages((P, n_pages), table, lens, refs, parent, grow)
        got = paged.update_pages(dp, *[_i32(v, dev) for v in (table, lens, refs, parent, grow)], page_scales=ds)
        torch.cuda.synchronize()
        assert [x.tolist() for x in got] == [t2, l2, r2, ok], k
        pool, sc = _apply(pool, copies, P), _apply(sc, copies, P)
        assert torch.equal(dp.cpu().view(torch.uint8), pool.view(torch.uint8)) and (sc is None or torch.equal(ds.cpu(), sc))
        table, lens, refs = t2, l2, r2
        _held(table, lens, refs, P)
    paged_empty = paged.update_pages(dp, *[_i32(v, dev) for v in (table, lens, refs, list(range(S)), [-n for n in lens])], page_scales=ds)
    assert not paged_empty[1].any() and not paged_empty[2].any() and (paged_empty[0] == -1).all() and paged_empty[3].all()


@pytest.mark.parametrize("capture", [False, True])
def test_drafts_rolled_back(dev, capture):
    """Steps of four draft tokens of which some are rejected, past page ends: the pool never loses a page, and the attention is
    that over the accepted rows."""
    from smla import paged
    announce(f"drafts rolled back, {'captured' if capture else 'eager'}")
    S, M, P, n_pages, H, D, n = 3, 8, 4, 18, 16, 512, 4
    r, g = random.Random(5), torch.Generator().manual_seed(5)
    cos, sin = _to(dev, *_tables(dev, M * P, 64))
    pages = torch.full((n_pages, P, D), float("nan"), dtype=torch.bfloat16, device=dev)
    state = [torch.full((S, M), -1, dtype=torch.int32, device=dev), _i32([0] * S, dev), _i32([0] * n_pages, dev)]
    parent, grow, cu = _i32(list(range(S)), dev), _i32([n] * S, dev), _i32(_cu([n] * S), dev)
    q, x = torch.zeros(S * n, H, D, device=dev), torch.zeros(S * n, D, device=dev)
    res = {}

    def step():
        t, l, f, ok = paged.update_pages(pages, *state, parent, grow)
        qs = paged.paged_append(q, x, pages, t, l, cu, cos, sin, kv_norm=True, q_norm=True, granted=ok)
        o = paged.paged_attn(qs, pages, t, l, cu, D ** -0.5, granted=ok)
        for a, b in zip(state, (t, l, f)):
            a.copy_(b)
        res.update(q=qs, o=o, ok=ok)

    if capture:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for a, v in zip(state, (-1, 0, 0)):
            a.fill_(v)
    lens, granted = [0] * S, 0
    for k in range(20):
        rejected = [r.randint(0, min(n, m)) if k else 0 for m in lens]
        base = [m - b for m, b in zip(lens, rejected)]
        parent.copy_(_i32([s if m + n <= M * P else -1 for s, m in enumerate(base)], dev))
        give = [n - b if p >= 0 else n for b, p in zip(rejected, parent.tolist())]
        base = [m if p >= 0 else 0 for m, p in zip(base, parent.tolist())]
        grow.copy_(_i32(give, dev))
        q.copy_(torch.randn(S * n, H, D, generator=g))
        x.copy_(torch.randn(S * n, D, generator=g))
        t_want, l_want, r_want, ok, _ = op.update_pages((P, n_pages), *[t.tolist() for t in state], parent.tolist(), give)
        base = [m if a else n for m, a, n in zip(base, ok, lens)]      # (the pool may run out: such a slot stays as it was)
        old = [pages[state[0][s].clamp(min=0).long()].reshape(-1, D)[:base[s]].clone() for s in range(S)]
        graph.replay() if capture else step()
        torch.cuda.synchronize()
        lens = [m + n if a else m for m, a in zip(base, ok)]
        granted += sum(ok)
        assert res["ok"].tolist() == ok and [t.tolist() for t in state] == [t_want, lens, r_want] and l_want == lens
        _held(t_want, lens, r_want, P)
        for s in range(S):
            now = pages[state[0][s].clamp(min=0).long()].reshape(-1, D)
            assert torch.equal(now[:base[s]], old[s])
        seen = [m if a else -1 for m, a in zip(lens, ok)]
        _check_attn(res["o"], res["q"].cpu(), pages.cpu(), None, state[0].cpu(), seen, _cu([n] * S), None, 0, 0)
    assert 20 < granted < 20 * S      # both happened


@pytest.mark.parametrize("n_pages", [20, 20000])
@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("net", [False, True])
def test_rows_given_back_past_a_fork(dev, n_pages, kv, net):
    """A slot that gives back rows of a page another slot holds, and appends: the other slot's rows keep their bits."""
    from smla import paged
    announce(f"rows given back past a fork, {n_pages} pages, {kv}, {'one call' if net else 'two calls'}")
    S, M, P, D = 3, 4, 8, 512
    cos, sin = _to(dev, *_tables(dev, M * P, 64))
    g = torch.Generator().manual_seed(3)
    pages = torch.zeros(n_pages, P, D, dtype=torch.uint8 if kv == "fp8" else torch.bfloat16, device=dev)
    scales = torch.zeros(n_pages, P, D // 64, device=dev) if kv == "fp8" else None
    state = torch.full((S, M), -1, dtype=torch.int32, device=dev), _i32([0] * S, dev), _i32([0] * n_pages, dev)

    def step(state, parent, grow, new):
        *state, ok = paged.update_pages(pages, *state, _i32(parent, dev), _i32(grow, dev), page_scales=scales)
        assert ok.tolist() == [1] * S
        if sum(new):
            x = torch.randn(sum(new), D, generator=g).to(dev)
            paged.paged_append(None, x, pages, state[0], state[1], _i32(_cu(new), dev), cos, sin, kv_norm=True, page_scales=scales,
                               granted=ok)
        torch.cuda.synchronize()
        return state

    def rows(state, s, n):
        at = state[0][s].clamp(min=0).long()
        return [t[at].flatten(0, 1)[:n].clone() for t in (pages, scales) if t is not None]

    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))  # noqa: E731
    state = step(state, [-1, -1, -1], [16, 0, 3], [16, 0, 3])
    state = step(state, [0, 0, 2], [0, 0, 0], [0, 0, 0])
    first, other, r0 = rows(state, 0, 16), rows(state, 2, 3), rows(state, 1, 12)
    assert state[0][0].tolist() == state[0][1].tolist() and state[2][:4].tolist() == [2, 2, 1, 0]
    if net:     # four rows back, one new
        state = step(state, [0, 1, 2], [0, -3, 0], [0, 1, 0])
    else:
        state = step(state, [0, 1, 2], [0, -4, 0], [0, 0, 0])
        state = step(state, [0, 1, 2], [0, 1, 0], [0, 1, 0])
    assert state[1].tolist() == [16, 13, 3]
    assert same(rows(state, 0, 16), first) and same(rows(state, 1, 12), r0) and same(rows(state, 2, 3), other)
    assert not same(rows(state, 1, 13), [t[:13] for t in first])
    assert int(state[0][0, 0]) == int(state[0][1, 0]) and int(state[0][0, 1]) != int(state[0][1, 1])
    _held(state[0].tolist(), state[1].tolist(), state[2].tolist(), P)
    # the page is its own now: it grows in place
    page = state[0][1].tolist()
    state = step(state, [0, 1, 2], [0, 2, 0], [0, 2, 0])
    assert state[0][1].tolist() == page and same(rows(state, 0, 16), first)


@pytest.mark.parametrize("length,n,D", [(45, 1, 512), (45, 4, 512), (128, 1, 576), (128, 9, 576), (1500, 1, 576), (1500, 5, 512)])
def test_attn_minus_infinity_counts_for_nothing(dev, length, n, D):
    """A row seen with a score of -inf has no share, whichever tokens are in the tile beside the one that sees it; where the
    same row scores +inf the token is NaN."""
    from smla import paged
    announce(f"paged_attn a row of +inf, {n} tokens at {length}, D={D}")
    pages, _, table = _cache(206, [length], 16, D)
    row = min(43, length - 2)
    pages[table[0, row // 16], row % 16, 5] = float("inf")
    q = torch.randn(n, 64, D, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16)
    dq, dp, dt = _to(dev, q, pages, table)
    lens = _i32([length], dev)
    out = paged.paged_attn(dq, dp, dt, lens, _i32([0, n], dev), D ** -0.5)
    kv, _ = op.rows(pages, None, table[0], length)
    kv[row] = 0.0
    for t in range(n):
        end = length - n + t + 1
        alone = paged.paged_attn(dq[t:t + 1], dp, dt, _i32([end], dev), _i32([0, 1], dev), D ** -0.5)[0].double().cpu()
        up = (q[t, :, 5] > 0) & (row < end)     # (an earlier token does not see it)
        assert alone[up].isnan().all() and out[t].cpu()[up].isnan().all()
        s = q[t].double() @ kv[:end].T * D ** -0.5
        if row < end:
            s[:, row] = float("-inf")
        want = torch.softmax(s, dim=-1) @ kv[:end, :512]
        for x in (alone, out[t].double().cpu()):
            err = (x - want).norm(dim=-1)[~up]
            assert (err <= 3 * BF16 * want.norm(dim=-1)[~up]).all(), (t, err)


def test_append_in_place(dev):
    """Dense bf16 queries may be their own output; a q_out over other parts of the inputs is refused."""
    from smla import _lib, paged
    announce("paged_append with q_out = q")
    T, H, D = 37, 5, 512
    g = torch.Generator().manual_seed(7)
    q = torch.randn(T, H, D, generator=g).to(torch.bfloat16).to(dev)
    kv = torch.randn(T, D, generator=g).to(torch.bfloat16).to(dev)
    cos, sin = _to(dev, *_tables(dev, 64, 64))
    table, lens, cu = _i32([[0, 1, 2, 3, 4]], dev), _i32([T], dev), _i32([0, T], dev)
    call = lambda q, out: paged.paged_append(q, kv, pages, table, lens, cu, cos, sin, q_norm=True, q_out=out)  # noqa: E731
    pages = torch.zeros(5, 8, D, dtype=torch.bfloat16, device=dev)
    want = call(q, None)
    mine = q.clone()
    assert call(mine, mine) is mine and torch.equal(mine, want)
    flat = torch.zeros((T + 1) * H * D, dtype=torch.bfloat16, device=dev)
    with pytest.raises(_lib.SmlaError):
        call(flat[:T * H * D].view(T, H, D), flat[H * D:].view(T, H, D))


@pytest.mark.parametrize("H,n", [(16, [1, 4, 3]), (64, [1, 40, 2])])
def test_attn_scales_of_any_value(dev, H, n):
    """e4m3 rows with scales that are no powers of two, beside such that are, negative and 0: rows are decode(code) * scale
    rounded to bf16, over which the oracle computes."""
    from smla import paged
    announce(f"paged_attn e4m3 rows of any scale, {H} heads")
    lens, D = [70, 333, 64], 576
    pages, scales, table = _cache(208, lens, 16, D, "fp8")
    g = torch.Generator().manual_seed(H)
    pick = torch.randint(0, 5, scales.shape, generator=g)
    scales = torch.where(pick == 0, scales, scales * (0.5 + torch.rand(scales.shape, generator=g)))
    scales[pick == 2] *= -1.0
    scales[(pick == 3) & (torch.rand(scales.shape, generator=g) < 0.1)] = 0.0
    rows = (pages.float() * scales.repeat_interleave(64, dim=-1)).to(torch.bfloat16)
    cu = _cu(n)
    q = torch.randn(cu[-1], H, D, generator=g).to(torch.bfloat16)
    dq, dp, ds, dt = _to(dev, q, pages, scales, table)
    out = paged.paged_attn(dq, dp, dt, _i32(lens, dev), _i32(cu, dev), D ** -0.5, page_scales=ds)
    torch.cuda.synchronize()
    _check_attn(out, q, rows, None, table, lens, cu, None, 0, 0)
    only = paged.paged_attn(dq, rows.to(dev), dt, _i32(lens, dev), _i32(cu, dev), D ** -0.5)
    assert torch.equal(out, only)

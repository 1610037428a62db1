"""GPU parity of the paged latent cache (``smla.paged``) with its float64 oracle: attention, append, slot
updates, compaction, and a run of them together.

Tolerances.  A rounding to bf16 is off by at most 2^-8 of the value.  paged_attn rounds the probabilities (each
enters numerator and denominator: the quotient moves by at most 2^-8 (sum p |v| / den + |out|)), the
partial sums of split tiles (2^-8 sum p |v| / den) and the result (2^-8 |out|); |out| <= sum p |v| / den = A, and the
fp32 scores of at most 576 products of unit variance move the weights by under 2^-9: elementwise 4 * 2^-8 A + 2^-8 A.
The roundings are independent, so over a token's values their 2-norms are each at most 2^-8 of the result's:
3 * 2^-8 of it in all, which a missing or additional row of up to a few thousand exceeds (its share of the 2-norm is
about n^-1/2)."""
import random

import pytest
import torch

from conftest import announce
from oracle import paged as op

pytestmark = pytest.mark.gpu

BF16 = 2.0 ** -8


def _cache(seed, lens, P, D, kv="bf16", extra=3, junk=0.0):
    """A pool with the sequences' pages in random order, on the CPU; rows past a length hold `junk`."""
    g = torch.Generator().manual_seed(seed)
    cols = max(1, max(-(-n // P) for n in lens))
    total = sum(-(-n // P) for n in lens) + extra
    perm = torch.randperm(total, generator=g).tolist()
    table = torch.full((len(lens), cols), -1, dtype=torch.int32)
    real = torch.zeros(total, P, dtype=torch.bool)
    for b, n in enumerate(lens):
        for c in range(-(-n // P)):
            table[b, c] = perm.pop()
            real[table[b, c], :min(P, n - c * P)] = True
    pages = torch.randn(total, P, D, generator=g)
    scales = None
    if kv == "fp8":
        scales = torch.exp2(torch.randint(-3, 3, (total, P, D // 64), generator=g).float())
        pages = (pages / scales.repeat_interleave(64, dim=-1)).clamp(-448, 448).to(torch.float8_e4m3fn)
        if junk:
            pages.view(torch.uint8)[~real] = 0x7f     # NaN
    else:
        pages = pages.to(torch.bfloat16)
        if junk:
            pages[~real] = junk
    return pages, scales, table


def _i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _cu(n):
    cu = [0]
    for k in n:
        cu.append(cu[-1] + k)
    return cu


def _to(dev, *ts):
    return [None if t is None else t.to(dev) for t in ts]


def _check_attn(out, q, pages, scales, table, lens, cu, sink, window, first):
    D = q.shape[-1]
    want, spread = op.paged_attn(q, pages, table, lens, cu, D ** -0.5, sink, window, first, scales=scales)
    got = out.double().cpu()[:cu[-1]]
    want, spread = want[:cu[-1]], spread[:cu[-1]]
    err = (got - want).abs()
    worst = (err - (5 * BF16 * spread + 1e-30)).max().item()
    assert worst <= 0, f"elementwise: {worst} past the bound"
    norm = want.norm(dim=-1)
    rel = (got - want).norm(dim=-1) - 3 * BF16 * norm
    assert rel.max().item() <= 0, f"a token's 2-norm is off by {((got - want).norm(dim=-1) / norm.clamp(min=1e-30)).max().item()}"
    assert (got[norm == 0] == 0).all()


def _run_attn(dev, n, lens, H, D, P, kv="bf16", window=0, first=0, sink=True, seed=0, junk=0.0, pad=0):
    from smla import paged
    pages, scales, table = _cache(seed, lens, P, D, kv, junk=junk)
    g = torch.Generator().manual_seed(seed + 1)
    cu = _cu(n)
    q = torch.randn(cu[-1] + pad, H, D, generator=g).to(torch.bfloat16)
    sk = torch.randn(H, generator=g) if sink else None
    dq, dp, ds, dt, dk = _to(dev, q, pages, scales, table, sk)
    out = paged.paged_attn(dq, dp, dt, _i32(lens, dev), _i32(cu, dev), D ** -0.5, dk, window, first, page_scales=ds)
    torch.cuda.synchronize()
    if pad:
        assert (out[cu[-1]:] == 0).all()
    _check_attn(out, q, pages, scales, table, lens, cu, sk, window, first)
    return out, (dq, dp, ds, dt, dk)


@pytest.mark.parametrize("H,D,P", [(64, 576, 64), (16, 512, 16), (1, 512, 1), (3, 576, 8), (128, 576, 128), (80, 512, 32),
                                   (65, 576, 24)])
@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_attn_head_layouts_and_pages(dev, H, D, P, kv):
    announce(f"paged_attn H={H} D={D} P={P} {kv}")
    _run_attn(dev, [1, 5, 2, 7], [1, 5, 67, 130], H, D, P, kv, seed=H + P)


@pytest.mark.parametrize("n", [2, 3, 4, 5, 6, 7])
@pytest.mark.parametrize("kv,D", [("bf16", 576), ("fp8", 512)])
def test_attn_tiles_of_both_sizes(dev, n, kv, D):
    """64 to 224 q rows a sequence: tiles of 64 and of 96, full and partly filled."""
    announce(f"paged_attn {n} tokens of 32 heads {kv}")
    _run_attn(dev, [n, n, n], [n, 150, 333], 32, D, 16, kv, seed=n)
    _run_attn(dev, [1, n, 2 * n - 1], [70, 150, 333], 32, D, 16, kv, window=50, first=3, seed=n + 10)


@pytest.mark.parametrize("lens", [[1], [2], [31], [32], [33], [63, 64, 65], [95, 96, 97, 127, 128, 129, 255, 256, 257]])
def test_attn_one_token_lengths(dev, lens):
    announce(f"paged_attn one token, lens={lens}")
    _run_attn(dev, [1] * len(lens), lens, 16, 576, 64, seed=sum(lens))


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("B,lens", [(1, [2111]), (3, [900, 5, 1777])])
def test_attn_split_over_workgroups(dev, kv, B, lens):
    """Few tiles over long rows: every tile's states are joined."""
    announce(f"paged_attn split {kv} {lens}")
    _run_attn(dev, [1] * B, lens, 64, 576, 64, kv, seed=B)
    _run_attn(dev, [3] * B, [x + 3 for x in lens], 16, 512, 16, kv, window=0, seed=B + 7)


def test_attn_more_tiles_than_compute_units(dev):
    """A chunk of many tiles beside one long sequence, whose tile is split."""
    announce("paged_attn 300 tokens of 64 heads and one token over 1500 rows")
    _run_attn(dev, [300, 1], [300, 1500], 64, 512, 64, seed=5)


def test_attn_long_tiles_in_parts(dev):
    """Few rounds of long tiles: parts of them go through states, equal to the same tokens asked one by one."""
    from smla import paged
    announce("paged_attn 600 tokens of 64 heads over 9000 rows")
    g = torch.Generator().manual_seed(8)
    T, L, P = 600, 9000, 64
    pages = torch.randn(L // P + 4, P, 512, generator=g).to(torch.bfloat16).to(dev)
    table = torch.randperm(L // P + 4, generator=g)[:-(-L // P)].to(torch.int32)[None].to(dev)
    q = torch.randn(T, 64, 512, generator=g).to(torch.bfloat16).to(dev)
    out = paged.paged_attn(q, pages, table, _i32([L], dev), _i32([0, T], dev), 512 ** -0.5)
    kv = pages[table[0].long()].reshape(-1, 512)[:L].float()
    for t in (0, 1, 299, 598, 599):
        n = L - T + t + 1
        one = paged.paged_attn(q[t:t + 1], pages, table, _i32([n], dev), _i32([0, 1], dev), 512 ** -0.5)[0]
        p = torch.softmax(q[t].float() @ kv[:n].T * 512 ** -0.5, dim=-1)
        want = p @ kv[:n]
        for x in (out[t], one):
            assert ((x.float() - want).norm(dim=-1) <= 3 * BF16 * want.norm(dim=-1)).all(), t


@pytest.mark.parametrize("L,P", [(8170, 15), (8160, 16), (8192, 64), (8224, 32)])
def test_attn_tiles_at_the_shortest_length_of_parts(dev, L, P):
    """Around the length from which tiles are cut into parts: every row is written, whichever way is taken."""
    from smla import paged
    announce(f"paged_attn 900 tokens of 64 heads over {L} rows in pages of {P}")
    g = torch.Generator().manual_seed(L)
    T, cols = 900, -(-L // P)
    pages = torch.randn(cols, P, 512, generator=g).to(torch.bfloat16).to(dev)
    table = torch.randperm(cols, generator=g).to(torch.int32)[None].to(dev)
    q = torch.randn(T, 64, 512, generator=g).to(torch.bfloat16).to(dev)
    out = torch.full_like(q, float("nan"))
    paged.paged_attn(q, pages, table, _i32([L], dev), _i32([0, T], dev), 512 ** -0.5, out=out)
    assert not out.isnan().any()
    kv = pages[table[0].long()].reshape(-1, 512)[:L].float()
    for t in (0, 1, 333, 698, 899):
        n = L - T + t + 1
        want = torch.softmax(q[t].float() @ kv[:n].T * 512 ** -0.5, dim=-1) @ kv[:n]
        assert ((out[t].float() - want).norm(dim=-1) <= 3 * BF16 * want.norm(dim=-1)).all(), t


@pytest.mark.parametrize("window,first", [(1, 0), (1, 1), (8, 0), (8, 4), (40, 37), (128, 4), (64, 500), (1000, 2), (1 << 29, 1 << 29)])
@pytest.mark.parametrize("H", [16, 64])
def test_attn_window_and_first_rows(dev, window, first, H):
    announce(f"paged_attn window={window} first={first} H={H}")
    _run_attn(dev, [9, 1, 70], [200, 300, 70], H, 512, 16, window=window, first=first, seed=window % 1000 + first % 1000)


def test_attn_many_sequences(dev):
    """More sequences than a wave's lanes, some without tokens."""
    r = random.Random(1)
    n = [r.choice([0, 1, 1, 2]) for _ in range(150)]
    lens = [max(k, r.randint(0, 90)) for k in n]
    announce(f"paged_attn {len(n)} sequences")
    _run_attn(dev, n, lens, 8, 512, 16, seed=11, pad=5)


def test_attn_rows_behind_the_last_sequence(dev):
    from smla import paged
    announce("paged_attn padded batch, out given")
    out, (dq, dp, ds, dt, dk) = _run_attn(dev, [2, 3], [40, 50], 64, 576, 16, seed=3, pad=9)
    mine = torch.full_like(out, 7.0)
    got = paged.paged_attn(dq, dp, dt, _i32([40, 50], dev), _i32([0, 2, 5], dev), 576 ** -0.5, dk, out=mine)
    torch.cuda.synchronize()
    assert got is mine and torch.equal(mine[:5], out[:5]) and (mine[5:] == 7.0).all()


@pytest.mark.parametrize("junk", [float("nan"), float("inf")])
@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_attn_unseen_rows_may_hold_anything(dev, junk, kv):
    """NaN and infinities behind a length, in page 0 (which entries without a page read) and in rows that later
    tokens of the same tile see: a token before them is untouched, one that sees them is NaN."""
    from smla import paged
    announce(f"paged_attn junk={junk} {kv}")
    _run_attn(dev, [4, 1, 2], [45, 20, 2], 16, 512, 16, kv, seed=21, junk=junk)
    _run_attn(dev, [6], [300], 16, 512, 16, kv, window=20, first=3, seed=22, junk=junk)
    pages, scales, table = _cache(23, [45], 16, 512, kv)
    lens, cu = [45], [0, 4]
    bad = pages.clone()
    if kv == "fp8":
        bad.view(torch.uint8)[table[0, 43 // 16], 43 % 16, 5] = 0x7f
    else:
        bad[table[0, 43 // 16], 43 % 16, 5] = junk
    q = torch.randn(4, 16, 512, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    dq, dp, ds, dt = _to(dev, q, bad, scales, table)
    out = paged.paged_attn(dq, dp, dt, _i32(lens, dev), _i32(cu, dev), 512 ** -0.5, page_scales=ds).cpu()
    _check_attn(out[:2], q[:2], pages, scales, table, [43], [0, 2], None, 0, 0)   # tokens at 41, 42
    seen = out[2:]
    if junk != junk or kv == "fp8":
        assert seen.isnan().all()
    else:  # +inf: NaN where the score is +inf; a score of -inf has no share but for 0 * inf
        up = (q[2:, :, 5].float() > 0)
        assert seen[up].isnan().all()


def test_attn_bad_tables_and_lengths(dev):
    """Page ids out of range, entries of -1 and lengths past the table are rows that are not there; no token
    before row 0 sees anything."""
    from smla import paged
    announce("paged_attn bad page ids")
    pages, _, table = _cache(31, [64, 64, 64], 16, 512)
    table[0, 1], table[1, 0], table[2, 3] = pages.shape[0], -7, 2 ** 31 - 1
    q = torch.randn(9, 16, 512, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    for lens in ([64, 64, 64], [64, 15, 100], [0, 2, 1]):
        cu = [0, 3, 6, 9]
        dq, dp, dt = _to(dev, q, pages, table)
        out = paged.paged_attn(dq, dp, dt, _i32(lens, dev), _i32(cu, dev), 512 ** -0.5)
        torch.cuda.synchronize()
        _check_attn(out, q, pages, None, table, lens, cu, None, 0, 0)
    out = paged.paged_attn(dq, dp, dt, _i32([-5, 64, 64], dev), _i32([0, 3, 6, 9], dev), 512 ** -0.5, _to(dev, torch.ones(16))[0])
    assert (out[:3] == 0).all()


def test_attn_scores_of_every_size(dev):
    """Large, equal and far-apart scores; a sink above and below them; scale 0."""
    from smla import paged
    announce("paged_attn score ranges")
    pages, _, table = _cache(41, [200], 32, 576)
    q = torch.randn(2, 16, 576, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    for factor, sink in ((1.0, 90.0), (1.0, -90.0), (30.0, None), (0.0, 0.0), (1.0, float("-inf"))):
        sk = None if sink is None else torch.full((16,), sink)
        dq, dp, dt, dk = _to(dev, q * factor, pages, table, sk)
        out = paged.paged_attn(dq, dp, dt, _i32([200], dev), _i32([0, 2], dev), 576 ** -0.5, dk)
        want, spread = op.paged_attn(q * factor, pages, table, [200], [0, 2], 576 ** -0.5, sk)
        # scores of up to `factor` times unit size carry that much of the fp32 sums' error
        tol = (5 + 2 * factor) * BF16 * spread + 1e-30
        assert ((out.double().cpu() - want).abs() <= tol).all(), (factor, sink)


def test_attn_same_bits_again_and_strided_inputs(dev):
    from smla import paged
    announce("paged_attn repeatable, strided table and q")
    n, lens = [1, 3, 1], [700, 900, 20]
    out, (dq, dp, ds, dt, dk) = _run_attn(dev, n, lens, 64, 576, 32, seed=51)
    wide = torch.full((3, dt.shape[1] + 9), 5, dtype=torch.int32, device=dev)
    wide[:, :dt.shape[1]] = dt
    qs = torch.zeros(dq.shape[0], 70, 576, dtype=torch.bfloat16, device=dev)
    qs[:, 3:67] = dq
    for _ in range(3):
        again = paged.paged_attn(qs[:, 3:67], dp, wide[:, :dt.shape[1]], _i32(lens, dev), _i32(_cu(n), dev), 576 ** -0.5, dk)
        assert torch.equal(again, out)


def test_attn_equals_the_dense_path(dev):
    """A decode step over pages against sparse_attn over the same rows as a list: the same sums in another order."""
    from smla import paged
    from smla import sparse_attn as ssa
    announce("paged_attn vs sparse_attn_batched")
    pages, _, table = _cache(61, [1024, 1024], 64, 576)
    q = torch.randn(2, 64, 576, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    dq, dp, dt = _to(dev, q, pages, table)
    out = paged.paged_attn(dq, dp, dt, _i32([1024, 1024], dev), _i32([0, 1, 2], dev), 576 ** -0.5)
    kv = dp[dt.long()].reshape(2, 1024, 576).contiguous()
    ids = torch.arange(1024, dtype=torch.int32, device=dev).expand(2, 1, 1024).contiguous()
    ref = ssa.sparse_attn_batched(dq[:, None], kv, None, ids, 576 ** -0.5, dv=512)[:, 0]
    rel = (out.float() - ref.float()).norm() / ref.float().norm()
    assert rel <= 6 * BF16


def test_attn_tokens_of_no_sequence(dev):
    """Before the first sequence and behind the last: 0 in a new tensor, as they were in one that is given."""
    from smla import paged
    announce("paged_attn cu from 3 to 8 of 13 tokens")
    pages, _, table = _cache(81, [200, 90], 16, 512)
    q = torch.randn(13, 16, 512, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16)
    dq, dp, dt = _to(dev, q, pages, table)
    lens, cu = _i32([200, 90], dev), _i32([3, 5, 8], dev)
    out = paged.paged_attn(dq, dp, dt, lens, cu, 512 ** -0.5)
    assert (out[:3] == 0).all() and (out[8:] == 0).all()
    _check_attn(out[3:8], q[3:8], pages, None, table, [200, 90], [0, 2, 5], None, 0, 0)
    mine = torch.full_like(out, 7.0)
    paged.paged_attn(dq, dp, dt, lens, cu, 512 ** -0.5, out=mine)
    assert (mine[:3] == 7).all() and (mine[8:] == 7).all() and torch.equal(mine[3:8], out[3:8])
    none = paged.paged_attn(dq, dp, dt, lens, _i32([0, 0, 0], dev), 512 ** -0.5)
    assert (none == 0).all() and paged.paged_attn(dq[:0], dp, dt, lens, _i32([0, 0, 0], dev), 512 ** -0.5).shape == (0, 16, 512)


def test_attn_signs_shared_tables_and_odd_addresses(dev):
    """A negative scale is the negated query's; sequences may share a table, a page may come twice in one; a query
    that is not on a 16-byte address is the same query."""
    from smla import paged
    announce("paged_attn scale < 0, an expanded table, a repeated page, q at an odd address")
    pages, _, _ = _cache(82, [160], 16, 576)
    g = torch.Generator().manual_seed(6)
    q = torch.randn(6, 3, 576, generator=g).to(torch.bfloat16)
    table = torch.tensor([[4, 1, 1, 7, 4, 0]], dtype=torch.int32)
    dq, dp, dt = _to(dev, q, pages, table)
    lens, cu = [90, 33, 96], [0, 1, 4, 6]
    args = (dp, dt.expand(3, 6), _i32(lens, dev), _i32(cu, dev))
    out = paged.paged_attn(dq, *args, 576 ** -0.5)
    _check_attn(out, q, pages, None, table.expand(3, 6), lens, cu, None, 0, 0)
    assert torch.equal(paged.paged_attn(-dq, *args, -(576 ** -0.5)), out)
    odd = torch.empty(dq.numel() + 1, dtype=torch.bfloat16, device=dev)[1:].view_as(dq)
    odd.copy_(dq)
    assert torch.equal(paged.paged_attn(odd, *args, 576 ** -0.5), out)


@pytest.mark.parametrize("kv,D,P,n_pages", [("bf16", 576, 64, 70000), ("fp8", 512, 64, 150000)])
def test_rows_past_32_bit_offsets(dev, kv, D, P, n_pages):
    """Append, attention, a fork and a compaction on pages that lie past 4 GiB from the pool's start."""
    from smla import paged
    announce(f"a pool of {n_pages * P * D * (1 if kv == 'fp8' else 2) / 2 ** 30:.1f} GiB, {kv}")
    g = torch.Generator().manual_seed(7)
    lens, H = [200, 130], 16
    small, sscale, stable = _cache(83, lens, P, D, kv, extra=0)
    n_small = small.shape[0]
    base = n_pages - n_small - 1        # the last page stays free for the fork
    assert base * P * D * (1 if kv == "fp8" else 2) > 1 << 32
    pages = torch.empty(n_pages, P, D, dtype=torch.uint8 if kv == "fp8" else torch.bfloat16, device=dev)
    scales = None if kv != "fp8" else torch.empty(n_pages, P, D // 64, device=dev)
    pages[base:base + n_small] = small.view(torch.uint8).to(dev) if kv == "fp8" else small.to(dev)
    if scales is not None:
        scales[base:base + n_small] = sscale.to(dev)
    table = torch.where(stable >= 0, stable + base, stable)
    q = torch.randn(3, H, D, generator=g).to(torch.bfloat16)
    cu = [0, 1, 3]
    dq, dt = _to(dev, q, table)
    out = paged.paged_attn(dq, pages, dt, _i32(lens, dev), _i32(cu, dev), D ** -0.5, page_scales=scales)
    _check_attn(out, q, small, sscale, stable, lens, cu, None, 0, 0)
    # the newest three rows again, by an append of the same token: rows of unit size, elsewhere as they were
    x = torch.randn(3, D, generator=g)
    cos, sin = _tables(dev, 256, 64)
    before = pages[base:base + n_small].clone()
    paged.paged_append(None, x.to(dev), pages, dt, _i32(lens, dev), _i32(cu, dev), *_to(dev, cos, sin), page_scales=scales)
    changed = (pages[base:base + n_small] != before).any(-1).cpu()
    want = torch.zeros_like(changed)
    for b, p in ((0, 199), (1, 128), (1, 129)):
        want[stable[b, p // P], p % P] = True
    assert torch.equal(changed, want)
    # slot 1 becomes a copy of slot 0, whose tail page goes to the pool's last page
    refs = torch.ones(n_pages, dtype=torch.int32, device=dev)
    refs[-1] = 0
    t2, l2, r2, ok = paged.update_pages(pages, dt, _i32(lens, dev), refs, _i32([0, 0], dev), _i32([0, 0], dev), page_scales=scales)
    assert ok.tolist() == [1, 1] and l2.tolist() == [200, 200] and int(t2[1, 3]) == n_pages - 1
    assert torch.equal(pages[-1, :8].view(torch.uint8), pages[int(dt[0, 3]), :8].view(torch.uint8))
    if scales is not None:
        assert torch.equal(scales[-1, :8], scales[int(dt[0, 3]), :8])
    # only the two slots' pages are live: they move to the pool's start
    refs = torch.zeros_like(refs)
    for page in t2[t2 >= 0].tolist():
        refs[page] += 1
    rows = [pages[t2[s].long()].reshape(-1, D)[:200].clone().view(torch.uint8) for s in range(2)]
    t3, r3, live = paged.compact_pages(pages, t2, refs, page_scales=scales)
    assert int(live) == int((refs > 0).sum()) == int(t3.max()) + 1 and int(r3.sum()) == int(refs.sum())
    for s in range(2):
        assert torch.equal(pages[t3[s].long()].reshape(-1, D)[:200].view(torch.uint8), rows[s])


def test_layers_past_32_bit_offsets(dev):
    """One launch over layers of more than 4 GiB together: a fork copies its tail page, and a compaction moves pages, in each."""
    from smla import paged
    announce("update and compact over 5 layers of 0.9 GiB")
    layers, n_pages, P, D = 5, 13000, 64, 576
    pages = torch.empty(layers, n_pages, P, D, dtype=torch.bfloat16, device=dev)
    fill = torch.randn(layers, 2, P, D, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).to(dev)
    pages[:, -2:] = fill
    table = _i32([[n_pages - 2, n_pages - 1], [-1, -1]], dev)
    refs = torch.zeros(n_pages, dtype=torch.int32, device=dev)
    refs[-2:] = 1
    args = table, _i32([100, 0], dev), refs, _i32([0, 0], dev), _i32([0, 3], dev)
    t2, l2, r2, ok = paged.update_pages(pages, *args)
    assert t2.tolist() == [[n_pages - 2, n_pages - 1], [n_pages - 2, 0]] and l2.tolist() == [100, 103] and ok.tolist() == [1, 1]
    assert torch.equal(pages[:, 0, :36], fill[:, 1, :36])
    t3, r3, live = paged.compact_pages(pages, t2, r2)
    assert t3.tolist() == [[1, 2], [1, 0]] and int(live) == 3 and r3[:3].tolist() == [1, 2, 1]
    assert torch.equal(pages[:, 1:3], fill) and torch.equal(pages[:, 0, :36], fill[:, 1, :36])


def test_two_graphs_and_several_calls_in_one(dev):
    """Two calls captured into one graph and one into another: every replay gives what the eager calls give, whichever ran
    before, with the lengths of the moment."""
    from smla import paged
    announce("paged_attn in two graphs")
    pages, _, table = _cache(84, [700, 300], 16, 576)
    q = torch.randn(2, 64, 576, generator=torch.Generator().manual_seed(8)).to(torch.bfloat16)
    dq, dp, dt = _to(dev, q, pages, table)
    lens, cu = _i32([700, 300], dev), _i32([0, 1, 2], dev)
    one = lambda: paged.paged_attn(dq, dp, dt, lens, cu, 576 ** -0.5)  # noqa: E731
    two = lambda: paged.paged_attn(dq, dp, dt, lens, cu, 576 ** -0.5, window=100, first=2)  # noqa: E731
    one(), two()
    torch.cuda.synchronize()
    a, b = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(a):
        a_one, a_two = one(), two()
    with torch.cuda.graph(b):
        b_one = one()
    for k, n in enumerate(([700, 300], [1, 300], [512, 33], [699, 0], [700, 300])):
        lens.copy_(_i32(n, dev))
        (a if k % 2 else b).replay()
        (b if k % 2 else a).replay()
        torch.cuda.synchronize()
        want = one(), two()
        assert torch.equal(a_one, want[0]) and torch.equal(a_two, want[1]) and torch.equal(b_one, want[0]), n


# ---------------------------------------------------------------------------------------------
def _tables(dev, n, rd):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rd, 2, dtype=torch.float64) / max(rd, 1))
    return a.cos().float(), a.sin().float()


def _run_append(dev, n, lens, H, D, P, xdt, kv, q_norm, kv_norm, rd=64, norm_dims=None, seed=0, pad=0, n_pos=None):
    """Norms and rotation are a few fp32 operations on values of unit size (2^-24 each, 2^-18 of the head's largest
    covers them); a bf16 result is off by 2^-8 of its value, an e4m3 one by 2^-4 of it or half a
    subnormal step (2^-10 of the scale), a round-tripped one by both roundings (the second is exact)."""
    from smla import paged
    pages, scales, table = _cache(seed, lens, P, D, "fp8" if kv == "fp8" else "bf16")
    g = torch.Generator().manual_seed(seed + 1)
    cu, T = _cu(n), sum(n) + pad
    nd = min(D, 512) if norm_dims is None else norm_dims
    q = torch.randn(T, H, D, generator=g).to(xdt)
    x = torch.randn(T, D + 128, generator=g).to(xdt)
    w = (1 + 0.1 * torch.randn(nd, generator=g)) if kv_norm == "w" else kv_norm
    qw = (1 + 0.1 * torch.randn(nd, generator=g)) if q_norm == "w" else q_norm
    cos, sin = _tables(dev, n_pos or max(lens), rd)
    dq, dx, dp, ds, dt, dc, dsn = _to(dev, q, x, pages, scales, table, cos, sin)
    dw, dqw = [t.to(dev) if isinstance(t, torch.Tensor) else t for t in (w, qw)]
    out = paged.paged_append(dq if H else None, dx[:, 128:], dp, dt, _i32(lens, dev), _i32(cu, dev), dc, dsn, kv_norm=dw, q_norm=dqw,
                             norm_dims=nd, page_scales=ds, fp8_sim=kv == "sim")
    torch.cuda.synchronize()
    got = dp.cpu() if kv != "fp8" else dp.cpu().view(torch.float8_e4m3fn)
    gsc = None if ds is None else ds.cpu()
    touched = torch.zeros(pages.shape[:2], dtype=torch.bool)
    for t, (b, p) in enumerate(op.positions(lens, cu)):
        if rd and p >= cos.shape[0] or p < 0:
            if H:
                assert (out[t] == 0).all()
            continue
        as_w = lambda v: v if isinstance(v, torch.Tensor) else None  # noqa: E731
        if H:
            y = op.norm_rope(q[t], as_w(qw), qw is not None and qw is not False, nd, cos[p], sin[p], 1e-6)
            tol = BF16 * y.abs() + 2.0 ** -18 * y.abs().amax(-1, keepdim=True)
            assert ((out[t].double().cpu() - y).abs() <= tol).all(), f"token {t} query"
        y = op.norm_rope(x[t, None, 128:], as_w(w), w is not None and w is not False, nd, cos[p], sin[p], 1e-6)[0]
        fine = 2.0 ** -18 * y.abs().max()
        page = int(table[b, p // P])
        touched[page, p % P] = True
        if kv == "bf16":
            assert ((got[page, p % P].double() - y).abs() <= BF16 * y.abs() + fine).all(), f"token {t} row"
            continue
        coded = D if kv == "fp8" else D - rd
        s = op.fp8_scale(y[:coded])
        if kv == "fp8":
            sg = gsc[page, p % P].double()
            amax = y.unflatten(-1, (-1, 64)).abs().amax(-1)
            edge = torch.log2(amax / 448.0)
            near = (edge - edge.round()).abs() < 1e-5      # a scale may go either way only on a power of two
            assert ((sg == s) | near).all()
            val = got[page, p % P].double() * sg.repeat_interleave(64)
        else:
            val = got[page, p % P].double()
        step = torch.zeros(D, dtype=torch.float64)
        step[:coded] = 2.0 ** -10 * 2 * s.repeat_interleave(64)
        rel = torch.full((D,), BF16, dtype=torch.float64)
        rel[:coded] = 2.0 ** -4
        assert ((val - y).abs() <= rel * y.abs() + step + fine).all(), f"token {t} coded row"
    # every other row is as it was
    raw = lambda t: t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t.view(torch.int16)  # noqa: E731
    assert torch.equal(raw(got)[~touched], raw(pages)[~touched])
    if gsc is not None:
        assert torch.equal(gsc[~touched], scales[~touched])
    if pad and H:
        assert (out[cu[-1]:] == 0).all()


@pytest.mark.parametrize("xdt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kv", ["bf16", "sim", "fp8"])
@pytest.mark.parametrize("H,D,P", [(64, 512, 64), (16, 576, 16), (1, 512, 1), (5, 128, 8), (3, 1024, 24), (2, 640, 32)])
def test_append_forms(dev, xdt, kv, H, D, P):
    announce(f"paged_append H={H} D={D} P={P} {xdt} {kv}")
    _run_append(dev, [1, 4, 9], [1, 33, 70], H, D, P, xdt, kv, True, "w", seed=H + D)


@pytest.mark.parametrize("q_norm,kv_norm", [(None, None), (False, True), ("w", "w"), (True, None)])
def test_append_norms(dev, q_norm, kv_norm):
    announce(f"paged_append norms {q_norm} {kv_norm}")
    _run_append(dev, [2, 0, 3], [20, 7, 3], 4, 576, 16, torch.float32, "bf16", q_norm, kv_norm, seed=3, pad=4)
    _run_append(dev, [2], [20], 4, 576, 16, torch.bfloat16, "bf16", q_norm, kv_norm, norm_dims=576, seed=4)
    _run_append(dev, [2], [20], 0, 192, 16, torch.bfloat16, "bf16", q_norm, kv_norm, norm_dims=100, rd=4, seed=5)


def test_append_without_rotation_and_past_the_tables(dev):
    announce("paged_append rd 0; positions past the rotation tables")
    _run_append(dev, [3, 2], [30, 2], 2, 128, 8, torch.float32, "bf16", True, True, rd=0, seed=6)
    _run_append(dev, [3, 2], [30, 2], 2, 128, 8, torch.float32, "bf16", True, True, n_pos=29, seed=7)


@pytest.mark.parametrize("xdt,T,kv", [(torch.bfloat16, 4100, "bf16"), (torch.float32, 2100, "fp8")])
def test_append_of_a_long_prompt(dev, xdt, T, kv):
    """A call of a long prompt gives the bits of the same tokens in three calls."""
    from smla import paged
    announce(f"paged_append {T} tokens of 64 heads, {xdt} {kv}")
    H, D, P = 64, 512, 64
    g = torch.Generator().manual_seed(T)
    q = torch.randn(T, H, D, generator=g).to(xdt).to(dev)
    x = torch.randn(T, D, generator=g).to(xdt).to(dev)
    cos, sin = _to(dev, *_tables(dev, T, 64))
    cols = -(-T // P)
    table = torch.randperm(cols, generator=g).to(torch.int32)[None].to(dev)
    pools = []
    for cuts in ([0, T], [0, T // 3, 2 * T // 3, T]):
        pages = torch.zeros(cols, P, D, dtype=torch.uint8 if kv == "fp8" else torch.bfloat16, device=dev)
        scales = torch.zeros(cols, P, D // 64, device=dev) if kv == "fp8" else None
        out = [paged.paged_append(q[a:b], x[a:b], pages, table, _i32([b], dev), _i32([0, b - a], dev), cos, sin, kv_norm=True,
                                  q_norm=True, page_scales=scales) for a, b in zip(cuts, cuts[1:])]
        pools.append((torch.cat(out), pages, scales))
    for one, three in zip(*pools):
        assert one is None or torch.equal(one, three)
    assert pools[0][0].isfinite().all() and (pools[0][0] != 0).any(-1).all()


def test_append_many_sequences(dev):
    r = random.Random(4)
    n = [r.choice([0, 1, 2]) for _ in range(200)]
    announce("paged_append 200 sequences")
    _run_append(dev, n, [k + r.randint(0, 20) for k in n], 2, 128, 4, torch.float32, "bf16", True, "w", seed=8, pad=3)


def test_append_bad_tables(dev):
    """Rows without a page are not stored anywhere; the queries are made all the same."""
    from smla import paged
    announce("paged_append bad page ids")
    pages = torch.ones(3, 4, 128, dtype=torch.bfloat16, device=dev)
    table = _i32([[0, -1], [3, 2], [2 ** 31 - 1, -(2 ** 31)]], dev)
    cos, sin = _to(dev, *_tables(dev, 64, 64))
    q, kv = torch.randn(6, 2, 128, device=dev), torch.randn(6, 128, device=dev)
    mine = torch.full((6, 2, 128), 3.0, dtype=torch.bfloat16, device=dev)
    out = paged.paged_append(q, kv, pages, table, _i32([6, 4, 40], dev), _i32([0, 2, 4, 6], dev), cos, sin, q_out=mine)
    torch.cuda.synchronize()
    assert (pages == 1).all() and out is mine and (mine != 3.0).any(-1).all()
    # a length below its tokens: those before row 0 write nothing
    mine.fill_(3.0)
    paged.paged_append(q, kv, pages, table, _i32([1, 0, -9], dev), _i32([0, 2, 4, 6], dev), cos, sin, q_out=mine)
    torch.cuda.synchronize()
    assert (mine[0] == 3).all() and (mine[1] != 3).any() and (mine[2:] == 3).all()
    assert (pages[0, 0] != 1).any() and (pages[0, 1:] == 1).all() and (pages[1:] == 1).all()


# ---------------------------------------------------------------------------------------------
def _state(r, S, M, P, n_pages):
    """A reachable state: the oracle's updates from an empty one."""
    t, lens, refs = [[-1] * M for _ in range(S)], [0] * S, [0] * n_pages
    for _ in range(6):
        parent = [r.choice([s, s, r.randrange(S), -1]) for s in range(S)]
        grow = [r.choice([0, 1, r.randrange(max(1, M * P // 3))]) for _ in range(S)]
        t, lens, refs, _, _ = op.update_pages((P, n_pages), t, lens, refs, parent, grow)
    return t, lens, refs


def _pool(seed, layers, n_pages, P, D, kv):
    g = torch.Generator().manual_seed(seed)
    shape = (layers, n_pages, P, D) if layers else (n_pages, P, D)
    if kv == "fp8":
        return torch.randint(0, 256, shape, generator=g, dtype=torch.uint8), torch.randn(*shape[:-1], D // 64, generator=g)
    return torch.randn(*shape, generator=g).to(torch.bfloat16), None


def _apply(pool, moves, P):
    """The pool after copies [(source, destination, rows)], read from the state before them."""
    if pool is None:
        return None
    new = pool.clone()
    for a, b, k in moves:
        new[..., b, :k, :] = pool[..., a, :k, :]
    return new


@pytest.mark.parametrize("S,M,P,n_pages,layers,D,kv", [
    (1, 1, 1, 1, 0, 512, "bf16"), (1, 4, 16, 6, 0, 576, "fp8"), (5, 7, 3, 20, 2, 64, "bf16"), (16, 9, 8, 70, 3, 128, "fp8"),
    (64, 12, 16, 400, 0, 512, "bf16"), (1500, 5, 4, 5000, 0, 64, "bf16"), (40, 300, 2, 9000, 1, 64, "fp8"),
    (1024, 32, 2, 16384, 0, 64, "bf16"), (9, 2500, 4, 20000, 0, 64, "bf16"), (7, 5000, 1, 33000, 2, 64, "fp8")])
def test_update_pages(dev, S, M, P, n_pages, layers, D, kv):
    from smla import paged
    r = random.Random(S + M)
    for k in range(3):
        announce(f"update_pages S={S} M={M} P={P} n_pages={n_pages} layers={layers} {kv} step {k}")
        table, lens, refs = _state(r, S, M, P, n_pages)
        parent = [r.choice([s, r.randrange(S), r.randrange(S), -1, -2 if r.random() < 0.1 else s, S if r.random() < 0.1 else s])
                  for s in range(S)]
        grow = [r.choice([0, 1, r.randrange(M * P + 2), -1 if r.random() < 0.2 else 0]) for _ in range(S)]
        pool, sc = _pool(k, layers, n_pages, P, D, kv)
        t2, l2, r2, ok, copies = op.update_pages((P, n_pages), table, lens, refs, parent, grow)
        dp, ds = _to(dev, pool, sc)
        ins = [_i32(v, dev) for v in (table, lens, refs, parent, grow)]
        for again in range(2):      # the inputs are as they were, so a second call gives the same
            got = paged.update_pages(dp, *ins, page_scales=ds)
            torch.cuda.synchronize()
            for name, x, y in zip(("table", "lens", "refs", "granted"), got, (t2, l2, r2, ok)):
                assert x.cpu().tolist() == y, name
            assert torch.equal(dp.cpu().view(torch.uint8), _apply(pool, copies, P).view(torch.uint8))
            if sc is not None:
                assert torch.equal(ds.cpu(), _apply(sc, copies, P))
        assert [x.cpu().tolist() for x in ins] == [table, lens, refs, parent, grow]


def test_update_pages_bad_entries(dev):
    """Page ids out of range in a table are neither copied nor counted; extreme lengths and growth are refused."""
    from smla import paged
    announce("update_pages bad entries")
    table = [[9, -5, 2], [0, 1, -1], [-1, -1, -1], [2 ** 31 - 1, 3, -1]]
    lens, refs = [10, 5, 0, 6], [1, 1, 1, 1, 0, 0, 0, 0, 0]
    for parent, grow in (([1, 0, 3, 0], [0, 0, 1, 2]), ([0, 1, 2, 3], [2 ** 31 - 1, 0, 2 ** 31 - 1, 1]),
                         ([-2 ** 31, 2 ** 31 - 1, 1, 1], [0, 0, -2 ** 31, 0])):
        pool, _ = _pool(1, 0, 9, 4, 64, "bf16")
        t2, l2, r2, ok, copies = op.update_pages((4, 9), table, lens, refs, parent, grow)
        dp = pool.to(dev)
        got = paged.update_pages(dp, *[_i32(v, dev) for v in (table, lens, refs, parent, grow)])
        for x, y in zip(got, (t2, l2, r2, ok)):
            assert x.cpu().tolist() == y
        assert torch.equal(dp.cpu(), _apply(pool, copies, 4))


@pytest.mark.parametrize("S,M,P,n_pages,layers,D,kv", [
    (1, 1, 1, 1, 0, 512, "bf16"), (3, 5, 16, 9, 2, 576, "fp8"), (8, 9, 8, 60, 0, 64, "bf16"), (30, 300, 2, 9000, 0, 64, "fp8"),
    (64, 64, 4, 20000, 1, 64, "bf16"), (9, 100, 2, 1025, 3, 64, "bf16"), (9, 2000, 1, 16384, 0, 64, "bf16"),
    (9, 2000, 1, 16385, 0, 64, "bf16"), (9, 6000, 1, 50000, 0, 64, "fp8")])
def test_compact_pages(dev, S, M, P, n_pages, layers, D, kv):
    from smla import paged
    r = random.Random(S)
    for k in range(3):
        announce(f"compact_pages S={S} M={M} n_pages={n_pages} layers={layers} {kv} step {k}")
        table, lens, refs = _state(r, S, M, P, n_pages)
        if k == 1:      # random ids over the pool, some without a page, others held by no table
            table = [[r.randrange(-2, n_pages + 2) for _ in range(M)] for _ in range(S)]
            refs = [r.choice([0, 0, 1, 3, -1 if r.random() < 0.1 else 0]) for _ in range(n_pages)]
        if k == 2:
            refs = [r.choice([0, 1]) if n_pages > 1 else 1] * n_pages   # all free or all live
        pool, sc = _pool(k, layers, n_pages, P, D, kv)
        t2, r2, live, moves = op.compact_pages(table, refs)
        moves = [(a, b, P) for a, b in moves]
        dp, ds = _to(dev, pool, sc)
        dt, dr = _i32(table, dev), _i32(refs, dev)
        for again in range(2):
            got = paged.compact_pages(dp, dt, dr, page_scales=ds)
            torch.cuda.synchronize()
            assert got[0].cpu().tolist() == t2 and got[1].cpu().tolist() == r2 and got[2].tolist() == [live]
            assert torch.equal(dp.cpu().view(torch.uint8), _apply(pool, moves, P).view(torch.uint8))
            if sc is not None:
                assert torch.equal(ds.cpu(), _apply(sc, moves, P))


# ---------------------------------------------------------------------------------------------
def _serve(dev, kv, capture):
    """Prompts, steps, forks and a compaction on one pool against the oracle's attention over each slot's own
    rows, kept on the host as a dense list."""
    from smla import paged
    S, M, P, n_pages, H, D = 6, 12, 8, 60, 16, 512
    g = torch.Generator().manual_seed(9)
    r = random.Random(9)
    cos, sin = _to(dev, *_tables(dev, M * P, 64))
    pages = torch.full((n_pages, P, D), float("nan"), dtype=torch.bfloat16, device=dev)
    scales = None
    if kv == "fp8":
        pages = torch.full((n_pages, P, D), 0x7f, dtype=torch.uint8, device=dev)
        scales = torch.full((n_pages, P, D // 64), float("nan"), device=dev)
    T = 40
    st = {"table": torch.full((S, M), -1, dtype=torch.int32, device=dev), "lens": torch.zeros(S, dtype=torch.int32, device=dev),
          "refs": torch.zeros(n_pages, dtype=torch.int32, device=dev), "parent": torch.zeros(S, dtype=torch.int32, device=dev),
          "grow": torch.zeros(S, dtype=torch.int32, device=dev), "cu": torch.zeros(S + 1, dtype=torch.int32, device=dev),
          "q": torch.zeros(T, H, D, device=dev), "x": torch.zeros(T, D, device=dev)}
    res = {}

    def step():
        t, n, f, ok = paged.update_pages(pages, st["table"], st["lens"], st["refs"], st["parent"], st["grow"], page_scales=scales)
        q = paged.paged_append(st["q"], st["x"], pages, t, n, st["cu"], cos, sin, kv_norm=True, q_norm=True, page_scales=scales)
        o = paged.paged_attn(q, pages, t, n, st["cu"], D ** -0.5, window=30, first=2, page_scales=scales)
        st["table"].copy_(t)
        st["lens"].copy_(n)
        st["refs"].copy_(f)
        res.update(q=q, o=o, ok=ok)

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
    for k in range(8):
        parent = list(range(S)) if k % 3 else [r.choice([s, r.randrange(S), -1]) for s in range(S)]
        have = [len(dense[p]) if p >= 0 else 0 for p in parent]
        grow = [min(r.choice([0, 1, 1, 5, 11]), M * P - h, T // S) for h in have]
        cu = _cu(grow)
        st["parent"].copy_(_i32(parent, dev))
        st["grow"].copy_(_i32(grow, dev))
        st["cu"].copy_(_i32(cu, dev))
        st["q"].copy_(torch.randn(T, H, D, generator=g))
        st["x"].copy_(torch.randn(T, D, generator=g))
        if graph is None:
            step()
        else:
            graph.replay()
        torch.cuda.synchronize()
        assert res["ok"].cpu().tolist() == [1] * S
        dense = [list(dense[p]) if p >= 0 else [] for p in parent]
        table, lens = st["table"].cpu(), st["lens"].tolist()
        host, hs = pages.cpu(), None if scales is None else scales.cpu()
        hp = host if scales is None else host.view(torch.float8_e4m3fn)
        for s in range(S):
            assert lens[s] == len(dense[s]) + grow[s]
            rows = [hp[table[s, j // P], j % P].double() * (1.0 if hs is None else hs[table[s, j // P], j % P].double().repeat_interleave(64))
                    for j in range(lens[s])]
            for j, old in enumerate(dense[s]):      # older rows are what they were, wherever they lie
                assert torch.equal(rows[j], old), (k, s, j)
            dense[s] = rows
        _check_attn(res["o"].cpu(), res["q"].cpu(), hp, hs, table, lens, cu, None, 30, 2)
        assert (res["o"][cu[-1]:] == 0).all()
        if k == 4:
            t, f, live = paged.compact_pages(pages, st["table"], st["refs"], page_scales=scales)
            st["table"].copy_(t)
            st["refs"].copy_(f)
            assert int(live) == int((f > 0).sum()) and not f[int(live):].any()


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_serving_run(dev, kv):
    announce(f"a run of updates, appends, attention and a compaction, {kv}")
    _serve(dev, kv, capture=False)


def test_serving_run_captured(dev):
    """The step captured once and replayed with other lengths, parents and tables, host work between."""
    announce("the run as replays of one graph")
    _serve(dev, "bf16", capture=True)


def test_two_streams(dev):
    """Calls on two streams at once have workspaces of their own."""
    from smla import paged
    announce("paged_attn on two streams")
    sets = []
    for k in range(2):
        pages, _, table = _cache(70 + k, [900, 700], 32, 576)
        q = torch.randn(2, 64, 576, generator=torch.Generator().manual_seed(k)).to(torch.bfloat16)
        sets.append(_to(dev, q, pages, table))
    lens, cu = _i32([900, 700], dev), _i32([0, 1, 2], dev)
    call = lambda s: paged.paged_attn(s[0], s[1], s[2], lens, cu, 576 ** -0.5)  # noqa: E731
    want = [call(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(10):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(call(sets[k]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[k]) for k in range(2) for x in got[k])

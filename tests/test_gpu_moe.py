"""GPU parity of the expert network (``smla.moe``) and the products with 4-bit weights with their float64 oracle.

Tolerances.  route: ids are equal; a weight is the float64 score rounded to fp32, at most 8 fp32 roundings of 2^-24.
linear_fp4: the products are exact in fp32 and K of them are summed in some order, (K + 1) 2^-24 of the sum of their
magnitudes, then the result's rounding (2^-8 of it for bf16, 2^-24 for fp32).  experts: the bound that the oracle derives."""
import math
import random

import pytest
import torch

from conftest import announce
from oracle import moe as om

pytestmark = pytest.mark.gpu


def _logits(seed, T, E, dtype):
    g = torch.Generator().manual_seed(seed)
    return (1.5 * torch.randn(T, E, generator=g) + 0.5 * torch.randn(E, generator=g)).to(dtype)


def _check_route(got, want):
    ids, w = got[0].cpu(), got[1].cpu().double()
    assert got[0].dtype == torch.int32 and got[1].dtype == torch.float32
    assert torch.equal(ids, want[0])
    assert torch.equal(w.isnan(), want[1].isnan())
    ok = ~want[1].isnan()
    assert ((w - want[1]).abs()[ok] <= 8 * 2.0 ** -24 * want[1].abs()[ok] + 1e-45).all()


ROUTES = [  # T, E, k, score, dtype, bias, groups, topk_groups, renorm, scale, shared
    (1, 256, 6, "sqrtsoftplus", "f32", True, 1, 1, True, 1.5, 1), (37, 256, 8, "sigmoid", "f32", True, 8, 4, True, 2.5, 0),
    (131, 100, 4, "softmax", "bf16", False, 1, 1, False, 1.0, 0), (3, 1, 1, "softmax", "f32", False, 1, 1, True, 1.0, 0),
    (5, 7, 7, "sigmoid", "bf16", True, 1, 1, False, 1.0, 2), (9, 1024, 32, "softmax", "f32", True, 16, 5, True, 1.0, 3),
    (70, 64, 2, "softmax", "bf16", False, 4, 1, True, 1.0, 0), (65, 65, 5, "sqrtsoftplus", "bf16", False, 1, 1, True, 1.0, 0),
    (12, 512, 16, "sigmoid", "bf16", False, 8, 3, False, 0.7, 0), (4, 1000, 64, "sqrtsoftplus", "f32", False, 1, 1, True, 1.0, 0),
    (17, 24, 3, "softmax", "f32", True, 24, 4, True, 1.0, 0), (600, 129, 6, "sigmoid", "f32", True, 1, 1, True, 1.0, 1),
    (300, 320, 9, "softmax", "f32", True, 2, 1, True, 1.0, 0),
]


@pytest.mark.parametrize("case", ROUTES, ids=lambda c: "-".join(map(str, c)))
def test_route(dev, case):
    from smla import moe
    T, E, k, score, dt, bias, groups, top, renorm, scale, shared = case
    announce(f"route {case}")
    x = _logits(T * 31 + E, T, E, torch.float32 if dt == "f32" else torch.bfloat16)
    b = 0.1 * torch.randn(E, generator=torch.Generator().manual_seed(E)) if bias else None
    kw = dict(score=score, groups=groups, topk_groups=top, renorm=renorm, scale=scale, shared=shared)
    want = om.route(x, k, bias=b, **kw)
    _check_route(moe.route(x.to(dev), k, bias=None if b is None else b.to(dev), **kw), want)


@pytest.mark.parametrize("score", ["softmax", "sigmoid", "sqrtsoftplus"])
@pytest.mark.parametrize("groups", [1, 4])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("E", [40, 64])
def test_route_ties_and_values_out_of_range(dev, score, groups, bias, E):
    """Equal logits, whole rows of one value, logits of -inf, +inf, NaN and the type's lowest, alone and together."""
    from smla import moe
    announce(f"route out of range {score} {groups} {bias} {E}")
    k = 7
    r = random.Random(5)
    low, inf, nan = torch.finfo(torch.float32).min, math.inf, math.nan
    rows = [[0.0] * E, [low] * E, [-inf] * E, [nan] * E, [1.0, 2.0] * (E // 2), [-inf] * (E - 3) + [1.0, -2.0, 1.0],
            [low] * (E - 2) + [3.0, 3.0], [nan] + [0.5] * (E - 1), [-inf, nan] * (E // 2), [-100.0] * 20 + [-101.0] * (E - 20),
            [80.0, 81.0] * (E // 2), [0.0, -0.0] * (E // 2)]
    rows += [[r.choice([0.25, -1.0, 3.0, -inf, low]) for _ in range(E)] for _ in range(20)]
    if score != "softmax":
        rows += [[r.choice([0.25, -1.0, nan, -inf]) for _ in range(E)] for _ in range(20)]
    if score == "sigmoid":
        rows += [[inf] * E, [r.choice([inf, -inf, 1.0]) for _ in range(E)]]
    x = torch.tensor(rows)
    b = torch.tensor([(e % 5) / 8 for e in range(E)]) if bias else None
    kw = dict(score=score, groups=groups, topk_groups=max(1, groups // 2), scale=1.5)
    _check_route(moe.route(x.to(dev), k, bias=None if b is None else b.to(dev), **kw), om.route(x, k, bias=b, **kw))
    if bias:
        b[3], b[17], b[30] = -inf, nan, inf
        _check_route(moe.route(x.to(dev), k, bias=b.to(dev), **kw), om.route(x, k, bias=b, **kw))


def test_route_order_next_to_a_border(dev):
    """Scores whose fp32 values would tie or trade places: neighbouring logits, with and without a bias that all but
    evens them out."""
    from smla import moe
    announce("route next to a border")
    E = 64
    step = torch.arange(E) * 2.0 ** -22 + 2.0      # one fp32 step apart
    x = torch.stack([step, step.flip(0), -step, 3 * step])
    for score in ("softmax", "sigmoid", "sqrtsoftplus"):
        _check_route(moe.route(x.to(dev), 9, score), om.route(x, 9, score))
        s = torch.tensor([om.scores(v, score) for v in x.double().tolist()], dtype=torch.float64)
        b = (1.0 - s[0]).float()                   # the sums differ by the bias' fp32 rounding
        _check_route(moe.route(x.to(dev), 9, score, bias=b.to(dev)), om.route(x, 9, score, bias=b))
        _check_route(moe.route(x.to(dev), 9, score, bias=b.to(dev), groups=8, topk_groups=3),
                     om.route(x, 9, score, bias=b, groups=8, topk_groups=3))


@pytest.mark.parametrize("groups", [1, 2])
def test_route_large_scores_that_the_bias_takes_away(dev, groups):
    """Scores of 100, whose fp32 steps are 2^-17, and biases that leave differences about as large; groups whose two
    largest values are large and opposite."""
    from smla import moe
    announce(f"route cancelled {groups}")
    E, k = 32, 3
    for seed in range(200):
        g = torch.Generator().manual_seed(seed)
        x = 10000 + torch.randn(1, E, generator=g)
        s = torch.tensor(om.scores(x.double().tolist()[0], "sqrtsoftplus"), dtype=torch.float64)
        b = -s.float()
        if seed % 2:                     # a few experts left near 0, all others far below
            b -= 1000.0 * (torch.arange(E) % 16 > 2 + seed % 3)
        if groups > 1:                   # two values of -+5100 to a group, which all but cancel
            b = -20000.0 - 100.0 * torch.arange(E)
            b[::16] = 5000.0
            b[1::16] = (-(s[::16] + 5000.0 + s[1::16])).float()
        kw = dict(bias=b, groups=groups, topk_groups=1)
        _check_route(moe.route(x.to(dev), k, "sqrtsoftplus", **{**kw, "bias": b.to(dev)}), om.route(x, k, "sqrtsoftplus", **kw))


def test_route_given_ids_strides_empty(dev):
    from smla import moe
    announce("route given ids")
    x = _logits(3, 33, 60, torch.float32)
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(-1, 62, (33, 5), generator=g, dtype=torch.int32)
    for score in ("softmax", "sigmoid", "sqrtsoftplus"):
        want = om.route(x, 5, score, ids=ids, scale=1.5, shared=1)
        _check_route(moe.route(x.to(dev), 5, score, ids=ids.to(dev), scale=1.5, shared=1), want)
    wide = torch.zeros(33, 200, dtype=torch.bfloat16)
    wide[:, 70:130] = x.to(torch.bfloat16)
    want = om.route(x.to(torch.bfloat16), 4, "sigmoid")
    wide = wide.to(dev)
    _check_route(moe.route(wide[:, 70:130], 4, "sigmoid"), want)
    _check_route(moe.route(wide[:, 70:130].t().contiguous().t(), 4, "sigmoid"), want)
    i, w = moe.route(wide[:0, :60], 4, shared=1)
    assert i.shape == w.shape == (0, 5)


def _packed(seed, *shape, scale=1.0):
    """Random codes of every value and scale bytes around K^-0.5 (CPU), and the float64 weights."""
    g = torch.Generator().manual_seed(seed)
    K = shape[-1]
    codes = torch.randint(0, 256, (*shape[:-1], K // 2), generator=g, dtype=torch.uint8)
    e = 125 - round(math.log2(K) / 2)
    scales = torch.randint(e - 2, e + 2, (*shape[:-1], K // 32), generator=g, dtype=torch.uint8)
    return codes, scales, om.unpack(codes, scales)


LINEARS = [  # T, N, K
    (1, 16, 32), (1, 1, 64), (1, 4096, 512), (1, 33, 4128), (2, 17, 96), (3, 100, 160), (7, 512, 1024), (8, 4096, 128),
    (15, 31, 2048), (16, 48, 8192), (17, 130, 384), (24, 2048, 1024), (31, 257, 288), (32, 64, 4096), (33, 129, 512),
    (64, 256, 256), (65, 300, 1184), (77, 1000, 4128), (128, 128, 128), (129, 513, 320), (200, 96, 64), (255, 1030, 640),
    (256, 256, 1024), (300, 77, 992), (700, 384, 1536), (1025, 640, 416),
    (16, 48, 4352), (5, 17, 14208), (6, 16, 12512), (6, 409, 11776), (20, 8383, 3296), (1722, 71, 2560), (3283, 66, 2240),
    (37, 11078, 2240), (784, 10036, 32), (719, 11074, 128), (17, 12932, 160), (1, 6848, 128), (18, 11030, 32),
]


@pytest.mark.parametrize("case", LINEARS, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_linear_fp4(dev, case, out):
    from smla import mla
    T, N, K = case
    announce(f"linear_fp4 {case} {out}")
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(T + K)).to(torch.bfloat16)
    codes, scales, w = _packed(N + K, N, K)
    dt = torch.bfloat16 if out == "bf16" else torch.float32
    y = mla.linear_fp4(x.to(dev), codes.to(dev), scales.to(dev), out_dtype=dt)
    assert y.dtype == dt and y.shape == (T, N)
    want = x.double() @ w.T
    tol = (K + 1) * 2.0 ** -24 * (x.double().abs() @ w.abs().T)
    tol = tol + (2.0 ** -8 if out == "bf16" else 2.0 ** -24) * (want.abs() + tol)
    assert ((y.cpu().double() - want).abs() <= tol).all()


def test_linear_fp4_every_code_and_scale(dev):
    """Identity rows pick single weights: all 16 codes under the scale bytes whose largest weight is finite (6 * 2^125 <
    2^128 <= 6 * 2^126, bytes up to 252) come out as they are.  Rows of the bytes above hold infinities, and the identity's
    zeros times those are NaN, as is all of byte 255."""
    from smla import mla
    announce("linear_fp4 codes and scales")
    N, K = 256, 64
    codes = torch.arange(K // 2, dtype=torch.uint8).repeat(N, 1) * 2 % 16
    codes = codes + 16 * (codes + 1)               # element i: code i mod 16
    scales = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 2)
    want = om.unpack(codes, scales)
    for T in (32, 64):
        x = torch.eye(K, dtype=torch.bfloat16)[:T]
        got = mla.linear_fp4(x.to(dev), codes.to(dev), scales.to(dev), out_dtype=torch.float32).cpu().double()
        w = want[:, :T].T
        inside = (w.abs() >= 2.0 ** -126) | (w == 0)
        inside[:, 253:] = False
        assert torch.equal(got[inside], w[inside])
        assert got[:, 253:].isnan().all() and not got[:, :253].isnan().any()


def test_linear_fp4_rows_stand_alone(dev):
    """A row of infinities or NaN changes no other row, whatever tile it shares; rows may lie apart; the batch a
    token is in changes its result by the sums' order at most."""
    from smla import mla
    announce("linear_fp4 rows")
    N, K = 200, 416
    codes, scales, w = _packed(9, N, K)
    codes, scales = codes.to(dev), scales.to(dev)
    for T in (2, 9, 40, 150, 400):
        x = torch.randn(T, K, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16).to(dev)
        clean = mla.linear_fp4(x, codes, scales, out_dtype=torch.float32)
        bad = x.clone()
        bad[T // 2] = math.nan
        bad[0, 3] = math.inf
        got = mla.linear_fp4(bad, codes, scales, out_dtype=torch.float32)
        keep = [t for t in range(T) if t not in (0, T // 2)]
        assert torch.equal(got[keep], clean[keep]) and got[T // 2].isnan().all()
        wide = torch.full((T, K + 24), math.nan, dtype=torch.bfloat16, device=dev)
        wide[:, 8:8 + K] = x
        assert torch.equal(mla.linear_fp4(wide[:, 8:8 + K], codes, scales, out_dtype=torch.float32), clean)
    lead = mla.linear_fp4(x.view(4, 100, K), codes, scales)
    assert lead.shape == (4, 100, N) and lead.dtype == torch.bfloat16
    assert mla.linear_fp4(x[:0], codes, scales).shape == (0, N)


def test_pack_fp4_is_the_oracles(dev):
    from smla import moe
    announce("pack_fp4")
    g = torch.Generator().manual_seed(11)
    for dt in (torch.float32, torch.bfloat16):
        w = torch.randn(5, 7, 96, generator=g).to(dt)
        codes, scales = moe.pack_fp4(w.to(dev))
        c, s = om.pack(w)
        assert torch.equal(codes.cpu(), c) and torch.equal(scales.cpu(), s)


EXPERTS = [  # T, E, of, k, K, I, weights, limit
    (1, 4, 4, 1, 32, 32, "fp4", None), (1, 64, 64, 6, 512, 256, "fp4", 10.0), (2, 8, 8, 3, 96, 160, "fp4", 1.0),
    (3, 16, 32, 4, 416, 96, "bf16", None), (8, 32, 32, 6, 1024, 128, "fp4", 10.0), (9, 5, 5, 5, 64, 32, "bf16", 0.5),
    (16, 128, 128, 8, 256, 64, "fp4", None), (17, 128, 128, 8, 256, 64, "fp4", None), (15, 1, 1, 1, 544, 320, "fp4", 7.0),
    (40, 8, 16, 2, 288, 96, "fp4", None), (64, 3, 3, 2, 128, 128, "bf16", 10.0), (100, 40, 40, 6, 160, 64, "fp4", 10.0),
    (130, 2, 2, 1, 64, 96, "fp4", None), (257, 7, 9, 3, 192, 224, "bf16", None), (300, 1000, 1000, 4, 64, 32, "fp4", 2.0),
    (513, 4, 4, 2, 384, 64, "fp4", 10.0), (600, 16, 16, 1, 96, 288, "bf16", 10.0),
    (16, 64, 64, 64, 64, 32, "fp4", None), (16, 1024, 1024, 64, 64, 32, "bf16", 10.0), (16, 2, 2, 2, 4096, 32, "fp4", 10.0),
    (16, 2, 2, 1, 4352, 64, "fp4", None), (5, 3, 3, 2, 32, 4096, "fp4", 10.0), (300, 2, 2, 2, 416, 352, "fp4", 10.0),
    (20, 64, 64, 64, 96, 64, "bf16", None), (900, 1024, 1024, 1, 128, 64, "fp4", None), (50, 2, 2, 1, 96, 4128, "bf16", 10.0),
]


def _experts_case(seed, T, E, of, k, K, I, kind):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, K, generator=g).to(torch.bfloat16)
    like = torch.randn(T, of, generator=g) + torch.randn(of, generator=g)
    ids = like.topk(k, dim=-1).indices.to(torch.int32)
    w = torch.rand(T, k, generator=g) + 0.1
    mats = []
    for i, (n, m) in enumerate(((I, K), (I, K), (K, I))):
        if kind == "fp4":
            mats.append(_packed(seed + i, E, n, m))
        else:
            v = (torch.randn(E, n, m, generator=g) * m ** -0.5).to(torch.bfloat16)
            mats.append((v, None, v.double()))
    return x, ids, w, mats


def _on(dev, mats):
    return [m[0].to(dev) if m[1] is None else (m[0].to(dev), m[1].to(dev)) for m in mats]


def _check_experts(y, want):
    y = y.cpu().double()
    assert not y.isnan().any()
    worst = ((y - want[0]).abs() / want[1].clamp(min=1e-30)).max().item()
    assert worst <= 1.0, worst


@pytest.mark.parametrize("case", EXPERTS, ids=lambda c: "-".join(map(str, c)))
def test_experts(dev, case):
    from smla import moe
    T, E, of, k, K, I, kind, limit = case
    announce(f"experts {case}")
    x, ids, w, mats = _experts_case(T + 7 * E, T, E, of, k, K, I, kind)
    want = om.experts(x, ids, w, *[m[2] for m in mats], limit or math.inf)
    y = moe.experts(x.to(dev), ids.to(dev), w.to(dev), *_on(dev, mats), limit=limit)
    assert y.dtype == torch.bfloat16 and y.shape == (T, K)
    _check_experts(y, want)


@pytest.mark.parametrize("T", [1, 9, 40, 400])
@pytest.mark.parametrize("kind", ["fp4", "bf16"])
@pytest.mark.parametrize("limit", [None, 10.0])
def test_experts_nan_and_infinity_stay(dev, T, kind, limit):
    """A token whose products are NaN, and an expert whose scales are, give NaN with a clamp too, to nobody else."""
    from smla import moe
    announce(f"experts nan {T} {kind} {limit}")
    E, k, K, I = 5, 2, 160, 96
    x, _, w, mats = _experts_case(T, T, E, E, k, K, I, kind)
    gate, up, down = _on(dev, mats)
    ids = torch.arange(T * k, dtype=torch.int32).view(T, k) % (E - 1)      # none has the last expert
    args = [w.to(dev), gate, up, down]
    want = moe.experts(x.to(dev), ids.to(dev), *args, limit=limit)
    assert want.isfinite().all()
    bad = x.clone()
    bad[T // 2, 7] = math.nan
    got = moe.experts(bad.to(dev), ids.to(dev), *args, limit=limit)
    assert got[T // 2].isnan().all()
    others = torch.arange(T) != T // 2
    assert torch.equal(got.cpu()[others], want.cpu()[others])
    last = gate[1] if kind == "fp4" else gate
    last[E - 1] = 255 if kind == "fp4" else math.nan
    assert torch.equal(moe.experts(x.to(dev), ids.to(dev), *args, limit=limit), want)
    ids[0, 1] = E - 1
    got = moe.experts(x.to(dev), ids.to(dev), *args, limit=limit)
    assert got[0].isnan().all() and got[1:].isfinite().all()   # (the sums' order goes with the ids)


@pytest.mark.parametrize("T", [3, 70])
def test_weights_that_begin_anywhere(dev, T):
    """Codes and scales of a product are taken at any address; the experts' have to be aligned, and are refused if not."""
    from smla import mla, moe
    announce(f"weights anywhere {T}")
    N, K = 40, 256
    codes, scales, _ = _packed(2, N, K)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16).to(dev)

    def moved(t, by):
        at = torch.empty(t.numel() + 16, dtype=t.dtype, device=dev)[by:by + t.numel()].view(t.shape)
        return at.copy_(t)
    want = mla.linear_fp4(x, codes.to(dev), scales.to(dev))
    assert torch.equal(mla.linear_fp4(x, moved(codes, 3), moved(scales, 5)), want)
    c, s, _ = _packed(3, 2, 64, 64)
    ids, w = torch.zeros(T, 1, dtype=torch.int32, device=dev), torch.ones(T, 1, device=dev)
    for pair in ((moved(c, 1), s.to(dev)), (c.to(dev), moved(s, 1))):
        with pytest.raises(ValueError, match="aligned"):
            moe.experts(x[:, :64], ids, w, pair, pair, pair)


@pytest.mark.parametrize("T", [1, 5, 16, 50, 300])
@pytest.mark.parametrize("kind", ["fp4", "bf16"])
def test_experts_ids_of_every_sort(dev, T, kind):
    """Tokens without an expert, ids out of range, the same expert twice or k times, one expert for all, negative and zero
    weights: and a token's NaN row, or an expert of NaN weights, stays with the tokens that have it."""
    from smla import moe
    announce(f"experts ids {T} {kind}")
    E, k, K, I = 6, 4, 128, 96
    x, _, w, mats = _experts_case(T, T, E, E, 1, K, I, kind)
    g = torch.Generator().manual_seed(T)
    w = torch.randn(T, k, generator=g)
    w[T // 2] = 0.0
    dense = [m[2] for m in mats]
    on = _on(dev, mats)
    sorts = [torch.randint(-2, E + 3, (T, k), generator=g), torch.randint(0, 2, (T, k), generator=g),
             torch.full((T, k), E - 1), torch.full((T, k), -1), torch.full((T, k), 2 ** 31 - 1)]
    for ids in sorts:
        ids = ids.to(torch.int32)
        y = moe.experts(x.to(dev), ids.to(dev), w.to(dev), *on, limit=10.0)
        _check_experts(y, om.experts(x, ids, w, *dense, 10.0))
    ids = torch.randint(0, E, (T, k), generator=g).to(torch.int32)
    clean = moe.experts(x.to(dev), ids.to(dev), w.to(dev), *on)
    bad = x.clone()
    bad[T - 1] = math.nan
    y = moe.experts(bad.to(dev), ids.to(dev), w.to(dev), *on)
    assert torch.equal(y[:-1], clean[:-1]) and y[-1].isnan().any()
    if kind == "fp4":
        on[0][1][2] = on[2][1][2] = 255        # expert 2 is NaN
    else:
        on[0][2], on[2][2] = math.nan, math.nan
    has = (ids == 2).any(1)
    y = moe.experts(x.to(dev), ids.to(dev), w.to(dev), *on).cpu()
    assert torch.equal(y[~has], clean.cpu()[~has]) and y[has].isnan().all()


def test_experts_largest_strides(dev):
    """Rows of x that lie apart, weights of fp64 and ids that are views; a token's result does not depend on what is
    beside it beyond its bound."""
    from smla import moe
    announce("experts strides")
    T, E, k, K, I = 70, 12, 3, 224, 96
    x, ids, w, mats = _experts_case(3, T, E, E, k, K, I, "fp4")
    on = _on(dev, mats)
    wide = torch.full((T, K + 40), math.nan, dtype=torch.bfloat16, device=dev)
    wide[:, 16:16 + K] = x.to(dev)
    clean = moe.experts(x.to(dev), ids.to(dev), w.to(dev), *on)
    ids2 = torch.full((T, 2 * k), -7, dtype=torch.int32, device=dev)
    ids2[:, ::2] = ids.to(dev)
    assert torch.equal(moe.experts(wide[:, 16:16 + K], ids2[:, ::2], w.to(dev).double(), *on), clean)
    assert moe.experts(x[:0].to(dev), ids[:0].to(dev), w[:0].to(dev), *on).shape == (0, K)
    want = om.experts(x, ids, w, *[m[2] for m in mats])
    for n in (1, 4, 16, 30):
        y = moe.experts(x[:n].to(dev), ids[:n].to(dev), w[:n].to(dev), *on)
        _check_experts(y, (want[0][:n], want[1][:n]))


def _layer(dev, E, k, K, I, shared, kind, table=None):
    from smla import moe
    g = torch.Generator().manual_seed(E + K)
    mats = []
    for i, (n, m) in enumerate(((I, K), (I, K), (K, I))):
        if kind == "fp4":
            mats.append(_packed(50 + i, E + shared, n, m))
        else:
            v = (torch.randn(E + shared, n, m, generator=g) * m ** -0.5).to(torch.bfloat16)
            mats.append((v, None, v.double()))
    router = (torch.randn(E, K, generator=g) * K ** -0.5).to(torch.bfloat16)
    bias = None if table is not None else 0.1 * torch.randn(E, generator=g)
    on = _on(dev, mats)
    w = moe.ExpertWeights(router.to(dev), *on, bias=None if bias is None else bias.to(dev),
                          table=None if table is None else table.to(dev))
    return moe.ExpertLayer(w, k=k), router, bias, [m[2] for m in mats]


@pytest.mark.parametrize("T", [1, 6, 33, 200])
@pytest.mark.parametrize("kind", ["fp4", "bf16"])
def test_layer(dev, T, kind):
    """Router product, routing, routed and shared experts as a layer runs them, the choice made by the layer's own logits."""
    announce(f"expert layer {T} {kind}")
    E, k, K, I = 24, 4, 192, 64
    layer, router, bias, dense = _layer(dev, E, k, K, I, 1, kind)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16)
    y = layer(x.to(dev))
    logits = layer.logits(x.to(dev)).cpu()
    ref = x.double() @ router.double().T
    assert ((logits.double() - ref).abs() <= (K + 1) * 2.0 ** -24 * (x.double().abs() @ router.double().abs().T)).all()
    ids, w = om.route(logits, k, "sqrtsoftplus", bias=bias, scale=1.5, shared=1)
    _check_experts(y, om.experts(x, ids, w.float(), *dense, 10.0))


def test_layer_by_token(dev):
    announce("expert layer by token")
    E, k, K, I = 16, 2, 128, 64
    table = torch.randint(0, E, (50, k), generator=torch.Generator().manual_seed(8), dtype=torch.int32)
    layer, _, _, dense = _layer(dev, E, k, K, I, 1, "fp4", table)
    x = torch.randn(3, 7, K, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16)
    tokens = torch.randint(0, 50, (3, 7), generator=torch.Generator().manual_seed(10))
    y = layer(x.to(dev), tokens.to(dev))
    assert y.shape == x.shape
    assert layer(x[:0].to(dev), tokens[:0].to(dev)).shape == (0, 7, K)
    flat = x.view(-1, K)
    ids, w = om.route(layer.logits(flat.to(dev)).cpu(), k, "sqrtsoftplus", ids=table[tokens.view(-1)], scale=1.5, shared=1)
    _check_experts(y.view(-1, K), om.experts(flat, ids, w.float(), *dense, 10.0))


@pytest.mark.parametrize("T", [1, 12, 90])
def test_layer_captured(dev, T):
    """A captured layer replayed with other tokens gives the eager results, with eager work between the replays; two
    graphs and a stream beside do not share anything."""
    announce(f"expert layer captured {T}")
    K = 192
    layer, *_ = _layer(dev, 24, 4, K, 64, 1, "fp4")
    codes, scales, _ = _packed(77, 130, K)
    codes, scales = codes.to(dev), scales.to(dev)
    from smla import mla

    def work(x):
        return layer(x), mla.linear_fp4(x, codes, scales, out_dtype=torch.float32)

    xs = [torch.randn(T, K, generator=torch.Generator().manual_seed(s)).to(torch.bfloat16).to(dev) for s in range(5)]
    want = [work(x) for x in xs]
    side = torch.cuda.Stream()
    graphs = []
    for i in range(2):
        x = xs[i].clone()
        with torch.cuda.stream(side):
            work(x)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = work(x)
        graphs.append((graph, x, y))
    for r in range(6):
        for i, (graph, x, y) in enumerate(graphs):
            x.copy_(xs[(r + i) % 5])
            graph.replay()
        for i, (graph, x, y) in enumerate(graphs):
            for a, b in zip(y, want[(r + i) % 5]):
                assert torch.equal(a, b)
        eager = work(xs[r % 5])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, want[r % 5]))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        a = work(xs[3])
    b = work(xs[4])
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(a + b, want[3] + want[4]))


def test_ops_are_registered(dev):
    """The calls are torch ops: fake tensors give shapes, and a leaf that asks for a gradient is refused as the
    framework's others are."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from smla import moe, ops
    announce("moe ops")
    with FakeTensorMode():
        x = torch.empty(6, 64, dtype=torch.bfloat16, device="cuda")
        i, w = ops.route_op(torch.empty(6, 8, device="cuda"), None, 3, 0, 1, 1, True, 1.0, 1, None)
        assert i.shape == w.shape == (6, 4) and i.dtype == torch.int32
        c, s = torch.empty(8, 32, 32, dtype=torch.uint8, device="cuda"), torch.empty(8, 32, 2, dtype=torch.uint8, device="cuda")
        assert ops.linear_fp4_op(x, c[0], s[0], torch.float32).shape == (6, 32)
        d, t = torch.empty(8, 64, 16, dtype=torch.uint8, device="cuda"), torch.empty(8, 64, 1, dtype=torch.uint8, device="cuda")
        assert ops.experts_op(x, i, w, c, c, d, s, s, t, 1.0).shape == (6, 64)
    for bad in (dict(k=9), dict(k=3, groups=3), dict(k=0)):
        with pytest.raises(Exception):
            moe.route(torch.zeros(2, 8, device=dev), **bad)

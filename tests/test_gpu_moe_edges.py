"""GPU tier: the expert network at the ends of what its entry points take.  Tolerances as in test_gpu_moe.py."""
import math

import pytest
import torch

from conftest import announce
from oracle import moe as om
from test_gpu_moe import _check_experts, _experts_case, _layer, _on, _packed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", [(70001, 2, 8, 64, 32, 20000), (300000, 6, 8, 32, 32, 100000), (1100000, 1, 4, 32, 32, 550000)],
                         ids=lambda c: "-".join(map(str, c)))
def test_experts_of_many_tokens(dev, case):
    """Tokens past one launch of the last sum (65535) and past the choices of one call (2^20): the same as in parts, bit for bit (of
    one tile form), and right at the borders."""
    from smla import moe
    T, k, E, K, I, part = case
    announce(f"experts of many tokens {case}")
    x, ids, w, mats = _experts_case(T, T, E, E, k, K, I, "fp4")
    on = _on(dev, mats)
    xd, idd, wd = x.to(dev), ids.to(dev), w.to(dev)
    y = moe.experts(xd, idd, wd, *on, limit=10.0)
    for t in range(0, T, part):
        assert torch.equal(y[t:t + part], moe.experts(xd[t:t + part], idd[t:t + part], wd[t:t + part], *on, limit=10.0))
    rows = [t for b in (0, 65535, 2 * 65535, T // 2, (1 << 20) // k, T) for t in range(b - 3, b + 3) if 0 <= t < T]
    _check_experts(y[rows], om.experts(x[rows], ids[rows], w[rows], *[m[2] for m in mats], 10.0))


def test_rows_that_lie_far_apart(dev):
    """Rows of x more than 2^20 (products: 2^22) elements apart, and 2^30 in all: as the packed ones."""
    from smla import mla, moe
    announce("rows far apart")
    E, k, K, I = 4, 2, 64, 32
    x, ids, w, mats = _experts_case(5, 1100, E, E, k, K, I, "fp4")
    on = _on(dev, mats)
    codes, scales, _ = _packed(6, 48, K)
    codes, scales = codes.to(dev), scales.to(dev)
    for T, ld in ((3, (1 << 20) + 8), (1100, 1 << 20), (3, (1 << 22) + 8)):
        far = torch.empty(T * ld, dtype=torch.bfloat16, device=dev).as_strided((T, K), (ld, 1))
        far.copy_(x[:T])
        near, i, v = x[:T].to(dev), ids[:T].to(dev), w[:T].to(dev)
        assert torch.equal(moe.experts(far, i, v, *on), moe.experts(near, i, v, *on))
        assert torch.equal(mla.linear_fp4(far, codes, scales), mla.linear_fp4(near, codes, scales))


def test_layer_of_tokens_outside_the_table(dev):
    """A padded batch's token ids (-1, the vocabulary's size, far past it) have the shared expert alone, the others their rows'
    experts; eager and captured."""
    announce("layer of tokens outside the table")
    E, k, K, I, V = 16, 2, 128, 64, 50
    table = torch.randint(0, E, (V, k), generator=torch.Generator().manual_seed(8), dtype=torch.int32)
    layer, _, _, dense = _layer(dev, E, k, K, I, 1, "fp4", table)
    x = torch.randn(2, 4, K, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16)
    tokens = torch.tensor([[0, V - 1, -1, V], [7, -V, 2 ** 31 - 1, -2 ** 31]])
    flat, t = x.view(-1, K), tokens.view(-1)
    inside = (t >= 0) & (t < V)
    given = torch.where(inside[:, None], table[t.clamp(0, V - 1)], -1).to(torch.int32)
    ids, w = om.route(layer.logits(flat.to(dev)).cpu(), k, "sqrtsoftplus", ids=given, scale=1.5, shared=1)
    want = om.experts(flat, ids, w.float(), *dense, 10.0)
    xd, td = x.to(dev), tokens.to(dev)
    y = layer(xd, td)
    _check_experts(y.view(-1, K), want)
    assert torch.equal(layer(xd, td.int()), y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = layer(xd, td)
    for _ in range(3):
        graph.replay()
        assert torch.equal(z, y)
        torch.cuda.synchronize()


@pytest.mark.parametrize("T", [1, 9, 60])
def test_layer_with_a_router_in_fp32(dev, T):
    """(The product of fp32 operands is within the bound that test_gpu_linear.py gives.)"""
    from smla import moe
    announce(f"layer with an fp32 router {T}")
    E, k, K, I = 24, 4, 192, 64
    layer, router, bias, dense = _layer(dev, E, k, K, I, 1, "fp4")
    g = torch.Generator().manual_seed(T)
    router = torch.randn(E, K, generator=g) * K ** -0.5
    layer = moe.ExpertLayer(moe.ExpertWeights(router.to(dev), layer.w.gate, layer.w.up, layer.w.down, bias=bias.to(dev)), k=k)
    x = torch.randn(T, K, generator=g).to(torch.bfloat16)
    logits = layer.logits(x.to(dev)).cpu()
    ref = x.double() @ router.double().T
    assert ((logits.double() - ref).abs() <= (K + 8) * 2.0 ** -23 * (x.double().abs() @ router.double().abs().T)).all()
    ids, w = om.route(logits, k, "sqrtsoftplus", bias=bias, scale=1.5, shared=1)
    _check_experts(layer(x.to(dev)), om.experts(x, ids, w.float(), *dense, 10.0))


def test_rows_up_to_the_last_that_a_call_addresses(dev):
    """1023 rows 2^20 elements apart: offsets up to 2^31 bytes, in the tiles and, first and last 16 rows, in the kernels for few."""
    from smla import mla, moe
    announce("rows up to 2^31 bytes")
    T, ld, E, k, K, I = 1023, 1 << 20, 4, 2, 64, 32
    x, ids, w, mats = _experts_case(5, T, E, E, k, K, I, "fp4")
    on = _on(dev, mats)
    codes, scales, _ = _packed(6, 48, K)
    codes, scales = codes.to(dev), scales.to(dev)
    far = torch.empty(T * ld, dtype=torch.bfloat16, device=dev).as_strided((T, K), (ld, 1))
    far.copy_(x)
    near, ids, w = x.to(dev), ids.to(dev), w.to(dev)
    for rows in (slice(0, T), slice(0, 16), slice(T - 16, T)):
        assert torch.equal(moe.experts(far[rows], ids[rows], w[rows], *on), moe.experts(near[rows], ids[rows], w[rows], *on))
        assert torch.equal(mla.linear_fp4(far[rows], codes, scales), mla.linear_fp4(near[rows], codes, scales))


def test_two_threads(dev):
    """Layers called from two threads at once, each on its own stream and with other sizes, give what they give alone."""
    import threading
    announce("two threads")
    K = 192
    layer, *_ = _layer(dev, 24, 4, K, 64, 1, "fp4")
    xs = [torch.randn(T, K, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16).to(dev) for T in (3, 17, 61, 300)]
    want = [layer(x) for x in xs]
    torch.cuda.synchronize()
    wrong, done = [], []

    def work(mine):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                for i in mine:
                    y = layer(xs[i])
                    torch.cuda.current_stream().synchronize()
                    if not torch.equal(y, want[i]):
                        wrong.append(i)
        done.append(mine)
    threads = [threading.Thread(target=work, args=(m,)) for m in ((0, 2), (3, 1))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(done) == 2 and not wrong


@pytest.mark.parametrize("T", [12, 40, 500])
@pytest.mark.parametrize("kind", ["fp4", "bf16"])
def test_experts_repeat_bit_for_bit(dev, T, kind):
    """The same call gives the same bits, whatever order its pairs are sorted in; past 16 tokens a token's result does not
    depend on the ids beside it either."""
    from smla import moe
    announce(f"experts repeat {T} {kind}")
    E, k, K, I = 6, 3, 544, 416
    x, ids, w, mats = _experts_case(T, T, E, E, k, K, I, kind)
    on = _on(dev, mats)
    xd, idd, wd = x.to(dev), ids.to(dev), w.to(dev)
    y = moe.experts(xd, idd, wd, *on)
    for _ in range(8):
        assert torch.equal(moe.experts(xd, idd, wd, *on), y)
    other = ids.clone()
    other[1::2] = other[1::2].flip(0)
    z = moe.experts(xd, other.to(dev), wd, *on)
    if T > 16:
        assert torch.equal(z[::2], y[::2])
    _check_experts(z, om.experts(x, other, w, *[m[2] for m in mats]))


@pytest.mark.parametrize("T", [1, 2, 40])
@pytest.mark.parametrize("kind", ["fp4", "bf16"])
def test_layer_of_inputs_that_begin_anywhere(dev, T, kind):
    """A layer takes its inputs at any address, one token (whose row is dense wherever it begins) as many."""
    announce(f"layer inputs anywhere {T} {kind}")
    K = 192
    layer, *_ = _layer(dev, 24, 4, K, 64, 1, kind)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16).to(dev)
    want = layer(x)
    for wide, at in ((K + 8, 3), (K + 5, 1), (K + 16, 8)):
        y = torch.full((T, wide), math.nan, dtype=torch.bfloat16, device=dev)[:, at:at + K]
        y.copy_(x)
        assert torch.equal(layer(y), want)
    flat = torch.empty(T * K + 1, dtype=torch.bfloat16, device=dev)[1:].view(T, K).copy_(x)
    assert torch.equal(layer(flat), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_packed_weights_that_are_not_finite(dev, dtype):
    """A block of 32 weights that holds a NaN or an infinity is NaN when packed, and the products with it; no other block changes."""
    from smla import mla, moe
    announce(f"packed weights not finite {dtype}")
    N, K = 24, 160
    g = torch.Generator().manual_seed(3)
    w = torch.randn(2, N, K, generator=g).to(dtype)
    clean_codes, clean_scales = moe.pack_fp4(w.to(dev))
    bad = w.clone()
    bad[0, 3, 40], bad[0, 5, 159], bad[1, 7, 0], bad[1, 7, 1] = math.nan, math.inf, -math.inf, math.nan
    codes, scales = moe.pack_fp4(bad.to(dev))
    hit = ~bad.isfinite().view(2, N, K // 32, 32).all(-1)
    assert hit.sum() == 3 and (scales.cpu()[hit] == 255).all()
    assert torch.equal(scales.cpu()[~hit], clean_scales.cpu()[~hit])
    assert torch.equal(codes.cpu().view(2, N, K // 32, 16)[~hit], clean_codes.cpu().view(2, N, K // 32, 16)[~hit])
    y = mla.linear_fp4(torch.randn(5, K, generator=g).to(torch.bfloat16).to(dev), codes[0], scales[0])
    assert y[:, [3, 5]].isnan().all() and y[:, 6:].isfinite().all()

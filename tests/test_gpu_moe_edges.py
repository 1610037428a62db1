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

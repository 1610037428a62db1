"""GPU tier: products with 4-bit weights and experts whose sums are long, in every tile form, past the reuse of the loop's rings; which
form a case takes is held in test_moe_plan.py.  The scales differ by powers of two from one group of 512 k to the next, so
that a group read from another's place shows.  Tolerances as in test_gpu_moe.py."""
import math

import pytest
import torch

from conftest import announce
from oracle import moe as om
from test_gpu_moe import _check_experts, _packed

pytestmark = pytest.mark.gpu

LONG_LINEARS = [  # T, N, K
    (65, 8192, 4096), (400, 4090, 2080), (257, 3000, 4160), (129, 8190, 2176),
    (129, 3000, 2080), (700, 1030, 4160), (1025, 1000, 4096),
    (3300, 2551, 2080), (3300, 2551, 4096), (5500, 1530, 4160),
]
LONG_EXPERTS = [  # T, E, k, K, I, weights
    (40, 3, 2, 2144, 2048, "fp4"), (33, 2, 1, 2048, 2080, "fp4"), (50, 3, 1, 2176, 2208, "fp4"),
    (70, 2, 1, 2144, 2048, "fp4"), (75, 2, 1, 2048, 2080, "fp4"), (140, 2, 1, 2176, 2208, "fp4"),
    (40, 2, 1, 1664, 1568, "bf16"), (130, 2, 1, 1600, 1632, "bf16"),
]


def _stepped(seed, *shape):
    """Codes, scales and float64 weights whose groups of 512 k differ by factors of 4."""
    codes, scales, _ = _packed(seed, *shape)
    scales = scales + (2 * (torch.arange(shape[-1] // 32) // 16 % 3)).to(torch.uint8)
    return codes, scales, om.unpack(codes, scales)


@pytest.mark.parametrize("case", LONG_LINEARS, ids=lambda c: "-".join(map(str, c)))
def test_long_products(dev, case):
    from smla import mla
    T, N, K = case
    announce(f"long product {case}")
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(T + K)).to(torch.bfloat16)
    codes, scales, w = _stepped(N + K, N, K)
    want = x.double() @ w.T
    tol = (K + 1) * 2.0 ** -24 * (x.double().abs() @ w.abs().T)
    for dt, half in ((torch.float32, 2.0 ** -24), (torch.bfloat16, 2.0 ** -8)):
        y = mla.linear_fp4(x.to(dev), codes.to(dev), scales.to(dev), out_dtype=dt).cpu().double()
        assert ((y - want).abs() <= tol + half * (want.abs() + tol)).all()


@pytest.mark.parametrize("case", LONG_EXPERTS, ids=lambda c: "-".join(map(str, c)))
def test_long_experts(dev, case):
    from smla import moe
    T, E, k, K, I, kind = case
    announce(f"long experts {case}")
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, K, generator=g).to(torch.bfloat16)
    ids = torch.rand(T, E, generator=g).topk(k, dim=-1).indices.to(torch.int32)
    w = torch.rand(T, k, generator=g) + 0.1
    mats, dense = [], []
    for i, (n, m) in enumerate(((I, K), (I, K), (K, I))):
        if kind == "fp4":
            c, s, d = _stepped(T + i, E, n, m)
            mats.append((c.to(dev), s.to(dev)))
        else:
            v = (torch.randn(E, n, m, generator=g) * m ** -0.5).to(torch.bfloat16)
            d = v.double()
            mats.append(v.to(dev))
        dense.append(d)
    y = moe.experts(x.to(dev), ids.to(dev), w.to(dev), *mats)
    _check_experts(y, om.experts(x, ids, w, *dense, math.inf))

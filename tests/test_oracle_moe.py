"""CPU tier: the oracle of the expert network against closed forms and torch's own operations."""
import math

import torch

from oracle import moe as om


def test_pack_unpack_grid_and_ties():
    w = torch.zeros(1, 32)
    w[0, :12] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0, 0.3, -6.0])
    codes, scales = om.pack(w)
    assert scales.tolist() == [[127]]
    assert om.unpack(codes, scales)[0, :12].tolist() == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -0.0, -4.0, 0.5, -6.0]


def test_unpack_scale_bytes():
    codes = torch.full((3, 16), 0x2a, dtype=torch.uint8)     # -1, 1
    v = om.unpack(codes, torch.tensor([[0], [130], [255]], dtype=torch.uint8))
    assert v[0, 0] == -2.0 ** -127 and v[1, 1] == 8.0 and v[2].isnan().all()


def test_route_softmax_is_torchs():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(20, 50, generator=g)
    ids, w = om.route(x, 5, "softmax", renorm=False)
    s = torch.softmax(x.double(), -1)
    top = s.topk(5)
    assert torch.equal(ids.long(), top.indices) and torch.allclose(w, top.values, rtol=1e-14, atol=0)


def test_route_groups_bias_ties():
    # groups {0, 1}, {2, 3}, {4, 5}; the bias lifts group 2; within it the tie goes to the lower id
    x = torch.zeros(1, 6)
    ids, w = om.route(x, 2, "sigmoid", bias=torch.tensor([0.0, 0.1, 0, 0, 0.2, 0.2]), groups=3, topk_groups=2, scale=3.0)
    assert ids.tolist() == [[4, 5]] and w.tolist() == [[1.5, 1.5]]
    ids, w = om.route(torch.full((1, 4), -math.inf), 2, "softmax", shared=1)
    assert ids.tolist() == [[0, 1, 4]] and w.tolist() == [[0.0, 0.0, 1.0]]
    ids, w = om.route(torch.tensor([[math.nan, 1.0, -math.inf, 0.0]]), 4, "sigmoid", renorm=False)
    assert ids.tolist() == [[1, 3, 0, 2]] and w[0, 2].isnan()


def test_experts_one_is_the_network():
    g = torch.Generator().manual_seed(2)
    gate, up, down = (torch.randn(1, a, b, generator=g).double() for a, b in ((8, 4), (8, 4), (4, 8)))
    x = torch.randn(3, 4, generator=g)
    y, bound = om.experts(x, torch.zeros(3, 1, dtype=torch.int32), torch.full((3, 1), 2.0), gate, up, down)
    xd = x.double()
    want = 2 * (torch.nn.functional.silu(xd @ gate[0].T) * (xd @ up[0].T)) @ down[0].T
    assert torch.allclose(y, want, rtol=1e-12) and (bound > 0).all()
    none, _ = om.experts(x, torch.full((3, 1), -1, dtype=torch.int32), torch.full((3, 1), 2.0), gate, up, down)
    assert (none == 0).all()

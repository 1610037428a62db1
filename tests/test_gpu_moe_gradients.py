"""GPU tier: the expert network's operators are forward only: a leaf that asks for a gradient never gets a result that is
silently cut off from it."""
import pytest
import torch

from conftest import announce
from test_gpu_moe import _packed

pytestmark = pytest.mark.gpu


def _refuses(y, leaf):
    assert y.requires_grad
    with pytest.raises(RuntimeError, match="no autograd formula|does not require grad|not implemented"):
        y.float().sum().backward()
    assert leaf.grad is None


def test_gradients_are_refused(dev):
    from smla import mla, moe
    announce("moe gradients refused")
    T, E, K, I = 5, 4, 64, 32
    g = torch.Generator().manual_seed(1)
    leaf = lambda *s, dt=torch.float32: torch.randn(*s, generator=g).to(dt).to(dev).requires_grad_()
    for logits, bias in ((leaf(T, E), None), (torch.zeros(T, E, device=dev), leaf(E))):
        ids, w = moe.route(logits, 2, "sigmoid", bias=bias)
        _refuses(w, logits if bias is None else bias)
        assert not ids.requires_grad
    codes, scales, _ = _packed(2, I, K)
    codes, scales = codes.to(dev), scales.to(dev)
    x = leaf(T, K, dt=torch.bfloat16)
    _refuses(mla.linear_fp4(x, codes, scales), x)
    ids = torch.zeros(T, 2, dtype=torch.int32, device=dev)
    w = torch.ones(T, 2, device=dev)
    mats = [torch.randn(E, *s, generator=g).to(torch.bfloat16).to(dev) for s in ((I, K), (I, K), (K, I))]
    for i in range(5):
        args = [x.detach(), w, *mats]
        args[i] = args[i].clone().requires_grad_()
        y = moe.experts(args[0], ids, args[1], *args[2:])
        _refuses(y, args[i])
        with torch.no_grad():
            assert torch.equal(moe.experts(args[0], ids, args[1], *args[2:]), y.detach())
            assert not moe.experts(args[0], ids, args[1], *args[2:]).requires_grad


@pytest.mark.parametrize("change", [dict(k=9), dict(k=3, groups=3), dict(k=0), dict(k=2, groups=4, topk_groups=5), dict(k=60, shared=5)])
def test_bad_choices_are_the_librarys_errors(dev, change):
    from smla import _lib, moe
    announce(f"route refuses {change}")
    with pytest.raises(_lib.SmlaError):
        moe.route(torch.zeros(2, 64 if change["k"] == 60 else 8, device=dev), **change)

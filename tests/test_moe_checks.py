"""CPU tier: the expert network's entry points refuse what their kernels cannot take, before any launch."""
import ctypes

import pytest
import torch

FAKE = ctypes.c_void_p(4096)    # never dereferenced: validation fails first
ODD = ctypes.c_void_p(4100)
F32, BF16, FP8, F16, FP4 = 0, 1, 2, 3, 5
OK, NULL, SHAPE, DTYPE, UNSUP, WS, RANGE = 0, -1, -2, -3, -4, -5, -6


def _call(name, names, defaults, **change):
    from smla import _lib
    lib = _lib.lib()
    assert set(change) <= set(names), change
    return getattr(lib, name)(*[change.get(n, defaults[n]) for n in names])


ROUTE = "logits dtype ld bias T E k score groups topk_groups renorm scale shared given ids weights stream".split()
ROUTE_OK = dict(logits=FAKE, dtype=F32, ld=64, bias=None, T=0, E=64, k=6, score=0, groups=1, topk_groups=1, renorm=1, scale=1.0,
                shared=0, given=None, ids=FAKE, weights=FAKE, stream=None)


@pytest.mark.parametrize("change,status", [
    ({}, OK),      # no tokens: nothing is launched
    (dict(dtype=F16), DTYPE), (dict(T=-1), SHAPE), (dict(E=0), SHAPE), (dict(k=0), SHAPE), (dict(shared=-1), SHAPE),
    (dict(T=2, ld=63), SHAPE), (dict(groups=0), SHAPE), (dict(groups=7), SHAPE), (dict(groups=8, topk_groups=9), SHAPE),
    (dict(groups=16, topk_groups=1, k=5), SHAPE), (dict(k=65), SHAPE), (dict(k=60, shared=5), UNSUP),
    (dict(E=1025, ld=1025), UNSUP), (dict(score=3), RANGE), (dict(score=-1), RANGE), (dict(scale=float("nan")), RANGE),
    (dict(T=1, logits=None), NULL), (dict(T=1, ids=None), NULL), (dict(T=1, weights=None), NULL),
    (dict(logits=None), OK), (dict(groups=7, given=FAKE), OK), (dict(T=1 << 26), UNSUP),
])
def test_route_status(change, status):
    assert _call("smla_route", ROUTE, ROUTE_OK, **change) == status


LINEAR = "x ldx codes scales T N K y y_dtype ws ws_bytes stream".split()
LINEAR_OK = dict(x=FAKE, ldx=64, codes=FAKE, scales=FAKE, T=0, N=10, K=64, y=FAKE, y_dtype=BF16, ws=None, ws_bytes=0, stream=None)


@pytest.mark.parametrize("change,status", [
    ({}, OK), (dict(T=-1), SHAPE), (dict(N=0), SHAPE), (dict(K=0), SHAPE), (dict(T=2, ldx=32), SHAPE),
    (dict(y_dtype=F16), DTYPE), (dict(y_dtype=FP8), DTYPE),
    (dict(T=1, x=None), NULL), (dict(T=1, codes=None), NULL), (dict(T=1, scales=None), NULL), (dict(T=1, y=None), NULL),
    (dict(T=1, K=80, ldx=80), UNSUP), (dict(T=1, ldx=68), UNSUP), (dict(T=1, x=ODD), UNSUP), (dict(T=1, codes=ODD), UNSUP),
    (dict(T=1, y=ODD), UNSUP), (dict(T=1, K=128, ldx=128, scales=ctypes.c_void_p(4097)), UNSUP),
    (dict(T=1 << 40), UNSUP), (dict(T=1, N=1 << 40), UNSUP), (dict(T=1, K=1 << 40, ldx=1 << 40), UNSUP),
])
def test_linear_fp4_status(change, status):
    assert _call("smla_linear_fp4", LINEAR, LINEAR_OK, **change) == status


EXPERTS = ("x ldx ids weights T k E K I gate gate_scales up up_scales down down_scales w_dtype limit y ws ws_bytes "
           "stream").split()
EXPERTS_OK = dict(x=FAKE, ldx=64, ids=FAKE, weights=FAKE, T=0, k=2, E=8, K=64, I=32, gate=FAKE, gate_scales=FAKE, up=FAKE,
                  up_scales=FAKE, down=FAKE, down_scales=FAKE, w_dtype=FP4, limit=10.0, y=FAKE, ws=FAKE, ws_bytes=1 << 40,
                  stream=None)


@pytest.mark.parametrize("change,status", [
    ({}, OK), (dict(w_dtype=F32), DTYPE), (dict(w_dtype=FP8), DTYPE), (dict(T=-1), SHAPE), (dict(k=0), SHAPE),
    (dict(E=0), SHAPE), (dict(K=0), SHAPE), (dict(I=0), SHAPE), (dict(T=2, ldx=32), SHAPE),
    (dict(T=1, K=80, ldx=80), UNSUP), (dict(T=1, I=48), UNSUP), (dict(T=1, E=1025), UNSUP), (dict(T=1, k=65), UNSUP),
    (dict(T=1, ldx=68), UNSUP), (dict(T=1, x=ODD), UNSUP), (dict(T=1, gate=ODD), UNSUP), (dict(T=1, up=ODD), UNSUP),
    (dict(T=1, down=ODD), UNSUP), (dict(T=1, y=ODD), UNSUP), (dict(T=1 << 40), UNSUP),
    *[(dict(T=1, **{n: ctypes.c_void_p(4097)}), UNSUP) for n in ("gate_scales", "up_scales", "down_scales")],
    (dict(T=1 << 20, ldx=1024), UNSUP), (dict(T=1 << 19, k=1, ldx=2048), UNSUP),
    *[(dict(T=1, **{n: None}), NULL) for n in ("x", "ids", "weights", "gate", "up", "down", "y", "gate_scales", "up_scales", "down_scales")],
    (dict(T=1, limit=0.0), RANGE), (dict(T=1, limit=-1.0), RANGE), (dict(T=1, limit=float("nan")), RANGE),
    (dict(T=1, ws=None), WS), (dict(T=1, ws_bytes=15), WS), (dict(T=1, ws=ctypes.c_void_p(4104)), WS),
])
def test_experts_status(change, status):
    assert _call("smla_experts", EXPERTS, EXPERTS_OK, **change) == status


def test_workspaces_of_bad_sizes_are_empty():
    from smla import _lib
    lib = _lib.lib()
    assert lib.smla_linear_fp4_workspace(0, 16, 64) == 0 and lib.smla_linear_fp4_workspace(64, 16, 33) == 0
    assert lib.smla_experts_workspace(1, 1, 2000, 64, 64, 5) == 0 and lib.smla_experts_workspace(0, 1, 20, 64, 64, 5) == 0


def _u8(*shape):
    return torch.zeros(*shape, dtype=torch.uint8)


@pytest.mark.parametrize("codes,scales", [
    (_u8(4, 32).float(), _u8(4, 2)), (_u8(5, 32), _u8(4, 2)), (_u8(4, 32), _u8(4, 1)), (_u8(4, 32), _u8(4, 2).float()),
    (_u8(4, 32), None), (_u8(4, 24), _u8(4, 1)), (_u8(4, 64)[:, ::2], _u8(4, 2)), (_u8(4, 32), _u8(4, 4)[:, ::2]),
])
def test_packed_weights_are_checked(codes, scales):
    from smla import ops
    assert ops._check_fp4(_u8(4, 32), _u8(4, 2), (4,), "w") == 64
    with pytest.raises(ValueError):
        ops._check_fp4(codes, scales, (4,), "w")


def test_rows_that_do_not_fit_are_packed():
    from smla import ops
    x = torch.zeros(6, 64, dtype=torch.bfloat16)
    assert ops._rows(x, 64, "x")[0] is x
    wide = torch.zeros(6, 80, dtype=torch.bfloat16)
    assert ops._rows(wide[:, :64], 64, "x")[1] == 80 and ops._rows(wide[:, 16:], 64, "x")[1] == 80
    for y in (wide[:, 1:65], torch.zeros(64, 6, dtype=torch.bfloat16).t(), torch.zeros(1, 64, dtype=torch.bfloat16).expand(6, 64)):
        packed, ld = ops._rows(y, 64, "x")
        assert ld == 64 and packed.is_contiguous()
    for bad in (x.float(), x[:, :32], x[0]):
        with pytest.raises(ValueError):
            ops._rows(bad, 64, "x")


def test_wrappers_refuse():
    from smla import mla, moe
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        moe.route(torch.zeros(2, 8), 2, score="relu")
    with pytest.raises(RuntimeError):      # not on a GPU
        moe.route(torch.zeros(2, 8), 2)
    with pytest.raises(RuntimeError):
        mla.linear_fp4(x, _u8(4, 32), _u8(4, 2))
    with pytest.raises(RuntimeError):
        moe.experts(x, torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, 1), *[(_u8(1, 64, 32), _u8(1, 64, 2))] * 3)
    with pytest.raises(ValueError):
        moe.pack_fp4(torch.zeros(4, 48))
    w = torch.zeros(2, 32, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):        # more routed experts than weights
        moe.ExpertLayer(moe.ExpertWeights(torch.zeros(3, 64, dtype=torch.bfloat16), w, w, w))
    layer = moe.ExpertLayer(moe.ExpertWeights(torch.zeros(2, 64, dtype=torch.bfloat16), w, w, w, table=torch.zeros(9, 6, dtype=torch.int32)))
    with pytest.raises(ValueError):        # a table without tokens
        layer(x)

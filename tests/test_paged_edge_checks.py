"""CPU tier: refusals and traces of the paged cache's calls beside those of ``test_paged_checks``."""
import ctypes

import pytest
import torch

from test_paged_checks import APPEND, APPEND_OK, ATTN, ATTN_OK, BF16, F32, FAKE, NULL, OK, RANGE, SHAPE, UNSUP, _call


def _with_granted(names, defaults):
    at = names.index("cu") + 1
    return names[:at] + ["granted"] + names[at:], defaults | dict(granted=FAKE)


@pytest.mark.parametrize("change,status", [({}, OK), (dict(granted=None), OK), (dict(cu=None), NULL), (dict(B=0), SHAPE),
                                           (dict(D=640), UNSUP), (dict(window=-1), RANGE)])
def test_paged_attn_granted_arguments(change, status):
    assert _call("smla_paged_attn_granted", *_with_granted(ATTN, ATTN_OK), **change) == status


@pytest.mark.parametrize("change,status", [({}, OK), (dict(granted=None), OK), (dict(cu=None), NULL), (dict(B=0), SHAPE),
                                           (dict(rd=6), UNSUP), (dict(flags=8), RANGE)])
def test_paged_append_granted_arguments(change, status):
    assert _call("smla_paged_append_granted", *_with_granted(APPEND, APPEND_OK), **change) == status


def test_granted_of_another_shape_or_type():
    from smla import ops
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    ops._check_batch(i32(2, 4), i32(2), i32(3), i32(2))
    for granted in (i32(3), i32(2, 1), i32(2).long(), i32(2).bool(), i32(4)[::2]):
        with pytest.raises(ValueError):
            ops._check_batch(i32(2, 4), i32(2), i32(3), granted)


def test_calls_with_granted_trace_as_their_ops():
    from smla import paged
    from torch._subclasses.fake_tensor import FakeTensorMode

    class Call(torch.nn.Module):
        def forward(self, q, x, p, t, n, c, cs, sn, ok):
            q = paged.paged_append(q, x, p, t, n, c, cs, sn, kv_norm=True, granted=ok)
            return paged.paged_attn(q, p, t, n, c, 0.04, granted=ok)

    with FakeTensorMode(allow_non_fake_inputs=True):
        i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
        f32 = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
        a = (f32(9, 16, 512), f32(9, 512), f32(20, 16, 512).bfloat16(), i32(3, 8), i32(3), i32(4), f32(128, 32), f32(128, 32), i32(3))
        assert tuple(Call()(*a).shape) == (9, 16, 512)
    program = torch.export.export(Call(), a, strict=False)
    called = [str(n.target) for n in program.graph.nodes if n.op == "call_function"]
    assert "smla.paged_append_.default" in called and "smla.paged_attn_.default" in called


def _at(n):
    return ctypes.c_void_p(1 << 20 | n)


# a bf16 q of 2 tokens of 16 heads of 512 at 0 (32768 bytes), kv behind it with 488 spare elements a row (2000 + 1024 bytes)
OVER = dict(T=2, x_dtype=BF16, q=_at(0), ldq=16 * 512, kv=_at(32768), ldkv=1000, B=1)


@pytest.mark.parametrize("change", [
    dict(q_out=_at(8)), dict(q_out=_at(32768 - 8)), dict(q_out=_at(32768)), dict(q_out=_at(32768 + 3024 - 8)),
    dict(x_dtype=F32, q_out=_at(0), kv=_at(1 << 19)),                           # fp32 q: written rows lie over others
    dict(q=_at(0), ldq=16 * 512 + 4, q_out=_at(0), kv=_at(1 << 19)),            # rows apart
])
def test_paged_append_refuses_queries_over_its_inputs(change):
    assert _call("smla_paged_append", APPEND, APPEND_OK | OVER, **change) == UNSUP

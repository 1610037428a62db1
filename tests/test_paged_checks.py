"""CPU tier: the paged cache's entry points refuse what their kernels cannot take, before any launch."""
import ctypes

import pytest
import torch

FAKE = ctypes.c_void_p(4096)    # never dereferenced: validation fails first
BF16, F32, FP8, F16 = 1, 0, 2, 3
OK, NULL, SHAPE, DTYPE, UNSUP, WS, RANGE = 0, -1, -2, -3, -4, -5, -6


def _call(name, names, defaults, **change):
    from smla import _lib
    lib = _lib.lib()
    assert set(change) <= set(names), change
    return getattr(lib, name)(*[change.get(n, defaults[n]) for n in names])


ATTN = ("q q_dtype pages page_dtype page_scales n_pages P table ld_table cols lens cu B T H D DV scale sink window first "
        "flags out out_dtype ws ws_bytes stream").split()
ATTN_OK = dict(q=FAKE, q_dtype=BF16, pages=FAKE, page_dtype=BF16, page_scales=None, n_pages=4, P=16, table=FAKE, ld_table=8,
               cols=8, lens=FAKE, cu=FAKE, B=2, T=0, H=16, D=576, DV=512, scale=1.0, sink=None, window=0, first=0, flags=0,
               out=FAKE, out_dtype=BF16, ws=FAKE, ws_bytes=1 << 40, stream=None)


@pytest.mark.parametrize("change,status", [
    ({}, OK),      # no tokens: nothing is launched
    (dict(q=None), NULL), (dict(pages=None), NULL), (dict(table=None), NULL), (dict(lens=None), NULL), (dict(cu=None), NULL),
    (dict(out=None), NULL), (dict(page_dtype=FP8), NULL),
    (dict(H=0), SHAPE), (dict(B=0), SHAPE), (dict(n_pages=0), SHAPE), (dict(P=0), SHAPE), (dict(cols=0), SHAPE),
    (dict(ld_table=7), SHAPE), (dict(T=-1), SHAPE), (dict(DV=577), SHAPE),
    (dict(q_dtype=F32), DTYPE), (dict(out_dtype=F32), DTYPE), (dict(page_dtype=F16), DTYPE),
    (dict(D=640), UNSUP), (dict(DV=256), UNSUP), (dict(q=ctypes.c_void_p(4104)), UNSUP),
    (dict(out=ctypes.c_void_p(4104)), UNSUP), (dict(pages=ctypes.c_void_p(4098)), UNSUP),
    (dict(window=-1), RANGE), (dict(first=-1), RANGE), (dict(window=1 << 30), RANGE), (dict(flags=1), RANGE),
    (dict(n_pages=1 << 20, P=1 << 12), RANGE), (dict(B=1 << 20), RANGE), (dict(T=1 << 30), RANGE), (dict(cols=1 << 31, ld_table=1 << 31), RANGE),
    (dict(ws=None), WS), (dict(ws_bytes=100), WS), (dict(ws=ctypes.c_void_p(4104)), WS),
    (dict(T=1), UNSUP), (dict(T=1, out=ctypes.c_void_p(4096 + 16 * 576 * 2 - 16)), UNSUP),    # out over q
    (dict(T=1, q=ctypes.c_void_p(4096 + 16 * 512 * 2 - 16)), UNSUP),
])
def test_paged_attn_arguments(change, status):
    assert _call("smla_paged_attn", ATTN, ATTN_OK, **change) == status


APPEND = ("q ldq kv ldkv x_dtype T H D norm_dims q_w kv_w cos sin n_pos rd eps sim flags q_out pages page_dtype scales n_pages "
          "P table ld_table cols lens cu B stream").split()
APPEND_OK = dict(q=FAKE, ldq=16 * 512, kv=FAKE, ldkv=512, x_dtype=F32, T=0, H=16, D=512, norm_dims=512, q_w=None, kv_w=FAKE,
                 cos=FAKE, sin=FAKE, n_pos=100, rd=64, eps=1e-6, sim=0, flags=7, q_out=FAKE, pages=FAKE, page_dtype=BF16,
                 scales=None, n_pages=4, P=16, table=FAKE, ld_table=8, cols=8, lens=FAKE, cu=FAKE, B=2, stream=None)


@pytest.mark.parametrize("change,status", [
    ({}, OK), (dict(q=None, q_out=None, H=0, ldq=0), OK), (dict(rd=0, cos=None, sin=None, n_pos=0), OK),
    (dict(q=None), NULL), (dict(q_out=None), NULL), (dict(kv=None), NULL), (dict(pages=None), NULL), (dict(cos=None), NULL),
    (dict(lens=None), NULL), (dict(cu=None), NULL), (dict(table=None), NULL), (dict(page_dtype=FP8), NULL),
    (dict(ldq=16 * 512 - 4), SHAPE), (dict(ldkv=508), SHAPE), (dict(norm_dims=516), SHAPE), (dict(norm_dims=0), SHAPE),
    (dict(rd=516), SHAPE), (dict(n_pos=0), SHAPE), (dict(B=0), SHAPE), (dict(P=0), SHAPE), (dict(ld_table=7), SHAPE),
    (dict(x_dtype=F16), DTYPE), (dict(page_dtype=F32), DTYPE),
    (dict(D=96, ldq=16 * 96, norm_dims=96), UNSUP), (dict(D=1088, ldq=16 * 1088, ldkv=1088), UNSUP), (dict(rd=6), UNSUP),
    (dict(norm_dims=510), UNSUP), (dict(ldkv=514), UNSUP), (dict(ldq=16 * 512 + 2), UNSUP), (dict(sim=2), UNSUP),
    (dict(sim=1, rd=32), UNSUP), (dict(sim=1, page_dtype=FP8, scales=FAKE), UNSUP), (dict(kv=ctypes.c_void_p(4104)), UNSUP),
    (dict(x_dtype=BF16, kv=ctypes.c_void_p(4100)), UNSUP), (dict(q_out=ctypes.c_void_p(4100)), UNSUP),
    (dict(flags=8), RANGE), (dict(T=1 << 28), RANGE),
])
def test_paged_append_arguments(change, status):
    assert _call("smla_paged_append", APPEND, APPEND_OK, **change) == status


UPDATE = ("table ld_table S M lens refs n_pages P parent grow table_out lens_out refs_out granted pages layers layer_bytes "
          "row_bytes scales scale_layer_bytes scale_row_bytes ws ws_bytes stream").split()
OTHER = ctypes.c_void_p(8192)
UPDATE_OK = dict(table=FAKE, ld_table=8, S=4, M=8, lens=FAKE, refs=FAKE, n_pages=20000, P=16, parent=FAKE, grow=FAKE, table_out=OTHER,
                 lens_out=OTHER, refs_out=OTHER, granted=OTHER, pages=FAKE, layers=1, layer_bytes=0, row_bytes=1024, scales=None,
                 scale_layer_bytes=0, scale_row_bytes=0, ws=FAKE, ws_bytes=(1 + 2 * 4 + 20000) * 4, stream=None)
BAD_POOL = [(dict(table=None), NULL), (dict(refs=None), NULL), (dict(pages=None), NULL), (dict(table_out=None), NULL),
            (dict(refs_out=None), NULL), (dict(S=0), SHAPE), (dict(M=0), SHAPE), (dict(n_pages=0), SHAPE), (dict(P=0), SHAPE),
            (dict(layers=0), SHAPE), (dict(row_bytes=0), SHAPE), (dict(ld_table=7), SHAPE), (dict(scales=FAKE), SHAPE),
            (dict(S=1 << 30), RANGE), (dict(n_pages=1 << 30), RANGE), (dict(layers=1 << 16), RANGE),
            (dict(table_out=FAKE), UNSUP), (dict(refs_out=FAKE), UNSUP), (dict(ws=None), WS), (dict(ws=ctypes.c_void_p(4098)), WS)]


@pytest.mark.parametrize("change,status", BAD_POOL + [
    (dict(lens=None), NULL), (dict(parent=None), NULL), (dict(grow=None), NULL), (dict(lens_out=None), NULL),
    (dict(granted=None), NULL), (dict(lens_out=FAKE), UNSUP), (dict(ws_bytes=(1 + 2 * 4 + 20000) * 4 - 1), WS)])
def test_update_pages_arguments(change, status):
    assert _call("smla_update_pages", UPDATE, UPDATE_OK, **change) == status


COMPACT = ("table ld_table S M refs n_pages P table_out refs_out live pages layers layer_bytes row_bytes scales "
           "scale_layer_bytes scale_row_bytes ws ws_bytes stream").split()
COMPACT_OK = {k: UPDATE_OK[k] for k in COMPACT if k in UPDATE_OK} | dict(live=OTHER, ws_bytes=60002 * 4)


@pytest.mark.parametrize("change,status", BAD_POOL + [(dict(live=None), NULL), (dict(ws_bytes=60002 * 4 - 1), WS)])
def test_compact_pages_arguments(change, status):
    assert _call("smla_compact_pages", COMPACT, COMPACT_OK, **change) == status


def test_workspace_sizes():
    from smla import _lib
    lib = _lib.lib()
    size = lib.smla_paged_attn_workspace
    assert size(-1, 16, 1, 64, 0, 0) == size(1, 0, 1, 64, 0, 0) == size(1, 16, 1, -1, 0, 0) == size(1, 16, 1, 64, -1, 0) == 0
    few, many, long = size(1, 64, 1, 4096, 0, 0), size(4096, 64, 1, 4096, 0, 0), size(4096, 64, 1, 1 << 20, 0, 0)
    assert 0 < few < many < long < 1 << 29
    assert size(4096, 64, 1, 1 << 20, 128, 4) == many       # a window keeps the tiles short
    update, compact = lib.smla_update_pages_workspace, lib.smla_compact_pages_workspace
    assert update(0, 1, 1) == update(1, 0, 1) == update(1, 1, 0) == compact(0) == 0
    # one launch, which needs none, up to one step of a scan, 1024 slots and 32768 entries
    assert update(1024, 32, 16384) == compact(16384) == 0
    assert update(4, 8, 16385) == 4 * (1 + 8 + 16385) and update(1025, 1, 8) == 4 * (1 + 2050 + 8)
    assert update(1024, 33, 8) == 4 * (1 + 2048 + 8) and compact(16385) == 4 * (2 + 3 * 16385)


def test_python_checks():
    from smla import ops, paged
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    with pytest.raises(RuntimeError):       # not on a GPU
        paged.paged_attn(bf(2, 4, 512), bf(3, 8, 512), i32(1, 2), i32(1), i32(2), 1.0)
    with pytest.raises(RuntimeError):
        paged.compact_pages(bf(3, 8, 512), i32(1, 2), i32(3))
    with pytest.raises(ValueError):
        paged.paged_attn(bf(2, 512), bf(3, 8, 512), i32(1, 2), i32(1), i32(2), 1.0)
    with pytest.raises(ValueError):
        paged.paged_append(None, bf(2, 512), bf(3, 8, 512), i32(1, 2), i32(1), i32(2), bf(1, 32), bf(1, 32), q_out=bf(2, 1, 512))
    assert ops._check_pool(bf(3, 8, 512), None, (3,)) == BF16
    assert ops._check_pool(torch.zeros(3, 8, 512, dtype=torch.uint8), torch.zeros(3, 8, 8), (3,)) == FP8
    for pool, scales, error in ((bf(3, 8, 512)[:, :4], None, ValueError), (bf(0, 8, 512), None, ValueError),
                                (torch.zeros(3, 8, 512), None, TypeError), (bf(3, 8, 512), torch.zeros(3, 8, 8), ValueError),
                                (torch.zeros(3, 8, 512, dtype=torch.uint8), None, ValueError),
                                (torch.zeros(3, 8, 512, dtype=torch.uint8), torch.zeros(3, 8, 9), ValueError),
                                (bf(3, 512), None, ValueError), (bf(2, 3, 8, 512), None, ValueError)):
        with pytest.raises(error):
            ops._check_pool(pool, scales, (3,))
    for table, lens, cu in ((i32(2, 0), i32(2), i32(3)), (i32(2), i32(2), i32(3)), (i32(2, 4).long(), i32(2), i32(3)),
                            (i32(2, 4), i32(3), i32(3)), (i32(2, 4), i32(2), i32(2)), (i32(2, 4), i32(2).long(), i32(3))):
        with pytest.raises(ValueError):
            ops._check_batch(table, lens, cu)


def _paged_calls():
    from smla import paged
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    bf = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    f32 = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
    yield ("attn", lambda q, p, t, n, c, s: paged.paged_attn(q, p, t, n, c, 0.04, s, 128, 4),
           lambda: (bf(9, 16, 576), bf(20, 16, 576), i32(3, 8), i32(3), i32(4), f32(16)), (9, 16, 512), "paged_attn_")
    yield ("append", lambda q, x, p, t, n, c, cs, sn: paged.paged_append(q, x, p, t, n, c, cs, sn, kv_norm=True),
           lambda: (f32(9, 16, 512), f32(9, 512), bf(20, 16, 512), i32(3, 8), i32(3), i32(4), f32(128, 32), f32(128, 32)),
           (9, 16, 512), "paged_append_")
    yield ("update", lambda p, t, n, r, a, g: paged.update_pages(p, t, n, r, a, g)[0],
           lambda: (bf(20, 16, 512), i32(3, 8), i32(3), i32(20), i32(3), i32(3)), (3, 8), "update_pages")
    yield ("compact", lambda p, t, r: paged.compact_pages(p, t, r)[0], lambda: (bf(20, 16, 512), i32(3, 8), i32(20)), (3, 8),
           "compact_pages")


@pytest.mark.parametrize("name,fn,args,shape,op", list(_paged_calls()), ids=lambda v: v if isinstance(v, str) else "")
def test_paged_calls_trace_as_their_ops(name, fn, args, shape, op):
    """Without memory behind the tensors nothing but the op itself may ask for a pointer."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    class Call(torch.nn.Module):
        def forward(self, *a):
            return fn(*a)

    with FakeTensorMode(allow_non_fake_inputs=True):
        a = args()
        assert tuple(fn(*a).shape) == shape
    program = torch.export.export(Call(), a, strict=False)
    assert f"smla.{op}.default" in [str(n.target) for n in program.graph.nodes if n.op == "call_function"]

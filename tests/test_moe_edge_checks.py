"""CPU tier: what the expert network's wrappers ask of the library, with the launches recorded instead of made."""
import pytest
import torch


@pytest.fixture
def calls(monkeypatch):
    """The arguments of every launch, from CPU tensors."""
    from smla import _lib, ops
    made = []
    monkeypatch.setattr(ops, "_one_device", lambda t, *rest: 0)
    monkeypatch.setattr(ops, "_launch", lambda dev, name, *args: made.append((name, args)))
    monkeypatch.setattr(ops, "_workspace", lambda dev, name, *sizes: getattr(_lib.lib(), name)(*sizes))
    return made


def _bf16(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("T,k,K,ld", [
    (1, 1, 32, 32), (16, 6, 64, 72), ((1 << 20) - 1, 1, 32, 32), (1 << 20, 1, 32, 32), ((1 << 20) + 1, 1, 32, 32), (174763, 6, 32, 32),
    (300000, 7, 32, 40), (33, 64, 32, 32), (16385, 64, 32, 32), (1100, 2, 32, 1 << 20), (1023, 2, 32, 1 << 20), (3, 2, 32, (1 << 20) + 8),
    (1 << 17, 1, 8192, 8192), ((1 << 17) - 1, 1, 8192, 8192), (300000, 1, 8192, 8192),
])
def test_experts_of_any_number_of_tokens(calls, T, k, K, ld):
    """Every call is within the library's limits, in order, and together they are all tokens; x stays where it is unless its rows
    lie too far apart."""
    from smla import ops
    inner, E = 32, 2
    x = torch.empty_strided((T, K), (ld, 1), dtype=torch.bfloat16)       # (never written: no memory behind it)
    ids, w = torch.zeros(T, k, dtype=torch.int32), torch.zeros(T, k)
    y = ops._experts(x, ids, w, _bf16(E, inner, K), _bf16(E, inner, K), _bf16(E, K, inner), None, None, None, 1.0)
    assert y.shape == (T, K)
    at = 0
    for name, a in calls:
        xp, ldx, ip, wp, n, kk, ee, KK, ii = a[:9]
        yp, _, wsb = a[-3:]
        assert name == "smla_experts" and (kk, ee, KK, ii) == (k, E, K, inner)
        assert 0 < n and n * k <= 1 << 20 and ldx <= 1 << 20 and ldx % 8 == 0 and (n == 1 or n * ldx < 1 << 30)
        if T * ld < 1 << 30 and ld <= 1 << 20:
            assert ldx == (ld if T > 1 else K) and xp == x.data_ptr() + 2 * ldx * at
        assert ip == ids.data_ptr() + 4 * k * at and wp == w.data_ptr() + 4 * k * at and yp == y.data_ptr() + 2 * K * at
        assert xp % 16 == yp % 16 == 0
        from smla import _lib
        assert wsb >= _lib.lib().smla_experts_workspace(n, k, E, K, inner, _lib.BF16)
        at += n
    assert at == T
    fewest = max(-(-T * k // (1 << 20)), -(-T * K // ((1 << 30) - 1)))
    assert len(calls) <= fewest + 1


def test_products_of_rows_that_lie_far_apart(calls):
    from smla import ops
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    for ld, want in (((1 << 22), 1 << 22), ((1 << 22) + 8, 64)):
        x = torch.empty_strided((3, 64), (ld, 1), dtype=torch.bfloat16)
        ops._linear_fp4(x, codes, scales, torch.float32)
        assert calls[-1][1][1] == want


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_tokens_outside_the_table_choose_nothing(monkeypatch, dtype):
    """A layer that chooses by token (a padded batch's -1, an id past the vocabulary): ids of -1, which add nothing, in place of a
    row that is another token's or no row at all."""
    from smla import moe, ops
    seen = []
    monkeypatch.setattr(ops, "linear_op", lambda x, w, groups, dt: torch.zeros(x.shape[0], w.shape[0], dtype=dt))
    monkeypatch.setattr(moe, "route", lambda logits, k, ids=None, **kw: (seen.append(ids), (ids, None))[1])
    monkeypatch.setattr(moe, "experts", lambda x, *rest: x.clone())
    w = _bf16(3, 32, 64)
    table = torch.arange(10, dtype=torch.int32).view(5, 2)
    layer = moe.ExpertLayer(moe.ExpertWeights(_bf16(3, 64), w, w, w, table=table), k=2)
    tokens = torch.tensor([[0, 4, -1, 3], [5, -5, 1, torch.iinfo(dtype).max]], dtype=dtype)
    assert layer(_bf16(2, 4, 64), tokens).shape == (2, 4, 64)
    assert seen[0].tolist() == [[0, 1], [8, 9], [-1, -1], [6, 7], [-1, -1], [-1, -1], [2, 3], [-1, -1]]
    assert table.tolist() == [[0, 1], [2, 3], [4, 5], [6, 7], [8, 9]] and seen[0].dtype == torch.int32


@pytest.mark.parametrize("current", [0, 1])
def test_a_layer_on_another_device(monkeypatch, current):
    """Every launch of a layer and of the packing of its weights is made with the tensors' GPU current, on a stream of it."""
    import contextlib
    from smla import _lib, moe, ops
    now, made = [current], []

    @contextlib.contextmanager
    def device(dev):
        before, now[0] = now[0], dev
        yield
        now[0] = before
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(ops, "_current_device", lambda: now[0])
    monkeypatch.setattr(ops, "_one_device", lambda t, *rest: 1)
    monkeypatch.setattr(ops, "_on_gpu", lambda *ts: None)
    monkeypatch.setattr(ops, "_raw_stream", lambda dev: ("stream", 1 if dev is None else dev))
    monkeypatch.setattr(_lib, "call", lambda name, *args: made.append((name, now[0], args[-1])))
    monkeypatch.setattr(ops, "linear_op", ops._linear)
    monkeypatch.setattr(ops, "route_op", ops._route)
    monkeypatch.setattr(ops, "experts_op", ops._experts)
    monkeypatch.setattr(ops, "rotate_fp4_op", ops.rotate_fp4_op._init_fn)
    gate, down = moe.pack_fp4(_bf16(3, 32, 64)), moe.pack_fp4(_bf16(3, 64, 32))
    for T in (1, 8, 40):
        for dt in (torch.bfloat16, torch.float32):
            moe.ExpertLayer(moe.ExpertWeights(torch.zeros(2, 64, dtype=dt), gate, gate, down), k=2)(_bf16(T, 64))
    assert [m[0] for m in made] == ["smla_rotate_fp4"] * 2 + ["smla_linear_ws", "smla_route", "smla_experts"] * 6
    assert all(m[1:] == (1, ("stream", 1)) for m in made), made


def test_rows_and_choices_of_nothing_are_the_librarys_errors(calls, monkeypatch):
    """Many tokens of no choices or of empty rows reach the library, which refuses them."""
    import ctypes
    from smla import _lib, ops
    monkeypatch.setattr(ops, "_launch", lambda dev, name, *args: _lib.call(name, *args, ctypes.c_void_p(0)))
    T = (1 << 20) + 1
    for k, K in ((1, 0), (0, 32)):
        x = torch.empty(T, K, dtype=torch.bfloat16)
        with pytest.raises(_lib.SmlaError):
            ops._experts(x, torch.zeros(T, k, dtype=torch.int32), torch.zeros(T, k), _bf16(2, 32, K), _bf16(2, 32, K),
                         _bf16(2, K, 32), None, None, None, 1.0)

"""CPU tier: which tile form a product with 4-bit weights and the experts take, restated from the constants in experts.hip and
held against the library's workspaces, so that the long cases of test_gpu_moe_long.py are known to run every form's loop past the
reuse of its rings (three groups of 512 k for the scales, two or three steps for the operands)."""
import os
import random
import re

import pytest

from test_gpu_moe_long import LONG_EXPERTS, LONG_LINEARS

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "deepseek-v4-flash-mlx_amd", "csrc")
CUS = 256


def _numbers(name):
    src = open(os.path.join(CSRC, "experts.hip")).read()
    return [float(v) for v in re.search(rf"\b{name}\[kForms\] = {{([^}}]*)}}", src).group(1).split(",")]


IDLE, ONE, BUSY = (_numbers(n) for n in ("kIdle", "kOne", "kBusy"))
BM, BN, KB = ([int(v) for v in _numbers(n)] for n in ("kFormBM", "kFormBN", "kFormKB"))


def _up(a, b):
    return -(-a // b)


def _few_lds(n, K, nw, r):
    steps = _up(K, 128)
    return n * (256 * steps + 16 * nw) + nw * r * (_up(_up(steps, nw), 4) * 256)


def linear_plan(T, N, K):
    """(form, splits, steps): form -1 is the kernel for few tokens."""
    best, bt = (2, 1), 1e30
    nw, tt = (4 if K <= 2048 else 8 if K <= 4096 else 16), _up(T, 16)
    lds = _few_lds(min(T, 16), K, nw, K % 128 == 0)
    if lds <= 144 * 1024 and tt <= 65535:
        wgs = _up(N, 16) * tt
        each = max(0.7, K * (2.0 * T / tt + 8.5) * 25.3e-6)
        more = _up(wgs, CUS) - 1 if 2 * (lds + 1024 * nw) > 160 * 1024 else max(0.0, wgs / CUS - 1)
        best, bt = (-1, 1), 3.6 + 0.35 * K / 1024 + more * each
    for f in range(3):
        tiles, steps, cap = _up(T, BM[f]) * _up(N, BN[f]), _up(K, KB[f]), CUS * (2 if f == 1 else 1)
        s = 1
        while s <= (1 if f == 2 else 8) and (s == 1 or steps // s >= 2):
            rest, t = tiles * s % cap, tiles * s // cap * BUSY[f]
            if rest > CUS:
                t += ONE[f] + (BUSY[f] - ONE[f]) * (rest - CUS) / CUS
            elif rest > 0:
                t += IDLE[f] + (ONE[f] - IDLE[f]) * rest / CUS
            t = max(3.6 + t * _up(steps, s), 2.5 + N * K * 0.53 / 5.5e6)
            t += (2.4 + s * T * N * 8 / 4.3e6 if s > 1 else 0) + (2.5 if K % 128 else 0)
            if t < bt:
                bt, best = t, (f, s)
            s *= 2
    return best


def expert_form(T, k, E, K, fp4):
    if T <= 16 and _few_lds(T, K, 4, 2) <= 144 * 1024:
        return -1
    per = T * k // min(E, T * k)
    return (0 if per <= 32 else 2) if fp4 else (1 if per <= 56 else 2)


def _16(n):
    return (n + 15) // 16 * 16


def linear_bytes(T, N, K):
    form, splits = linear_plan(T, N, K)
    return 0 if form < 0 else (_16(4 * splits * T * N) if splits > 1 else 0) + (_16(N * _up(K, 128) * 4) if K % 128 else 0)


def experts_bytes(T, k, E, K, inner, fp4):
    P, form = T * k, expert_form(T, k, E, K, fp4)
    if form < 0:
        return 16 * P + _16(2 * P * inner)
    room = (P // BM[form] + min(E, P)) // 8 + 3
    pad = lambda rows, n: _16(rows * _up(n, 128) * 4) if fp4 and n % 128 else 0
    return 2 * _16(4 * P) + _16(32 + 96 * room) + _16(2 * P * inner) + _16(4 * P * K) + 2 * pad(E * inner, K) + pad(E * K, inner)


def _log(r, lo, hi):
    return int(round(lo * (hi / lo) ** r.random()))


def test_the_restatement_is_the_librarys():
    from smla import _lib
    lib, r = _lib.lib(), random.Random(2)
    for _ in range(3000):
        T, N, K = _log(r, 1, 5000), _log(r, 1, 30000), 32 * _log(r, 1, 300)
        assert lib.smla_linear_fp4_workspace(T, N, K) == linear_bytes(T, N, K), (T, N, K)
        T, E, inner = _log(r, 1, 5000), _log(r, 1, 1024), 32 * _log(r, 1, 100)
        k, fp4 = r.randint(1, min(E, 64)), r.random() < 0.5
        want = experts_bytes(T, k, E, K, inner, fp4)
        assert lib.smla_experts_workspace(T, k, E, K, inner, 5 if fp4 else 1) == want, (T, k, E, K, inner, fp4)


def test_the_long_cases_reach_every_form():
    """Each form of 4-bit weights: K in whole steps and not, each past the scales' third group and past the ring's stages in one
    split; both products of the experts."""
    seen = set()
    for T, N, K in LONG_LINEARS:
        form, splits = linear_plan(T, N, K)
        assert form >= 0 and _up(K, KB[form]) * KB[form] // splits > 3 * 512, (T, N, K, form, splits)
        seen.add((form, K % 128 > 0, splits > 1))
    assert {(f, odd) for f, odd, _ in seen} == {(f, odd) for f in range(3) for odd in (False, True)}
    assert {f for f, _, split in seen if split} == {0, 1}
    seen = set()
    for T, E, k, K, inner, kind in LONG_EXPERTS:
        form = expert_form(T, k, E, K, kind == "fp4")
        assert form >= 0 and min(K, inner) > 3 * 512
        seen.add((kind, form, K % 128 > 0, inner % 128 > 0))
    assert {s[:2] for s in seen} == {("fp4", 0), ("fp4", 2), ("bf16", 1), ("bf16", 2)}
    for form in (0, 2):
        mine = [s for s in seen if s[:2] == ("fp4", form)]
        assert {s[2] for s in mine} == {s[3] for s in mine} == {False, True}

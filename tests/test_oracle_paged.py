"""CPU tier: the oracle of the paged cache against the reference-shaped attention oracle on contiguous rows,
closed forms, and the invariants its page tables have to keep."""
import random

import pytest
import torch

from oracle import norm_rope as onr
from oracle import paged as op
from oracle import sparse_attn as osa


def _cache(g, lens, P, D, extra=3):
    cols = max(-(-n // P) for n in lens)
    total = sum(-(-n // P) for n in lens) + extra
    perm = torch.randperm(total, generator=g).tolist()
    table = torch.full((len(lens), cols), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        for c in range(-(-n // P)):
            table[b, c] = perm.pop()
    return torch.randn(total, P, D, generator=g), table


@pytest.mark.parametrize("window,first", [(0, 0), (5, 0), (5, 3), (100, 2)])
def test_attention_is_the_reference_over_the_seen_rows(window, first):
    g = torch.Generator().manual_seed(1)
    lens, n = [7, 23], [7, 4]
    pages, table = _cache(g, lens, 4, 32)
    q, sink = torch.randn(sum(n), 3, 32, generator=g), torch.randn(3, generator=g)
    cu = [0, 7, 11]
    out, spread = op.paged_attn(q, pages, table, lens, cu, 32 ** -0.5, sink, window, first, dv=16)
    for b in range(2):
        kv = torch.stack([pages[table[b, j // 4], j % 4] for j in range(lens[b])])
        for i in range(n[b]):
            p = lens[b] - n[b] + i
            ids = [j if j <= p and (not window or j > p - window or j < first) else -1 for j in range(lens[b])]
            ref = osa.sparse_attn(q[cu[b] + i][None], kv, sink, torch.tensor([ids]), 32 ** -0.5, dv=16)
            assert torch.allclose(out[cu[b] + i].float(), ref[0], atol=1e-5)
    assert (spread + 1e-12 >= out.abs()).all()


def test_no_row_gives_zero():
    q = torch.ones(2, 1, 8)
    out, _ = op.paged_attn(q, torch.ones(1, 4, 8), torch.tensor([[-1], [0]]), [4, 1], [0, 1, 2], 1.0, dv=8)
    assert out[0].abs().max() == 0 and torch.equal(out[1], torch.ones(1, 8, dtype=torch.float64))


def test_norm_rope_matches_the_reference_form():
    g = torch.Generator().manual_seed(2)
    x, w = torch.randn(3, 64, generator=g), torch.randn(64, generator=g)
    freqs = onr.precompute_freqs_cis(16, 10, 0, 10000.0, 40, 32, 1)[7]
    y = op.norm_rope(x, w, True, 64, freqs.real, freqs.imag, 1e-6)
    ref = onr.rmsnorm(x, w, 1e-6)
    ref[:, -16:] = onr.apply_rotary_emb(ref[None, :, None, -16:].transpose(0, 1), freqs[None])[:, 0, 0]
    assert torch.allclose(y.float(), ref, atol=1e-5)


def _check_state(table, lens, refs, P):
    count = [0] * len(refs)
    for row, n in zip(table, lens):
        used = -(-n // P)
        assert all(p >= 0 for p in row[:used]) and all(p == -1 for p in row[used:])
        for p in row[:used]:
            count[p] += 1
    assert count == list(refs)
    # a page that two slots hold is whole in both
    for row, n in zip(table, lens):
        if n % P:
            assert refs[row[n // P]] == 1


def test_updates_keep_the_tables_sound():
    r = random.Random(3)
    P, S, M, n_pages = 4, 6, 8, 24
    table, lens, refs = [[-1] * M for _ in range(S)], [0] * S, [0] * n_pages
    data = [[None] * P for _ in range(n_pages)]     # what each row holds
    want = [[] for _ in range(S)]                   # each slot's rows in order
    seen = set()
    for step in range(300):
        parent = [r.choice([s, s, r.randrange(S), -1]) for s in range(S)]
        grow = [r.choice([0, 1, 1, r.randrange(12)]) for _ in range(S)]
        before = [list(w) for w in want]
        table, lens2, refs, granted, copies = op.update_pages((P, n_pages), table, lens, refs, parent, grow)
        for a, b, k in copies:
            data[b][:k] = data[a][:k]
        for s in range(S):
            seen.add(granted[s])
            if granted[s]:
                want[s] = list(before[parent[s]]) if parent[s] >= 0 else []
                for _ in range(grow[s]):
                    j = len(want[s])
                    want[s].append((step, s, j))
                    data[table[s][j // P]][j % P] = (step, s, j)
        lens = lens2
        _check_state(table, lens, refs, P)
        for s in range(S):
            assert [data[table[s][j // P]][j % P] for j in range(lens[s])] == want[s]
        if step % 7 == 0:
            table, refs, live, moves = op.compact_pages(table, refs)
            for a, b in moves:
                data[b] = list(data[a])
            assert all(x > 0 for x in refs[:live]) and not any(refs[live:])
            _check_state(table, lens, refs, P)
    assert seen == {0, 1}


def test_rows_given_back_free_their_pages():
    """Growth of either sign: a draft's pages past the accepted rows are free again, and refs counts what the tables name."""
    r = random.Random(4)
    P, S, M, n_pages = 4, 6, 8, 30
    table, lens, refs = [[-1] * M for _ in range(S)], [0] * S, [0] * n_pages
    shorter = 0
    for _ in range(400):
        parent = [r.choice([s, s, s, r.randrange(S), -1]) for s in range(S)]
        grow = [r.choice([0, 1, 5, -1, -5, -40, r.randrange(12)]) for _ in range(S)]
        before = lens
        table, lens, refs, granted, copies = op.update_pages((P, n_pages), table, lens, refs, parent, grow)
        for s, p in enumerate(parent):
            have = before[p] if p >= 0 else 0
            assert lens[s] == (have + grow[s] if granted[s] else before[s])
            shorter += granted[s] and grow[s] < 0 and p == s and -(-lens[s] // P) < -(-before[s] // P)
        count = [0] * n_pages
        for row, n in zip(table, lens):
            used = -(-n // P)
            assert all(p >= 0 for p in row[:used]) and all(p == -1 for p in row[used:])
            for p in row[:used]:
                count[p] += 1
        assert count == refs
        assert all(refs[b] == 1 and 0 < k < P for _, b, k in copies)
    assert shorter > 20
    t, n, f, ok, _ = op.update_pages((P, n_pages), table, lens, refs, list(range(S)), [-x for x in lens])
    assert not any(n) and not any(f) and all(ok)


def test_rows_given_back_past_a_fork_stay_the_other_slots():
    """Random forks, growth and rows given back: each slot's rows are its own however its pages are shared."""
    r = random.Random(5)
    P, S, M, n_pages = 4, 6, 8, 40
    table, lens, refs = [[-1] * M for _ in range(S)], [0] * S, [0] * n_pages
    data, want, own = [[None] * P for _ in range(n_pages)], [[] for _ in range(S)], 0
    for step in range(600):
        parent = [r.choice([s, s, s, r.randrange(S), -1 if r.random() < 0.3 else s]) for s in range(S)]
        grow = [r.choice([0, 1, 1, -1, -2, r.randrange(9), -r.randrange(9)]) for _ in range(S)]
        before = [list(w) for w in want]
        table, lens, refs, granted, copies = op.update_pages((P, n_pages), table, lens, refs, parent, grow)
        moved = [(b, k, list(data[a])) for a, b, k in copies]
        for b, k, was in moved:
            data[b][:k] = was[:k]
        for s in range(S):
            if granted[s]:
                have = before[parent[s]] if parent[s] >= 0 else []
                want[s] = list(have[:min(len(have), len(have) + grow[s])])
                for j in range(len(want[s]), lens[s]):
                    want[s].append((step, s, j))
                    data[table[s][j // P]][j % P] = (step, s, j)
        own += sum(granted[s] and parent[s] == s and any(table[s][len(want[s]) // P] == b for _, b, _ in copies)
                   for s in range(S) if len(want[s]) < M * P)
        for s in range(S):
            assert [data[table[s][j // P]][j % P] for j in range(lens[s])] == want[s], (step, s)
    assert own > 5

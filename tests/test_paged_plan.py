"""The plan of an attention over pages, on the CPU: every row meets every piece of a block that it sees exactly once, rows that are joined are
joined of all of their parts, and what is refused."""
import random

import numpy as np
import pytest


def plan(lens, table, open_, seq, counts, rep, H, D, causal, page, few_rows, few_work=1, cap=1 << 18):
    from kvq import _lib
    lens, seq, counts = (np.array(x, dtype=np.int64) for x in (lens, seq, counts))
    table, open_ = np.ascontiguousarray(table, dtype=np.int32), np.array(open_, dtype=np.uint8)
    info, words = np.zeros(12, dtype=np.int64), np.full(cap, -7, dtype=np.int32)
    _lib.call("kvq_paged_plan", lens.ctypes.data, table.ctypes.data, open_.ctypes.data, len(lens), table.shape[1], page, seq.ctypes.data,
              counts.ctypes.data, len(seq), rep, H, D, int(causal), few_rows, few_work, -(-512 // H), -(-256 // H), 16384 // H,
              words.ctypes.data, cap, info.ctypes.data)
    i = info.tolist()
    if cap < 12 * i[0] + 8 * i[1] + i[4]:      # nothing but the sizes
        assert (words == -7).all()
        return i, None, None, None
    items = words[:12 * i[0]].reshape(-1, 12)
    merges = words[12 * i[0]:12 * i[0] + 8 * i[1]].reshape(-1, 8)
    few = words[12 * i[0] + 8 * i[1]:12 * i[0] + 8 * i[1] + i[4]]
    assert (words[12 * i[0] + 8 * i[1] + i[4]:] == -7).all()
    return i, items, merges, few


def keys_of(table, slot, u0, u1, length, page):
    """What units [u0, u1) of a slot hold: (page, first token) of each piece of a block of 32 or 64 tokens."""
    full = length // page * page
    n_full, piece = -(-full // 64), min(page, 64)
    for u in range(u0, u1):
        if u < n_full:
            for t in range(64 * u, min(64 * u + 64, full), piece):
                yield int(table[slot][t // page]), t
        else:
            yield "open", slot, full + (u - n_full) * 64


def check(lens, table, open_, seq, counts, rep, H, D, causal, page, few_rows):
    i, items, merges, few = plan(lens, table, open_, seq, counts, rep, H, D, causal, page, few_rows)
    keys = lambda slot, u0, u1, length: keys_of(table, slot, u0, u1, length, page)
    rows = sum(counts)
    slot_of, sees = [], []
    for s, c in zip(seq, counts):
        for t in range(c):
            slot_of.append(s)
            sees.append(lens[s] - c + t + 1 if causal else lens[s])
    seen = [dict() for _ in range(rows)]       # (page or open block, token) -> times
    parts = [[] for _ in range(rows)]          # (part, row in the part) of each row, or "out"

    def add(row, slot, u0, u1, length, buf):
        if not length:
            return
        n_full = -(-(length // page * page) // 64)
        assert u1 <= n_full or buf == open_[slot] & 1
        for key in keys(slot, u0, u1, length):
            seen[row][key] = seen[row].get(key, 0) + 1

    per_tile = 32 * i[3] // rep
    for row0, toks, slot, u0, u1, vis0, step, length, buf, part, *_ in items.tolist():
        assert 0 <= toks <= per_tile and 0 <= row0 and row0 + toks <= rows and u0 <= u1 and part < i[2]
        assert length <= lens[slot]
        for t in range(toks):
            row = row0 + t
            add(row, slot, u0, u1, length, buf)
            assert min(vis0 + step * t, length) == min(sees[row], length)
            parts[row].append((part, t) if part >= 0 else "out")
    joined = [0] * rows
    for row0, toks, p0, n0, o0, p1, n1, o1 in merges.tolist():
        for t in range(toks):
            row = row0 + t
            joined[row] += 1
            assert sorted(parts[row]) == sorted([(p0 + k, o0 + t) for k in range(n0)] + [(p1 + k, o1 + t) for k in range(n1)])
        assert max(n0, n1) <= i[11]
    taken = [False] * rows
    if i[5]:
        n, head = i[5], few[:12].tolist()
        assert head[0] == n and head[2] == i[6] and head[6] == i[7] and head[7] == i[8] and head[10] == i[9]
        seqs, runs = few[12:12 + 8 * (n + 1)].reshape(-1, 8).tolist(), few[12 + 8 * (n + 1):12 + 8 * (n + 1) + 12 * (head[8] + 1)].reshape(-1, 12).tolist()
        assert sum(r[11] for r in runs[:-1]) == head[2] == runs[-1][5]
        for k, (slot, row0, tokens, u0, u1, split0, base, b, pos0, buf, front, count) in enumerate(runs[:-1]):
            assert count == -(-(u1 - u0) // head[3]) and split0 == sum(r[11] for r in runs[:k])
            for row in range(row0, row0 + tokens):
                if b >= 0:
                    assert seqs[b][3] == row0 and seqs[b][5] == k and not taken[row]
                    taken[row] = True
                length = u1 * 64 if b < 0 else pos0 + tokens if causal else pos0
                assert b < 0 or length == lens[slot]
                add(row, slot, u0, u1, length, buf)
    for row in range(rows):
        slot, n = slot_of[row], sees[row]
        n_all = -(-(lens[slot] // page * page) // 64) + -(-(lens[slot] % page) // 64)
        want = {key for key in keys(slot, 0, n_all, lens[slot]) if key[-1] < n}
        assert want <= set(seen[row]) and set(seen[row].values()) <= {1}, (row, slot)
        if taken[row]:
            assert not parts[row]
        elif joined[row]:
            assert joined[row] == 1 and "out" not in parts[row]
        else:
            assert parts[row] == ["out"]
    return i


@pytest.mark.parametrize("seed", range(30))
def test_every_row_meets_what_it_sees_once(seed):
    rng = random.Random(seed)
    page, rep, H = rng.choice([32, 64, 128]), rng.choice([1, 3, 4, 8, 40]), rng.choice([1, 2, 8, 70])
    slots, blocks, nxt = 10, 40, 0
    lens = [rng.choice([0, 1, page, rng.randint(0, 20 * page)]) for _ in range(slots)]
    table = np.zeros((slots, blocks), dtype=np.int32)
    for s in range(slots):
        origin = rng.randrange(s) if s and rng.random() < 0.7 else None
        shared = 0
        if origin is not None:
            shared = min(lens[origin] // page, rng.choice([blocks, rng.randint(0, blocks)]))
            lens[s] = shared * page + rng.choice([0, 1, rng.randint(0, 3 * page)])
            table[s, :shared] = table[origin, :shared]
        for j in range(shared, lens[s] // page):
            table[s, j], nxt = nxt, nxt + 1
    open_ = [rng.randrange(2) for _ in range(slots)]
    causal = rng.random() < 0.6
    seq = sorted(rng.choice(range(slots)) for _ in range(rng.randint(1, 9)))
    if rng.random() < 0.3:
        rng.shuffle(seq)
    counts = [min(rng.choice([0, 1, 2, rng.randint(0, 150)]), lens[s] if causal else 400) for s in seq]
    for few_rows in (0, 32, 1 << 30):
        check(lens, table, open_, seq, counts, rep, H, rng.choice([64, 128]), causal, page, few_rows)


def test_shared_texts_and_parts_are_used():
    table = np.tile(np.arange(70), (9, 1))
    for s in range(9):
        table[s, 64:] = 1000 + 10 * s + np.arange(6)
    lens = [64 * 64 + 10 + s for s in range(9)]
    i = check(lens, table, [0] * 9, list(range(8)), [9] * 8, 4, 8, 128, True, 64, 0)
    assert i[1] >= 8 and i[2] > 16             # joined, and the text in several parts
    assert i[0] * 8 <= 4 * 512
    i = check(lens, table, [0] * 9, list(range(8)), [1] * 8, 4, 8, 128, True, 64, 32)
    assert i[0] == 0 and i[5] == 8 and i[10]   # few rows: the decode's kernels, with the text read once
    i = check(lens, table, [0] * 9, [3, 3, 3], [1, 2, 60], 4, 8, 128, False, 64, 0)
    assert i[1] == 2 and i[2] == 2 * i[11]     # 63 rows of one slot are two tiles


def test_a_full_chip_takes_wider_tiles():
    table = np.arange(40 * 70).reshape(40, 70)
    lens = [64 * 60 + s for s in range(40)]
    assert check(lens, table, [0] * 40, list(range(40)), [320] * 40, 4, 8, 128, True, 64, 32)[3] == 8
    assert plan(lens, table, [0] * 40, list(range(40)), [320] * 40, 4, 8, 64, True, 64, 32)[0][3] == 4
    assert plan(lens, table, [0] * 40, list(range(4)), [320] * 4, 4, 8, 128, True, 64, 32)[0][3] == 4


def test_refusals_and_short_buffers():
    from kvq import _lib
    table = np.arange(40).reshape(2, 20)
    good = dict(lens=[100, 0], table=table, open_=[0, 0], seq=[0, 1], counts=[5, 0], rep=4, H=2, D=64, causal=True, page=64, few_rows=32)
    plan(**good)
    for bad, match in ((dict(seq=[0, 2]), "no slot"), (dict(seq=[-1, 1]), "no slot"), (dict(counts=[101, 0]), "last ones"), (dict(counts=[-1, 0]), "negative"),
                       (dict(counts=[1 << 31, 0], causal=False), "2\\^31"), (dict(rep=129), "sizes"), (dict(rep=0), "sizes"), (dict(H=0), None),
                       (dict(page=48), "sizes"), (dict(D=96), "sizes")):
        if match is None:
            continue
        with pytest.raises(_lib.KVQError, match=match):
            plan(**{**good, **bad})
    i, items, *_ = plan(**{**good, "few_rows": 0}, cap=4)
    assert i[0] == 1 and items is None
    lib = _lib.load()
    assert lib.kvq_paged_attention_workspace(3, 4, 2, 64) == 3 * 2 * 128 * 66 and lib.kvq_paged_attention_workspace(3, 8, 2, 128) == 3 * 2 * 256 * 130
    assert lib.kvq_paged_attention_workspace(3, 8, 2, 64) == -1 and lib.kvq_paged_attention_workspace(-1, 4, 2, 64) == -1
    one = 1 << 12
    call = lambda items, merges, parts, waves, floats, D=64, P=64, q=one: lib.kvq_paged_attention(
        q, 256, 64, 2, 8, 2, D, 0.1, one, items, merges, parts, 0, waves, one, 20, P, 0, one, one, one, one, one, one, one, floats, None)
    for args, match in (((1, 0, 1, 4, 10), b"workspace"), ((1, 0, 0, 8, 0), b"wavefronts"), ((1 << 24, 0, 0, 4, 0), b"too many"),
                        ((1, 1 << 24, 0, 4, 0), b"too many"), ((-1, 0, 0, 4, 0), b"bad sizes"), ((1, 0, 0, 4, 0, 96), b"head_dim"),
                        ((1, 0, 0, 4, 0, 64, 16), b"pages"), ((1, 0, 0, 4, 0, 64, 64, None), b"null"), ((1, 0, 0, 4, 0, 64, 64, one + 8), b"multiples")):
        assert call(*args) != 0 and match in lib.kvq_last_error(), (args, lib.kvq_last_error())
    assert call(0, 0, 0, 4, 0) == 0            # nothing to do


def test_device_tables_refusals():
    from kvq import _lib
    lib = _lib.load()
    assert lib.kvq_tables_step_words(64, 8, 100) == 12 + 8 * 9 + 12 * 17 + 8 * 3
    for bad in ((48, 8, 1), (64, 0, 1), (64, 8, 0), (64, 1 << 20, 1 << 12)):
        assert lib.kvq_tables_step_words(*bad) == -1
    one, words = 1 << 12, lib.kvq_tables_step_words(64, 8, 100)
    call = lambda n=8, most=100, page=64, tokens=1000, pages=50, blocks=16, splits=8, slots=one, w=words, scratch=8 + 24: lib.kvq_tables_extend(
        slots, one, n, most, page, tokens, pages, blocks, splits, one, one, one, one, one, one, w, one, scratch, one, one, None)
    for bad, match in ((dict(slots=None), b"null"), (dict(w=words - 1), b"short"), (dict(scratch=31), b"short"), (dict(tokens=1025), b"bad sizes"),
                       (dict(splits=7), b"split item"), (dict(page=16), b"bad sizes"), (dict(tokens=1 << 31, blocks=1 << 30), b"bad sizes")):
        assert call(**bad) != 0 and match in lib.kvq_last_error(), (bad, lib.kvq_last_error())
    assert lib.kvq_tables_free(one, None, 0, 64, 4, one, one, one, one, one, None) != 0
    assert lib.kvq_tables_free(None, None, 1, 64, 4, one, one, one, one, one, None) != 0

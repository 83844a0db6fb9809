"""The page accounts and the plans of the paged cache and of prompt attention, on the host: against a plain
model of the accounts, and everything that is refused."""
import ctypes
import random

import numpy as np
import pytest

from oracle.paged import Accounts


class Host:
    """The accounts as PagedCache keeps them, without a device."""

    def __init__(self, slots, pages, max_tokens, page):
        from kvq import _lib
        self.lib = _lib.load()
        self.slots, self.pages, self.page, self.max_tokens, self.blocks = slots, pages, page, max_tokens, -(-max_tokens // page)
        self.lens = np.zeros(slots, np.int64)
        self.table = np.zeros((slots, self.blocks), np.int32)
        self.refs = np.zeros(pages, np.int32)
        self.open = np.zeros(slots, np.uint8)
        self.account = np.array([pages, 0], np.int64)
        self.p = [x.ctypes.data for x in (self.lens, self.table, self.refs, self.open, self.account)]

    def extend(self, slots, counts, cap=64, words=None, run=1 << 31, tokens=1 << 31, few=(0, 0)):
        s, c = np.array(slots, np.int64), np.array(counts, np.int64)
        n = self.lib.kvq_pages_step_words(self.page, c.ctypes.data, len(c)) if words is None else words
        self.desc = np.zeros(max(n, 1), np.int32)
        return self.lib.kvq_pages_extend(*self.p, self.slots, self.pages, self.blocks, self.page, self.max_tokens, s.ctypes.data,
                                         c.ctypes.data, len(s), cap, *few, run, tokens, self.desc.ctypes.data, n, None, None)

    def fork(self, src, dst):
        s, d = np.array(src, np.int64), np.array(dst, np.int64)
        return self.lib.kvq_pages_fork(*self.p[:4], self.slots, self.blocks, self.page, s.ctypes.data, d.ctypes.data, len(s), 1, 1, 64,
                                       None, None, None, None)

    def free(self, slots):
        s = np.array(slots, np.int64)
        return self.lib.kvq_pages_free(*self.p, self.slots, self.blocks, self.page, s.ctypes.data, len(s))

    def move(self, end, pages, same):
        refs = self.refs if same else np.zeros(pages, np.int32)
        place = np.zeros(len(self.refs), np.int32)
        rc = self.lib.kvq_pages_move(*self.p[:3], refs.ctypes.data, self.p[4], self.slots, self.pages, pages, end, self.blocks, self.page,
                                     place.ctypes.data, 1, 1, 64, 16, 16, 16, *([16] * 3 if same else [32] * 3), None, None)
        if rc == 0:
            self.refs, self.pages = refs, pages
            self.p[2] = refs.ctypes.data
        return rc

    def error(self):
        return self.lib.kvq_last_error()

    def same(self, model):
        assert self.lens.tolist() == model.lens and self.refs.tolist() == model.refs
        for s, pages in enumerate(model.table):
            assert self.table[s, :len(pages)].tolist() == pages
        free = [i for i, r in enumerate(model.refs) if r == 0]
        assert self.account[0] == len(free) and (not free or self.account[1] <= free[0])


@pytest.mark.parametrize("page", [32, 64, 128])
def test_accounts_follow_the_model(page):
    rng = random.Random(page)
    host, model = Host(9, 40, 20 * page, page), Accounts(9, 40, page)
    for _ in range(300):
        op = rng.choice(["extend", "extend", "extend", "extend", "fork", "free", "move"])
        if op == "extend":
            slots = rng.sample(range(9), rng.randint(1, 4))
            counts = [rng.choice([0, 1, 2, page - 1, page, rng.randint(1, 3 * page)]) for _ in slots]
            need = sum((host.lens[s] + c) // page - host.lens[s] // page for s, c in zip(slots, counts))
            fits = need <= host.account[0] and all(host.lens[s] + c <= host.max_tokens for s, c in zip(slots, counts))
            rc = host.extend(slots, counts)
            assert (rc == 0) == fits, host.error()
            if fits:
                model.extend(slots, counts)
                _description(host, slots, counts)
            else:
                assert b"decode buffer exhausted" in host.error()
        elif op == "fork":
            empty = [s for s in range(9) if host.lens[s] == 0]
            held = [s for s in range(9) if host.lens[s]]
            if not empty or not held:
                continue
            dst = rng.sample(empty, rng.randint(1, len(empty)))
            src = [rng.choice(held) for _ in dst]
            assert host.fork(src, dst) == 0
            model.fork(src, dst)
        elif op == "move":
            used, same = host.pages - int(host.account[0]), rng.random() < 0.5
            end = rng.randint(used, host.pages) if same else max(1, used, rng.randint(20, 50))
            assert host.move(end, host.pages if same else end, same) == 0
            model.move(end, host.pages)
        else:
            slots = rng.sample(range(9), rng.randint(1, 3))
            assert host.free(slots + slots[:1]) == 0              # a slot named twice is empty the second time
            model.free(slots)
        host.same(model)


def _description(host, slots, counts, most=64):
    """Rows, items, the pages of what gets full; runs: every unit of every sequence in one, shared ones only in front."""
    n, d, page = len(slots), host.desc, host.page
    seq, nr = d[12:12 + 8 * (n + 1)].reshape(n + 1, 8), int(d[8])
    runs = d[12 + 8 * (n + 1):][:12 * (nr + 1)].reshape(nr + 1, 12)
    pages = d[int(d[9]):]
    assert seq[n, 5] == nr and d[9] == 12 + 8 * (n + 1) + 12 * (nr + 1)
    row = item = 0
    for i, (s, c) in enumerate(zip(slots, counts)):
        end = int(host.lens[s])
        pos0 = end - c
        assert seq[i, :5].tolist() == [s, pos0, c, row, item]
        for j in range(pos0 // page, (end - 1) // page + 1 if c else 0):
            want = host.table[s, j] if (j + 1) * page <= end else -1
            assert pages[item] == want
            item += 1
        full = end // page * page
        units = -(-full // 64) + -(-(end - full) // 64)
        own, front = runs[seq[i, 5]], seq[i, 7]
        assert own[[0, 1, 2, 7]].tolist() == [s, row, c, i] and own[4] == (units if c else own[3])
        assert own[3] == (runs[front - 1, 4] if front else 0) and own[8:11].tolist() == [pos0, seq[i, 6] >> 1, front]
        if front:
            f = runs[front - 1]
            assert c and f[3] == 0 and f[4] >= 4 and f[7] == -1 and f[1] <= row and row + c <= f[1] + f[2]
            blocks = f[4] * 64 // page
            assert f[4] * 64 <= pos0 // page * page
            assert np.array_equal(host.table[s, :blocks], host.table[f[0], :blocks])
        row += c
    split = base = 0
    assert d[10] == (nr > n or (runs[:nr, 11] > 1).any()) and d[11] == (runs[:nr, 11] == 1).all()
    for r in runs[:nr]:
        assert r[5] == split and r[6] == base
        k = -(-(r[4] - r[3]) // int(d[3]))
        assert r[11] == k
        split, base = split + k, base + k * r[2]
    assert runs[nr, 5:7].tolist() == [split, base]
    assert d[4] == all(b - a == 1 for a, b in zip(seq[:, 4], seq[1:, 4]))
    assert seq[n, 3:5].tolist() == [row, item] and d[:3].tolist() == [n, item, split] and split <= most
    assert d[5:8].tolist() == [max(counts), max(max(counts), *(int(r[2]) for r in runs[:nr])), base]


def test_few_units_take_few_items():
    host = Host(6, 2000, 64 * 400, 64)
    for slots, counts, few, want in (([0], [64 * 64], (16, 100), 16), ([1], [64 * 64], (16, 63), 16), ([2], [64 * 300], (16, 400), 16),
                                     ([3, 4, 5], [64 * 300, 64, 64], (3, 400), 64)):       # the last: one would hold nearly all
        assert host.extend(slots, counts, cap=64, few=few) == 0
        _description(host, slots, counts)
        assert want // 2 < int(host.desc[2]) <= want


def test_uneven_sequences_take_more_items():
    """64 sequences with a place each, the longest twice an even share: up to twice as many items; not for even ones, short
    ones, more sequences than places, or a step that has to fit an older one."""
    slots = list(range(64))
    uneven = [64 * (1 + i % 60) for i in slots]
    for counts, few, more in ((uneven, (32, 1), True), (uneven, (0, 0), False), (uneven, (31, 1), False),
                              ([64 * (50 + i % 10) for i in slots], (32, 1), False), ([64 * (1 + i % 14) for i in slots], (32, 1), False)):
        host = Host(64, 64 * 64, 64 * 64, 64)
        assert host.extend(slots, counts, cap=64, few=few) == 0
        _description(host, slots, counts, most=128)
        assert (int(host.desc[2]) > 64) == more
    host = Host(64, 64 * 64, 64 * 64, 64)      # few units, but not one item for each: the same
    assert host.extend(slots, uneven, cap=64, few=(32, 10000)) == 0 and int(host.desc[2]) > 64
    host = Host(64, 64 * 64, 64 * 64, 64)
    assert host.extend(slots, [64 * 10] * 64, cap=96, few=(32, 10000)) == 0 and int(host.desc[2]) == 64 and not host.desc[10]


def test_fronts_of_forks():
    """Forks named side by side share a run in front; where the step has to fit an older one they do not."""
    host = Host(8, 60, 60 * 64, 64)
    assert host.extend([0], [64 * 9 + 5]) == 0 and host.extend([1], [64 * 6]) == 0
    assert host.fork([0, 0, 0, 1], [2, 3, 4, 5]) == 0
    slots, counts = [2, 3, 0, 4, 1, 5, 6], [1, 2, 1, 64, 1, 1, 3]
    assert host.extend(slots, counts) == 0
    _description(host, slots, counts)
    seq = host.desc[12:12 + 8 * 8].reshape(8, 8)
    assert seq[:7, 7].tolist() == [1, 1, 1, 1, 6, 6, 0] and seq[7, 5] == 9
    host.free(range(8))
    assert host.extend([0], [64 * 9]) == 0 and host.fork([0], [1]) == 0
    for limit in (dict(run=1), dict(tokens=2), dict(cap=2)):
        assert host.extend([0, 1], [1, 1], **limit) == 0
        assert int(host.desc[8]) == 2
    assert host.extend([0, 1], [1, 1], run=2, tokens=64, cap=64) == 0
    assert int(host.desc[8]) == 3
    assert host.extend([0, 1], [1, 0]) == 0 and int(host.desc[8]) == 2      # nobody to share with


def test_refusals_change_nothing():
    host = Host(4, 5, 400, 64)
    assert host.extend([0, 1], [130, 70]) == 0
    before = [x.copy() for x in (host.lens, host.table, host.refs, host.open, host.account)]
    for slots, counts, message in (([0, 0], [1, 1], b"named twice"), ([4], [1], b"no slot"), ([-1], [1], b"no slot"),
                                   ([2, 3], [64, -1], b"bad counts"), ([2], [401], b"exhausted"),
                                   ([2, 3], [64, 128], b"exhausted")):
        assert host.extend(slots, counts) == 1 and message in host.error(), (slots, counts, host.error())
    assert host.extend([2], [1], cap=0) == 1 and host.extend([2], [1], words=10) == 1
    for src, dst, message in (([0], [1], b"in use"), ([0, 0], [2, 2], b"twice"), ([0], [4], b"no slot"), ([-1], [2], b"no slot"),
                              ([0], [0], b"in use"), ([2], [2], b"both"), ([0, 2], [2, 3], b"both")):
        assert host.fork(src, dst) == 1 and message in host.error(), (src, dst, host.error())
    assert host.move(1, 1, False) == 1 and b"in use" in host.error()
    assert host.free([0, 9]) == 1 and b"no slot" in host.error()
    for a, b in zip(before, (host.lens, host.table, host.refs, host.open, host.account)):
        assert np.array_equal(a, b)


def _plan(lib, lq, lk, rep, H, causal):
    lq, lk, info = np.array(lq, np.int64), np.array(lk, np.int64), np.zeros(3, np.int64)
    args = (lq.ctypes.data, lk.ctypes.data, len(lq), rep, H, causal)
    rc = lib.kvq_prompt_plan(*args, None, 0, info.ctypes.data)
    if rc:
        return rc, None, None
    words = np.zeros(max(8 * info[0] + 4 * info[1], 1), np.int32)
    assert lib.kvq_prompt_plan(*args, words.ctypes.data, words.size, info.ctypes.data) == 0
    return info, words[:8 * info[0]].reshape(-1, 8), words[8 * info[0]:8 * info[0] + 4 * info[1]].reshape(-1, 4)


def test_prompt_plan_covers_every_key_of_every_row_once():
    """Tiles of rows, cut along the keys where they are few: each visible (row, key) pair in one item, the parts of a
    tile joined by one merge."""
    from kvq import _lib
    lib = _lib.load()
    rng = random.Random(3)
    cut = 0
    for _ in range(80):
        n, rep, causal, H = rng.randint(1, 6), rng.choice([1, 2, 3, 4, 7, 8, 128]), rng.choice([0, 1]), rng.choice([1, 2, 8])
        lq = [rng.choice([0, 1, 31, 32, rng.randint(0, 300)]) for _ in range(n)]
        lk = [max(0, a + rng.choice([0, 0, 50, -3, rng.randint(0, 9000)])) for a in lq]
        info, items, merges = _plan(lib, lq, lk, rep, H, causal)
        rows, keys = np.concatenate([[0], np.cumsum(lq)]), np.concatenate([[0], np.cumsum(lk)])
        pairs = [np.zeros((a, b), np.int32) for a, b in zip(lq, lk)]
        parts = {}
        done = np.zeros(int(rows[-1]), np.int32)
        for row, toks, key, nk, vis0, step, part, _ in items.tolist():
            s = int(np.searchsorted(rows, row, "right") - 1)
            t = row - rows[s]
            assert 0 < toks * rep <= 128 and row + toks <= rows[s + 1] and nk >= 0 and step == causal
            first = key - keys[s]
            assert 0 <= first and first + nk <= lk[s]
            for i in range(toks):
                sees = max(0, min(nk, vis0 + step * i))
                pairs[s][t + i, first:first + sees] += 1
            if part < 0:
                done[row:row + toks] += 1
            else:
                parts[part] = (row, toks)
        for part, count, row, toks in merges.tolist():
            assert count > 1 and all(parts.pop(part + i) == (row, toks) for i in range(count))
            done[row:row + toks] += 1
            cut += 1
        assert not parts and (done == 1).all()
        assert info[2] == sum(m[1] for m in merges)
        for a, b, x in zip(lq, lk, pairs):
            t, j = np.arange(a)[:, None], np.arange(b)[None]
            assert np.array_equal(x, (j <= t + b - a).astype(np.int32) if causal else np.ones_like(x))
    assert cut > 20
    assert _plan(lib, [-1], [1], 1, 1, 1)[0] == 1 and _plan(lib, [1], [-1], 1, 1, 1)[0] == 1
    assert _plan(lib, [1], [1], 129, 1, 1)[0] == 1 and _plan(lib, [1 << 30] * 2, [1, 1], 1, 1, 1)[0] == 1


def test_kernel_entries_refuse_before_any_launch():
    from kvq import _lib
    lib = _lib.load()
    one = ctypes.c_void_p(16)
    rc = lib.kvq_prompt_attention(one, 64, 64, one, 64, 64, one, 64, 64, 2, 4, 2, 96, 0.1, one, 1, 0, 0, one, None, 0, None)
    assert rc == 1 and b"head_dim" in lib.kvq_last_error()
    rc = lib.kvq_prompt_attention(one, 64, 64, one, 64, 64, one, 64, 64, 0, 4, 2, 64, 0.1, one, 1, 0, 0, one, None, 0, None)
    assert rc == 1 and b"fp16 or bf16" in lib.kvq_last_error()
    rc = lib.kvq_prompt_attention(one, 64, 60, one, 64, 64, one, 64, 64, 2, 4, 2, 64, 0.1, one, 1, 0, 0, one, None, 0, None)
    assert rc == 1 and b"16 bytes" in lib.kvq_last_error()
    assert lib.kvq_prompt_workspace(3, 2, 64) == 3 * 2 * 128 * 66
    rc = lib.kvq_prompt_attention(one, 64, 64, one, 64, 64, one, 64, 64, 2, 4, 2, 64, 0.1, one, 3, 1, 3, one, one, 3 * 2 * 128 * 66 - 1, None)
    assert rc == 1 and b"workspace" in lib.kvq_last_error()
    rc = lib.kvq_prompt_attention(one, 64, 64, one, 1 << 24, 64, one, 64, 64, 2, 4, 2, 64, 0.1, one, 1, 0, 0, one, None, 0, None)
    assert rc == 1 and b"2^24" in lib.kvq_last_error()
    rc = lib.kvq_pages_append(one, 64, 64, one, 64, 64, 2, one, 1, one, 4, 2, 64, 48, 0, one, one, one, one, one, None)
    assert rc == 1 and b"page" in lib.kvq_last_error()
    rc = lib.kvq_pages_append(one, 64, 64, one, 64, 64, 2, one, 1, one, 4, 2, 64, 64, 3, one, one, one, one, one, None)
    assert rc == 1 and b"code" in lib.kvq_last_error()
    need = lib.kvq_paged_decode_workspace(4, 2, 2, 64)
    assert need == 4 * 2 * 2 * 66
    rc = lib.kvq_paged_decode(one, 256, 64, 2, 1, 4, 2, 64, 0.1, one, 1, 4, 1, 4, 1, one, 4, 64, 0, one, one, one, one, one, one, one, need - 1, None, None)
    assert rc == 1 and b"workspace" in lib.kvq_last_error()
    assert lib.kvq_paged_decode_workspace(4, 2, 2, 96) == -1


def test_accounts_move_without_a_device():
    """Without a table on the device the pools are not looked at: null ones do, for one pool and for another."""
    host, model = Host(3, 20, 640, 64), Accounts(3, 20, 64)
    for f in (host, model):
        f.extend([0, 1, 2], [200, 300, 130])
        f.free([0])
    for end, pages, same in ((6, 20, True), (9, 9, False), (30, 30, False)):
        place, refs = np.zeros(len(host.refs), np.int32), host.refs if same else np.zeros(pages, np.int32)
        assert host.lib.kvq_pages_move(*host.p[:3], refs.ctypes.data, host.p[4], 3, host.pages, pages, end, host.blocks, 64,
                                       place.ctypes.data, 1, 1, 64, *[None] * 8) == 0, host.error()
        host.refs, host.pages = refs, pages
        host.p[2] = refs.ctypes.data
        model.move(end, pages)
        host.same(model)
    # one pool of two sizes, or in two places
    place, refs = np.zeros(30, np.int32), np.zeros(30, np.int32)
    for to, pages, kc, kc_to in ((host.refs, 31, 16, 16), (host.refs, 30, 16, 32), (refs, 30, 16, 16)):
        assert host.lib.kvq_pages_move(*host.p[:3], to.ctypes.data, host.p[4], 3, 30, pages, 30, host.blocks, 64, place.ctypes.data, 1, 1,
                                       64, kc, kc, kc, kc_to, kc_to, kc_to, 16, None) == 1
        assert b"one size" in host.error()
    host.same(model)

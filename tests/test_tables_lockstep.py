"""The device accounts' kernels followed on the CPU: their source compiled for the host, a wavefront at a time between barriers, the
wavefronts in several orders.  What is read without a barrier behind another wavefront's write comes out wrong here in every run."""
import ctypes
import os
import random
import subprocess

import numpy as np
import pytest

from oracle.paged import Accounts

HERE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lockstep")


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    from kvq._lib import SIGNATURES
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    out = str(tmp_path_factory.mktemp("lockstep") / "tables.so")
    subprocess.run([f"{rocm}/llvm/bin/clang++", "-x", "c++", "-std=c++17", "-O1", "-fPIC", "-shared", "-Wno-unknown-pragmas", "-I", HERE,
                    os.path.join(HERE, "tables.cpp"), "-o", out], check=True)
    lib = ctypes.CDLL(out)
    for name in ("kvq_tables_step_words", "kvq_tables_extend", "kvq_tables_free"):
        f = getattr(lib, name)
        f.restype, f.argtypes = SIGNATURES[name]
    lib.lockstep_error.restype = ctypes.c_char_p
    return lib


class Tables:
    """A cache's accounts as the kernels have them, and their model."""

    def __init__(self, lib, slots, pages, page, max_tokens):
        self.lib, self.page, self.max_tokens, self.pages = lib, page, max_tokens, pages
        self.blocks = -(-max_tokens // page)
        self.lens, self.open = np.zeros(slots, np.int32), np.zeros(slots, np.int32)
        self.refs, self.account = np.zeros(pages, np.int32), np.array([pages, 0, 0], np.int32)
        self.table = np.zeros((slots, self.blocks), np.int32)
        self.model = Accounts(slots, pages, page)

    def step(self, slots, most, splits):
        n = len(slots)
        words = self.lib.kvq_tables_step_words(self.page, n, most)
        items = words - 32 * n - 32
        return dict(slots=np.array(slots, np.int32), most=most, splits=splits, desc=np.zeros(words, np.int32),
                    scratch=np.zeros(n + items, np.int32), positions=np.full(n * most, -7, np.int32), places=np.full(n * most, -7, np.int64))

    def extend(self, st, counts, fits=True):
        n, most, page = len(st["slots"]), st["most"], self.page
        c = np.array(counts, np.int32)
        at = lambda a: a.ctypes.data
        refused = int(self.account[2])
        assert self.lib.kvq_tables_extend(at(st["slots"]), at(c), n, most, page, self.max_tokens, self.pages, self.blocks, st["splits"], at(self.lens),
                                          at(self.refs), at(self.open), at(self.account), at(self.table), at(st["desc"]), st["desc"].size,
                                          at(st["scratch"]), st["scratch"].size, at(st["positions"]), at(st["places"]), None) == 0
        assert self.lib.lockstep_error() is None
        assert int(self.account[2]) == refused + (not fits)
        counts = counts if fits else [0] * n
        before = [self.model.lens[s] for s in st["slots"]]
        self.model.extend(st["slots"].tolist(), counts)
        self.same()
        seqs, head = st["desc"][12:12 + 8 * (n + 1)].reshape(-1, 8), st["desc"][:12].tolist()
        runs = st["desc"][12 + 8 * (n + 1):12 + 8 * (n + 1) + 12 * (n + 1)].reshape(-1, 12)
        item_pages, item, split = st["desc"][head[9]:], 0, 0
        for i, (s, b, t) in enumerate(zip(st["slots"].tolist(), before, counts)):
            pages = self.model.table[s]
            want = [b + j if j < t else -1 for j in range(most)]
            assert st["positions"][i * most:(i + 1) * most].tolist() == want
            assert st["places"][i * most:(i + 1) * most].tolist() == [pages[p // page] * page + p % page if p >= 0 and p // page < len(pages) else -1
                                                                      for p in want]
            assert seqs[i].tolist()[:6] == [s, b, t, i * most, item, i] and runs[i].tolist()[5] == split
            for j in range(b // page, (b + t - 1) // page + 1) if t else ():
                assert item_pages[item] == (pages[j] if j < len(pages) else -1)
                item += 1
            full = (b + t) // page * page
            units = -(-full // 64) + -(-(b + t - full) // 64) if t else 0
            assert runs[i].tolist()[4] == units and runs[i].tolist()[11] == -(-units // head[3])
            split += -(-units // head[3])
        assert head[0] == n and head[1] == item and head[2] == split <= st["splits"] and head[5] == max(counts)

    def free(self, st, which):
        n = len(st["slots"])
        w = np.array(which, np.uint8)
        assert self.lib.kvq_tables_free(st["slots"].ctypes.data, w.ctypes.data, n, self.page, self.blocks, self.lens.ctypes.data, self.refs.ctypes.data,
                                        self.open.ctypes.data, self.account.ctypes.data, self.table.ctypes.data, None) == 0
        assert self.lib.lockstep_error() is None
        self.model.free([s for s, x in zip(st["slots"].tolist(), which) if x])
        self.same()

    def same(self):
        assert self.lens.tolist() == self.model.lens and self.refs.tolist() == self.model.refs
        assert self.account[0] == self.model.refs.count(0)
        assert all(r for r in self.model.refs[:self.account[1]])
        for s, pages in enumerate(self.model.table):
            assert self.table[s, :len(pages)].tolist() == pages, s


@pytest.mark.parametrize("order", [0, -1, 1, 3], ids=["first to last", "last to first", "from the second", "from the fourth"])
@pytest.mark.parametrize("n,most,page,splits", [(8, 1, 32, 32), (5, 70, 32, 40), (200, 2, 64, 256), (300, 1, 128, 512), (6, 3000, 64, 20), (1100, 1, 32, 1500)],
                         ids=str)
def test_every_order_of_the_wavefronts(lib, n, most, page, splits, order):
    """Steps of a token, of drafts and of prompts, of fewer and more sequences than the workgroup has threads; steps that do not fit;
    slots given back between them."""
    lib.lockstep_order(order)
    rng = random.Random(n + most)
    max_tokens = 3 * most + 3 * page
    t = Tables(lib, n + 1, n * (max_tokens // page) * 2 // 3 + 2, page, max_tokens)
    grow = t.step(rng.sample(range(n), min(n, 40)), 2 * page - 1, max(splits, n))
    st = t.step(rng.sample(range(n + 1), n), most, splits)
    room = lambda s: max_tokens - t.model.lens[s]
    fitting = lambda x, c: sum((t.model.lens[s] + k) // page - t.model.lens[s] // page for s, k in zip(x["slots"].tolist(), c)) <= t.model.refs.count(0)
    for r in range(3 if n < 1000 else 1):
        for x in (grow, st, st):
            c = [min(room(s), rng.choice([x["most"], x["most"], rng.randint(0, x["most"])])) for s in x["slots"].tolist()]
            t.extend(x, c, fits=fitting(x, c))
        t.extend(st, [most + 1] + [0] * (n - 1), fits=False)
        t.free(st, [rng.random() < 0.4 for _ in range(n)])


@pytest.mark.parametrize("order", [0, -1, 1])
def test_pages_between_those_of_others(lib, order):
    """Free pages far apart in a large pool, more than one look finds."""
    lib.lockstep_order(order)
    t = Tables(lib, 3, 9000, 32, 32 * 8200)
    hold = t.step([2], 32 * 3, 4)
    t.extend(hold, [96])
    fill = t.step([0, 1], 32 * 4000, 16)
    t.extend(fill, [32 * 4000, 5])
    t.free(fill, [1, 0])
    t.extend(fill, [32 * 2000, 32 * 3990])
    t.extend(fill, [32 * 3500, 40], fits=False)

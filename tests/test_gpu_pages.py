"""The paged 8-bit cache against its oracle: filling, reading back and decoding in any order of steps, forked,
freed and moved pages, blocks that hold an infinity, replays, and what is refused."""
import random

import pytest
import torch

from attention_bounds import check
from oracle.paged import Accounts, attend, cached

pytestmark = pytest.mark.gpu

PAIR = 2.0 ** -17                              # a probability times a scale, kept as two bf16


class Mirror:
    """A PagedCache and what it should hold: each slot's tokens in host memory and the accounts' model."""

    def __init__(self, layers=1, slots=6, pages=40, max_tokens=700, Hkv=2, d=64, page=64, code="int8",
                 dtype=torch.bfloat16, seed=0):
        import kvq
        self.cache = kvq.PagedCache(layers, slots, pages, max_tokens, Hkv, d, page=page, code=code, dtype=dtype)
        self.model, self.g = Accounts(slots, pages, page), torch.Generator().manual_seed(seed)
        empty = torch.empty((0, Hkv, d), dtype=dtype)
        self.k = [[empty for _ in range(slots)] for _ in range(layers)]
        self.v = [[empty for _ in range(slots)] for _ in range(layers)]

    def rand(self, n, H):
        c = self.cache
        x = torch.randn(n, H, c.d, generator=self.g) * torch.exp(torch.randn(1, H, c.d, generator=self.g))
        return x.to(c.dtype)

    def extend(self, slots, counts, into=None):
        c = self.cache
        step = c.extend(slots, counts, into=into)
        self.model.extend(slots, counts)
        new = []
        for l in range(c.layers):
            k, v = self.rand(step.rows, c.Hkv), self.rand(step.rows, c.Hkv)
            a = 0
            for s, n in zip(slots, counts):
                self.k[l][s], self.v[l][s] = torch.cat([self.k[l][s], k[a:a + n]]), torch.cat([self.v[l][s], v[a:a + n]])
                a += n
            new.append((k, v))
        return step, new

    def push(self, slots, counts):
        step, new = self.extend(slots, counts)
        for l, (k, v) in enumerate(new):
            self.cache.append(l, k.cuda(), v.cuda(), step)
        return step

    def fork(self, src, dst):
        self.cache.fork(src, dst)
        self.model.fork(src, dst)
        for kv in (*self.k, *self.v):
            for a, b in zip(src, dst):
                kv[b] = kv[a]

    def free(self, slots):
        self.cache.free(slots)
        self.model.free(slots)
        for kv in (*self.k, *self.v):
            for s in slots:
                kv[s] = kv[s][:0]

    def check(self, what=""):
        """Accounts, table and every token: what is read back is code * scale in float32, rounded once."""
        c = self.cache
        assert c.lengths == self.model.lens and c.free_pages == self.model.refs.count(0)
        table = c.table.cpu()
        for s, pages in enumerate(self.model.table):
            assert table[s, :len(pages)].tolist() == pages, (what, s)
        used = [s for s, n in enumerate(c.lengths) if n]
        if not used:
            return
        for l in range(c.layers):
            got = c.rows(l, used)
            for x, held in zip(got, (self.k[l], self.v[l])):
                want = torch.cat([cached(held[s], c.page, c.code).float().to(c.dtype) for s in used])
                assert torch.equal(x.cpu(), want), (what, l)

    def decode(self, step, Hq, layer=0, what=""):
        import kvq
        c = self.cache
        q = self.rand(step.rows, Hq)
        out = kvq.paged_decode(q.cuda(), c.d ** -0.5, c, layer, step)
        a = 0
        for s, n in zip(step.slots.tolist(), step.counts.tolist()):
            if n == 0:
                continue
            k, v = cached(self.k[layer][s], c.page, c.code), cached(self.v[layer][s], c.page, c.code)
            ref = attend(q[a:a + n], k, v, c.d ** -0.5)
            check(out[a:a + n], ref, float(v.abs().max()), k.shape[0], c.d, c.dtype, PAIR, f"{what} slot {s}, {n} of {k.shape[0]}")
            a += n
        return q, out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("page,d,Hkv", [(32, 64, 2), (64, 128, 2), (128, 64, 1), (32, 128, 1), (128, 128, 1)])
def test_any_order_of_steps(page, d, Hkv, code, dtype):
    """Tokens that come one by one, in pieces and in long prompts: the same codes, and the decode over them."""
    m = Mirror(page=page, d=d, Hkv=Hkv, code=code, dtype=dtype, seed=page + d)
    m.push([0, 2], [1, page])
    m.push([2, 0, 4], [1, page - 1, 3 * page + 5])
    m.check("prompts")
    step = m.push([0, 1, 2, 4], [1, 0, 1, 1])                       # nothing for one of them
    m.check("tokens")
    m.decode(step, 4 * Hkv, what="one token")
    step = m.push([4, 0], [page - 3, 5])
    m.check("over a border")
    m.decode(step, Hkv, what="many tokens")
    for _ in range(3):
        m.push([0, 2], [1, page // 2])
    m.check("more")


@pytest.mark.parametrize("rep", [1, 3, 7, 8, 16, 20])
def test_decode_heads_and_drafts(rep):
    """Query heads per KV head and drafted tokens beyond one tile of 16 rows, uneven, causal within the step."""
    m = Mirror(Hkv=2, d=64, page=32, seed=rep)
    m.push([0, 1, 2, 3], [33, 1, 200, 95])
    step = m.push([3, 0, 1, 2], [1, 6, 2, 17])
    m.decode(step, 2 * rep, what=f"rep {rep}")


@pytest.mark.parametrize("n", [1, 63, 64, 65, 128, 640, 4099])
def test_decode_lengths(n):
    m = Mirror(slots=2, pages=80, max_tokens=4200, Hkv=1, d=128, page=64, seed=n)
    if n > 1:
        m.push([1], [n - 1])
    m.decode(m.push([1], [1]), 4, what=f"length {n}")


def test_split_sequences_beside_short_ones():
    """One long sequence in many items beside short ones of one, and the same answer alone."""
    import kvq
    m = Mirror(slots=5, pages=400, max_tokens=9000, Hkv=1, d=64, page=32, seed=8)
    m.push([0, 1, 2, 3], [8200, 40, 1, 700])
    step = m.push([0, 1, 2, 3], [2, 1, 1, 3])
    q, out = m.decode(step, 8, what="split")
    again = kvq.paged_decode(q.cuda(), 64 ** -0.5, m.cache, 0, step)
    assert torch.equal(out, again)


def test_fork_free_and_moves():
    m = Mirror(layers=3, slots=8, pages=30, max_tokens=600, Hkv=2, d=64, page=32, seed=4)
    m.push([0, 1, 2], [100, 64, 31])
    m.push([1, 0, 2], [70, 33, 1])
    m.fork([0, 0, 1, 7], [3, 4, 5, 6])
    m.check("forked")
    step = m.push([0, 3, 4, 5], [3, 28, 40, 1])
    m.check("grown apart")
    for l in range(3):
        m.decode(step, 4, layer=l, what=f"layer {l}")
    m.free([0, 1])
    m.check("freed")
    used = m.cache.compact()
    m.model.move(used, 30)
    assert used == 30 - m.cache.free_pages
    m.check("compacted")
    step = m.push([0, 4], [50, 1])
    m.check("reused")
    m.cache.resize(25)
    m.model.move(25, 25)
    m.check("smaller")
    m.decode(step, 4, layer=2, what="after moving")
    m.free([3, 5, 2])
    m.cache.resize(60)
    m.model.move(60, 60)
    m.push([5], [500])
    m.check("larger")
    m.free([0, 4, 5, 6, 7])
    m.check("empty")
    m.cache.resize(1)
    assert m.cache.free_pages == 1


@pytest.mark.parametrize("page,d,Hkv,rep", [(32, 64, 2, 4), (64, 128, 1, 3), (128, 64, 1, 8)])
def test_shared_fronts(page, d, Hkv, rep):
    """Forks side by side read their shared pages once: uneven drafts, growth over block borders, and others between."""
    import kvq
    m = Mirror(slots=12, pages=200, max_tokens=2500, Hkv=Hkv, d=d, page=page, seed=page)
    m.push([0, 1, 2], [1500, 700, 40])
    m.fork([0, 0, 0, 1, 2, 0], [3, 4, 5, 6, 7, 8])
    step = m.push([0, 3, 4, 1, 6, 2, 7, 5], [1, 3, 1, 2, 1, 1, 1, 1])
    assert step.fronts
    m.decode(step, rep * Hkv, what="forks")
    step = m.push([8, 3, 4], [page + 5, 1, 2 * page])
    q, out = m.decode(step, rep * Hkv, what="apart")
    assert step.fronts and torch.equal(out, kvq.paged_decode(q.cuda(), d ** -0.5, m.cache, 0, step))
    step = m.push([3, 2, 4], [1, 1, 1])                             # not side by side
    assert not step.fronts
    m.decode(step, rep * Hkv, what="between")
    m.free([0, 8])
    step = m.push([4, 3], [1, 2])
    assert step.fronts
    m.decode(step, rep * Hkv, what="freed")


def test_a_step_written_over_one_without_forks():
    """A captured decode of two sequences runs a later step whose slots have come to share pages."""
    import kvq
    m = Mirror(slots=4, pages=90, max_tokens=1300, Hkv=1, d=64, page=32, seed=17)
    m.push([0, 1], [600, 300])
    step = m.push([0, 1], [2, 1])
    floats = kvq.paged_workspace_floats(step, 4, 1, 64)
    m.free([1])
    m.fork([0], [1])
    step, [(k, v)] = m.extend([0, 1], [2, 1], into=step)
    m.cache.append(0, k.cuda(), v.cuda(), step)
    assert kvq.paged_workspace_floats(step, 4, 1, 64) == floats
    m.decode(step, 4, what="rewritten")


def test_a_captured_step_without_fronts_keeps_to_none():
    """Three sequences of three, one and one new tokens, captured when nothing was shared: a later step over forks side by
    side runs in the same graph, which joins no shared fronts."""
    import kvq
    m = Mirror(slots=3, pages=90, max_tokens=1300, Hkv=1, d=64, page=32, seed=18)
    m.push([0, 1, 2], [400, 600, 500])
    step, [(k, v)] = m.extend([0, 1, 2], [3, 1, 1])
    kd, vd, q = k.cuda(), v.cuda(), m.rand(5, 4).cuda()
    out, ws = torch.empty_like(q), torch.empty(kvq.paged_workspace_floats(step, 4, 1, 64), device="cuda")
    m.cache.append(0, kd, vd, step)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        m.cache.append(0, kd, vd, step)
        kvq.paged_decode(q, 0.125, m.cache, 0, step, out=out, workspace=ws)
    m.free([2])
    m.fork([1], [2])
    for i in range(3):
        step, [(k, v)] = m.extend([0, 1, 2], [3, 1, 1], into=step)
        kd.copy_(k)
        vd.copy_(v)
        _ = (q.float() * 2).sum()
        gr.replay()
        torch.cuda.synchronize()
        a = 0
        for s, n in ((0, 3), (1, 1), (2, 1)):
            kk, vv = cached(m.k[0][s], 32, "int8"), cached(m.v[0][s], 32, "int8")
            check(out[a:a + n], attend(q[a:a + n].cpu(), kk, vv, 0.125), float(vv.abs().max()), kk.shape[0], 64, torch.bfloat16, PAIR,
                  f"replay {i}, slot {s}")
            a += n
    # a new step of the same slots shares
    assert m.push([0, 1, 2], [3, 1, 1]).fronts


def test_another_stream_and_expanded_rows():
    """Steps on a side stream; one token's rows expanded over a step (strides of zero)."""
    import kvq
    m = Mirror(slots=2, Hkv=2, d=64, page=32, seed=19)
    m.push([0], [70])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step = m.push([0, 1], [3, 40])
        q = m.rand(1, 4)
        out = kvq.paged_decode(q.cuda().expand(43, -1, -1), 0.125, m.cache, 0, step)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, kvq.paged_decode(q.expand(43, -1, -1).contiguous().cuda(), 0.125, m.cache, 0, step))
    m.check("side stream")
    step, _ = m.extend([1], [50])
    k = m.rand(1, 2)
    m.k[0][1] = torch.cat([m.k[0][1][:-50], k.expand(50, -1, -1)])
    m.v[0][1] = torch.cat([m.v[0][1][:-50], k.expand(50, -1, -1)])
    kd = k.cuda().expand(50, -1, -1)
    m.cache.append(0, kd, kd, step)
    m.check("expanded")


def test_resize_on_another_stream():
    """The old pools are read by a stream that is busy; what the pools' own stream allocates next is other memory."""
    m = Mirror(slots=2, pages=40, max_tokens=1000, Hkv=2, d=64, page=32, seed=21)
    m.push([0, 1], [600, 300])
    x = torch.ones(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(20):
            x = x @ x * 1e-4
        m.cache.resize(60)
    m.model.move(60, 60)
    size = 40 * 2 * 32 * 64
    held = [torch.full((size,), 77, dtype=torch.int8, device="cuda") for _ in range(4)]
    torch.cuda.current_stream().wait_stream(side)
    m.check("resized")
    assert all(bool((h == 77).all()) for h in held)


@pytest.mark.parametrize("rep,T", [(1, 1), (2, 2), (4, 1), (3, 1), (5, 1), (7, 1), (4, 2), (8, 2)])
def test_joins_within_the_launch(rep, T):
    """A step's items joined by the last workgroup, where it has few rows, and by a launch; counters are zeros again."""
    import kvq
    m = Mirror(slots=3, pages=200, max_tokens=7000, Hkv=2, d=128, page=64, seed=22)
    m.push([0, 1, 2], [6000, 900, 1])
    step = m.push([0, 1, 2], [T] * 3)
    assert step.joins
    q, out = m.decode(step, 2 * rep, what="joined")
    for _ in range(3):
        assert torch.equal(out, kvq.paged_decode(q.cuda(), 128 ** -0.5, m.cache, 0, step))
    assert not m.cache._counters.any()
    m.cache._tickets = [None]
    m.decode(step, 2 * rep, what="joined by a launch")


def test_a_captured_step_without_joins():
    """As many sequences as there are places: an item each and no launch for joins, in later steps of the graph neither, however
    long some of them have grown; nothing new for one sequence."""
    import kvq
    n = 66
    m = Mirror(slots=n, pages=900, max_tokens=1200, Hkv=8, d=64, page=32, seed=23)
    m.push(list(range(n)), [1 + 5 * i % 90 for i in range(n)])
    counts = [0 if i == 7 else 1 for i in range(n)]
    # 96 places at head_dim 64: short sequences take one item all the same
    step, [(k, v)] = m.extend(list(range(n)), counts)
    assert step.joins == 0 and step.splits == n - 1
    kd, vd, q = k.cuda(), v.cuda(), m.rand(n - 1, 16).cuda()
    out, ws = torch.empty_like(q), torch.empty(kvq.paged_workspace_floats(step, 16, 8, 64), device="cuda")
    m.cache.append(0, kd, vd, step)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        m.cache.append(0, kd, vd, step)
        kvq.paged_decode(q, 0.125, m.cache, 0, step, out=out, workspace=ws)
    assert ws.numel() == 0
    for i in range(3):
        m.push([3, 40], [300, 33])
        if i == 2:                             # neighbours that share pages
            m.free([4])
            m.fork([3], [4])
        step, [(k, v)] = m.extend(list(range(n)), counts, into=step)
        kd.copy_(k)
        vd.copy_(v)
        _ = (q.float() * 2).sum()
        gr.replay()
        torch.cuda.synchronize()
        a = 0
        for s, c in enumerate(counts):
            if c:
                kk, vv = cached(m.k[0][s], 32, "int8"), cached(m.v[0][s], 32, "int8")
                check(out[a:a + 1], attend(q[a:a + 1].cpu(), kk, vv, 0.125), float(vv.abs().max()), kk.shape[0], 64, torch.bfloat16,
                      PAIR, f"replay {i}, slot {s}")
                a += 1


def test_uneven_sequences():
    """A step of sequences that are cut finer than the places, and of long ones whose joins take a workgroup each."""
    m = Mirror(slots=66, pages=1200, max_tokens=9000, Hkv=8, d=64, page=64, seed=24)
    m.push(list(range(60)), [3 + 41 * i % 1500 for i in range(60)])
    m.decode(m.push(list(range(60)), [1 + i % 2 for i in range(60)]), 16, what="uneven")
    m.push([64], [8500])
    m.decode(m.push([64], [2]), 40, what="one long")
    m.decode(m.push([64, 65], [1, 3]), 16, what="long and short")


def test_a_scaling_of_nothing():
    import kvq
    m = Mirror(slots=2, pages=60, max_tokens=1000, Hkv=1, d=64, page=32, seed=25)
    m.push([0, 1], [900, 20])
    step = m.push([0, 1], [3, 2])
    q = m.rand(5, 2)
    out = kvq.paged_decode(q.cuda(), 0.0, m.cache, 0, step)
    for s, a, b in ((0, 0, 3), (1, 3, 5)):
        kk, vv = cached(m.k[0][s], 32, "int8"), cached(m.v[0][s], 32, "int8")
        check(out[a:b], attend(q[a:b], kk, vv, 0.0), float(vv.abs().max()), kk.shape[0], 64, torch.bfloat16, PAIR, f"slot {s}")


def test_random_life():
    """A few hundred random steps, forks, frees and moves."""
    rng = random.Random(11)
    m = Mirror(layers=2, slots=7, pages=50, max_tokens=500, Hkv=1, d=64, page=32, seed=11)
    for i in range(120):
        op = rng.choice(["push", "push", "push", "fork", "free", "move"])
        empty = [s for s, n in enumerate(m.model.lens) if n == 0]
        held = [s for s in range(7) if s not in empty]
        if op == "push":
            slots = rng.sample(range(7), rng.randint(1, 4))
            counts = [rng.choice([1, 1, 31, 32, 33, rng.randint(1, 120)]) for _ in slots]
            need = sum((m.model.lens[s] + c) // 32 - m.model.lens[s] // 32 for s, c in zip(slots, counts))
            if need <= m.cache.free_pages and all(m.model.lens[s] + c <= 500 for s, c in zip(slots, counts)):
                step = m.push(slots, counts)
                if i % 5 == 0:
                    m.decode(step, 3, layer=1, what=f"step {i}")
        elif op == "fork" and empty and held:
            m.fork([rng.choice(held)], [empty[0]])
        elif op == "free" and held:
            m.free(rng.sample(held, 1))
        elif op == "move":
            used = m.cache.pages - m.cache.free_pages
            if rng.random() < 0.5:
                m.cache.compact()
                m.model.move(used, m.cache.pages)
            else:
                n = max(used, 40) + rng.randint(0, 20)
                m.cache.resize(n)
                m.model.move(n, n)
        if i % 10 == 9:
            m.check(f"step {i}")


def test_many_slots():
    """More sequences than go with one launch by value."""
    n = 300
    m = Mirror(slots=2 * n, pages=700, max_tokens=100, Hkv=1, d=64, page=32, seed=14)
    m.push(list(range(n)), [1 + (7 * i) % 90 for i in range(n)])
    m.fork(list(range(n)), list(range(n, 2 * n)))
    step = m.push(list(range(2 * n)), [1] * (2 * n))
    m.check("many")
    m.decode(step, 2, what="many")


def test_append_again_writes_the_same():
    """A step that fills a block and opens the next one, appended twice."""
    m = Mirror(seed=6, page=32)
    m.push([0, 1], [20, 31])
    step, [(k, v)] = m.extend([0, 2, 1], [25, 0, 1])
    for _ in range(3):
        m.cache.append(0, k.cuda(), v.cuda(), step)
        m.check("again")


def test_captured_steps():
    """A captured append and decode, replayed for step after step written into the same description."""
    import kvq
    m = Mirror(slots=3, pages=60, max_tokens=900, Hkv=2, d=64, page=32, seed=12)
    m.push([0, 1, 2], [30, 62, 500])
    step, [(k, v)] = m.extend([2, 0, 1], [1, 1, 1])
    kd, vd, q = k.cuda(), v.cuda(), torch.zeros((3, 8, 64), dtype=torch.bfloat16, device="cuda")
    out = torch.empty_like(q)
    ws = torch.empty(kvq.paged_workspace_floats(step, 8, 2, 64), device="cuda")
    m.cache.append(0, kd, vd, step)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        m.cache.append(0, kd, vd, step)
        kvq.paged_decode(q, 64 ** -0.5, m.cache, 0, step, out=out, workspace=ws)
    for i in range(40):
        if i:
            step, [(k, v)] = m.extend([2, 0, 1], [1, 1, 1], into=step)
        kd.copy_(k)
        vd.copy_(v)
        q.copy_(m.rand(3, 8))
        _ = (q.float() * 2).sum()
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, kvq.paged_decode(q, 64 ** -0.5, m.cache, 0, step)), i
        if i % 13 == 0:
            m.check(f"replay {i}")
            a = 0
            for s in (2, 0, 1):
                kk, vv = cached(m.k[0][s], 32, "int8"), cached(m.v[0][s], 32, "int8")
                check(out[a:a + 1], attend(q[a:a + 1].cpu(), kk, vv, 64 ** -0.5), float(vv.abs().max()), kk.shape[0], 64, torch.bfloat16,
                      PAIR, f"replay {i}, slot {s}")
                a += 1


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_infinities_and_nan(bad, dtype):
    """A full block with one reads as NaN for those who see it, and no other; in the open block it is hidden from the
    drafted tokens before it."""
    import kvq
    m = Mirror(slots=3, Hkv=1, d=64, page=32, dtype=dtype, seed=3)
    m.push([0, 1], [70, 20])
    step, [(k, v)] = m.extend([0, 1, 2], [4, 4, 30])
    kb, vb = k.clone(), v.clone()
    kb[2], vb[2, :, 5] = bad, bad                                  # third draft of slot 0, open block
    vb[6, :, 5] = bad                                              # third draft of slot 1
    m.cache.append(0, k.cuda(), v.cuda(), step)
    q = m.rand(38, 2).cuda()
    clean = kvq.paged_decode(q, 0.125, m.cache, 0, step)
    m.cache.append(0, kb.cuda(), vb.cuda(), step)
    got = kvq.paged_decode(q, 0.125, m.cache, 0, step)
    assert torch.equal(got[:2], clean[:2]) and torch.equal(got[4:6], clean[4:6]) and torch.equal(got[8:], clean[8:])
    assert not torch.isfinite(got[2:4, :, 5].float()).any() and not torch.isfinite(got[6:8, :, 5].float()).any()
    assert torch.equal(got[6:8, :, :5], clean[6:8, :, :5])
    # the block of slot 1 gets full: it reads as NaN; slots 0 and 2 do not change
    step = m.push([1, 2], [8, 2])
    got = kvq.paged_decode(m.rand(10, 2).cuda(), 0.125, m.cache, 0, step)
    assert torch.isnan(got[:8].float()).all() and torch.isfinite(got[8:].float()).all()
    k1, v1 = m.cache.rows(0, [1])
    assert torch.isnan(v1.float()).all() and torch.isfinite(k1.float()).all()


def test_hidden_nan_block():
    """Drafts that fill a block with a NaN among them: the drafts before the block do not see it."""
    import kvq
    m = Mirror(slots=1, Hkv=1, d=64, page=32, seed=2)
    m.push([0], [30])
    step, [(k, v)] = m.extend([0], [40])
    vb = v.clone()
    vb[5] = float("nan")
    q = m.rand(40, 4).cuda()
    m.cache.append(0, k.cuda(), vb.cuda(), step)
    got = kvq.paged_decode(q, 0.125, m.cache, 0, step).float()
    assert torch.isfinite(got[:2]).all() and torch.isnan(got[2:]).all()


def test_extreme_magnitudes():
    """Blocks of tiny and of the largest values, and of zeros, beside ordinary ones."""
    for dtype, big in ((torch.bfloat16, 1e30), (torch.bfloat16, 3.3e38), (torch.float16, 6e4)):
        m = Mirror(slots=1, Hkv=1, d=64, page=32, dtype=dtype, seed=9)
        for scale in (1.0, 1e-30, 0.0, big):
            step, [(k, v)] = m.extend([0], [32])
            v = (torch.randn(32, 1, 64, generator=m.g) * scale).clamp(-big, big).to(dtype)
            m.v[0][0] = torch.cat([m.v[0][0][:-32], v])
            m.cache.append(0, k.cuda(), v.cuda(), step)
        m.check("magnitudes")


def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes a side: pages at its end are filled, read, decoded and moved."""
    import kvq
    m = Mirror(layers=2, slots=3, pages=70000, max_tokens=64 * 70000, Hkv=8, d=128, page=64, seed=1)
    filler = m.cache.extend([0], [64 * 69990])                     # claimed, never written
    m.model.extend([0], [64 * 69990])
    assert filler.rows == 64 * 69990
    step = m.push([1], [200])
    table = m.cache.table.cpu()
    assert table[1, :3].tolist() == [69990, 69991, 69992]
    for l in (0, 1):
        got = m.cache.rows(l, [1])
        for x, held in zip(got, (m.k[l][1], m.v[l][1])):
            assert torch.equal(x.cpu(), cached(held, 64, "int8").float().to(torch.bfloat16))
    step = m.push([1], [1])
    m.decode(step, 16, layer=1, what="end of the pool")
    m.free([0])
    assert m.cache.compact() == 3
    m.model.move(3, 70000)
    m.check("moved")


def test_gpu_refusals():
    import kvq
    with pytest.raises(kvq.KVQError, match="head_dim"):
        kvq.PagedCache(1, 1, 1, 10, 1, 96)
    with pytest.raises(ValueError, match="page"):
        kvq.PagedCache(1, 1, 1, 10, 1, 64, page=16)
    with pytest.raises(TypeError):
        kvq.PagedCache(1, 1, 1, 10, 1, 64, dtype=torch.float32)
    with pytest.raises(ValueError, match="code"):
        kvq.PagedCache(1, 1, 1, 10, 1, 64, code="int4")
    with pytest.raises(kvq.KVQError):
        kvq.PagedCache(1, 1, 1, 10, 1, 64, device="cpu")
    c = kvq.PagedCache(2, 3, 4, 300, 2, 64, page=64)
    with pytest.raises(kvq.KVQError, match="exhausted"):
        c.extend([0], [301])
    with pytest.raises(kvq.KVQError, match="exhausted"):
        c.extend([0, 1], [192, 128])
    with pytest.raises(ValueError):
        c.extend([], [])
    none = c.extend([0, 2], [0, 0])
    c.extend([0, 2], [0, 0], into=none)
    empty = torch.empty((0, 2, 64), dtype=torch.bfloat16, device="cuda")
    c.append(1, empty, empty, none)
    assert kvq.paged_decode(torch.empty((0, 4, 64), dtype=torch.bfloat16, device="cuda"), 0.1, c, 0, none).shape == (0, 4, 64)
    with pytest.raises(kvq.KVQError, match="twice"):
        c.extend([1, 1], [1, 1])
    assert c.lengths == [0, 0, 0] and c.free_pages == 4
    step = c.extend([0, 1], [3, 1])
    k = torch.zeros((4, 2, 64), dtype=torch.bfloat16, device="cuda")
    q = torch.zeros((4, 4, 64), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(IndexError):
        c.append(2, k, k, step)
    with pytest.raises(ValueError):
        c.append(0, k[:3], k[:3], step)
    with pytest.raises(TypeError):
        c.append(0, k.half(), k.half(), step)
    with pytest.raises(kvq.KVQError):
        c.append(0, k.cpu(), k.cpu(), step)
    c.append(0, k, k, step)
    with pytest.raises(ValueError):
        kvq.paged_decode(q[:, :3], 0.1, c, 0, step)
    with pytest.raises(TypeError):
        kvq.paged_decode(q.half(), 0.1, c, 0, step)
    # a step of another cache; of a slot that has been freed and holds as many tokens again
    other = kvq.PagedCache(2, 3, 4, 300, 2, 64, page=64)
    same = other.extend([0, 1], [3, 1])
    with pytest.raises(ValueError, match="another cache"):
        c.append(0, k, k, same)
    with pytest.raises(ValueError, match="another cache"):
        kvq.paged_decode(q, 0.1, c, 0, same)
    with pytest.raises(ValueError, match="own cache"):
        c.extend([0, 1], [3, 1], into=same)
    other.extend([2], [0])
    other.append(0, k, k, same)                # what changed were other slots, or nothing
    other.extend([0], [0])
    other.append(1, k, k, same)
    other.free([0])
    other.extend([0], [3])
    with pytest.raises(ValueError, match="changed"):
        other.append(1, k, k, same)
    with pytest.raises(ValueError, match="changed"):
        kvq.paged_decode(q, 0.1, other, 1, same)
    long = kvq.PagedCache(1, 1, 11, 700, 2, 64)
    long.extend([0], [690])
    many = long.extend([0], [4])               # several items: their results need room
    with pytest.raises(kvq.KVQError, match="workspace"):
        kvq.paged_decode(q, 0.1, long, 0, many, workspace=torch.empty(10, device="cuda"))
    with pytest.raises(kvq.KVQError, match="no slot"):
        c.rows(0, [0, 3])
    with pytest.raises(ValueError, match="same counts"):
        c.extend([0, 1], [1, 1], into=step)
    c.extend([1], [1])
    with pytest.raises(ValueError, match="changed"):
        kvq.paged_decode(q, 0.1, c, 0, step)
    with pytest.raises(ValueError, match="changed"):
        c.append(0, k, k, step)
    with pytest.raises(kvq.KVQError, match="in use"):
        c.fork([0], [1])
    with pytest.raises(ValueError, match="in use"):
        c.extend([0], [128]) and c.resize(1)
    step = c.extend([2], [4])
    c.resize(9)
    with pytest.raises(ValueError, match="moved"):
        c.append(0, k, k, step)


def test_a_step_is_not_rewritten_after_resize():
    """The graphs that were captured with a step hold the pools of then, which resize gives back; compact keeps them."""
    import kvq
    m = Mirror(slots=2, pages=20, max_tokens=300, Hkv=1, d=64, page=32, seed=31)
    m.push([0, 1], [70, 40])
    step, [(k, v)] = m.extend([0, 1], [3, 1])
    m.cache.append(0, k.cuda(), v.cuda(), step)
    m.cache.compact()
    m.model.move(3, 20)
    step, [(k, v)] = m.extend([0, 1], [3, 1], into=step)
    m.cache.append(0, k.cuda(), v.cuda(), step)
    m.cache.resize(30)
    m.model.move(30, 30)
    with pytest.raises(ValueError, match="resize"):
        m.cache.extend([0, 1], [3, 1], into=step)
    m.check("refused")
    m.decode(step, 2, what="the last step, over the new pools")
    step = m.push([0, 1], [3, 1])              # a new one
    step, [(k, v)] = m.extend([0, 1], [3, 1], into=step)
    m.cache.append(0, k.cuda(), v.cuda(), step)
    m.decode(step, 2, what="a new step")
    m.check("a new step")


def test_a_step_dropped_before_another_stream_is_done():
    """Append and decode on a stream that is busy, step and cache gone: what their own stream allocates next is other memory."""
    import kvq
    m = Mirror(slots=2, pages=40, max_tokens=1000, Hkv=2, d=64, page=32, seed=32)
    m.push([0, 1], [600, 40])
    step, [(k, v)] = m.extend([0, 1], [40, 1])
    k, v, q = k.cuda(), v.cuda(), m.rand(41, 4).cuda()
    m.cache.append(0, k, v, step)
    want, size = kvq.paged_decode(q, 0.125, m.cache, 0, step), step.desc.numel()
    out, ws = torch.empty_like(want), torch.empty(kvq.paged_workspace_floats(step, 4, 2, 64), device="cuda")
    x = torch.ones(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(20):
            x = x @ x * 1e-4
        m.cache.append(0, k, v, step)
        kvq.paged_decode(q, 0.125, m.cache, 0, step, out=out, workspace=ws)
    del step
    held = [torch.zeros(size, dtype=torch.int32, device="cuda") for _ in range(64)]
    parts = (m.cache.table, m.cache.kc, m.cache.vc, m.cache.sc, m.cache.k_open, m.cache.v_open, m.cache._counters)
    like = [torch.empty_like(p, device="meta") for p in parts]
    del parts
    m.cache = None
    held += [torch.zeros_like(p, device="cuda") for p in like for _ in range(4)]
    torch.cuda.synchronize()
    assert torch.equal(out, want) and not any(bool(h.any()) for h in held)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf")])
@pytest.mark.parametrize("page,d,dtype", [(32, 64, torch.bfloat16), (64, 128, torch.float16), (128, 64, torch.bfloat16), (128, 128, torch.float16)])
def test_a_visible_infinity_of_the_open_block_stays(page, d, dtype, bad):
    """However small its weight beside what other tokens, wavefronts and items hold: the rows that see it have it in that
    channel.  Joined in the launch, by a launch, and behind a shared front."""
    import kvq
    m = Mirror(slots=4, pages=160, max_tokens=30 * page + 10, Hkv=1, d=d, page=page, dtype=dtype, seed=33)
    n = 23 * page + page - 4                   # page - 4 tokens in the open block, then three more
    for big in (3, 12 * page, 23 * page + 1, 23 * page + page - 5, n + 2):
        step, [(k, v)] = m.extend([0], [n])
        k[..., 0] = 0
        if big < n:
            k[big, :, 0] = 25.0 * d ** 0.5
        at = 23 * page + (0 if big % 2 else page - 6)
        vb = v.clone()
        vb[at, :, 5] = bad
        m.cache.append(0, k.cuda(), vb.cuda(), step)
        m.fork([0], [1])
        for slots, counts in (([0], [1]), ([1], [2]), ([0, 1], [2, 1])):
            step, [(k, v)] = m.extend(slots, counts)
            k[..., 0] = 0
            if big >= n:
                k[:, :, 0] = 25.0 * d ** 0.5
            m.cache.append(0, k.cuda(), v.cuda(), step)
            q = m.rand(sum(counts), 4)
            q[..., 0] = 16.0
            tickets = m.cache._tickets
            for way in (tickets, [None]):
                m.cache._tickets = way
                out = kvq.paged_decode(q.cuda(), d ** -0.5, m.cache, 0, step).float()
                what = (big, at, slots, way[0] is None)
                assert (out[..., 5] == bad).all(), what
                assert torch.isfinite(out[..., :5]).all() and torch.isfinite(out[..., 6:]).all(), what
            m.cache._tickets = tickets
        assert step.fronts
        m.free([0, 1])


@pytest.mark.parametrize("late", [50, 70000, 100010])
@pytest.mark.parametrize("tickets", [True, False])
def test_joins_of_more_items_than_a_wavefront_has_lanes(tickets, late):
    """A sequence of more than 64 items beside 39 short ones: two rounds of maxima, the largest score in an early and in a
    late one."""
    m = Mirror(slots=40, pages=1750, max_tokens=100100, Hkv=1, d=128, page=64, seed=34)
    if not tickets:
        m.cache._tickets = [None]
    q = _one_strong_key(m, 0, 100020, late, 4)
    m.push(list(range(1, 40)), [40 + i for i in range(39)])
    step = m.push(list(range(40)), [1] * 40)
    first = step.host[12 + 8 * 41:].reshape(-1)[:12]
    assert first[7] == 0 and first[11] > 64
    _check_rows(m, step, q, 40, 4)


@pytest.mark.parametrize("late", [50, 70000, 131060])
@pytest.mark.parametrize("rows", [1, 3])
def test_joins_with_a_workgroup_for_each_row(rows, late):
    """One long sequence of many items, whose rows are joined by four wavefronts each, 32 partial results on their way."""
    m = Mirror(slots=1, pages=2100, max_tokens=131100, Hkv=1, d=128, page=64, seed=35)
    q = _one_strong_key(m, 0, 131070, late, 8)
    step = m.push([0], [rows])
    assert step.splits >= 160 and step.joins
    _check_rows(m, step, q, rows, 8)


def _one_strong_key(m, slot, n, at, Hq):
    """n tokens for the slot, the one at ``at`` along the query that is returned."""
    step, [(k, v)] = m.extend([slot], [n])
    q = m.rand(1, Hq)
    k[at] = (30 * q[0, :1] / q[0, :1].float().norm()).to(k.dtype)
    m.k[0][slot] = k
    m.cache.append(0, k.cuda(), v.cuda(), step)
    return q


def _check_rows(m, step, q, rows, Hq):
    import kvq
    c = m.cache
    qs = torch.cat([q, m.rand(rows - 1, Hq)])
    out = kvq.paged_decode(qs.cuda(), c.d ** -0.5, c, 0, step)
    a = 0
    for s, n in zip(step.slots.tolist(), step.counts.tolist()):
        kk, vv = cached(m.k[0][s], c.page, c.code), cached(m.v[0][s], c.page, c.code)
        check(out[a:a + n], attend(qs[a:a + n], kk, vv, c.d ** -0.5), float(vv.abs().max()), kk.shape[0], c.d, c.dtype, PAIR, f"slot {s}")
        a += n


def test_a_step_beyond_every_slot_takes_no_memory():
    """Counts that no slot can hold are refused before their description is allocated (268 MB for 2^31 - 1 tokens)."""
    import kvq
    c = kvq.PagedCache(1, 2, 4, 300, 2, 64, page=32)
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    for counts in ([(1 << 31) - 1], [301], [1, 1 << 30], [(1 << 31) - 1] * 2):
        with pytest.raises(kvq.KVQError, match="exhausted"):
            c.extend(list(range(len(counts))), counts)
    assert torch.cuda.max_memory_allocated() - before < 1 << 20
    assert c.lengths == [0, 0] and c.free_pages == 4
    assert c.extend([0, 1], [64, 64]).rows == 128

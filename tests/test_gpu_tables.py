"""The paged cache's accounts in device memory against their model: tables, slot maps, appended and decoded tokens, pages given
back, steps that do not fit, a captured loop without the host, and what is refused."""
import random

import pytest
import torch

from attention_bounds import check
from oracle.paged import attend, cached
from test_gpu_pages import PAIR, Mirror

pytestmark = pytest.mark.gpu


def dev(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def extend(m, acc, step, counts, fits=True):
    """One step on both sides, its positions, places and table; returns the rows' tokens per layer."""
    c, n, most = m.cache, len(counts), step.most
    acc.extend(step, dev(counts))
    slots, counts = step.slots.tolist(), counts if fits else [0] * n
    before = [m.model.lens[s] for s in slots]
    m.model.extend(slots, counts)
    positions, places = step.positions.cpu().view(n, most), step.places.cpu().view(n, most)
    for i, (s, b, k) in enumerate(zip(slots, before, counts)):
        pages = m.model.table[s]
        want = [b + j if j < k else -1 for j in range(most)]
        assert positions[i].tolist() == want
        assert places[i].tolist() == [pages[p // c.page] * c.page + p % c.page if p >= 0 and p // c.page < len(pages) else -1 for p in want]
    same(m, acc)
    new = []
    for l in range(c.layers):
        k, v = m.rand(step.rows, c.Hkv), m.rand(step.rows, c.Hkv)
        for i, (s, t) in enumerate(zip(slots, counts)):
            a = i * most
            m.k[l][s], m.v[l][s] = torch.cat([m.k[l][s], k[a:a + t]]), torch.cat([m.v[l][s], v[a:a + t]])
        new.append((k, v))
    return new


def same(m, acc):
    c = m.cache
    assert acc.lengths.tolist() == m.model.lens and int(acc.free_pages) == m.model.refs.count(0)
    table = c.table.cpu()
    for s, pages in enumerate(m.model.table):
        assert table[s, :len(pages)].tolist() == pages, s


def free(m, acc, step, which=None):
    acc.free(step, None if which is None else dev(which, torch.bool))
    slots = [s for i, s in enumerate(step.slots.tolist()) if which is None or which[i]]
    m.model.free(slots)
    for kv in (*m.k, *m.v):
        for s in slots:
            kv[s] = kv[s][:0]
    same(m, acc)


def decode(m, step, counts, Hq, layer=0):
    import kvq
    c = m.cache
    q = m.rand(step.rows, Hq)
    out = kvq.paged_decode(q.cuda(), c.d ** -0.5, c, layer, step)
    for i, (s, t) in enumerate(zip(step.slots.tolist(), counts)):
        a = i * step.most
        assert not out[a + t:a + step.most].any()                   # rows that are none's
        if t:
            k, v = cached(m.k[layer][s], c.page, c.code), cached(m.v[layer][s], c.page, c.code)
            check(out[a:a + t], attend(q[a:a + t], k, v, c.d ** -0.5), float(v.abs().max()), k.shape[0], c.d, c.dtype, PAIR, f"slot {s}")
    return q, out


@pytest.mark.parametrize("page,d,Hkv,code,dtype", [(32, 64, 2, "int8", torch.bfloat16), (64, 128, 1, "e4m3", torch.float16),
                                                    (128, 64, 1, "int8", torch.float16)])
def test_steps_as_on_the_host(page, d, Hkv, code, dtype):
    """Prompts and tokens of random counts in steps of two sizes, sequences that end and others that take their slots, shared pages;
    and on the host again."""
    import kvq
    rng = random.Random(page)
    m = Mirror(layers=2, slots=7, pages=70, max_tokens=900, Hkv=Hkv, d=d, page=page, code=code, dtype=dtype, seed=page)
    m.push([5, 0], [300, 2 * page + 3])
    m.fork([5], [6])
    m.free([0])
    acc = kvq.DeviceAccounts(m.cache)
    same(m, acc)
    big, small = acc.step([3, 0, 6, 1], 3 * page), acc.step([0, 1, 3, 6, 5], 3)
    for r in range(4):
        for step in (big, small, small):
            counts = [rng.choice([0, 1, step.most, rng.randint(0, step.most)]) for _ in step.slots]
            counts = [min(c, 900 - m.model.lens[s]) for c, s in zip(counts, step.slots.tolist())]
            need = sum((m.model.lens[s] + c) // page - m.model.lens[s] // page for c, s in zip(counts, step.slots.tolist()))
            assert need <= m.model.refs.count(0)
            for l, (k, v) in enumerate(extend(m, acc, step, counts)):
                m.cache.append(l, k.cuda(), v.cuda(), step)
            if step is small:
                decode(m, step, counts, 4 * Hkv, layer=r % 2)
        free(m, acc, big, [rng.random() < 0.5 for _ in range(4)])
    acc.close()
    m.check("on the host")
    step = m.push([1, 2, 5], [1, 40, 1])
    m.decode(step, 4 * Hkv, layer=1, what="on the host")
    m.check("later")


def test_many_rows_of_a_slot_over_the_pages():
    """A device step's prompts, then the rows over the pages once the accounts are back."""
    import kvq
    from test_gpu_paged_attention import run
    m = Mirror(slots=3, pages=60, max_tokens=1200, Hkv=2, d=64, page=32, seed=3)
    with kvq.DeviceAccounts(m.cache) as acc:
        step = acc.step([2, 0], 700)
        for k, v in extend(m, acc, step, [700, 333]):
            m.cache.append(0, k.cuda(), v.cuda(), step)
    run(m, [0, 2], [40, 7], 8)


def test_a_step_that_does_not_fit():
    """Counts out of range, a full slot, too few pages: nothing changes but the number of such steps."""
    import kvq
    m = Mirror(slots=4, pages=12, max_tokens=200, Hkv=1, d=64, page=32, seed=5)
    m.push([0], [150])
    acc = kvq.DeviceAccounts(m.cache)
    step = acc.step([0, 1, 2], 120)
    for k, v in extend(m, acc, step, [40, 100, 31]):
        m.cache.append(0, k.cuda(), v.cuda(), step)
    for i, counts in enumerate(([11, 0, 0], [1, -1, 0], [1, 121, 0], [1, 100, 120])):
        extend(m, acc, step, counts, fits=False)
        assert int(acc.refused) == i + 1
        m.cache.append(0, m.rand(360, 1).cuda(), m.rand(360, 1).cuda(), step)
        decode(m, step, [0, 0, 0], 4)
    for k, v in extend(m, acc, step, [10, 60, 1]):
        m.cache.append(0, k.cuda(), v.cuda(), step)
    decode(m, step, [10, 60, 1], 4)
    with pytest.raises(kvq.KVQError, match="4 steps"):
        acc.close()
    m.check("handed back")
    with pytest.raises(kvq.KVQError, match="handed back"):
        acc.extend(step, dev([0, 0, 0]))


@pytest.mark.parametrize("n,most,page", [(1, 1, 32), (1, 5000, 32), (64, 70, 64), (1500, 2, 32), (1025, 40, 128)])
def test_sizes(n, most, page):
    """One sequence and more than a workgroup has threads, rows beyond one piece, more new pages than one look finds; pages held by others
    between them."""
    import kvq
    rng = random.Random(n)
    tokens = max(3 * most, 200)
    pages = n * (tokens // page + 1) + 300
    cache = kvq.PagedCache(1, n + 1, pages, max(tokens, 200 * page), 1, 64, page=page)
    m = Mirror.__new__(Mirror)
    from oracle.paged import Accounts
    m.cache, m.model = cache, Accounts(n + 1, pages, page)
    for _ in range(3):                         # pages of the last slot between the others'
        cache.extend([0, n], [page * 5, page * 50])
        m.model.extend([0, n], [page * 5, page * 50])
    cache.free([0])
    m.model.free([0])
    m.k = m.v = []
    acc = kvq.DeviceAccounts(cache)
    step = acc.step(rng.sample(range(n), n), most)
    for _ in range(2):
        counts = [rng.choice([0, most, rng.randint(0, most)]) for _ in range(n)]
        acc.extend(step, dev(counts))
        slots = step.slots.tolist()
        before = [m.model.lens[s] for s in slots]
        fast_extend(m.model, slots, counts)
        same(m, acc)
        positions = torch.tensor([[b + j if j < k else -1 for j in range(most)] for b, k in zip(before, counts)]).view(-1)
        assert torch.equal(step.positions.cpu().long(), positions)
    free(m, acc, step)
    acc.close()
    assert cache.lengths == m.model.lens and cache.free_pages == m.model.refs.count(0)


def fast_extend(model, slots, counts):
    """Accounts.extend with the search for free pages going on where it was."""
    low = 0
    for s, c in zip(slots, counts):
        model.lens[s] += c
        while len(model.table[s]) < model.lens[s] // model.page:
            low = model.refs.index(0, low)
            model.refs[low] = 1
            model.table[s].append(low)


@pytest.mark.parametrize("n,Hkv", [(3, 2), (40, 8)])
def test_a_captured_loop(n, Hkv):
    """extend, append and decode in one graph, counts changed on the device between replays: two sequences end and a new one takes the
    first one's slot."""
    import kvq
    m = Mirror(slots=n, pages=40 * n, max_tokens=700, Hkv=Hkv, d=64, page=32, seed=7)
    m.push(list(range(n)), [20 + 37 * i % 300 for i in range(n)])
    with kvq.DeviceAccounts(m.cache) as acc:
        step, prompt = acc.step(list(range(n)), 2), acc.step([0], 100)
        counts = dev([0] * n)
        q, k, v = m.rand(2 * n, 4 * Hkv).cuda(), m.rand(2 * n, Hkv).cuda(), m.rand(2 * n, Hkv).cuda()
        out, ws = torch.zeros_like(q), torch.empty(kvq.paged_workspace_floats(step, 4 * Hkv, Hkv, 64), device="cuda")
        gr = torch.cuda.CUDAGraph()
        acc.extend(step, counts)
        m.cache.append(0, k, v, step)
        kvq.paged_decode(q, 0.125, m.cache, 0, step, out=out, workspace=ws)
        torch.cuda.synchronize()
        with torch.cuda.graph(gr):
            acc.extend(step, counts)
            m.cache.append(0, k, v, step)
            kvq.paged_decode(q, 0.125, m.cache, 0, step, out=out, workspace=ws)
        for r in range(5):
            c = [(i + r) % 3 if not (r > 1 and i < 2) else 0 for i in range(n)]
            if r == 3:
                free(m, acc, prompt)
                for kk, vv in extend(m, acc, prompt, [77]):
                    m.cache.append(0, kk.cuda(), vv.cuda(), prompt)
                c[0] = 2
            counts.copy_(dev(c))
            kk, vv, qq = m.rand(2 * n, Hkv), m.rand(2 * n, Hkv), m.rand(2 * n, 4 * Hkv)
            k.copy_(kk)
            v.copy_(vv)
            q.copy_(qq)
            gr.replay()
            _ = (out.float() * 2).sum()
            torch.cuda.synchronize()
            m.model.extend(list(range(n)), c)
            same(m, acc)
            for s, t in enumerate(c):
                m.k[0][s], m.v[0][s] = torch.cat([m.k[0][s], kk[2 * s:2 * s + t]]), torch.cat([m.v[0][s], vv[2 * s:2 * s + t]])
                if t and s < 6:
                    a, b = (cached(x[0][s], 32, "int8") for x in (m.k, m.v))
                    check(out[2 * s:2 * s + t], attend(qq[2 * s:2 * s + t], a, b, 0.125), float(b.abs().max()), a.shape[0], 64, m.cache.dtype,
                          PAIR, f"replay {r}, slot {s}")
    m.check("handed back")


@pytest.mark.parametrize("slots,most", [([1], 1), ([1], 40), ([2, 0, 1], 1), ([2, 0, 1], 40)])
def test_a_step_before_its_first_extend(slots, most):
    """Describes no tokens: nothing is appended, and its rows of a decode are zeros."""
    import kvq
    m = Mirror(slots=3, pages=20, max_tokens=300, Hkv=2, d=64, page=32, seed=12)
    m.push([0, 1], [70, 33])
    acc = kvq.DeviceAccounts(m.cache)
    step = acc.step(slots, most)
    assert not (step.positions + 1).any() and not (step.places + 1).any()
    new = m.rand(step.rows, 2).cuda()
    m.cache.append(0, new, new, step)
    decode(m, step, [0] * len(slots), 4)
    same(m, acc)
    acc.close()
    m.check("before")


def test_another_stream():
    import kvq
    m = Mirror(slots=3, pages=20, max_tokens=300, Hkv=1, d=64, page=32, seed=9)
    acc = kvq.DeviceAccounts(m.cache)
    step = acc.step([2, 1], 50)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for k, v in extend(m, acc, step, [50, 33]):
            m.cache.append(0, k.cuda(), v.cuda(), step)
        decode(m, step, [50, 33], 4)
        acc.close()
    m.check("side stream")


def test_refusals():
    import kvq
    m = Mirror(slots=3, Hkv=2, d=64, page=32)
    c = m.cache
    old = m.push([0], [40])
    plan = kvq.PagedPlan(c, [0], [3], 4)
    acc = kvq.DeviceAccounts(c)
    q = m.rand(40, 4).cuda()
    for call in (lambda: kvq.DeviceAccounts(c), lambda: c.extend([0], [1]), lambda: c.rows(0, [0]), lambda: c.fork([0], [1]),
                 lambda: c.free([0]), lambda: c.compact(), lambda: c.resize(50), lambda: c.lengths, lambda: c.length(0),
                 lambda: c.free_pages, lambda: kvq.PagedPlan(c, [0], [1], 4), lambda: kvq.PagedCtl(c, [0]).begin(1)):
        with pytest.raises(kvq.KVQError, match="on the device"):
            call()
    for call in (lambda: kvq.paged_decode(q, 0.1, c, 0, old), lambda: kvq.paged_attention(q[:3], 0.1, c, 0, plan),
                 lambda: c.append(0, q[:, :2], q[:, :2], old)):
        with pytest.raises(ValueError, match="changed"):
            call()
    for slots, most, error in (([], 1, ValueError), ([3], 1, kvq.KVQError), ([-1], 1, kvq.KVQError), ([0, 0], 1, kvq.KVQError),
                               ([0], 0, ValueError), ([0], 701, kvq.KVQError), ([0, 1], 1 << 30, ValueError)):
        with pytest.raises(error):
            acc.step(slots, most)
    step = acc.step([0, 1], 4)
    good = dev([1, 2])
    for bad, error in ((good.long(), ValueError), (good[:1], ValueError), (good.cpu(), kvq.KVQError), (dev([1, 0, 2, 0])[::2], ValueError)):
        with pytest.raises(error):
            acc.extend(step, bad)
    with pytest.raises(ValueError, match="bool"):
        acc.free(step, good)
    other = kvq.DeviceAccounts(Mirror(slots=3, Hkv=2, d=64, page=32).cache)
    for call in (lambda: other.extend(step, good), lambda: other.free(step), lambda: acc.extend(old, good[:1])):
        with pytest.raises(ValueError, match="other accounts"):
            call()
    acc.extend(step, good)
    two = acc.step([1], 1)
    acc.extend(two, good[:1])
    with pytest.raises(ValueError, match="changed"):
        kvq.paged_decode(m.rand(8, 4).cuda(), 0.1, c, 0, step)       # slot 1 has had another step
    acc.free(two)
    with pytest.raises(ValueError, match="changed"):
        kvq.paged_decode(m.rand(1, 4).cuda(), 0.1, c, 0, two)
    acc.close()
    assert c.lengths == [41, 0, 0]
    with pytest.raises(kvq.KVQError, match="handed back"):
        acc.close()
    with pytest.raises(ValueError, match="changed"):
        kvq.paged_decode(m.rand(8, 4).cuda(), 0.1, c, 0, step)
    with pytest.raises(ValueError):
        c.extend([0, 1], [4, 4], into=step)

"""Attention of many rows over the paged cache against the float64 oracle: chunks of prompts, questions behind a shared text,
cross attention; cut and joined rows, values that a row must not see, replays and other streams, and what is refused."""
import pytest
import torch

from attention_bounds import HALF, check
from oracle.paged import attend, cached
from test_gpu_pages import Mirror

pytestmark = pytest.mark.gpu

# A weight times its block's value scale is one number of the type, rounded to nearest once: off by at most half a step, 2^-8 (bf16) or
# 2^-11 (fp16) of itself, 2^-32 of the block's largest value where it is below fp16's normal range (the bound has 2^-25 of it)
# The rounded weights p (1 + e), |e| <= h, are summed: the output is off by sum p e (v - o) / (1 + sum p e), at most h (sum p |v| + |o|) / (1 - h), and |o| is
# no more than sum p |v|
WEIGHT = {t: 2 * h / (1 - h) for t, h in HALF.items()}


@pytest.fixture(params=[0, None, 1 << 30], ids=["tiles", "by rows", "16 rows"], autouse=True)
def few_rows(request, monkeypatch):
    """Every call by the kernels of many rows, by those that it gets, and by the decode's."""
    import kvq.paged
    if request.param is not None:
        monkeypatch.setattr(kvq.paged, "FEW_ROWS", request.param)
    else:
        monkeypatch.setattr(kvq.paged, "FEW_WORK", 1)                # however short they are
    return request.param


def run(m, slots, counts, Hq, causal=True, layer=0, what="", scaling=None, q=None):
    """One call, every row checked; returns (plan, q, out)."""
    import kvq
    c = m.cache
    scaling = c.d ** -0.5 if scaling is None else scaling
    plan = kvq.PagedPlan(c, slots, counts, Hq, causal=causal)
    q = m.rand(sum(counts), Hq) if q is None else q
    out = kvq.paged_attention(q.cuda(), scaling, c, layer, plan)
    a = 0
    for s, n in zip(slots, counts):
        if n:
            k, v = cached(m.k[layer][s], c.page, c.code), cached(m.v[layer][s], c.page, c.code)
            ref = attend(q[a:a + n], k, v, scaling, causal)
            check(out[a:a + n], ref, float(v.abs().max()) if len(v) else 0.0, k.shape[0], c.d, c.dtype, WEIGHT[c.dtype],
                  f"{what} slot {s}, {n} of {k.shape[0]}")
        a += n
    return plan, q, out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("page,d,Hkv,rep", [(32, 64, 2, 4), (64, 128, 1, 3), (128, 64, 1, 7), (32, 128, 1, 1), (128, 128, 2, 2), (64, 64, 1, 8)])
def test_chunks(page, d, Hkv, rep, code, dtype):
    """Chunks from one token to all of the slot's, lengths around the blocks' borders, nothing for one of them."""
    m = Mirror(page=page, d=d, Hkv=Hkv, code=code, dtype=dtype, seed=page + d + rep)
    m.push([0, 1, 2, 3, 4], [1, page, 2 * page + 40, 3 * page - 1, 64])
    run(m, [0, 1, 2, 3, 4], [1, page, 41, 60, 0], rep * Hkv, what="chunks")
    run(m, [4, 2], [64, 1], rep * Hkv, what="whole")
    m.push([0, 1], [70, 33])
    run(m, [1, 0], [33, 70], rep * Hkv, what="later")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,d,Hkv,rep", [(32, 64, 2, 4), (64, 128, 1, 3), (128, 64, 1, 8)])
def test_shared_text(page, d, Hkv, rep, dtype, few_rows):
    """Questions of forks side by side, others between, uneven; and the same rows again, and each alone."""
    import kvq
    m = Mirror(slots=10, pages=200, max_tokens=1500, Hkv=Hkv, d=d, page=page, dtype=dtype, seed=page)
    m.push([0, 1], [900, 333])
    m.fork([0] * 5 + [1] * 2, [2, 3, 4, 5, 6, 7, 8])
    counts = [1, 5, 17, 3, 90, 2, 40, 8]
    m.push([0, 2, 3, 4, 5, 7, 8, 9], [1, 5, 17, 3, 90, 2, 40, 8])
    plan, q, out = run(m, [0, 2, 3, 4, 5, 7, 8, 9], counts, rep * Hkv, what="forks")
    # the seven that share a text are joined, a tile of their rows at a time
    assert (few_rows != 0 or plan.merges >= 7) and torch.equal(out, kvq.paged_attention(q.cuda(), d ** -0.5, m.cache, 0, plan))
    run(m, [2, 9, 3, 6, 4], [5, 0, 17, 9, 3], rep * Hkv, what="between")
    run(m, [6, 6], [900, 30], Hkv, what="the text itself, twice")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("page,d,Hkv,rep", [(32, 64, 2, 1), (64, 128, 1, 4), (128, 128, 1, 2)])
def test_cross(page, d, Hkv, rep, code, dtype):
    """Every row sees every token: beams of one encoder, one without states, single tokens and prompts, shared pages."""
    m = Mirror(slots=8, pages=100, max_tokens=900, Hkv=Hkv, d=d, page=page, code=code, dtype=dtype, seed=page + rep)
    m.push([0, 1, 2, 3], [750, 1, page, 200])
    m.fork([0, 0], [5, 6])
    m.push([5], [70])
    run(m, [0, 0, 0, 4, 1, 2, 3], [1, 1, 1, 2, 3, 1, 100], rep * Hkv, causal=False, what="beams")
    run(m, [0, 5, 6, 3], [7, 1, 2, 0], rep * Hkv, causal=False, what="shared pages")
    run(m, [4, 4], [1, 0], rep * Hkv, causal=False, what="none")
    # forks of a whole number of units: nothing of their own
    m.free([0, 5, 6])
    m.push([0], [512])
    m.fork([0, 0], [5, 6])
    run(m, [0, 5, 6, 4], [3, 1, 40, 1], rep * Hkv, causal=False, what="all shared")


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n,rep,d", [(4099, 4, 64), (2600, 1, 128), (5000, 2, 64)])
def test_cut_along_the_tokens(n, rep, d, causal, few_rows):
    """Few rows over many tokens: parts and their joins, with and without a shared text."""
    m = Mirror(slots=4, pages=300, max_tokens=5200, Hkv=1, d=d, page=64, seed=n)
    m.push([0, 1], [n, 700])
    plan, _, _ = run(m, [0, 1], [3, 2], rep, causal, what="cut")
    if few_rows == 0:
        assert plan.parts > 2 and plan.merges == 2 and not plan.sequences
    else:
        assert not plan.items and plan.sequences == 2
    m.fork([0, 0], [2, 3])
    m.push([2, 3], [5, 40])
    run(m, [2, 3], [5, 7], rep, causal, what="cut text")


@pytest.mark.parametrize("page,code,dtype,causal", [(32, "int8", torch.bfloat16, True), (64, "e4m3", torch.float16, True),
                                                     (128, "int8", torch.float16, False), (64, "int8", torch.bfloat16, False)])
def test_a_full_chip(page, code, dtype, causal):
    """As many tiles as the chip has places: workgroups of 256 rows, alone and with a text that is shared; some heads of all rows."""
    import kvq
    H, d, heads = 64, 128, [0, 31, 63]
    m = Mirror(slots=9, pages=9 * (1100 // page + 1), max_tokens=1100, Hkv=H, d=d, page=page, code=code, dtype=dtype, seed=page)
    lens = [300, 256, 290, 300]
    m.push([0, 1, 2, 3, 4], [*lens, 640])
    m.fork([4] * 4, [5, 6, 7, 8])
    m.push([5, 6, 7, 8], lens)
    for slots in ([0, 1, 2, 3], [5, 6, 7, 8]):
        plan = kvq.PagedPlan(m.cache, slots, [256] * 4, H, causal=causal)
        assert plan.sequences or plan.waves == 8
        q = m.rand(1024, H)
        out = kvq.paged_attention(q.cuda(), d ** -0.5, m.cache, 0, plan)
        for i, s in enumerate(slots):
            k, v = (cached(x[0][s][:, heads], page, code) for x in (m.k, m.v))
            rows = slice(256 * i, 256 * (i + 1))
            check(out[rows][:, heads], attend(q[rows][:, heads], k, v, d ** -0.5, causal), float(v.abs().max()), k.shape[0], d, dtype,
                  WEIGHT[dtype], f"slot {s}")


def test_one_query_head_to_many():
    """128 query heads over one KV head: a tile for each token."""
    m = Mirror(Hkv=1, d=64, page=32, seed=5)
    m.push([0], [150])
    run(m, [0], [3], 128, what="128 heads")
    run(m, [0], [2], 20, what="20 heads")


def test_layers_after_moves():
    m = Mirror(layers=3, slots=4, pages=30, max_tokens=600, Hkv=2, d=64, page=32, seed=4)
    m.push([0, 1, 2], [100, 164, 31])
    m.free([0])
    import kvq
    plan = kvq.PagedPlan(m.cache, [1, 2], [50, 31], 4)               # made before the pages move
    m.cache.compact()
    for l in range(3):
        _, q, out = run(m, [1, 2], [50, 31], 4, layer=l, what=f"layer {l}")
        assert torch.equal(out, kvq.paged_attention(q.cuda(), 0.125, m.cache, l, plan))
    m.cache.resize(20)
    assert torch.equal(out, kvq.paged_attention(q.cuda(), 0.125, m.cache, 2, plan))
    run(m, [2, 1], [3, 164], 4, layer=2, what="resized")


@pytest.mark.parametrize("scaling", [0.0, -0.3, 2.5])
def test_scaling(scaling):
    m = Mirror(Hkv=1, d=64, page=32, seed=6)
    m.push([0], [150])
    run(m, [0], [40], 4, what=f"scaling {scaling}", scaling=scaling)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page", [32, 64, 128])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("side", ["k", "v"])
def test_hidden_values_change_nothing(side, value, page, dtype):
    """An infinity or a NaN behind what a row sees, in a block that was coded (its scale is NaN) and in the open one: the rows in
    front of the block are as without it; in the open block a visible value is its channel's result."""
    import kvq
    d, n = 64, 3 * page + 20
    m = Mirror(slots=2, Hkv=1, d=d, page=page, dtype=dtype, max_tokens=600, seed=7)
    k, v = m.rand(n, 1), m.rand(n, 1)
    q = m.rand(n, 2)
    for slot, bad in ((0, [2 * page + 5]), (1, [3 * page + 11])):
        kk, vv = k.clone(), v.clone()
        for j in bad:
            (kk if side == "k" else vv)[j, 0, 3] = value
        step = m.cache.extend([slot], [n])
        m.cache.append(0, kk.cuda(), vv.cuda(), step)
        plan = kvq.PagedPlan(m.cache, [slot], [n], 2)
        out = kvq.paged_attention(q.cuda(), d ** -0.5, m.cache, 0, plan).cpu()
        first = bad[0] // page * page if slot == 0 else bad[0]       # rows in front of the block, or of the token
        if slot == 0:
            first = 2 * page                                        # row i sees the block's first token from i = first on
        ref = attend(q, cached(k, page, "int8"), cached(v, page, "int8"), d ** -0.5)
        vmax = float(v.abs().max())
        check(out[:first], tuple(x[:first] for x in ref), vmax, n, d, dtype, WEIGHT[dtype], f"slot {slot}")
        late = out[first:].float()
        if slot == 0 or side == "k" and value != value:
            assert late.isnan().all()
        elif side == "v":
            hit = late[..., 3]
            assert bool(hit.isnan().all()) if value != value else bool((hit == value).all())
            rest = [i for i in range(d) if i != 3]
            check(out[first:][..., rest], tuple(x[first:][..., rest] if x.shape[-1] == d else x[first:] for x in ref), vmax, n, d, dtype,
                  WEIGHT[dtype], "other channels")


def test_few_and_many_rows_in_one_call(few_rows):
    """Single tokens, drafts and long chunks side by side, nothing for one, a shared text among the chunks, a slot named twice."""
    m = Mirror(slots=9, pages=200, max_tokens=1500, Hkv=2, d=64, page=32, seed=12)
    m.push([0, 1, 2, 3, 4], [900, 31, 640, 70, 1])
    m.fork([2, 2], [5, 6])
    m.push([5, 6], [100, 60])
    slots, counts = [4, 0, 2, 5, 6, 3, 7, 1], [1, 2, 50, 100, 60, 70, 0, 1]
    plan, _, _ = run(m, slots, counts, 8, what="mixed")
    assert few_rows is not None or plan.items and plan.sequences == 7
    run(m, [1, 4, 0], [1, 1, 100], 8, what="few in front")
    run(m, [0, 4, 1], [100, 1, 1], 8, what="many in front")
    run(m, [0, 0, 1, 0, 7, 3], [2, 1, 3, 40, 2, 1], 8, causal=False, what="cross")
    run(m, [0, 1, 0], [1, 1, 1], 8, causal=False, what="named twice")


def test_replays_streams_and_strides():
    """A captured call replayed with other rows, another stream, expanded rows, the caller's output and workspace."""
    import kvq
    m = Mirror(slots=4, pages=120, max_tokens=3100, Hkv=2, d=64, page=32, seed=8)
    m.push([0], [3001])
    m.fork([0, 0], [1, 2])
    m.push([1, 2], [4, 9])
    plan = kvq.PagedPlan(m.cache, [1, 2], [4, 9], 8)
    assert plan.workspace_floats()
    q = m.rand(13, 8).cuda()
    out = torch.empty_like(q)
    ws = torch.full((plan.workspace_floats(),), float("nan"), device="cuda")
    kvq.paged_attention(q, 0.125, m.cache, 0, plan, out=out, workspace=ws)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        kvq.paged_attention(q, 0.125, m.cache, 0, plan, out=out, workspace=ws)
    for i in range(3):
        q.copy_(m.rand(13, 8))
        _ = (q.float() * 2).sum()
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, kvq.paged_attention(q, 0.125, m.cache, 0, plan)), i
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one = m.rand(1, 8).cuda()
        got = kvq.paged_attention(one.expand(13, -1, -1), 0.125, m.cache, 0, plan)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, kvq.paged_attention(one.expand(13, -1, -1).contiguous(), 0.125, m.cache, 0, plan))
    wide = torch.empty((13, 8, 96), dtype=q.dtype, device="cuda")
    wide[..., 32:] = q
    assert torch.equal(kvq.paged_attention(wide[..., 32:], 0.125, m.cache, 0, plan), out)
    odd = torch.empty((13, 8, 67), dtype=q.dtype, device="cuda")
    odd[..., 3:] = q
    assert torch.equal(kvq.paged_attention(odd[..., 3:], 0.125, m.cache, 0, plan), out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_through_the_router(dtype):
    """Prompts, tokens, questions and branches of a batch through router_attention, questions straight over the pages."""
    from types import SimpleNamespace
    import kvq
    m = Mirror(layers=2, slots=6, pages=90, max_tokens=900, Hkv=2, d=64, page=32, dtype=dtype, seed=13)
    c = m.cache

    def step(ctl, counts, T):
        begins = [c.length(s) == 0 for s in ctl.slots]
        with kvq.routed(ctl):
            ctl.begin(counts)
            for l in range(2):
                q, k, v = (torch.randn(len(counts), h, T, 64, generator=m.g).to(dtype) for h in (8, 2, 2))
                out, _ = kvq.router_attention(SimpleNamespace(layer_idx=l, scaling=0.125), q.cuda(), k.cuda(), v.cuda(), None)
                for b, (s, n) in enumerate(zip(ctl.slots, counts)):
                    assert not out[b, :T - n].any()
                    kk, vv = (x[b].transpose(0, 1)[T - n:] for x in (k, v))
                    m.k[l][s], m.v[l][s] = torch.cat([m.k[l][s], kk]), torch.cat([m.v[l][s], vv])
                    if n == 0:
                        continue
                    kk, vv = m.k[l][s], m.v[l][s]
                    if not begins[b]:
                        kk, vv = cached(kk, 32, "int8"), cached(vv, 32, "int8")
                    check(out[b, T - n:], attend(q[b].transpose(0, 1)[T - n:], kk, vv, 0.125), float(vv.abs().max()), kk.shape[0], 64, dtype,
                          WEIGHT[dtype], f"layer {l} slot {s}")

    ctl = kvq.PagedCtl(c, [0, 1, 2], over_pages=True)
    step(ctl, [300, 131, 64], 300)
    step(ctl, [1, 1, 1], 1)
    step(ctl, [60, 0, 49], 60)
    c.fork([0, 0], [3, 4])
    for l in range(2):
        for x in (m.k[l], m.v[l]):
            x[3] = x[4] = x[0]
    step(kvq.PagedCtl(c, [0, 3, 4, 5, 1], over_pages=True), [20, 33, 1, 70, 50], 70)
    step(ctl, [2, 1, 3], 3)


def test_blocks_of_very_different_scales():
    """Value scales that grow and fall from block to block by factors of up to 2^60 (bf16) and 2^14 (fp16), blocks of zeros between: each
    row against the blocks that it sees."""
    import kvq
    for dtype, big in ((torch.bfloat16, 60), (torch.float16, 14)):
        for page in (32, 64):
            n, d = 9 * page + 7, 64
            m = Mirror(slots=1, Hkv=1, d=d, page=page, dtype=dtype, max_tokens=1000, seed=page)
            k, v = m.rand(n, 1), torch.randn(n, 1, d, generator=m.g)
            for j, e in enumerate([0, -big, 0, None, big // 2, -big // 2, 3, None, -big, 0]):
                v[j * page:(j + 1) * page] *= 0.0 if e is None else 2.0 ** (e - (big if dtype == torch.bfloat16 else 0))
            v, q = v.to(dtype), m.rand(n, 2)
            step = m.cache.extend([0], [n])
            m.cache.append(0, k.cuda(), v.cuda(), step)
            out = kvq.paged_attention(q.cuda(), d ** -0.5, m.cache, 0, kvq.PagedPlan(m.cache, [0], [n], 2))
            vv = cached(v, page, "int8")
            ref = attend(q, cached(k, page, "int8"), vv, d ** -0.5)
            for a in range(0, n, page):        # a row's bound has the largest value that it sees
                b = min(n, a + page)
                check(out[a:b], tuple(x[a:b] for x in ref), float(vv[:b].abs().max()), b, d, dtype, WEIGHT[dtype], f"{dtype} page {page} rows {a}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,d", [(32, 128), (64, 64), (128, 128)])
@pytest.mark.parametrize("way", ["climb", "jumps", "from far below", "down"])
def test_scores_that_climb(way, page, d, dtype):
    """Scores that climb along the text, for some rows slowly, for others fast, for others not: by less than a weight has room for,
    by far more from one block to the next, and from far below the others."""
    import kvq
    n = 640 + 9
    at = torch.arange(n, dtype=torch.float64)
    c = {"climb": at * 0.06, "jumps": 45.0 * (at // 130), "from far below": torch.where(at < 200, -150.0, 20.0), "down": 120.0 - at * 0.2}[way]
    m = Mirror(slots=1, Hkv=2, d=d, page=page, dtype=dtype, max_tokens=1000, seed=page + d)
    u = torch.randint(0, 2, (2, d), generator=m.g).double() * 2 - 1
    k = (c[:, None, None] * u + 0.3 * torch.randn(n, 2, d, generator=m.g)).to(dtype)
    v = m.rand(n, 2)
    q = torch.tensor([1.0, -1.0, 0.25, 0.0, 0.5] * 8, dtype=torch.float64)[:, None, None] * u.repeat_interleave(2, 0)
    m.cache.append(0, k.cuda(), v.cuda(), m.cache.extend([0], [n]))
    m.k[0][0], m.v[0][0] = k, v
    run(m, [0], [40], 4, what=way, scaling=1.0 / d, q=q.to(dtype))
    run(m, [0], [40], 4, causal=False, what=way, scaling=1.0 / d, q=q.to(dtype))


def test_scores_of_minus_infinity():
    """A text whose first block gives a row scores of -inf alone (keys and queries near the type's largest): the row is what the
    rest of it gives."""
    import kvq
    d, n = 64, 64 * 5 + 3
    m = Mirror(slots=1, Hkv=1, d=d, page=64, max_tokens=600, seed=3)
    k, v, q = m.rand(n, 1), m.rand(n, 1), m.rand(40, 2)
    k[:64] = -3e37
    k[:, 0, 1:] = 0
    q[:, :, 0] = torch.where(torch.arange(40)[:, None] % 2 == 0, 3e37, 1.0)
    k[64:, 0, 0] = 0
    m.cache.append(0, k.cuda(), v.cuda(), m.cache.extend([0], [n]))
    out = kvq.paged_attention(q.cuda(), 1.0, m.cache, 0, kvq.PagedPlan(m.cache, [0], [40], 2))
    kk, vv = cached(k, 64, "int8"), cached(v, 64, "int8")
    # the others of the first block weigh exp(-3e37), nothing
    ref = attend(q, kk[64:], vv[64:], 1.0)
    check(out, ref, float(vv.abs().max()), n, d, torch.bfloat16, WEIGHT[torch.bfloat16], "-inf in front")


def test_refusals():
    import kvq
    m = Mirror(slots=3, Hkv=2, d=64, page=32)
    m.push([0, 1], [40, 10])
    c = m.cache
    for slots, counts, what in (([], [], "length"), ([0], [1, 2], "length"), ([3], [1], "slot"), ([-1], [1], "slot"), ([0], [-1], "negative"),
                                ([0], [41], "last"), ([2], [1], "last")):
        with pytest.raises((ValueError, kvq.KVQError), match=what):
            kvq.PagedPlan(c, slots, counts, 4)
    for Hq in (0, 3, 2 * 129):
        with pytest.raises(ValueError, match="query heads"):
            kvq.PagedPlan(c, [0], [1], Hq)
    plan = kvq.PagedPlan(c, [0, 1], [5, 2], 4)
    q = m.rand(7, 4).cuda()
    ws = torch.empty(0, device="cuda")
    call = lambda q=q, layer=0, cache=c, p=plan, **kw: kvq.paged_attention(q, 0.1, cache, layer, p, **kw)
    call()
    for bad, error in ((dict(layer=1), IndexError), (dict(layer=-1), IndexError), (dict(q=q[:6]), ValueError), (dict(q=q[..., :32]), ValueError),
                       (dict(q=q.half()), TypeError), (dict(q=q.cpu()), kvq.KVQError), (dict(out=torch.empty_like(q)[:6]), ValueError),
                       (dict(out=torch.empty(7, 4, 64, device="cuda")), ValueError), (dict(workspace=ws.double()), ValueError)):
        with pytest.raises(error):
            call(**bad)
    other = Mirror(slots=3, Hkv=2, d=64, page=32).cache
    with pytest.raises(ValueError, match="another cache"):
        call(cache=other)
    long = Mirror(slots=1, pages=200, max_tokens=6000, Hkv=1, d=64, page=32)
    long.push([0], [5000])
    cut = kvq.PagedPlan(long.cache, [0], [2], 4)
    assert cut.workspace_floats() > 0
    with pytest.raises(ValueError, match="workspace"):
        kvq.paged_attention(long.rand(2, 4).cuda(), 0.1, long.cache, 0, cut, workspace=ws)
    m.push([2], [3])
    call()                                     # another slot's tokens
    m.push([1], [1])
    with pytest.raises(ValueError, match="changed"):
        call()

"""Attention over packed prompts against the float64 oracle: lengths from none to many, chunks behind a past,
rows without a key, grouped heads, strides, values that a row must not see, replays and other streams."""
import math

import pytest
import torch

from attention_bounds import HALF, check
from oracle.paged import attend

pytestmark = pytest.mark.gpu


def _inputs(lens, lens_k, Hq, Hkv, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randn(n, h, d, generator=g).to(dtype) for n, h in ((sum(lens), Hq), (sum(lens_k), Hkv), (sum(lens_k), Hkv)))


def _check(out, q, k, v, lens, lens_k, causal, dtype, what):
    a = x = 0
    d = q.shape[2]
    for t, n in zip(lens, lens_k):
        if t:
            ref = attend(q[a:a + t], k[x:x + n], v[x:x + n], d ** -0.5, causal)
            vmax = float(v[x:x + n].abs().max()) if n else 0.0
            check(out[a:a + t], ref, vmax, n, d, dtype, HALF[dtype], f"{what} {t} of {n}")
        a, x = a + t, x + n


SHAPES = [
    # lens, lens_k, Hq, Hkv, d, causal
    ([1], [1], 1, 1, 64, True),
    ([20], [20], 32, 8, 128, True),
    ([63, 1, 64, 65, 0, 2], [63, 1, 64, 65, 0, 2], 4, 2, 64, True),
    ([130, 7], [130, 7], 2, 2, 128, True),                   # one query head per KV head
    ([37, 50], [37, 50], 7, 1, 128, True),                   # seven: tiles of 18 tokens
    ([33, 5], [33, 5], 6, 2, 64, True),
    ([4, 30, 1], [70, 200, 129], 8, 2, 64, True),            # behind a past
    ([9, 3, 5], [4, 0, 5], 4, 1, 128, True),                 # more queries than keys: rows without a key
    ([9, 3, 0], [77, 0, 5], 4, 4, 128, False),
    ([5, 2], [0, 0], 4, 2, 64, True),
    ([0, 0], [0, 7], 4, 2, 64, True),
    ([2], [300], 128, 1, 64, True),                          # a tile per token
    ([150], [150], 3, 1, 64, False),
    ([3, 1, 40], [5000, 700, 1300], 4, 1, 128, True),        # few rows: cut along the keys
    ([1, 2], [6000, 513], 2, 2, 64, False),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_prompt_attention(case, dtype):
    import kvq
    lens, lens_k, Hq, Hkv, d, causal = SHAPES[case]
    q, k, v = _inputs(lens, lens_k, Hq, Hkv, d, dtype, 100 + case)
    plan = kvq.PromptPlan(lens, Hq, Hkv, lens_k=lens_k, causal=causal)
    out = torch.full(q.shape, float("nan"), dtype=dtype, device="cuda")
    got = kvq.prompt_attention(q.cuda(), k.cuda(), v.cuda(), d ** -0.5, plan, out=out)
    assert got.data_ptr() == out.data_ptr()
    _check(got, q, k, v, lens, lens_k, causal, dtype, f"case {case}")


def test_large_scores_and_constant_rows():
    """Scores of several hundred (one key takes all the weight, its maximum late) and equal scores."""
    import kvq
    lens, Hq, Hkv, d = [200], 4, 1, 128
    q, k, v = _inputs(lens, lens, Hq, Hkv, d, torch.bfloat16, 5)
    k[150] = 40 * q[180, 0] / q[180, 0].norm()
    q[180] = q[180] * 8
    q[10] = 0
    out = kvq.prompt_attention(q.cuda(), k.cuda(), v.cuda(), d ** -0.5, kvq.PromptPlan(lens, Hq, Hkv))
    _check(out, q, k, v, lens, lens, True, torch.bfloat16, "large")


@pytest.mark.parametrize("layout", ["fused", "head_major", "odd"])
def test_strides(layout):
    """Rows of a fused projection, head-major rows, and rows the kernels cannot read in 16-byte pieces."""
    import kvq
    lens, Hq, Hkv, d = [70, 31], 8, 2, 64
    q, k, v = _inputs(lens, lens, Hq, Hkv, d, torch.bfloat16, 9)
    n = sum(lens)
    if layout == "fused":
        x = torch.cat([q, k, v], 1).cuda()
        a, b, c = x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]
    elif layout == "head_major":
        a, b, c = (x.transpose(0, 1).contiguous().cuda().transpose(0, 1) for x in (q, k, v))
    else:
        a, b, c = (torch.zeros((n, x.shape[1], d + 3), dtype=x.dtype, device="cuda")[:, :, 1:1 + d].copy_(x) for x in (q, k, v))
    plan = kvq.PromptPlan(lens, Hq, Hkv)
    got = kvq.prompt_attention(a, b, c, d ** -0.5, plan)
    assert torch.equal(got, kvq.prompt_attention(q.cuda(), k.cuda(), v.cuda(), d ** -0.5, plan))
    _check(got, q, k, v, lens, lens, True, torch.bfloat16, layout)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_values_that_a_row_does_not_see(bad, dtype):
    """Keys and values behind a row, infinite or NaN, leave it as it is; a row that sees one does not hide it."""
    import kvq
    lens, Hq, Hkv, d, at = [90, 40], 4, 2, 64, 50
    q, k, v = _inputs(lens, lens, Hq, Hkv, d, dtype, 21)
    plan = kvq.PromptPlan(lens, Hq, Hkv)
    clean = kvq.prompt_attention(q.cuda(), k.cuda(), v.cuda(), d ** -0.5, plan)
    # the same behind a past that is cut into parts
    past = [torch.cat([x[:0], torch.randn(3000, Hkv, d).to(dtype), x[:90]]) for x in (k, v)]
    late = kvq.PromptPlan([90], Hq, Hkv, lens_k=[3090])
    assert late.parts
    for s in (0, 1):
        dirty = [x.clone() for x in past]
        before = kvq.prompt_attention(q[:90].cuda(), past[0].cuda(), past[1].cuda(), d ** -0.5, late)
        dirty[s][3000 + at] = bad
        after = kvq.prompt_attention(q[:90].cuda(), dirty[0].cuda(), dirty[1].cuda(), d ** -0.5, late)
        assert torch.equal(after[:at], before[:at])
        assert s == 0 or not torch.isfinite(after[at:].float()).any()
    kb, vb = k.clone(), v.clone()
    kb[at + 5], vb[at, :, 3] = bad, bad
    got = kvq.prompt_attention(q.cuda(), kb.cuda(), vb.cuda(), d ** -0.5, plan)
    assert torch.equal(got[:at], clean[:at]) and torch.equal(got[90:], clean[90:])
    seen = got[at:at + 5].float()
    assert not torch.isfinite(seen[:, :, 3]).any()
    assert torch.equal(seen[:, :, :3], clean[at:at + 5, :, :3].float())
    assert torch.equal(seen[:, :, 4:], clean[at:at + 5, :, 4:].float())


def test_expanded_rows_and_a_negative_scaling():
    import kvq
    lens, Hq, Hkv, d = [90, 3], 4, 2, 128
    q, k, v = _inputs(lens, lens, Hq, Hkv, d, torch.float16, 51)
    plan = kvq.PromptPlan(lens, Hq, Hkv)
    one = k[:1].cuda().expand(93, -1, -1)
    assert torch.equal(kvq.prompt_attention(q.cuda(), one, v.cuda(), 0.1, plan),
                       kvq.prompt_attention(q.cuda(), one.contiguous(), v.cuda(), 0.1, plan))
    assert torch.equal(kvq.prompt_attention(q.cuda(), k.cuda(), v.cuda(), -0.1, plan),
                       kvq.prompt_attention(-q.cuda(), k.cuda(), v.cuda(), 0.1, plan))


@pytest.mark.parametrize("scaling", [0.0, -0.0, 1e-45])
def test_a_scaling_of_nothing(scaling):
    """Every visible value weighs the same; hidden ones nothing."""
    import kvq
    lens, lens_k = [70, 3], [70, 900]
    q, k, v = _inputs(lens, lens_k, 4, 2, 64, torch.bfloat16, 52)
    out = kvq.prompt_attention(q.cuda(), k.cuda(), v.cuda(), scaling, kvq.PromptPlan(lens, 4, 2, lens_k=lens_k))
    a = x = 0
    for t, n in zip(lens, lens_k):
        ref = attend(q[a:a + t], k[x:x + n], v[x:x + n], 0.0)
        check(out[a:a + t], ref, float(v[x:x + n].abs().max()), n, 64, torch.bfloat16, HALF[torch.bfloat16], f"{t} of {n}")
        a, x = a + t, x + n


def test_offsets_past_32_bits():
    """Rows whose offsets pass 2^32 bytes and 2^31 elements."""
    import kvq
    lens, Hq, Hkv, d = [2100], 2, 1, 64
    q, k, v = _inputs(lens, lens, Hq, Hkv, d, torch.bfloat16, 33)
    step = 1 << 20
    flat = torch.empty((2100 * step + d * 4,), dtype=torch.bfloat16, device="cuda")
    rows = [flat.as_strided((2100, h, d), (step, d, 1), o * d) for o, h in ((0, 2), (2, 1), (3, 1))]
    for r, x in zip(rows, (q, k, v)):
        r.copy_(x)
    plan = kvq.PromptPlan(lens, Hq, Hkv)
    got = kvq.prompt_attention(*rows, d ** -0.5, plan)
    assert torch.equal(got, kvq.prompt_attention(q.cuda(), k.cuda(), v.cuda(), d ** -0.5, plan))


def test_replays_and_another_stream():
    import kvq
    lens, Hq, Hkv, d = [300, 41, 7], 8, 2, 128
    q, k, v = (x.cuda() for x in _inputs(lens, lens, Hq, Hkv, d, torch.bfloat16, 41))
    plan = kvq.PromptPlan(lens, Hq, Hkv)
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = kvq.prompt_attention(q, k, v, d ** -0.5, plan)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, kvq.prompt_attention(q, k, v, d ** -0.5, plan))
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        kvq.prompt_attention(q, k, v, d ** -0.5, plan, out=out)
    few = kvq.PromptPlan([2, 3], Hq, Hkv, lens_k=[4000, 900])      # cut along the keys: with scratch of its own
    assert few.parts
    k2, v2 = (torch.randn((4900, Hkv, d), dtype=torch.bfloat16, device="cuda") for _ in (0, 1))
    ws, out2 = torch.empty(few.workspace_floats(d), device="cuda"), torch.empty_like(q[:5])
    gr2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr2):
        kvq.prompt_attention(q[:5], k2, v2, d ** -0.5, few, out=out2, workspace=ws)
    for i in range(3):
        q.copy_(torch.randn_like(q))
        _ = (q.float() * 2).sum()
        torch.cuda.synchronize()
        gr.replay()
        gr2.replay()
        torch.cuda.synchronize()
        assert torch.equal(out2, kvq.prompt_attention(q[:5], k2, v2, d ** -0.5, few)), i
        assert torch.equal(out, kvq.prompt_attention(q, k, v, d ** -0.5, plan)), i


def test_refusals():
    import kvq
    q = torch.zeros((5, 4, 64), dtype=torch.bfloat16, device="cuda")
    k = torch.zeros((5, 2, 64), dtype=torch.bfloat16, device="cuda")
    plan = kvq.PromptPlan([5], 4, 2)
    with pytest.raises(ValueError, match="plan"):
        kvq.prompt_attention(q[:4], k, k, 0.1, plan)
    with pytest.raises(ValueError, match="plan"):
        kvq.prompt_attention(q, k[:4], k[:4], 0.1, plan)
    with pytest.raises(TypeError):
        kvq.prompt_attention(q.float(), k.float(), k.float(), 0.1, plan)
    with pytest.raises(TypeError):
        kvq.prompt_attention(q, k.half(), k.half(), 0.1, plan)
    with pytest.raises(kvq.KVQError, match="head_dim"):
        kvq.prompt_attention(q[..., :32], k[..., :32], k[..., :32], 0.1, plan)
    with pytest.raises(ValueError, match="out"):
        kvq.prompt_attention(q, k, k, 0.1, plan, out=torch.empty((5, 64, 4), dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(kvq.KVQError):
        kvq.prompt_attention(q.cpu(), k, k, 0.1, plan)


def test_a_plan_dropped_before_another_stream_is_done():
    """A call on a stream that is busy, its plan gone: what the plan's own stream allocates next is other memory."""
    import kvq
    lens, lens_k, Hq, Hkv, d = [30, 4], [3000, 70], 4, 2, 64
    q, k, v = (x.cuda() for x in _inputs(lens, lens_k, Hq, Hkv, d, torch.bfloat16, 65))
    plan = kvq.PromptPlan(lens, Hq, Hkv, lens_k=lens_k)
    want, size = kvq.prompt_attention(q, k, v, 0.125, plan), plan.words.numel()
    out, ws = torch.empty_like(want), torch.empty(plan.workspace_floats(d), device="cuda")
    x = torch.ones(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(20):
            x = x @ x * 1e-4
        kvq.prompt_attention(q, k, v, 0.125, plan, out=out, workspace=ws)
    del plan
    held = [torch.zeros(size, dtype=torch.int32, device="cuda") for _ in range(64)]
    torch.cuda.synchronize()
    assert torch.equal(out, want) and not any(bool(h.any()) for h in held)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,lens_k", [([40], [40]), ([40], [3040])])
def test_rows_whose_scores_are_all_minus_infinity(lens, lens_k, dtype):
    """Visible keys with scores of -inf only leave a row without a sum, a NaN, whether its tile is cut along the keys or not;
    one finite score takes all the weight."""
    import kvq
    q, k, v = _inputs(lens, lens_k, 4, 2, 64, dtype, 61)
    q[..., 0], k[..., 0] = 1.0, float("-inf")
    plan = kvq.PromptPlan(lens, 4, 2, lens_k=lens_k)
    assert bool(plan.parts) == (lens_k[0] > 512)
    out = kvq.prompt_attention(q.cuda(), k.cuda(), v.cuda(), 0.125, plan)
    assert torch.isnan(out).all()
    k[lens_k[0] - 30, :, 0] = 0.0
    out = kvq.prompt_attention(q.cuda(), k.cuda(), v.cuda(), 0.125, plan).cpu()
    assert torch.isnan(out[:10]).all() and torch.equal(out[10:], v[-30].repeat_interleave(2, 0).expand(30, -1, -1))


def _far_query_and_key(q, k, at):
    """The key ``at`` takes all the weight: by e^400 and more over every other visible one."""
    q[..., 0], k[..., 0] = 16.0, 0.0
    k[at, :, 0] = 25.0 * q.shape[2] ** 0.5


@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float16, 64), (torch.float16, 128)])
@pytest.mark.parametrize("t,n,ats", [(300, 300, (10, 130, 299)), (90, 3090, (5, 1000, 2990, 3040))])
def test_a_visible_infinity_is_its_channels_result(t, n, ats, dtype, d, bad, far):
    """In tiles that every row sees and in those that some see in part, in whole sequences and in parts, and however small its
    weight: the rows that see an infinite value have it in that channel, the others and other channels do not change."""
    import kvq
    lens, lens_k, Hq, Hkv = [t], [n], 4, 2
    q, k, v = _inputs(lens, lens_k, Hq, Hkv, d, dtype, 62)
    if far:
        _far_query_and_key(q, k, 700 % n)
    plan = kvq.PromptPlan(lens, Hq, Hkv, lens_k=lens_k)
    assert bool(plan.parts) == (n > 512)
    run = lambda x: kvq.prompt_attention(q.cuda(), k.cuda(), x.cuda(), d ** -0.5, plan).cpu()
    clean = run(v)
    assert torch.isfinite(clean).all()
    for at in ats:
        for channel in (1, d - 1):
            vb, want = v.clone(), clean.clone()
            vb[at, 1, channel] = bad
            want[max(0, at - (n - t)):, 2:, channel] = bad
            assert torch.equal(torch.nan_to_num(run(vb), 7.0, 8.0, 9.0), torch.nan_to_num(want, 7.0, 8.0, 9.0)), (at, channel)
    vb = v.clone()
    vb[0, 0, 3], vb[n - t // 2, 0, 3] = float("inf"), float("-inf")
    out = run(vb)[:, :2, 3]
    assert torch.isposinf(out[:t - t // 2]).all() and torch.isnan(out[t - t // 2:]).all()


def test_many_small_fp16_weights():
    """A key without a value takes nearly all the weight, 200000 keys of value one 2^-26 of it each: 0.003 together, in tiles
    that are not cut."""
    import kvq
    t, n, d = 600, 200000, 64
    q, k, v = torch.zeros(t, 128, d), torch.zeros(n, 1, d), torch.ones(n, 1, d)
    q[..., 0], k[0, :, 0], v[0] = 1.0, 26.0, 0.0
    q, k, v = (x.half().cuda() for x in (q, k, v))
    plan = kvq.PromptPlan([t], 128, 1, lens_k=[n])
    assert plan.items == t and not plan.parts
    out = kvq.prompt_attention(q, k, v, math.log(2.0), plan).double().cpu()
    w = torch.arange(n - t, n, dtype=torch.float64)[:, None, None] * 2.0 ** -26
    # a weight of 2^-26 is rounded by 2^-6 of itself at most (2^-25 as a number of the type, 2^-19 with the reference at 2^7), the
    # sums by n roundings each, the result by half a step
    tol = 2.0 ** -6 + 2 * n * 2.0 ** -24 + 2.0 ** -11
    worst = float((out / (w / (1 + w)) - 1).abs().max())
    print(f"relative error {worst:.2e}, bound {tol:.2e}")
    assert worst <= tol


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,n,Hq,Hkv,d", [(600, 20000, 128, 1, 64), (530, 4333, 128, 1, 128), (1050, 1050, 64, 1, 64)])
def test_long_loops_of_many_tiles(t, n, Hq, Hkv, d, dtype):
    """More tiles of rows than places, so that each goes over all of its keys: up to 313 key tiles a workgroup, the largest
    score early, late and in between."""
    import kvq
    q, k, v = _inputs([t], [n], Hq, Hkv, d, dtype, 63)
    plan = kvq.PromptPlan([t], Hq, Hkv, lens_k=[n])
    assert plan.items * Hkv > 512 and not plan.parts
    rows = [0, 1, t // 2, t - 2, t - 1]
    for i, at in zip(rows, (n - t, 100, n - t, n - t + t // 2, 0)):
        k[at] = 6 * q[i, 0] / q[i, 0].norm()
        q[i] = q[i] * 4
    out = kvq.prompt_attention(q.cuda(), k.cuda(), v.cuda(), d ** -0.5, plan)
    for i in rows:
        m = n - t + i + 1
        check(out[i:i + 1], attend(q[i:i + 1], k[:m], v[:m], d ** -0.5), float(v[:m].abs().max()), m, d, dtype, HALF[dtype], f"row {i}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("late", [0, 12000, 39990])
def test_more_parts_than_a_wavefront_has_lanes(late, dtype):
    """A tile in more than 64 parts, joined in two rounds of maxima, the largest score in an early and in a late one."""
    import kvq
    n, d = 40000, 128
    q, k, v = _inputs([1], [n], 4, 1, d, dtype, 64)
    k[late] = 30 * q[0, 0] / q[0, 0].norm()
    plan = kvq.PromptPlan([1], 4, 1, lens_k=[n])
    assert plan.merges == 1 and plan.parts > 64
    out = kvq.prompt_attention(q.cuda(), k.cuda(), v.cuda(), d ** -0.5, plan)
    _check(out, q, k, v, [1], [n], True, dtype, f"late {late}")

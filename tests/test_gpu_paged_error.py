"""Attention over pages by the kernels of many rows: hidden infinities and NaN change no bit in front of them, for both codes; and the
error of weights that are one number of the type, against what their rounding alone can do."""
import pytest
import torch

from attention_bounds import HALF, bound
from oracle.paged import cached

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def tiles(monkeypatch):
    import kvq.paged
    monkeypatch.setattr(kvq.paged, "FEW_ROWS", 0)
    monkeypatch.setattr(kvq.paged, "FEW_WORK", 1)


def call(k, v, q, page, code, causal=True):
    import kvq
    n, H, d = k.shape
    c = kvq.PagedCache(1, 1, n // page + 1, n, H, d, page=page, code=code, dtype=k.dtype)
    c.append(0, k.cuda(), v.cuda(), c.extend([0], [n]))
    plan = kvq.PagedPlan(c, [0], [q.shape[0]], q.shape[1], causal=causal)
    assert plan.items and not plan.sequences
    return kvq.paged_attention(q.cuda(), d ** -0.5, c, 0, plan).cpu()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,d", [(32, 64), (64, 128), (128, 64)])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("side", ["k", "v"])
def test_rows_in_front_of_a_bad_block(side, value, page, d, dtype, code):
    """A block that holds an infinity or a NaN is NaN to the rows that see it, and the others are bit for bit what they are without it."""
    g = torch.Generator().manual_seed(page + d)
    n = 5 * page + 20
    k, v, q = (torch.randn(n, h, d, generator=g).to(dtype) for h in (1, 1, 4))
    good = call(k, v, q, page, code)
    for j in (1, 2, 4):
        x = {"k": k.clone(), "v": v.clone()}
        x[side][j * page + 7, 0, 3] = value
        out = call(x["k"], x["v"], q, page, code)
        assert torch.equal(out[:j * page], good[:j * page]) and out[j * page:].isnan().all(), j


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,d,sharp", [(32, 64, 1.0), (32, 128, 4.0), (64, 128, 0.2), (64, 64, 4.0), (128, 64, 1.0), (128, 128, 4.0)])
def test_error_of_the_rounded_weights(page, d, sharp, dtype, code, causal):
    """Weights p (1 + e), |e| <= h, half a step, that are summed as they are rounded give sum p (1 + e) v / (1 + sum p e): off from o by
    sum p e (v - o) / (1 + sum p e), at most h / (1 - h) sum p |v - o|.  The other roundings as everywhere."""
    g = torch.Generator().manual_seed(page + d)
    n, t, Hq = 7 * page + 19, 90, 4
    k, v, q = (torch.randn(m, h, d, generator=g, dtype=torch.float64) for m, h in ((n, 1), (n, 1), (t, Hq)))
    k, v, q = k.to(dtype), (v + 0.5).to(dtype), (sharp * q).to(dtype)
    got = call(k, v, q, page, code, causal).double()
    kk, vv = (cached(x, page, code)[:, 0] for x in (k, v))
    qq, scaling, h = q.double(), d ** -0.5, HALF[dtype]
    seen = torch.arange(n)[None] <= (torch.arange(t)[:, None] + n - t if causal else n)
    s = (qq.reshape(-1, d) @ kk.T * scaling).view(t, Hq, n).masked_fill(~seen[:, None], -torch.inf)
    p = torch.softmax(s, -1)
    out, mass = p @ vv, p @ vv.abs()
    apart = torch.stack([(p[i].unsqueeze(-1) * (vv[None] - out[i].unsqueeze(1)).abs()).sum(1) for i in range(t)])
    score = (qq.abs().reshape(-1, d) @ kk.abs().T).view(t, Hq, n).masked_fill(~seen[:, None], 0.0).amax(-1, keepdim=True) * scaling
    tol = bound(out, mass, score, float(vv.abs().max()), n, d, dtype, 0.0) + (1 + h) * h / (1 - h) * apart
    worst = float(((got - out).abs() / tol).max())
    print(f"{worst:.3f} of the bound", flush=True)
    assert worst <= 1.0

"""Attention over pages where the value blocks' scales lie far apart or near the format's end, against the float64 oracle: both codes, every
page size, rows by the kernels of many and of few."""
import pytest
import torch

from attention_bounds import HALF, check
from oracle.paged import attend, cached

pytestmark = pytest.mark.gpu

# As in the tests of ordinary values: a weight is rounded by h, and so is the sum that divides by it, at most 2 h / (1 - h) of
# sum p |v|
WEIGHT = {t: 2 * h / (1 - h) for t, h in HALF.items()}


@pytest.fixture(params=[(0, 1), (0, 64), (1 << 30, 1)], ids=["cut", "whole", "16 rows"], autouse=True)
def heads(request, monkeypatch):
    """Tiles that are cut along the text, tiles that are not (64 KV heads of them fill the chip), the decode's kernels."""
    import kvq.paged
    monkeypatch.setattr(kvq.paged, "FEW_ROWS", request.param[0])
    monkeypatch.setattr(kvq.paged, "FEW_WORK", 1)
    return request.param[1]


class Text:
    """A text in one slot: blocks of `run` tokens with values of 2^e each, and scores near c; the same for all KV heads."""

    def __init__(self, exponents, scores, run, page, code, dtype, heads, rest=7, seed=0):
        import kvq
        d = 128 if page == 64 else 64
        g = torch.Generator().manual_seed(seed)
        self.n, self.d, self.page, self.code, self.dtype = len(exponents) * run + rest, d, page, code, dtype
        at = torch.arange(self.n)
        pick = lambda x: torch.tensor([*x, x[-1]], dtype=torch.float64)[at.clamp(max=len(exponents) * run) // run]
        self.u = torch.randint(0, 2, (1, d), generator=g).double() * 2 - 1
        # values up to twice the power of two, one of them in each block, so that a block's largest is known
        v = torch.rand(self.n, 1, d, generator=g, dtype=torch.float64) * 4 - 2
        v[at % 32 == 5, :, 3] = 2.0
        self.v = (v * torch.exp2(pick(exponents))[:, None, None]).to(dtype)
        self.k = ((pick(scores)[:, None] * self.u)[:, None] + 0.3 * torch.randn(self.n, 1, d, generator=g)).to(dtype)
        self.heads, self.rep = heads, 4 if heads == 1 else 8
        self.q = (self.u * (1 + 0.1 * torch.randn(self.n, heads * self.rep, 1, generator=g))).to(dtype)
        self.cache = kvq.PagedCache(1, 1, self.n // page + 1, self.n, heads, d, page=page, code=code, dtype=dtype)
        self.cache.append(0, *(x.cuda().expand(-1, heads, -1) for x in (self.k, self.v)), self.cache.extend([0], [self.n]))

    def check(self, rows, causal=True, what=""):
        """The last `rows` rows, those of each page against the largest value that they see; in units of it, so that the bound's
        floor for numbers near zero means what it does for ordinary ones."""
        import kvq
        n, page = self.n, self.page
        q = self.q[n - rows:]
        plan = kvq.PagedPlan(self.cache, [0], [rows], q.shape[1], causal=causal)
        out = kvq.paged_attention(q.cuda(), 1.0 / self.d, self.cache, 0, plan).cpu()
        assert torch.isfinite(out).all() and (self.heads == 1 or not plan.parts)
        some = [0, 1, 2, 3] if self.heads == 1 else [0, 3, q.shape[1] - 1]
        out, q = out[:, some], q[:, some]
        k, v = cached(self.k, page, self.code), cached(self.v, page, self.code)
        ref = attend(q, k, v, 1.0 / self.d, causal)
        for a in [0, *range(-(n - rows) % page or page, rows, page)]:
            b = min(rows, a + page - (n - rows + a) % page)
            mass = float(ref[1][a:b].max())
            unit = 2.0 ** -round(torch.log2(torch.tensor(mass)).item()) if self.dtype == torch.bfloat16 else 1.0
            got, (o, m, s) = out[a:b].double() * unit, (x[a:b] for x in ref)
            vmax = float(v[:n - rows + b].abs().max()) if causal else float(v.abs().max())
            check(got, (o * unit, m * unit, s), vmax * unit, n, self.d, self.dtype, WEIGHT[self.dtype], f"{what} rows {a}")


CODES = ["int8", "e4m3"]
PAGES = [32, 64, 128]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("dtype,small,big", [(torch.float16, -9, 14), (torch.float16, -6, 12), (torch.bfloat16, -60, 60), (torch.bfloat16, -70, 70)])
def test_large_values_that_a_row_does_not_see(dtype, small, big, page, code, heads):
    """Rows of a prompt in front of a block of far larger values, in the same unit and in the same tile: as exact as without it."""
    for at in (1, 2, 3, 4, 5):                 # the large block among six
        e = [big if i == at else small for i in range(6)]
        t = Text(e, [0] * 6, page, page, code, dtype, heads, seed=page + at)
        t.check(t.n, what=f"large block {at}")


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("e", [[83, 0, -63], [95, 30, -40, -85], [60, -80, 60, -80]], ids=str)
def test_values_that_fall_again_and_again(e, page, code, heads):
    """bf16 values that fall by more than 2^100 in several steps: sums of the large ones stay finite in units of the small."""
    bf16 = torch.bfloat16
    Text(e, [0] * len(e), 128, page, code, bf16, heads, seed=page).check(130, what="even")
    Text([e[0]] * 2 + e, [0] * 2 + [8.0] * len(e), 128, page, code, bf16, heads, seed=page + 1).check(130, what="heavier later")


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("e", [-94, -97, -103, -106])
def test_small_values(e, page, code, heads):
    """bf16 values down to where a block's codes are all zero, alone, between ordinary ones, and between ordinary ones that weigh nothing."""
    bf16 = torch.bfloat16
    Text([e] * 6, [0] * 6, 128, page, code, bf16, heads, seed=page).check(200, what="alone")
    Text([0, e, e, 0, e, 0, e], [0] * 7, 128, page, code, bf16, heads, seed=page + 1).check(200, what="between")
    t = Text([0, e, e, 0, e], [-60, 0, 0, -60, 0], 128, page, code, bf16, heads, rest=0, seed=page + 2)
    t.check(128, what="heavy between light")
    t.check(128, False, what="heavy between light")


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("e", [[100, 30, -40, -80, -105], [-100, 100, -100], [0, -130, 90, -130, -60]], ids=str)
def test_small_values_behind_large_ones(e, page, code, heads):
    """bf16 values up to 2^205 of the smallest, blocks whose codes are all zero."""
    bf16 = torch.bfloat16
    Text(e, [0] * len(e), 128, page, code, bf16, heads, seed=page).check(130, what="even")
    Text([e[0]] * 2 + e, [0] * 2 + [8.0] * len(e), 128, page, code, bf16, heads, seed=page + 1).check(130, what="heavier later")


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype,apart", [(torch.float16, 12), (torch.float16, 20), (torch.float16, 24), (torch.float16, 27), (torch.float16, 30),
                                         (torch.bfloat16, 60), (torch.bfloat16, 90), (torch.bfloat16, 99)])
def test_neighbours_that_share_a_unit(dtype, apart, code, heads):
    """Pages of 32 tokens whose values are 2^apart of each other's in one unit of 64, the small ones with nearly all of the weight: it counts
    in the softmax's sum whatever is left of it in the products."""
    big = 9 if dtype == torch.float16 else apart // 2
    for first in (0, 1):
        e = [big, big - apart] if first else [big - apart, big]
        for light in (-2.0, -5.0, -9.0):
            c = [light, 0] if first else [0, light]
            t = Text(e * 2, c * 2, 32, 32, code, dtype, heads, seed=apart + first)
            for causal in (True, False):
                t.check(128, causal, what=f"light {light}")


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("small,big", [(-60, 30), (-20, 70), (-94, 0)])
def test_neighbours_of_which_the_small_one_is_all(small, big, code, heads):
    """bf16, pages of 32 tokens in one unit, the far larger one of next to no weight, in front or behind."""
    for first in (0, 1):
        for light in (-25.0, -60.0, -90.0):
            e, c = ([big, small], [light, 0]) if first else ([small, big], [0, light])
            t = Text(e * 3, c * 3, 32, 32, code, torch.bfloat16, heads, rest=0 if first else 7, seed=first)
            t.check(64, causal=False, what=f"light {light}")
            t.check(32, what=f"light {light}")


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("small,big", [(-70, 70), (-80, 90)])
def test_tiles_over_the_border_of_a_large_block(small, big, page, code, heads):
    """bf16 rows of one tile on both sides of where a far larger block begins, the tile's units in even and odd numbers."""
    run = max(page, 64)
    for at in (1, 2, 3):
        t = Text([small] * at + [big], [0] * (at + 1), run, page, code, torch.bfloat16, heads, rest=0, seed=page + at)
        for offset in (8, 20):
            t.check(t.n - offset, what=f"large block {at}, rows from {offset}")

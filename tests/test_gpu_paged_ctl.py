"""The router over a paged cache: a prompt, single tokens, drafted tokens, a long question and a branch of one batch
through router_attention, against the float64 oracle over what the cache holds; and a small model through it."""
from types import SimpleNamespace

import pytest
import torch

from attention_bounds import HALF, check
from oracle.paged import attend, cached

pytestmark = pytest.mark.gpu
PAIR = 2.0 ** -17


class Served:
    def __init__(self, B, Hq, Hkv, d, layers, dtype, page=64, code="int8"):
        import kvq
        self.cache = kvq.PagedCache(layers, 2 * B, 60, 900, Hkv, d, page=page, code=code, dtype=dtype)
        self.ctl = kvq.PagedCtl(self.cache, range(B))
        self.g = torch.Generator().manual_seed(B + Hq)
        self.Hq, self.layers, self.dtype, self.d = Hq, layers, dtype, d
        empty = torch.empty((0, Hkv, d), dtype=dtype)
        self.k, self.v = ([[empty] * B for _ in range(layers)] for _ in (0, 1))

    def step(self, counts, T=None, what=""):
        import kvq
        from kvq.paged_ctl import MANY_ROWS
        n = self.ctl.slots
        c = [counts] * len(n) if isinstance(counts, int) else counts
        T = max(c) if T is None else T
        fresh = all(self.cache.length(s) == 0 for s in n)
        with kvq.routed(self.ctl):
            self.ctl.begin(counts)
            for l in range(self.layers):
                q, k, v = (torch.randn(len(n), h, T, self.d, generator=self.g).to(self.dtype)
                           for h in (self.Hq, self.cache.Hkv, self.cache.Hkv))
                out, none = kvq.router_attention(SimpleNamespace(layer_idx=l, scaling=self.d ** -0.5), q.cuda(), k.cuda(), v.cuda(), None)
                assert none is None and out.shape == (len(n), T, self.Hq, self.d) and out.dtype == self.dtype
                for b, m in enumerate(c):
                    assert not out[b, :T - m].any()
                    kk, vv = (x[b].transpose(0, 1)[T - m:] for x in (k, v))
                    self.k[l][b], self.v[l][b] = torch.cat([self.k[l][b], kk]), torch.cat([self.v[l][b], vv])
                    if m == 0:
                        continue
                    kk, vv = self.k[l][b], self.v[l][b]
                    if not fresh:
                        kk, vv = (cached(x, self.cache.page, self.cache.code) for x in (kk, vv))
                    # read back for prompt_attention the cache's rows are rounded once more: u of each key and value
                    many = not fresh and self.Hq // self.cache.Hkv * max(c) >= MANY_ROWS
                    if many:
                        kk, vv = kk.to(self.dtype), vv.to(self.dtype)
                    ref = attend(q[b].transpose(0, 1)[T - m:], kk, vv, self.d ** -0.5)
                    check(out[b, T - m:], ref, float(vv.abs().max()), kk.shape[0], self.d, self.dtype,
                          HALF[self.dtype] if fresh or many else PAIR, f"{what} layer {l} sequence {b}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_batch_through_the_router(dtype):
    s = Served(3, 8, 2, 64, 2, dtype)
    s.step([70, 131, 64], what="prompt")                     # padded on the left to 131
    s.step(1, what="token")
    s.step(3, what="drafts")
    s.step([1, 0, 2], T=4, what="uneven")
    s.step(33, what="question")
    s.step([60, 49, 1], what="long question")
    s.step(1, what="token")


def test_refusals():
    import kvq
    cache = kvq.PagedCache(1, 2, 10, 300, 2, 64)
    ctl = kvq.PagedCtl(cache, [0, 1])
    q, k = torch.zeros((2, 4, 3, 64), dtype=torch.bfloat16, device="cuda"), torch.zeros((2, 2, 3, 64), dtype=torch.bfloat16, device="cuda")
    m = SimpleNamespace(layer_idx=0, scaling=0.1)
    with pytest.raises(RuntimeError, match="begin"):
        ctl.attend(m, q, k, k, None, {})
    with pytest.raises(ValueError, match="counts"):
        ctl.begin([1])
    ctl.begin(4)
    with pytest.raises(ValueError, match="new tokens"):
        ctl.attend(m, q, k, k, None, {})
    with pytest.raises(kvq.KVQError, match="exhausted"):
        ctl.begin(400)
    with pytest.raises(RuntimeError, match="begin"):
        ctl.attend(m, q, k, k, None, {})
    with pytest.raises(IndexError):
        kvq.PagedCtl(cache, [5]).begin(1)


def test_a_model_through_the_router():
    """A small model with random weights: its logits through the paged cache are near those through SDPA, prompt and
    decoded tokens, and a branch of the sequence continues like the sequence itself."""
    import kvq
    from transformers import LlamaConfig, LlamaForCausalLM
    name = kvq.register()
    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=97, hidden_size=256, intermediate_size=320, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=64, max_position_embeddings=512)
    models = [LlamaForCausalLM._from_config(cfg, attn_implementation=a, dtype=torch.bfloat16).cuda().eval() for a in ("sdpa", name)]
    models[1].load_state_dict(models[0].state_dict())
    ids = torch.randint(0, 97, (2, 150), device="cuda")
    cache = kvq.PagedCache(2, 4, 12, 300, 2, 64, page=32)
    ctl = kvq.PagedCtl(cache, [0, 1])
    with torch.no_grad():
        want = models[0](input_ids=ids, use_cache=False).logits.float()
        got = []
        with kvq.routed(ctl):
            for a, b in ((0, 140), (140, 141), (141, 145), (145, 150)):
                ctl.begin(b - a)
                pos = torch.arange(a, b, device="cuda").expand(2, -1)
                got.append(models[1](input_ids=ids[:, a:b], position_ids=pos, use_cache=False).logits.float())
            cache.fork([0, 1], [2, 3])
            nxt, pos = ids[:, :1], torch.full((2, 1), 150, device="cuda")
            ctl.begin(1)
            one = models[1](input_ids=nxt, position_ids=pos, use_cache=False).logits
            other = kvq.PagedCtl(cache, [2, 3])
            with kvq.routed(other):
                other.begin(1)
                two = models[1](input_ids=nxt, position_ids=pos, use_cache=False).logits
    got = torch.cat(got, 1)
    assert torch.equal(one, two)
    assert torch.isfinite(got).all() and got.shape == want.shape
    print("logits: largest difference", float((got - want).abs().max()), "of", float(want.abs().max()))


def test_a_forward_pass_without_begin():
    """A layer that comes a second time in a step is refused, and the step's rows stay; begin claims the next one."""
    import kvq
    cache = kvq.PagedCache(2, 2, 10, 300, 2, 64)
    ctl = kvq.PagedCtl(cache, [0, 1])
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(2, h, 3, 64, generator=g).bfloat16().cuda() for h in (4, 2, 2))
    layers = [SimpleNamespace(layer_idx=l, scaling=0.125) for l in (0, 1)]
    for _ in range(2):
        ctl.begin(3)
        with pytest.raises(ValueError):
            ctl.attend(layers[0], q[:, :, :2], k[:, :, :2], v[:, :, :2], None, {})
        for m in layers:                       # the one that was refused has not come yet
            ctl.attend(m, q, k, v, None, {})
        held = [x.clone() for l in (0, 1) for x in cache.rows(l, [0, 1])]
        for m in layers:
            with pytest.raises(RuntimeError, match="begin"):
                ctl.attend(m, q, -k, -v, None, {})
        assert all(torch.equal(a, b) for a, b in zip(held, [x for l in (0, 1) for x in cache.rows(l, [0, 1])]))
    assert cache.lengths == [6, 6]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts", [[1, 70, 0, 131], [1, 5, 0, 6], [60, 33, 2, 8], [0, 70, 0, 3]])
def test_prompts_that_begin_beside_running_sequences(counts, dtype):
    """A prompt attends its own exact keys, whoever else is in the batch; the running sequences attend what the cache holds."""
    import kvq
    from kvq.paged_ctl import MANY_ROWS
    Hq, Hkv, d = 8, 2, 64
    cache = kvq.PagedCache(1, 4, 40, 500, Hkv, d, page=32, dtype=dtype)
    ctl = kvq.PagedCtl(cache, [3, 0, 1, 2])    # slots 3 and 1 hold tokens when the others begin
    g = torch.Generator().manual_seed(5)
    rand = lambda T: tuple(torch.randn(4, h, T, d, generator=g).to(dtype) for h in (Hq, Hkv, Hkv))
    m = SimpleNamespace(layer_idx=0, scaling=0.125)
    first = [90, 0, 40, 0]
    held = []
    for c in (first, counts):
        T = max(c)
        q, k, v = rand(T)
        ctl.begin(c)
        out, _ = ctl.attend(m, q.cuda(), k.cuda(), v.cuda(), None, {})
        held.append((k, v))
    many = Hq // Hkv * max(counts) >= MANY_ROWS
    for b, n in enumerate(counts):
        if n == 0:
            continue
        kk, vv = (x[b].transpose(0, 1)[T - n:] for x in (k, v))
        if first[b]:
            kk, vv = (cached(torch.cat([x[b].transpose(0, 1)[90 - first[b]:], y]), 32, "int8") for x, y in zip(held[0], (kk, vv)))
            if many:
                kk, vv = kk.to(dtype), vv.to(dtype)
        weight = PAIR if first[b] and not many else HALF[dtype]
        check(out[b, T - n:], attend(q[b].transpose(0, 1)[T - n:], kk, vv, 0.125), float(vv.abs().max()), kk.shape[0], d, dtype,
              weight, f"sequence {b}: {n} behind {first[b]}")
        assert not out[b, :T - n].any()

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


class Kept:
    """The router's controller as it should be, on the CPU: every step attends over what a paged cache holds by then, the first one
    over its own keys.  ``mistake``: one that the comparison has to see."""

    def __init__(self, page, mistake=None, dtype=torch.bfloat16):
        self.page, self.mistake, self.dtype, self.held = page, mistake, dtype, {}

    def attend(self, module, q, k, v, mask, kwargs):
        kv = [x.to(self.dtype).transpose(1, 2) for x in (k, v)]        # (B, T, H, d)
        layer = module.layer_idx
        if self.mistake == "layer" and layer in self.held:
            layer = 1 - layer
        first = layer not in self.held
        past = [] if first else self.held[layer]
        self.held[layer] = kv = kv if first else [torch.cat(x, 1) for x in zip(past, kv)]
        out = []
        for b in range(q.shape[0]):
            kk, vv = (x[b].double() if first else cached(x[b], self.page, "int8") for x in kv)
            if self.mistake == "heads":
                kk, vv = kk.flip(1), vv.flip(1)
            if self.mistake == "offset" and not first:
                kk, vv = kk[:-1], vv[:-1]
            scaling = module.scaling * (0.5 if self.mistake == "scaling" else 1.0)
            out.append(attend(q[b].transpose(0, 1), kk, vv, scaling)[0])
        return torch.stack(out).to(q.dtype), None


def test_a_models_logits_through_the_router():
    """The logits of a small bf16 model through the paged cache, prompt and later steps, lie as near those of the same weights in
    float32 with attention in 64 bits as the logits of bf16 arithmetic with SDPA do: both carry the same roundings, so within
    twice their largest distance.  Mistakes move the logits by four times that and more."""
    import kvq
    name = kvq.register()
    exact_sdpa, exact = (x.float() for x in _small_models(name))
    ids = torch.randint(0, 97, (2, 150), generator=torch.Generator().manual_seed(7))
    cuts = ((0, 140), (140, 141), (141, 145), (145, 150))

    def steps(model, ctl, device):
        logits = []
        with torch.no_grad(), kvq.routed(ctl):
            for a, b in cuts:
                if hasattr(ctl, "begin"):
                    ctl.begin(b - a)
                pos = torch.arange(a, b, device=device).expand(2, -1)
                logits.append(model(input_ids=ids[:, a:b].to(device), position_ids=pos, use_cache=False).logits.double().cpu())
        return torch.cat(logits, 1)

    with torch.no_grad():
        plain = exact_sdpa(input_ids=ids, use_cache=False).logits.double()
    # the oracle's prompt is SDPA's, where it keeps float32 keys and values
    assert float((steps(exact, Kept(32, dtype=torch.float32), "cpu") - plain)[:, :140].abs().max()) < 1e-4
    want = steps(exact, Kept(32), "cpu")
    whole, parts = (x.cuda() for x in _small_models(name))
    with torch.no_grad():
        near = whole(input_ids=ids.cuda(), use_cache=False).logits.double().cpu()
    got = steps(parts, kvq.PagedCtl(kvq.PagedCache(2, 2, 12, 300, 2, 64, page=32), [0, 1]), "cuda")
    noise = float((near - plain).abs().max())
    first, later = (float((got - want)[:, s].abs().max()) for s in (slice(0, 140), slice(140, 150)))
    print(f"bf16 arithmetic {noise:.4f}, prompt {first:.4f}, later steps {later:.4f}")
    assert max(first, later) <= 2 * noise
    for mistake in ("layer", "heads", "offset", "scaling"):            # what these bounds can tell
        wrong = float((steps(exact, Kept(32, mistake), "cpu") - want)[:, 140:].abs().max())
        print(f"{mistake}: {wrong:.4f}")
        assert wrong > 4 * noise, mistake


def _small_models(name):
    from transformers import LlamaConfig, LlamaForCausalLM
    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=97, hidden_size=256, intermediate_size=320, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=64, max_position_embeddings=512, initializer_range=0.05)
    models = [LlamaForCausalLM._from_config(cfg, attn_implementation=a, dtype=torch.bfloat16).eval() for a in ("sdpa", name)]
    models[1].load_state_dict(models[0].state_dict())
    return models


def test_a_step_run_again_and_captured():
    """A step's pass repeated on purpose, then captured; its replays run the steps that are written into it."""
    import kvq
    cache = kvq.PagedCache(1, 2, 20, 300, 2, 64, page=32)
    ctl = kvq.PagedCtl(cache, [0, 1])
    m = SimpleNamespace(layer_idx=0, scaling=0.125)
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda T: [torch.randn(2, h, T, 64, generator=g, device="cuda").bfloat16() for h in (4, 2, 2)]
    ctl.begin([70, 33])
    ctl.attend(m, *rand(70), None, {})
    ctl.begin(1)
    q, k, v = rand(1)
    first, _ = ctl.attend(m, q, k, v, None, {})
    ctl.seen.clear()
    again, _ = ctl.attend(m, q, k, v, None, {})
    assert torch.equal(first, again)
    ctl.seen.clear()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out, _ = ctl.attend(m, q, k, v, None, {})
    for i in range(4):
        if i:
            cache.extend([0, 1], [1, 1], into=ctl.step)
            for x, y in zip((q, k, v), rand(1)):
                x.copy_(y)
        _ = (q.float() * 2).sum()
        gr.replay()
        torch.cuda.synchronize()
        want = kvq.paged_decode(q.transpose(1, 2).reshape(2, 4, 64), 0.125, cache, 0, ctl.step)
        assert torch.equal(out.view(2, 4, 64), want), i
        kk, vv = cache.rows(0, [0, 1])
        assert torch.equal(kk[70 + i], k[0, :, 0]) and torch.equal(vv[-1], v[1, :, 0])
    assert cache.lengths == [74, 37]

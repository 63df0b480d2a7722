"""GPU tests of decoding from a paged cache through the decoder
(MixtralDecoder.forward_paged, generate_paged): the logits of ragged steps against the same
texts alone in a dense cache, and the loop around them.

Bar on fp16 logits: |got - ref| <= 3e-2 + 1e-2 |ref|, the decoder tests' bar: the two
passes run different kernels (experts by numbers of rows, attention with and without fp16
scores), whose roundings compound over the layers."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
V = 512


@pytest.fixture(scope="module")
def model():
    from hydranet_amd.model.decoder import MixtralDecoderConfig, build_synthetic_decoder
    cfg = MixtralDecoderConfig(num_layers=2, hidden_dim=512, intermediate_dim=1024,
                               num_attention_heads=8, num_kv_heads=2, head_dim=128,
                               vocab_size=V, num_experts=8, experts_per_token=2,
                               max_position_embeddings=256)
    return build_synthetic_decoder(cfg, DEV, decode_top_k=2, seed=3)


def _prompts(lengths, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, V, (n,), generator=g).tolist() for n in lengths]


def _alone(model, text):
    """The logits after each token of one text, from a dense cache."""
    ids = torch.tensor([text], device=DEV)
    return model.forward(ids, model.new_cache(1, -(-len(text) // 8) * 8), top_k=2)[0].float()


def _close(got, want):
    err = (got.float() - want.float()).abs()
    # (a router's near-tie may fall either way at a few rows)
    assert not err.numel() or \
        float((err <= 3e-2 + 1e-2 * want.float().abs()).float().mean()) >= 0.98


def test_ragged_steps_equal_each_text_alone(model):
    """Prompts of several lengths in one step, then a chunk of some beside single tokens of
    others, then one token each."""
    from hydranet_amd.model.paged import PagedBatch, PagedKVCache
    texts = _prompts([90, 7, 40, 130])
    want = [_alone(model, t) for t in texts]
    cache = PagedKVCache(2, 40, 2, 128, 16, DEV)
    table = cache.table([cache.take(cache.pages_for(len(t))) for t in texts])
    at = [0] * 4
    for step in ([50, 6, 1, 64], [39, 1, 10, 65], None, [0, 0, 28, 0]):
        lens = torch.tensor(at if step else [a if a < len(t) else -1 for a, t in zip(at, texts)],
                            device=DEV)
        m = step or [1] * 4
        rows = [t[a:a + n] + [0] * (n - len(t[a:a + n])) for t, a, n in zip(texts, at, m)]
        flat = torch.tensor(sum(rows, []), device=DEV)
        if step is None:
            one = PagedBatch(table, lens, 130)
        else:
            starts = torch.tensor([0] + m, device=DEV).cumsum(0).int()
            one = PagedBatch(table, lens, 130, starts, sum(m), max(m))
        logits = model.forward_paged(flat, one, cache, top_k=2)
        row = 0
        for b in range(4):
            n = min(m[b], len(texts[b]) - at[b])
            _close(logits[row:row + n], want[b][at[b]:at[b] + n])
            row += m[b]
            at[b] += n
    assert at == [90, 7, 40, 130]


def test_int4_projections():
    """The same with the attention's projections in INT4, stacked into one launch."""
    from hydranet_amd.model.decoder import (MixtralDecoderConfig, build_synthetic_decoder,
                                            convert_dense_to_int4)
    from hydranet_amd.model.paged import PagedBatch, PagedKVCache
    cfg = MixtralDecoderConfig(num_layers=2, hidden_dim=512, intermediate_dim=1024,
                               num_attention_heads=8, num_kv_heads=2, head_dim=128, vocab_size=V,
                               num_experts=8, experts_per_token=2, max_position_embeddings=256)
    m = convert_dense_to_int4(build_synthetic_decoder(cfg, DEV, decode_top_k=2, seed=4))
    texts = _prompts([30, 12])
    cache = PagedKVCache(2, 8, 2, 128, 16, DEV)
    table = cache.table([cache.take(2), cache.take(1)])
    starts = torch.tensor([0, 30, 42], dtype=torch.int32, device=DEV)
    one = PagedBatch(table, torch.zeros(2, dtype=torch.int64, device=DEV), 30, starts, 42, 30)
    got = m.forward_paged(torch.tensor(sum(texts, []), device=DEV), one, cache, 2)
    _close(got, torch.cat([_alone(m, t) for t in texts]))


def test_logits_of_chosen_rows(model):
    from hydranet_amd.model.paged import PagedBatch, PagedKVCache
    texts = _prompts([20, 33])
    cache = PagedKVCache(2, 8, 2, 128, 16, DEV)
    table = cache.table([cache.take(2), cache.take(3)])
    starts = torch.tensor([0, 20, 53], dtype=torch.int32, device=DEV)
    one = PagedBatch(table, torch.zeros(2, dtype=torch.int64, device=DEV), 33, starts, 53, 33)
    flat = torch.tensor(sum(texts, []), device=DEV)
    last = torch.tensor([52, 19], device=DEV)
    some = model.forward_paged(flat, one, cache, 2, last)
    assert tuple(some.shape) == (2, V)
    _close(some, model.forward_paged(flat, one, cache, 2)[last])


def _check_greedy(model, prompts, out, samples=1):
    """Every token is a largest logit of a plain pass over the text, within the bar."""
    for i, tokens in enumerate(out):
        p = prompts[i % len(prompts)]
        lg = _alone(model, p + tokens[:-1])[len(p) - 1:]
        chosen, top = lg.gather(1, torch.tensor(tokens, device=DEV)[:, None])[:, 0], lg.amax(1)
        ok = chosen >= top - 2 * (3e-2 + 1e-2 * top.abs())
        assert float(ok.float().mean()) >= 0.9, (i, ok.tolist())


@pytest.mark.parametrize("graph", [True, False])
@pytest.mark.parametrize("samples,options", [
    (1, {}), (3, {"page_size": 32}), (1, {"max_batch": 2}), (2, {"chunk": 10, "max_batch": 3})])
def test_generate_greedy(model, graph, samples, options):
    prompts = _prompts([5, 64, 33, 1, 100])
    out = model.generate_paged(prompts, 12, samples=samples, graph=graph, **options)
    assert len(out) == 5 * samples and all(len(t) == 12 for t in out)
    _check_greedy(model, prompts, out)


def test_generate_from_few_pages(model):
    """Texts wait for pages; all come back."""
    from hydranet_amd.model.paged import PagedKVCache
    prompts = _prompts([40, 50, 30, 60, 16])
    cache = PagedKVCache(2, 9, 2, 128, 16, DEV)
    mine = cache.take(2)
    out = model.generate_paged(prompts, 9, cache=cache, samples=2)
    assert cache.free_pages == 7
    cache.give(mine)
    _check_greedy(model, prompts, out)
    with pytest.raises(RuntimeError, match="KV cache full"):
        model.generate_paged(_prompts([20, 150]), 9, cache=cache)
    assert cache.free_pages == 9


def test_generate_stops_and_samples(model):
    prompts = _prompts([9, 30])
    g = torch.Generator(device=DEV).manual_seed(5)
    out = model.generate_paged(prompts, 40, temperature=1.0, samples=8, generator=g,
                               stop=range(0, V, 10))
    for t in out:
        assert all(x % 10 for x in t[:-1]) and (t[-1] % 10 == 0 or len(t) == 40)
    assert len({tuple(t) for t in out}) == 16  # (its own uniforms for each sample)
    g.manual_seed(5)
    assert out == model.generate_paged(prompts, 40, temperature=1.0, samples=8, generator=g,
                                       stop=range(0, V, 10))


def test_generate_with_penalties_and_grammar(model):
    prompts = _prompts([9, 30, 70])
    # a presence penalty above any logit's spread: no token twice
    out = model.generate_paged(prompts, 30, presence=1e3)
    assert all(len(set(t)) == 30 for t in out)
    # frequency: all of 8 tokens in turn, when a bias leaves only those
    out = model.generate_paged(prompts, 16, frequency=1e3, bias={i: 1e4 for i in range(8)})
    assert all(sorted(t) == sorted(list(range(8)) * 2) for t in out)
    out = model.generate_paged(prompts, 5, bias={7: 1e4})
    assert out == [[7] * 5] * 3

    def grammar(text):
        """The token after the last one, modulo the vocabulary; anything at first."""
        if text in prompts:
            return None
        t = (text[-1] + 1) % V
        w = torch.zeros(V // 32, dtype=torch.int64)
        w[t // 32] = 1 << t % 32
        return torch.where(w >= 2 ** 31, w - 2 ** 32, w).int()
    for graph in (True, False):
        out = model.generate_paged(prompts, 9, allowed=grammar, samples=2, graph=graph)
        assert all(t == [(t[0] + i) % V for i in range(9)] for t in out)
    from hydranet_amd.model.paged import PagedKVCache
    cache = PagedKVCache(2, 20, 2, 128, 16, DEV)
    with pytest.raises(RuntimeError, match="no logit is finite"):
        model.generate_paged(prompts, 9, cache=cache,
                             allowed=lambda text: torch.zeros(V // 32, dtype=torch.int32))
    assert cache.free_pages == 20


@pytest.mark.parametrize("P,n", [(250, 7), (256, 1), (200, 57)])
def test_generate_up_to_the_models_last_position(model, P, n):
    prompts = _prompts([P, 3])
    out = model.generate_paged(prompts, n)
    _check_greedy(model, prompts, out)
    with pytest.raises(AssertionError, match="256 positions"):
        model.generate_paged(prompts, n + 1)


def test_generate_refuses(model):
    for kw in (dict(prompts=[[]]), dict(prompts=[[V]]), dict(prompts=[[-1]]),
               dict(max_new_tokens=0), dict(samples=0), dict(samples=65), dict(chunk=0)):
        a = dict(prompts=[[1, 2]], max_new_tokens=3)
        a.update(kw)
        with pytest.raises(AssertionError):
            model.generate_paged(**a)
    assert model.generate_paged([], 3) == []


def test_a_position_past_the_angles(model):
    """A row whose position is past the angles is NaN in its own logits alone."""
    from hydranet_amd.model.paged import PagedBatch, PagedKVCache
    cache = PagedKVCache(2, 40, 2, 128, 16, DEV)
    table = cache.table([cache.take(18), cache.take(18)])
    lens = torch.tensor([256, 10], device=DEV)
    logits = model.forward_paged(torch.tensor([3, 4], device=DEV), PagedBatch(table, lens, 257),
                                 cache)
    assert not math.isfinite(float(logits[0].sum())) and logits[1].isfinite().all()

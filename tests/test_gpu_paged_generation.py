"""GPU tests of paged steps and generation place by place: the first and last rows of every
run, every token index over many texts, so that a fault at one place of every text shows.

The bar on a logit is the decoder tests' (3e-2 + 1e-2 of it: other kernels, whose roundings
compound over the layers); a router's near-tie may fall the other way at a row, about one
in fifty, so a place may miss the bar in one text of eight."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
V = 512


def _model(device, seed=3):
    from hydranet_amd.model.decoder import MixtralDecoderConfig, build_synthetic_decoder
    cfg = MixtralDecoderConfig(num_layers=2, hidden_dim=512, intermediate_dim=1024,
                               num_attention_heads=8, num_kv_heads=2, head_dim=128,
                               vocab_size=V, num_experts=8, experts_per_token=2,
                               max_position_embeddings=256)
    return build_synthetic_decoder(cfg, device, decode_top_k=2, seed=seed)


@pytest.fixture(scope="module")
def model():
    return _model(DEV)


def _prompts(lengths, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, V, (n,), generator=g).tolist() for n in lengths]


def _alone(model, text):
    ids = torch.tensor([text], device=DEV)
    return model.forward(ids, model.new_cache(1, -(-len(text) // 8) * 8), top_k=2)[0].float()


def _few(missed, n, what):
    assert missed <= n // 8, f"{what}: {missed} of {n} miss the bar"


@pytest.mark.parametrize("page", [16, 64])
def test_first_and_last_rows_of_runs(model, page):
    """16 texts in four steps: chunks, then single tokens, then what is left."""
    from hydranet_amd.model.paged import PagedBatch, PagedKVCache
    lengths = [20 + 11 * i for i in range(16)]
    texts = _prompts(lengths, 2)
    want = [_alone(model, t) for t in texts]
    cache = PagedKVCache(2, 16 * 13, 2, 128, page, DEV)
    table = cache.table([cache.take(cache.pages_for(n)) for n in lengths])
    at = [0] * 16
    for step in (0.4, 0.3, None, 1.0):
        m = [1 if step is None else max(1, int(step * (n - a))) for n, a in zip(lengths, at)]
        lens = torch.tensor(at, device=DEV)
        flat = torch.tensor(sum([t[a:a + n] for t, a, n in zip(texts, at, m)], []), device=DEV)
        starts = torch.tensor([0] + m, device=DEV).cumsum(0).int()
        one = PagedBatch(table, lens, 200) if step is None else \
            PagedBatch(table, lens, 200, starts, sum(m), max(m))
        logits = model.forward_paged(flat, one, cache, top_k=2).float()
        first = last = row = 0
        for b in range(16):
            w = want[b][at[b]:at[b] + m[b]]
            ok = ((logits[row:row + m[b]] - w).abs() <= 3e-2 + 1e-2 * w.abs()).float().mean(1)
            first, last = first + int(ok[0] < 0.95), last + int(ok[-1] < 0.95)
            row += m[b]
            at[b] += m[b]
        _few(first, 16, f"first rows of step {step}")
        _few(last, 16, f"last rows of step {step}")
    assert at == lengths


@pytest.mark.parametrize("graph", [True, False])
@pytest.mark.parametrize("samples,options", [
    (1, {}), (3, {"page_size": 32}), (1, {"max_batch": 5}), (2, {"chunk": 50, "max_batch": 9})])
def test_every_token_index(model, graph, samples, options):
    """Greedy texts: each token a largest logit of a plain pass over what is before it, at
    every index and in every sample."""
    prompts = _prompts([1 + 5 * i for i in range(16)] + [16, 32, 48, 64, 96, 15, 17, 65], 4)
    n = 10
    out = model.generate_paged(prompts, n, samples=samples, graph=graph, **options)
    assert len(out) == 24 * samples and all(len(t) == n for t in out)
    missed = torch.zeros(samples, n, dtype=torch.int64)
    for i, tokens in enumerate(out):
        p = prompts[i % 24]
        lg = _alone(model, p + tokens[:-1])[len(p) - 1:]
        chosen = lg.gather(1, torch.tensor(tokens, device=DEV)[:, None])[:, 0]
        top = lg.amax(1)
        ok = chosen >= top - 2 * (3e-2 + 1e-2 * top.abs())
        missed[i // 24] += (~ok).cpu().long()
    for s in range(samples):
        for i in range(n):
            _few(int(missed[s, i]), 24, f"sample {s}, token {i}")

@pytest.mark.parametrize("shape", [(1,), (1, V // 32), (V // 32 + 1,)])
@pytest.mark.parametrize("first", [True, False])
def test_words_of_another_number_are_refused(model, shape, first):
    """Of the first token and of a later one (where one word stood for all the others)."""
    from hydranet_amd.model.paged import PagedKVCache
    cache = PagedKVCache(2, 6, 2, 128, 16, DEV)
    prompt = _prompts([9])[0]

    def allowed(text):
        return None if not first and text == prompt else torch.full(shape, -1, dtype=torch.int32)
    with pytest.raises(AssertionError, match="allowed"):
        model.generate_paged([prompt], 5, allowed=allowed, cache=cache)
    assert cache.free_pages == 6


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_a_model_on_another_device_than_the_current_one():
    """The decode step's graph is captured where the model is."""
    model = _model(torch.device("cuda:1"))
    prompts = _prompts([9, 30], 6)
    assert torch.cuda.current_device() == 0
    out = model.generate_paged(prompts, 8)
    with torch.cuda.device(1):
        assert out == model.generate_paged(prompts, 8, graph=False)

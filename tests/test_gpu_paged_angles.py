"""GPU tests of what a decoder keeps between paged steps (the angles' table, the stacked
projections): first steps inside a capture, angles changed afterwards, weights that record
no changes."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
V = 512


def _model(seed=3):
    from hydranet_amd.model.decoder import MixtralDecoderConfig, build_synthetic_decoder
    cfg = MixtralDecoderConfig(num_layers=1, hidden_dim=512, intermediate_dim=1024,
                               num_attention_heads=8, num_kv_heads=2, head_dim=128,
                               vocab_size=V, num_experts=8, experts_per_token=2,
                               max_position_embeddings=256)
    return build_synthetic_decoder(cfg, DEV, decode_top_k=2, seed=seed)


def _step(model):
    """A step of two texts over pages of random numbers: a call that gives its logits."""
    from hydranet_amd.model.paged import PagedBatch, PagedKVCache
    cache = PagedKVCache(1, 10, 2, 128, 16, DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    for t in cache.k + cache.v:
        t.normal_(generator=g)
    table = cache.table([cache.take(5), cache.take(3)])
    lens, tokens = torch.tensor([70, 31], device=DEV), torch.tensor([5, 77], device=DEV)
    batch = PagedBatch(table, lens, 80)
    return lambda: model.forward_paged(tokens, batch, cache)


def test_first_step_inside_a_capture():
    want = _step(_model())()  # (also: library handles)
    model = _model()
    step = _step(model)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    eager = step()  # before the first replay
    assert torch.equal(eager, want)
    for _ in range(3):
        held.zero_()
        graph.replay()
        assert torch.equal(held, want) and torch.equal(step(), want)


def test_angles_changed_after_a_capture():
    model = _model()
    step = _step(model)
    first = step().clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.no_grad():
        model.rotary.cos_cached.copy_(model.rotary.cos_cached.flip(0))
        model.rotary.sin_cached.copy_(model.rotary.sin_cached.flip(0))
    other = step().clone()
    assert not torch.equal(other, first)
    junk = [torch.full((256, 64), 9.0, device=DEV) for _ in range(8)]  # (where a table was)
    for _ in range(3):
        graph.replay()
        assert torch.equal(held, other) and torch.equal(step(), other)
    del junk


@pytest.mark.parametrize("inside", [True, False])
def test_weights_made_in_inference_mode(inside):
    """Tensors that record no changes: nothing made of them is kept."""
    want = _step(_model())()
    with torch.inference_mode():
        model = _model()
    with torch.inference_mode(inside):
        step = _step(model)
        assert torch.equal(step(), want) and torch.equal(step(), want)
    with torch.inference_mode():
        model.rotary.cos_cached.neg_()
        other = _step(model)()
    assert not torch.equal(other, want)


def test_a_model_used_inside_and_outside_of_inference_mode():
    model = _model()
    with torch.inference_mode():
        want = _step(model)()
    assert torch.equal(_step(model)(), want)
    model.rotary.cos_cached.neg_()
    assert not torch.equal(_step(model)(), want)

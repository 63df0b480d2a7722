"""GPU tests of generation from a paged cache."""
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


def _prompts(lengths, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, V, (n,), generator=g).tolist() for n in lengths]


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_a_model_on_another_device_than_the_current_one():
    """The decode step's graph is captured where the model is."""
    model = _model(torch.device("cuda:1"))
    prompts = _prompts([9, 30], 6)
    assert torch.cuda.current_device() == 0
    out = model.generate_paged(prompts, 8)
    with torch.cuda.device(1):
        assert out == model.generate_paged(prompts, 8, graph=False)

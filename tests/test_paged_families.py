"""The paged decoder against HF models of each family that it runs, dense and
random, with windows and scaled frequencies (GPU)."""

import pytest
import torch

pytestmark = pytest.mark.gpu

TINY = dict(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=4, num_attention_heads=4,
            num_key_value_heads=2, max_position_embeddings=256, pad_token_id=0, bos_token_id=1, eos_token_id=2)
LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 32, "rope_theta": 1e4}
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64, "mscale": 1.0, "mscale_all_dim": 0.3,
        "rope_theta": 1e4}
# Either side rounds some 20 times per layer to fp16 (2^-11 of the residual's
# size, in no order): 4 layers, 4 standard deviations.
TOL = 4 * (4 * 20) ** 0.5 * 2.0 ** -11


@pytest.mark.parametrize("family,kw", [
    ("llama", {}), ("llama", {"attention_bias": True, "mlp_bias": True, "rope_scaling": LLAMA3}), ("llama", {"rope_scaling": YARN}),
    ("mistral", {"sliding_window": 6}), ("mistral", {"sliding_window": None}),
    ("qwen2", {"use_sliding_window": True, "sliding_window": 6, "max_window_layers": 2}),
    ("qwen3", {"use_sliding_window": True, "sliding_window": 6, "max_window_layers": 1, "head_dim": 64})])
def test_logits_match_the_hf_model(cuda, family, kw):
    from transformers import AutoConfig, AutoModelForCausalLM
    from turbopress_amd.paged_decode import PagedDecoder
    torch.manual_seed(5)
    model = AutoModelForCausalLM.from_config(AutoConfig.for_model(family, **TINY, **kw))
    for p in model.parameters():  # (scores and outputs of a size that positions and windows show in)
        p.data.mul_(4) if p.dim() > 1 else p.data.add_(0.1 * torch.randn_like(p))
    model = model.half().to(cuda).eval()
    dec = PagedDecoder(model, 2, 64, page_size=16, fp8_head=False)
    prompts = [torch.randint(0, 512, (n,), device=cuda) for n in (21, 4)]

    def near(logits, tokens):
        with torch.inference_mode():
            want = model(input_ids=tokens[None], use_cache=False).logits[0, -1].float()
        assert (logits.float() - want).abs().max() <= TOL * want.abs().max()

    for s, p in enumerate(prompts):
        near(dec.prefill(s, p)[0], p)
        dec.cache.reserve(s, len(p) + 4)
    for i in range(4):
        prompts = [torch.cat((p, dec.tokens[s:s + 1])) for s, p in enumerate(prompts)]
        logits = dec.step(graph=i % 2 == 1)
        for s, p in enumerate(prompts):
            near(logits[s], p)

"""The paged decoder against the HF decoder over its own cache, on a small
random packed model (GPU)."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(cuda, tmp_path_factory):
    from turbopress_amd.artifact import load_packed_model
    from turbopress_amd.synthetic import tiny_qwen3_config, write_synthetic_artifact
    root = tmp_path_factory.mktemp("tiny")
    write_synthetic_artifact(root, tiny_qwen3_config(), bits=3, seed=3)
    return load_packed_model(root, device="cuda", mode="hip")[0]


def _prompts(lengths):
    g = torch.Generator().manual_seed(1)
    return [torch.randint(0, 1024, (n,), generator=g).cuda() for n in lengths]


@torch.inference_mode()
def _hf_logits(model, tokens):
    return model(input_ids=tokens[None], use_cache=False).logits[0, -1].float()


def _near(got, want, tol):
    assert (got.float() - want).abs().max() <= tol * want.abs().max()


# Either side rounds some 20 times per layer to fp16 (2^-11 of the residual's
# size, in no order): 2 layers, 4 standard deviations.
TOL = 4 * (2 * 20) ** 0.5 * 2.0 ** -11
# The 8-bit head: codes and weights off by up to 2^-4 of themselves, 256 terms of
# either sign; a sixth of that bound for each (an even spread is 2^-4 / sqrt(12)
# at most), 5 standard deviations of their sum over the largest of 1024 logits
# (3 standard deviations of a logit)
TOL8 = TOL + 5 * (2 * (2.0 ** -4) ** 2 / 12) ** 0.5 / 3


@pytest.mark.parametrize("fp8_head,tol", [(False, TOL), (True, TOL8)])
def test_logits_match_the_hf_decoder(model, fp8_head, tol):
    from turbopress_amd.paged_decode import PagedDecoder
    prompts = _prompts([5, 40, 1, 17])
    dec = PagedDecoder(model, 5, 64, page_size=16, fp8_head=fp8_head)
    for s, p in enumerate(prompts):
        _near(dec.prefill(s, p)[0], _hf_logits(model, p), tol)
        dec.cache.reserve(s, len(p) + 4)
    for i in range(4):
        prompts = [torch.cat((p, dec.tokens[s:s + 1])) for s, p in enumerate(prompts)]
        logits = dec.step(graph=i % 2 == 1)
        for s, p in enumerate(prompts):
            _near(logits[s], _hf_logits(model, p), tol)
    assert dec.positions.tolist() == [9, 44, 5, 21, -1] and dec.lengths.tolist() == [10, 45, 6, 22, 0]


def test_graph_and_eager_tokens_match(model):
    from turbopress_amd.paged_decode import PagedDecoder
    prompts = _prompts([3, 8, 6])
    dec = PagedDecoder(model, 3, 64, page_size=4)
    eager, _ = dec.generate(prompts, 20, graph=False)
    assert len(eager) == 3 and all(len(t) == 20 for t in eager)
    for _ in range(2):
        assert dec.generate(prompts, 20, graph=True)[0] == eager
    # a sequence alone has the tokens that it has beside others
    assert PagedDecoder(model, 3, 64, page_size=32).generate(prompts[1:2], 20)[0] == eager[1:2]


def test_pages_are_handed_out_and_taken_back(cuda):
    from turbopress_amd.paged_decode import PagedCache
    c = PagedCache(1, 3, 20, 1, 8, page_size=4, n_pages=7)
    c.reserve(0, 9)
    c.reserve(1, 16)
    c.reserve(1, 3)
    held = c.block_table.cpu()
    assert (held[0] >= 0).tolist() == [True] * 3 + [False] * 2 and (held[1] >= 0).tolist() == [True] * 4 + [False]
    assert sorted(held[held >= 0].tolist()) == list(range(7))
    with pytest.raises(RuntimeError, match="full"):
        c.reserve(2, 1)
    with pytest.raises(ValueError):
        c.reserve(0, 21)
    c.release(0)
    c.reserve(2, 12)
    assert c.block_table[0].max() == -1 and sorted(c.block_table[2, :3].tolist()) == sorted(held[0, :3].tolist())


def test_sliding_window_layers_match_the_hf_decoder(cuda, tmp_path):
    from turbopress_amd.artifact import load_packed_model
    from turbopress_amd.paged_decode import PagedDecoder
    from turbopress_amd.synthetic import tiny_qwen3_config, write_synthetic_artifact
    cfg = tiny_qwen3_config()
    cfg.use_sliding_window, cfg.sliding_window = True, 6
    cfg.layer_types = ["sliding_attention", "full_attention"] * (cfg.num_hidden_layers // 2)
    write_synthetic_artifact(tmp_path, cfg, bits=3, seed=3)
    windowed = load_packed_model(tmp_path, device="cuda", mode="hip")[0]
    assert windowed.model.layers[0].self_attn.sliding_window == 6
    dec = PagedDecoder(windowed, 2, 64, page_size=16, fp8_head=False)
    for s, p in enumerate(_prompts([21, 4])):
        _near(dec.prefill(s, p)[0], _hf_logits(windowed, p), TOL)
        dec.cache.reserve(s, len(p) + 1)
        tokens = torch.cat((p, dec.tokens[s:s + 1]))
        logits = dec.step(graph=False)
        _near(logits[s], _hf_logits(windowed, tokens), TOL)
        dec.stop(s)


def test_what_the_decoder_does_not_run_is_refused(model):
    from turbopress_amd.paged_decode import PagedDecoder
    act = model.config.hidden_act
    model.config.hidden_act = "gelu"
    try:
        with pytest.raises(ValueError, match="hidden_act"):
            PagedDecoder(model, 1, 64)
    finally:
        model.config.hidden_act = act

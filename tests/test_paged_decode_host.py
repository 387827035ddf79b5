"""What the paged decoder and its tables decide on the host (no GPU)."""

import pytest
import torch


@pytest.mark.parametrize("keys", [{"mscale": 0.707, "mscale_all_dim": 0.707}, {"mscale": 1.0, "mscale_all_dim": 0.5},
                                  {"mscale": 0.7}, {"mscale_all_dim": 0.7}, {"mscale": 0.0, "mscale_all_dim": 1.0},
                                  {"mscale": 1.0, "mscale_all_dim": 0.4, "attention_factor": 1.2}, {"truncate": False}])
@pytest.mark.parametrize("factor", [8.0, 1.0])
def test_yarn_keys_match_transformers(keys, factor):
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    from turbopress_amd.paged import rotary_frequencies
    scaling = dict({"rope_type": "yarn", "factor": factor, "original_max_position_embeddings": 4096}, **keys)
    cfg = LlamaConfig(hidden_size=256, num_attention_heads=4, head_dim=64, max_position_embeddings=int(4096 * factor),
                      rope_theta=1e4, rope_scaling=dict(scaling, rope_theta=1e4))
    want, want_factor = ROPE_INIT_FUNCTIONS["yarn"](cfg, "cpu")
    got, got_factor = rotary_frequencies(64, 1e4, scaling)
    assert abs(got_factor - want_factor) < 1e-6
    assert ((got - want.double()).abs() <= 2.0 ** -21 * want.double()).all()


TINY = dict(vocab_size=64, hidden_size=64, intermediate_size=128, num_hidden_layers=4, num_attention_heads=4,
            num_key_value_heads=2, max_position_embeddings=128, pad_token_id=0, bos_token_id=1, eos_token_id=2)


def tiny_model(family, **kw):
    from transformers import AutoConfig, AutoModelForCausalLM
    return AutoModelForCausalLM.from_config(AutoConfig.for_model(family, **TINY, **kw)).half()


@pytest.mark.parametrize("family", ["smollm3", "granite", "ernie4_5", "olmo2", "phi3", "cohere", "seed_oss"])
def test_families_with_other_layers_are_refused(family):
    from turbopress_amd.paged_decode import PagedDecoder
    with pytest.raises(ValueError, match=family):
        PagedDecoder(tiny_model(family), 1, 64, fp8_head=False)


@pytest.mark.parametrize("family,kw,windows", [
    ("llama", {}, [0] * 4), ("mistral", {"sliding_window": 6}, [6] * 4), ("mistral", {"sliding_window": None}, [0] * 4),
    ("qwen2", {"use_sliding_window": True, "sliding_window": 6, "max_window_layers": 2}, [0, 0, 6, 6]),
    ("qwen3", {"use_sliding_window": True, "sliding_window": 6, "max_window_layers": 1, "head_dim": 16}, [0, 6, 6, 6])])
def test_windows_of_the_layers(family, kw, windows):
    from turbopress_amd.paged_decode import PagedDecoder
    assert PagedDecoder(tiny_model(family, **kw), 1, 64, fp8_head=False).windows == windows


def test_a_rotary_share_that_the_family_ignores_is_refused():
    from turbopress_amd.paged_decode import PagedDecoder
    with pytest.raises(ValueError, match="partial_rotary_factor"):
        PagedDecoder(tiny_model("llama", partial_rotary_factor=0.5), 1, 64, fp8_head=False)


@pytest.fixture
def stubbed(monkeypatch):
    """A decoder of three sequences whose layers and head are not run."""
    from turbopress_amd.paged_decode import PagedDecoder
    dec = PagedDecoder(tiny_model("llama"), 3, 32, page_size=8, fp8_head=False)
    ran = []
    monkeypatch.setattr(dec, "_rows", lambda tokens, *a: ran.append(len(tokens)) or (torch.zeros(len(tokens), 64),) * 2)
    monkeypatch.setattr(dec, "_logits", lambda x, h: torch.zeros(len(x), 64))
    dec.ran = ran
    return dec


def test_a_step_without_a_page_is_refused(stubbed):
    """Before anything runs, and without moving the other sequences."""
    dec = stubbed
    dec.prefill(0, torch.arange(7))
    dec.prefill(2, torch.arange(12))
    dec.step(graph=False)  # tokens 7 and 12: in the prompts' pages
    for graph in (False, True):
        with pytest.raises(RuntimeError, match="token 8 of sequence 0"):
            dec.step(graph=graph)
    assert dec.ran == [7, 12, 3] and dec.positions.tolist() == [8, -1, 13] and dec.lengths.tolist() == [9, 0, 14]
    dec.cache.reserve(0, 9)
    dec.step(graph=False)
    dec.stop(0)
    for _ in range(2):
        dec.step(graph=False)
    with pytest.raises(RuntimeError, match="token 16 of sequence 2"):
        dec.step(graph=False)
    assert dec.positions.tolist() == [-1, -1, 16]


def test_a_step_past_the_longest_length_is_refused(stubbed):
    dec = stubbed
    dec.prefill(1, torch.arange(31))
    dec.step(graph=False)
    with pytest.raises(RuntimeError, match="token 32 of sequence 1"):
        dec.step(graph=False)
    with pytest.raises(ValueError):
        dec.cache.reserve(1, 33)
    dec.stop(1)
    dec.step(graph=False)


@pytest.mark.parametrize("sequence", [-1, 3])
def test_sequences_that_do_not_exist_are_refused(stubbed, sequence):
    """-1 too: its rows were the last sequence's on the host and no one's on the device."""
    dec = stubbed
    dec.prefill(2, torch.arange(4))
    before = dec.cache.block_table.clone()
    for call in (lambda: dec.prefill(sequence, torch.arange(3)), lambda: dec.stop(sequence),
                 lambda: dec.cache.reserve(sequence, 9), lambda: dec.cache.release(sequence), lambda: dec.cache.room(sequence)):
        with pytest.raises(IndexError, match="outside"):
            call()
    assert dec.ran == [4] and dec.positions.tolist() == [-1, -1, 4] and torch.equal(dec.cache.block_table, before)


def test_generate_fills_the_longest_length(stubbed, monkeypatch):
    """A prompt and its new tokens but the last, which nothing reads, take max_len places."""
    dec = stubbed
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: None)
    tokens, _ = dec.generate([torch.arange(20), torch.arange(2)], 13, graph=False)
    assert len(tokens) == 2 and all(len(t) == 13 for t in tokens)
    assert dec.positions.tolist() == [32, 14, -1] and dec.cache.room(0) == 32 and dec.cache.room(1) == 16
    with pytest.raises(ValueError):
        dec.generate([torch.arange(20)], 14, graph=False)


def test_the_head_is_the_models_own_unless_asked():
    from turbopress_amd.paged_decode import PagedDecoder
    model = tiny_model("llama")
    assert PagedDecoder(model, 1, 32).head is None
    codes, scales = PagedDecoder(model, 1, 32, fp8_head=True).head
    assert codes.shape == (64, 64) and codes.dtype == torch.float8_e4m3fn and scales.shape == (1, 1)


def test_runs_from_one_beginning(stubbed, monkeypatch):
    """Both runs of the command decode from the same prefill: the second one
    finds the first one's beginning, whatever its prefill would have been."""
    dec = stubbed
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: None)
    tokens = iter(range(1000))
    monkeypatch.setattr(dec, "_logits", lambda x, h: torch.nn.functional.one_hot(
        torch.tensor([next(tokens) % 64] * len(x)), 64).float())
    begin = dec._begin([torch.arange(20), torch.arange(2)], 5)
    assert dec.ran == [20, 2]
    first = dec._decode(begin, 5, graph=False)[0]
    assert dec.positions.tolist() == [24, 6, -1] and dec._next == [24, 6, -1]
    second = dec._decode(begin, 5, graph=False)[0]
    assert [t[0] for t in first] == [t[0] for t in second] == [0, 1]
    assert dec.positions.tolist() == [24, 6, -1] and dec.lengths.tolist() == [25, 7, 0] and dec.ran == [20, 2] + [3] * 8

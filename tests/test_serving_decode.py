"""The paged decoder's drafted steps, adapters, windows with first tokens, chunked
prompts and scores, against the HF decoder on a small random packed model (GPU),
and what they decide and refuse on the host."""

import ctypes
import json
import random

import pytest
import torch

from test_paged_decode import TOL, _hf_logits, _near, _prompts
from test_paged_decode_host import tiny_model


@pytest.fixture(scope="module")
def model(cuda, tmp_path_factory):
    from turbopress_amd.artifact import load_packed_model
    from turbopress_amd.synthetic import tiny_qwen3_config, write_synthetic_artifact
    root = tmp_path_factory.mktemp("tiny")
    write_synthetic_artifact(root, tiny_qwen3_config(), bits=3, seed=3)
    return load_packed_model(root, device="cuda", mode="hip")[0]


# ---------------------------------------------------------------------------
# on the host
# ---------------------------------------------------------------------------
def test_lookup_draft():
    from turbopress_amd.paged_decode import lookup_draft
    assert lookup_draft([1, 2, 3, 9, 1, 2, 3], 2) == ([9, 1], [-1, 0])
    # two occurrences, the latest first: one trunk, two branches
    tokens, parents = lookup_draft([5, 6, 7, 1, 5, 6, 8, 2, 5, 6], 6)
    assert tokens == [8, 2, 5, 6, 7, 1] and parents == [-1, 0, 1, 2, -1, 4]
    # the branches share what they begin with
    assert lookup_draft([4, 1, 2, 9, 4, 1, 3, 9, 4], 5, longest=1) == ([1, 3, 9, 4, 2], [-1, 0, 1, 2, 0])
    assert lookup_draft([1, 2, 3], 4) == lookup_draft([], 4) == lookup_draft([1], 4) == lookup_draft([1, 1], 0) == ([], [])
    assert lookup_draft([1, 1], 4) == ([1], [-1])
    assert lookup_draft([7, 7, 7, 7], 2, branches=1) == ([7], [-1])


@pytest.fixture
def drafting(monkeypatch):
    """A decoder of three sequences that checks 4 tokens of each; its layers are
    not run, the most likely token behind t at any place is (3 t + 1) % 64."""
    from turbopress_amd.paged_decode import PagedDecoder
    dec = PagedDecoder(tiny_model("llama"), 3, 32, page_size=8, draft=4)
    monkeypatch.setattr(dec, "_rows", lambda tokens, *a: (torch.zeros(len(tokens), 64),) * 2)
    monkeypatch.setattr(dec, "_logits", lambda x, h: torch.nn.functional.one_hot(torch.tensor([5] * len(x)), 64).float())
    dec.ran = []

    def verify():
        dec.ran.append(dec._drafted.clone())
        return (3 * dec._drafted[0] + 1) % 64, -0.5 * dec._drafted[0].float()

    monkeypatch.setattr(dec, "_verify", verify)
    for c in (dec.cache.k, dec.cache.v):
        c.copy_(torch.arange(c.numel()).view(c.shape) % 1013)
    return dec


def _cached(dec, s, t):
    page = dec.cache.block_table[s, t // 8]
    return dec.cache.k[:, page, t % 8].clone(), dec.cache.v[:, page, t % 8].clone()


def test_drafts_are_accepted_along_their_path(drafting):
    dec = drafting
    dec.prefill(0, torch.arange(7))
    dec.prefill(2, torch.arange(3))
    for s, n in ((0, 16), (2, 16)):
        dec.cache.reserve(s, n)
    # 5 -> 16 -> 49 -> 20 -> 61: the second branch is right, its last token is not
    before = {(s, t): _cached(dec, s, t) for s in (0, 2) for t in range(16)}
    gained = dec.verify([([9, 16, 49, 7], [-1, -1, 1, 2]), None, ([9], [-1])], graph=False)
    assert gained == [([16, 49, 20], [-2.5, -8.0, -24.5]), ([], []), ([16], [-2.5])]
    state = dec.ran[0]
    assert state[0].tolist() == [[5, 9, 16, 49, 7], [0] * 5, [5, 9, 0, 0, 0]]
    assert state[1].tolist() == [[7, 8, 8, 9, 10], [-1] * 5, [3, 4, -1, -1, -1]]
    assert state[2].tolist() == [[7, 8, 9, 10, 11], [-1] * 5, [3, 4, -1, -1, -1]]
    assert state[3].tolist() == [[1, 3, 5, 13, 29], [0] * 5, [1, 3, 0, 0, 0]]
    assert state[4, :, 0].tolist() == [7, 0, 3]
    assert dec.tokens.tolist()[::2] == [20, 16] and dec.positions.tolist() == [10, -1, 4] and dec.lengths.tolist() == [11, 0, 5]
    for (s, t), was in before.items():  # 16 and 49 lie behind 5 now, nothing else has moved
        want = before[0, t + 1] if s == 0 and t in (8, 9) else was
        assert all(torch.equal(a, b) for a, b in zip(_cached(dec, s, t), want))
    # a chain that is right to its end
    assert dec.verify([([61, 56, 41, 60], [-1, 0, 1, 2]), None, None], graph=False)[0][0] == [61, 56, 41, 60, 53]
    assert dec.positions.tolist() == [15, -1, 5] and dec._next == [15, -1, 5]


def test_63_drafted_tokens(monkeypatch):
    """The last one's bit is the sign's."""
    from turbopress_amd.paged import tree_ancestors
    from turbopress_amd.paged_decode import PagedDecoder
    dec = PagedDecoder(tiny_model("llama"), 1, 100, page_size=8, draft=63)
    dec.cache.reserve(0, 80)
    dec._next, seen = [2], []
    monkeypatch.setattr(dec, "_verify", lambda: seen.append(dec._drafted.clone()) or (torch.full((1, 64), 3), torch.zeros(1, 64)))
    r = random.Random(0)
    parents = [-1] + [r.randrange(-1, j) for j in range(1, 63)]
    dec.verify([([1] * 63, parents)], graph=False)
    assert torch.equal(seen[0][3], tree_ancestors(torch.tensor([[-1] + [p + 1 for p in parents]])))
    assert seen[0][1, 0].tolist() == [1 + bin(m & (1 << 64) - 1).count("1") for m in seen[0][3, 0].tolist()]


def test_drafts_that_are_none_are_refused(drafting):
    from turbopress_amd.paged_decode import PagedDecoder
    dec = drafting
    dec.prefill(1, torch.arange(6))
    state = dec.cache.block_table.clone()
    for draft in (([1] * 5, [-1] * 5), ([1, 2], [-1]), ([1, 2], [-1, 1]), ([1], [-2]), ([64], [-1]), ([-1], [-1])):
        with pytest.raises(ValueError, match=r"drafts\[1\]"):
            dec.verify([None, draft, None], graph=False)
    with pytest.raises(ValueError, match="2 drafts for 3"):
        dec.verify([None, None])
    with pytest.raises(RuntimeError, match="token 8 of sequence 1"):  # (the page ends at 8)
        dec.verify([None, ([1, 2], [-1, 0]), None])
    assert not dec.ran and dec.positions.tolist() == [-1, 6, -1] and torch.equal(dec.cache.block_table, state)
    dec.verify([None, ([1], [-1]), None], graph=False)
    with pytest.raises(RuntimeError, match="checks no drafts"):
        PagedDecoder(tiny_model("llama"), 1, 32).verify([None])
    for kw in (dict(draft=-1), dict(draft=64), dict(window=-1), dict(sinks=-1)):
        with pytest.raises(ValueError):
            PagedDecoder(tiny_model("llama"), 1, 32, **kw)
    with pytest.raises(RuntimeError, match="is decoding"):
        dec.score(torch.arange(4), sequence=1)
    with pytest.raises(ValueError, match="two tokens"):
        dec.score(torch.arange(1))
    with pytest.raises(ValueError, match="adapter 0"):
        dec.prefill(0, torch.arange(4), adapter=0)
    for moves in ([(1, 0, 8)], [(1, -1, 0)], [(0, 0, 0)]):
        with pytest.raises(ValueError, match="hold"):
            dec.cache.move(moves)


def test_generate_drafted_fills_the_longest_length(drafting, monkeypatch):
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: None)
    dec, want = drafting, [5]
    for _ in range(12):
        want.append((3 * want[-1] + 1) % 64)
    r = random.Random(1)

    def drafter(history, count):  # right to some place, with a wrong branch first
        good = [(3 * history[-1] + 1) % 64]
        while len(good) < count:
            good.append((3 * good[-1] + 1) % 64 if r.random() < 0.7 else 0)
        return ([0, *good][:count], [-1, -1, *range(1, count)][:count])

    prompts = [torch.arange(20), torch.arange(2)]
    for _ in range(3):
        tokens, _, gain = dec.generate_drafted(prompts, 13, drafter, graph=False)
        assert tokens == [want, want] and gain > 1
        assert dec.positions.tolist() == [32, 14, -1] and dec.lengths.tolist() == [33, 15, 0] and dec._next == [32, 14, -1]
    with pytest.raises(ValueError):
        dec.generate_drafted([torch.arange(20)], 14, drafter, graph=False)


def test_windows_given_cut_the_layers_own():
    from turbopress_amd.paged_decode import PagedDecoder
    kw = {"use_sliding_window": True, "sliding_window": 6, "max_window_layers": 2}
    assert PagedDecoder(tiny_model("qwen2", **kw), 1, 64, window=4).windows == [4] * 4
    assert PagedDecoder(tiny_model("qwen2", **kw), 1, 64, window=9, sinks=2).windows == [9, 9, 6, 6]


def _pair(g, rank, k, n, dtype=torch.float16):
    return torch.randn(rank, k, generator=g).to(dtype), torch.randn(n, rank, generator=g).to(dtype)


def _write(root, modules, config=None, extra=None):
    from safetensors.torch import save_file
    root.mkdir()
    rank = next(iter(modules.values()))[0].shape[0]
    (root / "adapter_config.json").write_text(json.dumps({"peft_type": "LORA", "r": rank, "lora_alpha": 16, **(config or {})}))
    tensors = {f"base_model.model.{name}.lora_{x}.weight": t.contiguous() for name, pair in modules.items() for x, t in zip("AB", pair)}
    save_file({**tensors, **(extra or {})}, root / "adapter_model.safetensors")
    return root


def test_adapters_are_loaded_and_stacked(tmp_path):
    from turbopress_amd.lora import LoraAdapters
    g = torch.Generator().manual_seed(0)
    q, o = "model.layers.0.self_attn.q_proj", "model.layers.1.self_attn.o_proj"
    one, two = {q: _pair(g, 4, 6, 10), o: _pair(g, 4, 8, 6)}, {q: _pair(g, 9, 6, 10)}
    got = LoraAdapters.load([_write(tmp_path / "a", one), _write(tmp_path / "b", two, {"use_rslora": True})], torch.float16, "cpu")
    assert got.count == 2 and got.scales.tolist() == [4.0, pytest.approx(16 / 3)]
    a, b = got.stacks[q]
    assert a.shape == (2, 9, 6) and b.shape == (2, 10, 9)
    for i, (wa, wb) in enumerate((one[q], two[q])):
        r = wa.shape[0]
        assert torch.equal(a[i, :r], wa) and torch.equal(b[i, :, :r], wb) and not a[i, r:].any() and not b[i, :, r:].any()
    a, b = got.stacks[o]
    assert a.shape == (2, 4, 8) and not a[1].any() and not b[1].any()
    got.check({q: (10, 6), o: (6, 8)}, torch.float16, torch.device("cpu"))
    for shapes, dtype in (({q: (10, 6)}, torch.float16), ({q: (6, 10), o: (6, 8)}, torch.float16),
                          ({q: (10, 6), o: (6, 8)}, torch.bfloat16)):
        with pytest.raises(ValueError):
            got.check(shapes, dtype, torch.device("cpu"))


def test_adapters_that_are_more_than_two_products_are_refused(tmp_path):
    from turbopress_amd.lora import LoraAdapters
    g = torch.Generator().manual_seed(0)
    name = "model.layers.0.self_attn.q_proj"
    pair = {name: _pair(g, 4, 6, 10)}
    for i, config in enumerate(({"use_dora": True}, {"rank_pattern": {"q_proj": 8}}, {"bias": "all"}, {"peft_type": "IA3"},
                                {"modules_to_save": ["lm_head"]})):
        with pytest.raises(ValueError):
            LoraAdapters.load([_write(tmp_path / str(i), pair, config)], torch.float16, "cpu")
    for i, extra in enumerate(({"base_model.model.lm_head.weight": torch.zeros(2)},
                               {"base_model.model.x.lora_A.weight": torch.zeros(2, 3)})):
        with pytest.raises(ValueError):
            LoraAdapters.load([_write(tmp_path / f"x{i}", pair, None, extra)], torch.float16, "cpu")
    f16 = torch.float16
    for adapters, scales, dtype in (([], [], f16), ([pair], [1, 2], f16), ([pair], [1], torch.float32),
                                    ([pair, {name: _pair(g, 4, 7, 10)}], [1, 1], f16), ([{name: _pair(g, 257, 6, 10)}], [1], f16),
                                    ([{name: (pair[name][0], _pair(g, 5, 6, 10)[1])}], [1], f16)):
        with pytest.raises(ValueError):
            LoraAdapters(adapters, scales, dtype, "cpu")


def test_c_entry_points_refuse_on_the_host(built_lib):
    from turbopress_amd import _lib as L
    lib, p, odd = built_lib, ctypes.c_void_p(256), ctypes.c_void_p(257)
    i3 = (ctypes.c_int64 * 3)(1024, 64, 8)

    def rot(tokens=2, kc=p, slots=p, pos=p, d=8, k=p):
        return lib.tp_rotary_slots(0, tokens, 2, 1, d, 8, 0, p, 16, 8, k, 8, 8, p, 4, pos, p, p, 8, 8, kc, i3, kc, i3, 3, 4, p, 1, 2,
                                   None, slots, None)

    assert rot(tokens=0) == L.TP_OK and rot(d=7) == rot(tokens=-1) == L.TP_ERR_BAD_DIMS
    assert rot(kc=None) == rot(slots=None) == rot(pos=None) == rot(k=None) == L.TP_ERR_NULL_POINTER
    assert rot(slots=ctypes.c_void_p(260)) == L.TP_ERR_MISALIGNED

    one = lib.tp_paged_attention_workspace_bytes(2, 4, 2, 64), lib.tp_paged_attention_counter_bytes(2, 4, 2, 64)

    def sinks(dtype=0, batch=2, window=8, sinks=4, q=p, size=one[0], csize=one[1]):
        return lib.tp_paged_attention_sinks(dtype, batch, 4, 2, 64, q, 256, 64, p, i3, p, i3, 5, 16, p, 1, p, 1.0, window, sinks, p, p,
                                            size, p, csize, None)

    assert sinks(batch=0) == L.TP_OK and sinks(dtype=2) == L.TP_ERR_BAD_TYPE
    assert sinks(sinks=-1) == sinks(window=-1) == L.TP_ERR_BAD_DIMS and sinks(q=None) == L.TP_ERR_NULL_POINTER
    assert sinks(size=one[0] - 1) == sinks(csize=one[1] - 1) == L.TP_ERR_WORKSPACE

    need, count = lib.tp_paged_tree_attention_workspace_bytes(2, 5, 4, 2, 64), lib.tp_paged_tree_attention_counter_bytes(2, 5, 4, 2, 64)
    assert need > 0 and count == 16
    # 256 rows of a cache head: a group of 256, or, of heads of more than 128 columns, of 32 each
    assert lib.tp_paged_tree_attention_counter_bytes(3, 64, 8, 2, 64) == 3 * 2 * 4
    assert lib.tp_paged_tree_attention_counter_bytes(3, 64, 8, 2, 256) == 3 * 2 * 8 * 4

    def tree(dtype=0, batch=2, tokens=5, hq=4, hkv=2, d=64, q=p, token=256, seen=p, page=16, window=0, sinks=0, size=need, csize=count,
             kc=p, out=p):
        return lib.tp_paged_tree_attention(dtype, batch, tokens, hq, hkv, d, q, 5 * 256, token, 64, kc, i3, kc, i3, 5, page, p, 1, p, seen,
                                           1.0, window, sinks, out, p, size, p, csize, None)

    assert tree(batch=0) == L.TP_OK and tree(dtype=2) == L.TP_ERR_BAD_TYPE
    assert tree(tokens=0) == tree(tokens=65) == tree(d=60) == tree(hq=5) == tree(page=0) == tree(window=-1) == tree(sinks=-1) \
        == tree(batch=-1) == tree(batch=1 << 20, hq=64, hkv=64) == L.TP_ERR_BAD_DIMS
    assert lib.tp_paged_tree_attention_workspace_bytes(1, 65, 2, 2, 64) == lib.tp_paged_tree_attention_counter_bytes(1, 0, 2, 2, 64) == -1
    assert tree(q=None) == tree(kc=None) == tree(out=None) == L.TP_ERR_NULL_POINTER
    assert tree(token=252) == tree(seen=ctypes.c_void_p(260)) == tree(q=odd) == L.TP_ERR_MISALIGNED
    assert tree(size=need - 1) == tree(csize=count - 1) == L.TP_ERR_WORKSPACE

    need, count = lib.tp_token_logprobs_workspace_bytes(3, 1000, 5), lib.tp_token_logprobs_counter_bytes(3, 1000, 5)
    assert need > 0 and count == 12 and lib.tp_token_logprobs_workspace_bytes(0, 1000, 5) == 0

    def lp(dtype=0, rows=3, vocab=1000, logits=p, ld=1000, tokens=p, out=p, entropy=p, top=5, tl=p, tt=p, ws=p, size=need, csize=count):
        return lib.tp_token_logprobs(dtype, rows, vocab, logits, ld, tokens, out, entropy, top, tl, tt, ws, size, p, csize, None)

    assert lp(rows=0) == L.TP_OK and lp(dtype=4) == L.TP_ERR_BAD_TYPE
    assert lp(vocab=0) == lp(rows=-1) == lp(top=65) == lp(top=-1) == lp(vocab=4) == lp(ld=-1) == lp(rows=1 << 40) == L.TP_ERR_BAD_DIMS
    assert lp(logits=None) == lp(entropy=None) == lp(out=None) == lp(tl=None) == lp(tt=None) == L.TP_ERR_NULL_POINTER
    assert lp(logits=odd) == lp(tokens=ctypes.c_void_p(260)) == lp(ws=ctypes.c_void_p(264)) == L.TP_ERR_MISALIGNED
    assert lp(ws=None) == lp(size=need - 1) == lp(csize=count - 1) == L.TP_ERR_WORKSPACE
    assert lib.tp_token_logprobs_workspace_bytes(1, 0, 0) == lib.tp_token_logprobs_counter_bytes(1, 8, 9) == -1

    need = lib.tp_lora_workspace_bytes(3, 100, 50, 8, 2)
    assert need > 0 and lib.tp_lora_workspace_bytes(3, 100, 50, 8, 0) == 0

    def lora(dtype=0, rows=3, k=100, n=50, rank=8, count=2, x=p, ldx=100, a=p, b=p, ids=p, scales=p, y=p, ldy=50, out=p, ws=p, size=need):
        return lib.tp_lora_add(dtype, rows, k, n, rank, count, x, ldx, a, 800, 100, b, 400, 8, ids, scales, y, ldy, out, ws, size, None)

    assert lora(rows=0) == L.TP_OK and lora(dtype=2) == L.TP_ERR_BAD_TYPE
    assert lora(k=0) == lora(n=0) == lora(rank=0) == lora(rank=257) == lora(rows=-1) == lora(count=-1) == lora(ldx=-1) == lora(ldy=-1) \
        == lora(rows=1 << 24, n=1 << 20) == L.TP_ERR_BAD_DIMS
    assert lora(x=None) == lora(a=None) == lora(b=None) == lora(ids=None) == lora(y=None) == lora(out=None) == L.TP_ERR_NULL_POINTER
    assert lora(x=odd) == lora(ids=ctypes.c_void_p(258)) == lora(scales=ctypes.c_void_p(258)) == lora(ws=ctypes.c_void_p(264)) \
        == L.TP_ERR_MISALIGNED
    assert lora(ws=None) == lora(size=need - 1) == L.TP_ERR_WORKSPACE
    assert lib.tp_lora_workspace_bytes(1, 1, 1, 257, 1) == -1


# ---------------------------------------------------------------------------
# on the device
# ---------------------------------------------------------------------------
@torch.inference_mode()
def _hf_all(model, tokens, window=0, sinks=0):
    """Logits behind every token, each seeing the last `window` and the first `sinks`."""
    n = len(tokens)
    mask = None
    if window:
        at = torch.arange(n, device=tokens.device)
        sees = (at[None] <= at[:, None]) & ((at[None] > at[:, None] - window) | (at[None] < sinks))
        mask = torch.where(sees, 0.0, torch.finfo(torch.float16).min).half()[None, None]
    return model(input_ids=tokens[None], attention_mask=mask, use_cache=False).logits[0].float()


def _greedy(model, prompt, tokens, logprobs=None):
    """Each token is the most likely one behind those before it, as far as either
    side's rounding (TOL of the largest logit) tells, and so is its log probability
    (off by the token's logit and the sum's, each)."""
    text = torch.cat((prompt, torch.tensor(tokens, device=prompt.device)))
    logits = _hf_all(model, text)[len(prompt) - 1:-1].double()
    tol = 2 * TOL * logits.abs().amax(1)
    got = logits.gather(1, text[len(prompt):, None])[:, 0]
    assert (got >= logits.amax(1) - tol).all()
    if logprobs is not None:
        want = logits.log_softmax(1).gather(1, text[len(prompt):, None])[:, 0]
        assert ((torch.tensor(logprobs, device=want.device) - want).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("draft", [1, 4, 7])
@pytest.mark.parametrize("branches", [1, 2])
def test_drafted_tokens_are_the_greedy_ones(model, draft, branches):
    """Drafts that hold the plain decoder's own tokens, and wrong branches."""
    from turbopress_amd.paged_decode import PagedDecoder
    # (a packed projection's sums are not always in one order for 17 to 32 rows)
    prompts = _prompts([5, 9] if draft == 7 else [5, 33, 12])
    dec = PagedDecoder(model, len(prompts), 96, page_size=16, draft=draft)
    plain, _ = dec.generate(prompts, 24, graph=False)
    texts = [p.tolist() + t for p, t in zip(prompts, plain)]
    r = random.Random(draft)

    def drafter(history, count):
        text = next((t for t in texts if t[:len(history)] == history), [0] * 200)
        tokens, parents, node = [], [], -1
        for t in text[len(history):]:
            if branches == 2 and len(tokens) + 1 < count and r.random() < 0.5:
                tokens.append((t + 1) % 1024)
                parents.append(node)
            if len(tokens) < count:
                tokens.append(t if r.random() < 0.9 else 7)
                parents.append(node)
                node = len(tokens) - 1
        return tokens, parents

    for graph in (False, True, True):
        got, _, gain = dec.generate_drafted(prompts, 24, drafter, graph=graph)
        assert [len(t) for t in got] == [24] * len(prompts) and gain > 1.2
        for p, t in zip(prompts, got):
            _greedy(model, p, t)
    got, _, _ = dec.generate_drafted(prompts, 24)  # (its own drafts)
    for p, t in zip(prompts, got):
        _greedy(model, p, t)


@pytest.mark.gpu
def test_a_captured_pass_is_replayed_beside_other_work(model):
    from turbopress_amd.paged_decode import PagedDecoder, lookup_draft
    prompts = _prompts([40, 3])  # (not 17 to 32 rows: a packed projection's sums are not always in one order there)
    dec = PagedDecoder(model, 3, 128, page_size=16, draft=4)
    runs = []
    for graph in (False, True):
        for s in range(3):
            dec.stop(s)
        for s, p in enumerate(prompts):
            dec.prefill(s, p)
            dec.cache.reserve(s, 120)
        texts, logprobs = [p.tolist() + [dec.tokens[s].item()] for s, p in enumerate(prompts)], [[], []]
        for i in range(12):
            drafts = [lookup_draft(t, 4) for t in texts] + [None]
            if i % 4 == 2:  # a plain step and a score between two passes
                assert dec.score(prompts[0], sequence=2).logprobs.shape == (39,)
                torch.cuda.synchronize()
                logits = dec.step(graph).float().log_softmax(1)
                for s in range(2):
                    texts[s].append(dec.tokens[s].item())
                    logprobs[s].append(logits[s, texts[s][-1]].item())
            else:
                for s, (t, l) in enumerate(dec.verify(drafts, graph)[:2]):
                    texts[s] += t
                    logprobs[s] += l
        for s, p in enumerate(prompts):
            _greedy(model, p, texts[s][len(p):], [_first(model, p), *logprobs[s]])
        runs.append(texts)
    assert runs[0] == runs[1]


def _first(model, prompt):
    return _hf_all(model, prompt)[-1].log_softmax(0).max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[5, 64, 1], [130, 63], [65]])
def test_chunked_prompts_and_scores(model, lengths):
    from turbopress_amd.paged_decode import PagedDecoder
    dec = PagedDecoder(model, len(lengths), 160, page_size=16)
    for s, p in enumerate(_prompts(lengths)):
        _near(dec.prefill(s, p, chunked=True)[0], _hf_logits(model, p), TOL)
        dec.cache.reserve(s, len(p) + 1)
    tokens = dec.tokens.clone()
    logits = dec.step(graph=False)
    for s, p in enumerate(_prompts(lengths)):
        text = torch.cat((p, tokens[s:s + 1]))
        _near(logits[s], _hf_logits(model, text), TOL)
        dec.stop(s)
        got = dec.score(text, top=3, sequence=s)
        want = _hf_all(model, text)[:-1].double()
        tol = 2 * TOL * want.abs().amax(1)
        lp = want.log_softmax(1)
        assert ((got.logprobs - lp.gather(1, text[1:, None])[:, 0]).abs() <= tol).all()
        assert ((got.top_logprobs - lp.topk(3).values).abs() <= tol[:, None]).all()
        # (logits off by e: |dH| = |cov(log p, e)| <= 2 e standard deviations of log p)
        mean = (lp.exp() * lp).sum(1)
        spread = (lp.exp() * (lp - mean[:, None]) ** 2).sum(1).sqrt()
        assert ((got.entropy + mean).abs() <= 2 * tol * spread + tol ** 2).all()
        assert dec._next[s] == -1 and dec.cache.room(s) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(9, 0), (9, 3), (1, 1), (40, 4)])
def test_windows_and_first_tokens(model, window, sinks):
    from turbopress_amd.paged_decode import PagedDecoder
    prompts = _prompts([33, 70])
    dec = PagedDecoder(model, 2, 96, page_size=16, window=window, sinks=sinks, draft=3)
    for chunked in (False, True):
        for s, p in enumerate(prompts):
            _near(dec.prefill(s, p, chunked=chunked)[0], _hf_all(model, p, window, sinks)[-1], TOL)
            dec.cache.reserve(s, len(p) + 6)
        tokens = dec.tokens.clone()
        logits = dec.step()
        texts = [torch.cat((p, t[None])) for p, t in zip(prompts, tokens)]
        for s, t in enumerate(texts):
            _near(logits[s], _hf_all(model, t, window, sinks)[-1], TOL)
        texts = [torch.cat((p, t[None])) for p, t in zip(texts, dec.tokens.clone())]
        gained = dec.verify([([3, 4, 5], [-1, 0, 1])] * 2)
        for s, t in enumerate(texts):
            want = _hf_all(model, t, window, sinks)[-1].double()
            tol = 2 * TOL * want.abs().max()
            assert want[gained[s][0][0]] >= want.max() - tol
            assert abs(want.log_softmax(0)[gained[s][0][0]].item() - gained[s][1][0]) <= tol


# (beside the plain decoder's roundings one more of each of seven projections)
TOLA = 4 * (2 * 27) ** 0.5 * 2.0 ** -11


@pytest.mark.gpu
def test_adapters_of_each_sequence(model):
    from turbopress_amd.lora import LoraAdapters
    from turbopress_amd.paged_decode import PagedDecoder, _projections
    g = torch.Generator().manual_seed(7)
    adapters = []
    for i, rank in enumerate((4, 24)):
        one = {}
        for j, layer in enumerate(model.model.layers):
            for name, m in _projections(layer):
                if i == 0 or "mlp" not in name:  # (the second changes attention alone)
                    a, b = _pair(g, rank, m.in_features, m.out_features, torch.float32)
                    one[f"model.layers.{j}.{name}"] = (a / m.in_features ** 0.5, 0.3 * b / rank ** 0.5)
        adapters.append(one)
    stack = LoraAdapters(adapters, [1.5, 0.5], torch.float16)
    prompts, each = _prompts([5, 40, 12]), [1, -1, 0]
    dec = PagedDecoder(model, 4, 96, page_size=16, adapters=stack, draft=3)

    def hf(text, which):
        hooks = []
        if which >= 0:
            for j, layer in enumerate(model.model.layers):
                for name, m in _projections(layer):
                    pair = stack.stacks.get(f"model.layers.{j}.{name}")

                    def hook(module, args, out, pair=pair):
                        a, b = (t[which].float() for t in pair)
                        return (out.float() + stack.scales[which] * (args[0].float() @ a.T @ b.T)).to(out.dtype)

                    hooks.append(m.register_forward_hook(hook))
        try:
            return _hf_all(model, text)
        finally:
            for h in hooks:
                h.remove()

    for graph in (False, True):
        texts = []
        for s, (p, which) in enumerate(zip(prompts, each)):
            _near(dec.prefill(s, p, adapter=which, chunked=graph)[0], hf(p, which)[-1], TOLA)
            dec.cache.reserve(s, len(p) + 8)
            texts.append(torch.cat((p, dec.tokens[s:s + 1])))
        logits = dec.step(graph)
        for s, t in enumerate(texts):
            _near(logits[s], hf(t, each[s])[-1], TOLA)
        texts = [torch.cat((t, dec.tokens[s:s + 1])) for s, t in enumerate(texts)]
        gained = dec.verify([([9, 9], [-1, -1])] * 3 + [None], graph)
        for s, t in enumerate(texts):
            want = hf(t, each[s])[-1].double()
            tol = 2 * TOLA * want.abs().max()
            assert want[gained[s][0][0]] >= want.max() - tol
            assert abs(want.log_softmax(0)[gained[s][0][0]].item() - gained[s][1][0]) <= tol
    # the adapters do change what is answered, and end with their sequence
    base = dec.score(prompts[1], sequence=3).logprobs
    assert (dec.score(prompts[1], adapter=0, sequence=3).logprobs - base).abs().max() > 0.1
    assert torch.equal(dec.score(prompts[1], sequence=3).logprobs, base)
    assert dec.adapter_of.tolist() == [1, -1, 0, -1]


@pytest.mark.gpu
def test_tensors_on_another_device_than_the_current_one(cuda, monkeypatch):
    """Each entry point goes to its tensors' device before it looks for a stream."""
    from test_serving_ops import _gen, _serve
    from turbopress_amd import logprobs, lora, paged
    _, run = _serve(_gen(3))
    want = [t.clone() for t in run()]
    entered, asked = [], []

    class Device(torch.cuda.device):
        def __enter__(self):
            entered.append(self.idx)
            super().__enter__()

    def elsewhere(index):
        asked.append(index)
        return len(asked) > len(entered) * 2  # (once for each call, not again inside)

    monkeypatch.setattr(torch.cuda, "device", Device)
    for module in (paged, logprobs, lora):
        monkeypatch.setattr(module, "_elsewhere", elsewhere)
    got = run()
    assert len(entered) >= 4 and len(asked) == 2 * len(entered) and set(entered) == {0}
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_calls_with_nothing_to_do(cuda):
    import turbopress_amd as T

    def z(*shape, dtype=torch.float16):
        return torch.zeros(*shape, dtype=dtype, device=cuda)

    i32 = torch.int32
    cache = z(3, 4, 2, 8)
    assert T.paged_tree_attention(z(0, 3, 4, 8), cache, cache, z(0, 2, dtype=i32), z(0, dtype=i32)).shape == (0, 3, 4, 8)
    # no pages at all, and a table of no columns
    q = torch.ones(2, 3, 4, 8, dtype=torch.float16, device=cuda)
    n = torch.tensor([5, 0], dtype=i32, device=cuda)
    assert not T.paged_tree_attention(q, z(0, 4, 2, 8), z(0, 4, 2, 8), z(2, 2, dtype=i32), n).any()
    assert not T.paged_tree_attention(q, cache, cache, z(2, 0, dtype=i32), n).any()
    got = T.token_logprobs(z(0, 9), z(0, dtype=torch.int64), top=2)
    assert got.logprobs.shape == got.entropy.shape == (0,) and got.top_tokens.shape == (0, 2)
    assert T.lora_add(z(0, 6), z(0, 5), z(3, 2, 5), z(3, 6, 2), z(0, dtype=i32)).shape == (0, 6)
    y, ids = torch.rand(4, 6, device=cuda).half(), torch.tensor([0, -1, 2 ** 31 - 1, -2 ** 31], dtype=i32, device=cuda)
    assert torch.equal(T.lora_add(y, z(4, 5), z(0, 2, 5), z(0, 6, 2), ids), y)
    assert torch.equal(T.lora_add(y, torch.ones_like(z(4, 5)), z(1, 2, 5), z(1, 6, 2), ids), y)

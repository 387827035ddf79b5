"""What a decoder's sequences are after a drafter, or a check of what it drafted,
has raised (on the host)."""

import pytest
import torch

from test_serving_decode import drafting  # noqa: F401 (a fixture)


def _good(history, count):
    tokens = [(3 * history[-1] + 1) % 64]
    while len(tokens) < count:
        tokens.append((3 * tokens[-1] + 1) % 64)
    return tokens[:count], [-1, *range(count - 1)][:count]


@pytest.mark.parametrize("bad", ["raise", ([64], [-1]), ([1], [0]), ([1] * 5, [-1] * 5), ([1, 2], [-1])])
def test_finished_sequences_live_on_where_a_drafter_fails(drafting, monkeypatch, bad):  # noqa: F811
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: None)
    dec = drafting

    def drafter(history, count):
        if len(history) < 12:  # (the short prompts' sequence fails late)
            return [], []
        if bad == "raise":
            raise KeyError("no draft")
        return bad

    def first(history, count):  # the first sequence has all its tokens after two passes, the second goes on
        return _good(history, count) if history[0] == 9 else drafter(history, count)

    prompts = [torch.tensor([9, *range(19)]), torch.arange(3)]
    with pytest.raises(KeyError if bad == "raise" else ValueError):
        dec.generate_drafted(prompts, 11, first, graph=False)
    assert dec._next[0] == 30 and dec.positions.tolist() == [30, dec._next[1], -1]
    assert dec.lengths.tolist() == [31, dec._next[1] + 1, 0]
    assert 3 <= dec._next[1] < 14
    with pytest.raises(RuntimeError, match="sequence 0 is decoding"):
        dec.score(torch.arange(4), sequence=0)
    # both go on from where they are
    at, last = list(dec._next), dec.tokens.tolist()
    dec.cache.reserve(0, 32)
    assert dec.verify([([], []), None, None], graph=False) == [([(3 * t + 1) % 64], [-0.5 * t]) for t in last[:2]] + [([], [])]
    assert dec._next == [at[0] + 1, at[1] + 1, -1]


def test_a_drafter_that_gives_more_than_is_asked_for(drafting, monkeypatch):  # noqa: F811
    """Never more than n_new tokens of a prompt: with 4 drafted at each pass, right ones, more would come."""
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: None)
    with pytest.raises(ValueError, match="4 tokens, up to [123] were asked for"):
        drafting.generate_drafted([torch.arange(5)], 9, lambda history, count: _good(history, 4), graph=False)
    tokens, _, _ = drafting.generate_drafted([torch.arange(5), torch.arange(7)], 9, _good, graph=False)
    assert [len(t) for t in tokens] == [9, 9]

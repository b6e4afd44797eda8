"""What CachedGpt refuses, and that a refusal moves nothing: the sequences go
on afterwards as if it had not been asked.  Going on means the same operators
on the same inputs, so results are equal bit for bit."""

import numpy as np
import pytest

from grokking_abmod_b200 import CachedGpt, GptConfig, MeshGpt, ops

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    return MeshGpt(0, GptConfig(vocab_size=17, context=12, width=128, heads=4, layers=2), 7)


PROMPTS = [[3, 1, 4], [1, 5]]


@pytest.mark.parametrize("tokens", [[[], [1, 2]], [[1, 2], []], [[], []]])
def test_every_sequence_needs_a_token_to_follow(model, tokens):
    """An empty list has no row of its own whose logits could be used."""
    run = CachedGpt(model, 2)
    run.extend(PROMPTS)
    with pytest.raises(ValueError):
        run.score(tokens, [0, 0])
    with pytest.raises(ValueError):
        run.generate(tokens, 1)
    assert run.lengths.tolist() == [3, 2]
    fresh = CachedGpt(model, 2)
    fresh.extend(PROMPTS)
    assert all((a == b).all() for a, b in zip(run.score([[7], [8]], [1, 2], 3), fresh.score([[7], [8]], [1, 2], 3)))


def test_a_step_that_fails_leaves_the_sequences_as_they_were(model, monkeypatch):
    run, fresh = CachedGpt(model, 2), CachedGpt(model, 2)
    for r in (run, fresh):
        r.extend(PROMPTS)
    attention, calls = ops.cache_attention, []

    def fails(*args, **kw):
        calls.append(1)
        if len(calls) == 2:  # the second layer's
            raise RuntimeError("no memory")
        return attention(*args, **kw)

    monkeypatch.setattr(ops, "cache_attention", fails)
    with pytest.raises(RuntimeError):
        run.extend([[7], [8, 9]])
    monkeypatch.undo()
    assert run.lengths.tolist() == [3, 2]
    assert (run.extend([[7], [8, 9]]) == fresh.extend([[7], [8, 9]])).all()
    assert run.lengths.tolist() == [4, 4]


def _moves_nothing(model, asked):
    run, fresh = CachedGpt(model, 2), CachedGpt(model, 2)
    for r in (run, fresh):
        r.extend(PROMPTS)
    with pytest.raises((ValueError, ops._lib.MeshError)):
        asked(run)
    assert run.lengths.tolist() == [3, 2] and int(run.status.item()) == 0
    assert (run.extend([[7], [8, 9]]) == fresh.extend([[7], [8, 9]])).all()


def test_generation_past_the_context_is_refused_before_it_begins(model):
    """Steps that cannot all be done would be lost with the exception."""
    _moves_nothing(model, lambda run: run.generate([[7], [8, 9]], 10))  # 3 + 1 + 9 > 12
    run = CachedGpt(model, 2)
    run.extend(PROMPTS)
    assert len(run.generate([[7], [8, 9]], 9)) == 9 and run.lengths.tolist() == [12, 12]


@pytest.mark.parametrize("asked", [lambda r: r.score([[7], [8]], [1]), lambda r: r.score([[7], [8]], [1, 17]),
                                   lambda r: r.score([[7], [8]], [1, -2]), lambda r: r.score([[7], [8]], [1, 2], 18),
                                   lambda r: r.score([[7], [8]], [1, 2], -1), lambda r: r.generate([[7], [8]], 2, 33),
                                   lambda r: r.generate([[7], [17]], 2), lambda r: r.generate([[7]], 2)])
def test_what_cannot_be_answered_is_refused_before_anything_moves(model, asked):
    _moves_nothing(model, asked)

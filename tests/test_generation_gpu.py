"""Generation over the 8-bit cache against the model's own forward.

A cached key or value is off by at most half its page's scale, amax / 127 (keys
are unit-RMS rows: about 0.02 a channel, 0.014 RMS).  A score then errs by
about 0.014, an attention output by 2% of its size, and the logits, whose
residual stream carries most of their size, by less: 5% of their norm bounds
it.  What goes into a cache in one piece or token by token differs by the
same kind of rounding."""

import numpy as np
import pytest

from grokking_abmod_b200 import CachedGpt, GptConfig, MeshGpt

pytestmark = pytest.mark.gpu

CASES = [dict(vocab_size=17, context=40, width=128, heads=4, layers=2),
         dict(vocab_size=31, context=70, width=256, heads=2, layers=3, connectivity="butterfly"),
         dict(vocab_size=11, context=33, width=64, heads=8, layers=1, embedding="table")]


def _rel(a, b):
    return np.linalg.norm(a - b) / np.linalg.norm(b)


@pytest.mark.parametrize("kw", CASES)
def test_cached_logits_follow_the_models(kw):
    config = GptConfig(**kw)
    model = MeshGpt(0, config, 7)
    rng = np.random.default_rng(1)
    n = config.context
    tokens = rng.integers(0, config.vocab_size, (3, n))
    want = model.logits(tokens.reshape(-1), n).reshape(3, n, -1)

    whole = CachedGpt(model, 3)
    got = whole.extend(tokens.tolist()).cpu().numpy().reshape(3, n, -1)
    assert _rel(got, want) < 0.05

    # a prompt each of another length, then a token at a time, one sequence pausing
    run = CachedGpt(model, 3, page_tokens=32)
    starts = [n // 2, 1, n - 3]
    parts = [[row] for row in run.extend([tokens[b, :s].tolist() for b, s in enumerate(starts)]).cpu().numpy()]
    rows = [[], [], []]
    at = 0
    for b, s in enumerate(starts):
        rows[b] = [p[0] for p in parts[at:at + s]]
        at += s
    for step in range(n):
        feed = [tokens[b, len(rows[b]):len(rows[b]) + (0 if b == 1 and step % 3 == 2 else 1)].tolist() for b in range(3)]
        if not any(feed):
            break
        logits = iter(run.extend(feed).cpu().numpy())
        for b in range(3):
            rows[b] += [next(logits) for _ in feed[b]]
    for b in range(3):
        assert len(rows[b]) > starts[b]
        assert _rel(np.stack(rows[b]), want[b, :len(rows[b])]) < 0.05
    with pytest.raises(ValueError):
        whole.extend([[0], [], []])
    with pytest.raises(ValueError):
        CachedGpt(model, 1).extend([[config.vocab_size]])


def test_scores_and_greedy_tokens():
    """Of a model trained to certainty on a few equations the cached path
    gives the same answers, and their log-probabilities."""
    from grokking_abmod_b200.data import EquationDataset
    data = EquationDataset(7, "add", 0.5, 1)
    model = MeshGpt(0, GptConfig(vocab_size=data.vocab_size, context=8, width=128, heads=4, layers=2), 7)
    x, y = data.batch(False, np.arange(len(data.training)))
    for _ in range(600):
        loss = model.train_batch(x, y, 4, 0.01, 0.0)
    assert loss < 0.1
    prompts, answers = x.reshape(-1, 4).tolist(), y.reshape(-1, 4)[:, 3].astype(np.int64)
    scored = CachedGpt(model, len(prompts)).score(prompts, answers, top=2)
    assert float(-scored.logprob.mean()) < 0.3
    assert np.array_equal(scored.top_index[:, 0].cpu().numpy(), answers)
    steps = CachedGpt(model, len(prompts)).generate(prompts, 2, top=3)
    assert np.array_equal(steps[0].top_index[:, 0].cpu().numpy(), answers)
    assert np.array_equal(steps[0].logprob.cpu().numpy(), steps[0].top_logprob[:, 0].cpu().numpy())

"""Log-probabilities keep their digits whatever the logits' size: with m the
largest logit and s the sum of e^(x - m), x_t - m rounds once (2^-24 of it), ln s
is off by the sum's few 2^-24 and its own rounding, whatever m is: 1e-6 and
2^-22 of the value bound it.  (x_t - lse would carry lse's rounding: 2^-24 of it.)"""

import numpy as np
import pytest

from grokking_abmod_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shift", [0.0, 100.0, -3000.0, 40000.0])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,vocab,top", [(40, 64, 0), (40, 97, 0), (40, 97, 3), (40, 61, 20), (5, 1000, 7),
                                            (3, 5000, 0), (3, 5000, 2), (2, 70001, 5), (900, 1700, 1)])
def test_large_logits(rows, vocab, top, dtype, shift):
    """Likely and unlikely tokens; every other row has one that is nearly certain."""
    import torch
    rng = np.random.default_rng(vocab)
    x = rng.normal(0, 3, (rows, vocab))
    tokens = rng.integers(0, vocab, rows).astype(np.int32)
    x[np.arange(0, rows, 2), tokens[::2]] += 24
    t = torch.from_numpy((x + shift).astype(np.float32)).to(getattr(torch, dtype))
    x = t.double().numpy()
    r = ops.token_logprobs(t.cuda(), torch.from_numpy(tokens).cuda(), top)
    m = x.max(1)
    logp = x - m[:, None] - np.log(np.exp(x - m[:, None]).sum(1))[:, None]
    want = logp[np.arange(rows), tokens]
    got = r.logprob.double().cpu().numpy()
    assert np.all(np.abs(got - want) <= 1e-6 + 2.0 ** -22 * np.abs(want)), np.abs(got - want).max()
    best = np.take_along_axis(logp, r.top_index.cpu().numpy().astype(np.int64), 1)
    got = r.top_logprob.double().cpu().numpy()
    assert np.all(np.abs(got - best) <= 1e-6 + 2.0 ** -22 * np.abs(best))

"""Token log-probabilities, entropy, top tokens and their gradient
(mb_op_token_logprobs*) against float64.

Tolerances, from the arithmetic: a term 2^-t with t = (m - x) log2 e carries
2^-22 (the exponential) and t 2^-23 (t itself); lse is off by that average and
its own rounding, 2e-6 (1 + |lse|); the entropy weighs each term with
t + log s, 1e-5 (1 + H) for the logits used here (within 60 of each other); a
gradient is p times at most |g| + |h| (60 + H) with p off by 6e-6, plus the
output type's half unit."""

import numpy as np
import pytest

from grokking_abmod_b200 import MeshError, ops

pytestmark = pytest.mark.gpu

DTYPES = ("float32", "bfloat16", "float16")
UNIT = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def _torch():
    import torch
    return torch


def _case(rng, rows, vocab, dtype, masked=False, stride=None, shift=0):
    """(float64 array, CUDA tensor whose rows are `stride` apart and begin `shift` elements in)."""
    torch = _torch()
    x = rng.normal(0, 3, (rows, vocab)).astype(np.float32)
    if masked:
        x[rng.random((rows, vocab)) < 0.4] = -np.inf
        x[0] = -np.inf
        if rows > 2:
            x[2] = -np.inf
            x[2, vocab - 1] = 5.0
    t = torch.from_numpy(x).to(getattr(torch, dtype))
    stride = stride or vocab
    room = torch.zeros(rows * stride + shift, dtype=t.dtype, device="cuda")
    view = room[shift:shift + rows * stride].view(rows, stride)[:, :vocab]
    view.copy_(t)
    return t.double().numpy(), view


def _plain(x, tokens, top):
    with np.errstate(divide="ignore", invalid="ignore"):
        m = np.where(np.isneginf(x.max(1)), 0, x.max(1))
        e = np.exp(x - m[:, None])
        s = e.sum(1)
        lse = m + np.log(s)
        logp = x - lse[:, None]
        p = np.where(s[:, None] > 0, np.exp(logp), 0)
        entropy = -np.where(p > 0, p * logp, 0).sum(1)
    none = s == 0
    lp = np.where(none, -np.inf, logp[np.arange(len(x)), np.maximum(tokens, 0)])
    lp = np.where(tokens < 0, 0, lp)
    order = np.argsort(-x, axis=1, kind="stable")[:, :top]
    best = np.take_along_axis(x, order, 1)
    with np.errstate(invalid="ignore"):
        best = np.where(np.isneginf(best), best, best - lse[:, None])
    return lp, entropy, lse, best, order, p


def _near(name, got, want, tol):
    got = got.double().cpu().numpy()
    finite = np.isfinite(want)
    assert np.array_equal(got[~finite], want[~finite]), name
    assert np.all(np.isfinite(got[finite])), name
    tol = np.broadcast_to(tol, want.shape)
    err = np.abs(got - want)[finite] - tol[finite]
    assert not err.size or err.max() <= 0, (name, err.max())


def _tokens(rng, rows, vocab, ignored=True):
    t = rng.integers(0, vocab, rows).astype(np.int32)
    if ignored and rows > 1:
        t[1] = -1
    return t


SHAPES = [(1, 1, 1), (5, 2, 2), (33, 64, 5), (70, 97, 20), (9, 255, 32), (4, 513, 32), (3, 1024, 7), (3, 1025, 32),
          (2, 4099, 1), (7, 8192, 20), (1, 32003, 32), (3, 65537, 5), (1, 131071, 32), (700, 1500, 3)]


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top", SHAPES)
def test_forward_and_backward(rows, vocab, top, dtype, masked):
    torch = _torch()
    rng = np.random.default_rng(rows + vocab)
    x, logits = _case(rng, rows, vocab, dtype, masked)
    tokens = _tokens(rng, rows, vocab)
    t = torch.from_numpy(tokens).cuda()
    status = ops.new_status()
    r = ops.token_logprobs(logits, t, top, status=status)
    lp, entropy, lse, best, order, p = _plain(x, tokens, top)
    flse = np.where(np.isfinite(lse), np.abs(lse), 0)
    _near("lse", r.lse, lse, 2e-6 * (1 + flse))
    _near("logprob", r.logprob, lp, 2e-6 * (1 + flse) + 2.0 ** -23 * np.where(np.isfinite(lp), np.abs(lp), 0))
    _near("entropy", r.entropy, entropy, 1e-5 * (1 + entropy))
    _near("top", r.top_logprob, best, (2e-6 * (1 + flse))[:, None] + 2.0 ** -23 * np.where(np.isfinite(best), np.abs(best), 0))
    assert np.array_equal(r.top_index.cpu().numpy(), order)

    g, h = rng.normal(0, 1, rows), rng.normal(0, 1, rows)
    g, h = g.astype(np.float32).astype(np.float64), h.astype(np.float32).astype(np.float64)
    tg, th = (torch.from_numpy(a.astype(np.float32)).cuda() for a in (g, h))
    none = np.isneginf(lse)
    use = np.where((tokens >= 0) & ~none, g, 0)
    with np.errstate(invalid="ignore"):
        logp = np.where(p > 0, x - lse[:, None], 0)
    d_lp = -p * use[:, None]
    d_lp[np.arange(rows), np.maximum(tokens, 0)] += use
    d_h = -h[:, None] * p * (logp + entropy[:, None])
    bound = 6e-6 * p * (np.abs(g) + np.abs(h) * (60 + entropy))[:, None]
    for dl, de, want in ((tg, th, d_lp + d_h), (tg, None, d_lp), (None, th, d_h)):
        d = ops.token_logprobs_backward(logits, t, r.lse, r.entropy, dl, de, status=status)
        # float16's subnormals: half of 2^-24
        _near("gradient", d, want, bound + UNIT[dtype] * np.abs(want) + 2.0 ** -25 * (dtype == "float16") + 2.0 ** -23 * np.abs(use)[:, None])
        assert d.dtype == logits.dtype
    ops.check_status(status)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("stride,shift", [(5003, 0), (5001, 1), (5008, 3), (5008, 8)])
def test_strided_rows_of_every_alignment(dtype, stride, shift):
    torch = _torch()
    rng = np.random.default_rng(stride + shift)
    x, logits = _case(rng, 13, 4999, dtype, True, stride, shift)
    tokens = _tokens(rng, 13, 4999)
    t = torch.from_numpy(tokens).cuda()
    r = ops.token_logprobs(logits, t, 9)
    lp, entropy, lse, best, order, p = _plain(x, tokens, 9)
    assert np.array_equal(r.top_index.cpu().numpy(), order)
    _near("lse", r.lse, lse, 2e-6 * (1 + np.where(np.isfinite(lse), np.abs(lse), 0)))
    d = ops.token_logprobs_backward(logits, t, r.lse, r.entropy, None, torch.ones(13, device="cuda"))
    whole = ops.token_logprobs_backward(logits.contiguous(), t, r.lse, r.entropy, None, torch.ones(13, device="cuda"))
    assert torch.equal(d, whole)


@pytest.mark.parametrize("vocab", [64, 1000, 3000, 70001])
@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_and_orders_that_are_hard_for_the_top_list(vocab, dtype):
    """All equal, few distinct values, rising, falling, -0 and +0."""
    torch = _torch()
    rng = np.random.default_rng(vocab)
    i = np.arange(vocab)
    x = np.stack([np.zeros(vocab), rng.integers(0, 3, vocab), i * 40.0 / vocab, -i * 40.0 / vocab,
                  np.where(i % 2, 0.0, -0.0), np.where(i == vocab - 1, 1.0, -np.inf), np.full(vocab, -3e38)])
    t = torch.from_numpy(x.astype(np.float32)).to(getattr(torch, dtype))
    r = ops.token_logprobs(t.cuda(), torch.zeros(len(x), dtype=torch.int32, device="cuda"), 32)
    order = np.argsort(-t.double().numpy(), axis=1, kind="stable")[:, :32]
    assert np.array_equal(r.top_index.cpu().numpy(), order)


def test_nan_and_infinity_stay_in_their_rows():
    torch = _torch()
    for vocab in (100, 20000):
        x = torch.randn(5, vocab, device="cuda")
        clean = ops.token_logprobs(x, torch.zeros(5, dtype=torch.int32, device="cuda"), 4)
        x[1, 7] = float("nan")
        x[3, 9] = float("inf")
        r = ops.token_logprobs(x, torch.zeros(5, dtype=torch.int32, device="cuda"), 4)
        for a, b in zip(r, clean):
            assert torch.equal(a[::2], b[::2])
            if a.dtype == torch.float32:
                assert torch.isnan(a[1::2]).all()
        assert r.top_index[1, 0] == 7 and r.top_index[3, 0] == 9
        ones = torch.ones(5, device="cuda")
        d = ops.token_logprobs_backward(x, torch.zeros(5, dtype=torch.int32, device="cuda"), r.lse, r.entropy, ones,
                                        ones)
        assert torch.isfinite(d[::2]).all() and torch.isnan(d[1::2]).all()


@pytest.mark.parametrize("rows,vocab", [(6, 97), (2, 5000)])
def test_gradient_against_differences(rows, vocab):
    """Central differences of the float64 forward along random directions:
    their error is the third derivative's, below 1e-7 at this step."""
    torch = _torch()
    rng = np.random.default_rng(vocab)
    x, logits = _case(rng, rows, vocab, "float32")
    tokens = _tokens(rng, rows, vocab)
    g, h = (rng.normal(0, 1, rows).astype(np.float32) for _ in range(2))
    t = torch.from_numpy(tokens).cuda()
    r = ops.token_logprobs(logits, t)
    d = ops.token_logprobs_backward(logits, t, r.lse, r.entropy, torch.from_numpy(g).cuda(),
                                    torch.from_numpy(h).cuda()).double().cpu().numpy()

    def f(y):
        lp, entropy, *_ = _plain(y, tokens, 0)
        return (g * lp + h * entropy).sum()

    for _ in range(4):
        u = rng.normal(0, 1, x.shape)
        eps = 1e-4
        slope = (f(x + eps * u) - f(x - eps * u)) / (2 * eps)
        assert abs((d * u).sum() - slope) <= 2e-5 * (np.abs(d * u).sum() + 1)


def test_refusals():
    torch = _torch()
    x = torch.zeros((3, 50), device="cuda")
    t = torch.zeros(3, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        ops.token_logprobs(x.double(), t)
    with pytest.raises(ValueError):
        ops.token_logprobs(x.t(), t)
    with pytest.raises(ValueError):
        ops.token_logprobs(x, t.long())
    with pytest.raises(ValueError):
        ops.token_logprobs(x, t[:2])
    with pytest.raises(ValueError):
        ops.token_logprobs(x.cpu(), t)
    with pytest.raises(MeshError):
        ops.token_logprobs(x, t, 33)
    with pytest.raises(MeshError):
        ops.token_logprobs(x[:, :4], t, 5)
    with pytest.raises(ValueError):
        ops.token_logprobs_backward(x, t, torch.zeros(2, device="cuda"), None)
    with pytest.raises(MeshError):  # the entropy's gradient needs the entropy
        ops.token_logprobs_backward(x, t, torch.zeros(3, device="cuda"), None, None, torch.zeros(3, device="cuda"))
    # a token out of range is reported, and its row is NaN
    status = ops.new_status()
    t[1] = 50
    r = ops.token_logprobs(x, t, status=status)
    assert int(status.item()) == 2 and torch.isnan(r.logprob[1]) and torch.isfinite(r.logprob[::2]).all()
    assert ops.token_logprobs(x[:0], t[:0], 2).top_index.shape == (0, 2)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top", [(515, 1025, 32), (750, 1499, 0), (1031, 1030, 5), (1100, 2197, 1), (2050, 4097, 20)])
def test_many_rows_of_longer_vocabularies(rows, vocab, top, dtype, masked):
    test_forward_and_backward(rows, vocab, top, dtype, masked)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_long_rows_with_ties_and_nan(dtype):
    """A warp a row: more equal values than its list holds, few kinds, NaN."""
    torch = _torch()
    rows, vocab = 1600, 3001
    rng = np.random.default_rng(11)
    i = np.arange(vocab)
    kinds = np.stack([np.zeros(vocab), rng.integers(0, 3, vocab), i * 40.0 / vocab, -i * 40.0 / vocab,
                      np.where(i == vocab - 1, 1.0, -np.inf), np.full(vocab, -3e38), np.full(vocab, -np.inf),
                      rng.normal(0, 3, vocab)]).astype(np.float32)
    x = torch.from_numpy(np.tile(kinds, (rows // 8, 1))).to(getattr(torch, dtype))
    order = np.argsort(-x.double().numpy(), axis=1, kind="stable")[:, :32]
    t = torch.zeros(rows, dtype=torch.int32, device="cuda")
    clean = ops.token_logprobs(x.cuda(), t, 32)
    assert np.array_equal(clean.top_index.cpu().numpy(), order)
    x[9, 7] = float("nan")
    r = ops.token_logprobs(x.cuda(), t, 32)
    keep = torch.arange(rows) != 9
    for a, b in zip(r, clean):
        assert torch.equal(a.cpu()[keep], b.cpu()[keep])
    assert torch.isnan(r.lse[9]) and r.top_index[9, 0] == 7
